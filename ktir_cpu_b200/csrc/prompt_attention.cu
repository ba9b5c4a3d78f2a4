// Attention over packed prompts with grouped heads, on the tensor cores.
//
// Query i of a sequence's n sees keys j <= i + m - n of its m when causal, all
// of them otherwise; o = softmax(scale q K^T) V over those.
//
// Bound by the tensor pipe and, about as tightly, by the exponentials: a tile
// of 128 rows x 128 keys costs 2 x 128^2 x dim products (1,024 cycles at dim
// 128) and 128^2 exponentials (16 per cycle and SM: 1,024 cycles).  So a CTA
// (one per SM, persistent) works on two row tiles at once, one in the softmax
// while the other is in the tensor pipe.
//
// A row is a (token, head) pair: the g = heads / kv_heads queries that share a
// kv head lie side by side, 128 / g tokens per row tile, so that every row of a
// tile uses the same K and V whatever g is, and a short prompt fills more of a
// tile.
//
// Which row tiles a CTA takes depends on how many there are (see plan()):
//   pairs    two that follow each other in a sequence, sharing its K and V blocks
//   singles  two of any sequences and heads, each with blocks of its own, where
//            most sequences have but one row tile per head
//   parts    no more row tiles than SMs: one per CTA, half of its keys to each group
//            of softmax warps, or, where its keys are many, a stretch of them; the
//            stretches' (m, l, O) are left in the workspace and the last CTA of a row
//            tile joins them in their order
//
// Roles, meeting only at mbarriers:
//   warps 0-3, 4-7  the softmax of row tile 0 and 1, one row per thread:
//                   S from TMEM, mask, running maximum and sum, P = 2^(x - m)
//                   rounded to the element type into TMEM, and at a tile's end
//                   O / l to memory
//   warps 8, 10     (MMA) S_w(j) = Q_w K_j^T and O_w += P_w(j) V_j, P read from
//                   TMEM; S_w(j+1) runs as soon as S_w(j) is in registers, so the
//                   softmax goes from block to block without waiting for it
//   warp 9 (TMA)    Q tiles, and K_j, V_j through one ring
//   warp 11         finds the next tile: tiles are taken in order of falling
//                   key counts over all sequences, back and forth over the
//                   CTAs, so that the last ones to finish are the shortest
// V rows past a sequence's last key belong to another sequence, and a weight of 0
// does not cancel an infinity there: a softmax warp sets them to zero in shared
// memory before the last block's product.
// TMEM holds S, P and O of both row tiles apart, which at dim 128 leaves room for
// blocks of 80 keys (128 at dim 64).
// The running maximum moves only when a row's maximum exceeds it by more than
// 2^8; O's rows are then rescaled in TMEM, after the product before.  In f16 it is kept
// 2^7 lower than it is (Elem::LIFT).
// Precision: S, O, m and l in f32; P is rounded to the element type for the
// second product (tcgen05 wants one type for both operands), half an ulp per
// weight (in f16 2^-32 of a row's largest where that is more); l adds the unrounded
// weights.
// Measured, 8192 tokens of 32 heads over 8, causal: dim 128 449 us in a short burst
// (1,220 TFLOP/s) and 505 to 520 under the power cap, dim 64 360 us.  Of a block's 2,100
// cycles (80 keys, both row tiles) the exponentials take 1,300; both groups of softmax
// warps run in step, so nothing else overlaps them.  A change of tiles costs 4,500
// cycles: the last product, the outputs, the next tile's S.
// Every wait is bounded; one that runs out raises the CTA's abort flag, every
// role then leaves its loop, waits for its own copies and products, and the
// CTA still frees its TMEM.
#include <cuda.h>

#include <type_traits>

#include "serve_common.cuh"
#include "tc_common.cuh"

using namespace ktir::serve;
using namespace ktir::tc;

namespace {

constexpr int BQ = 128;              // rows of a row tile
constexpr int THREADS = 384;
constexpr int SCHED = 4;             // tiles announced ahead
constexpr int WEIGHTS = 512;         // weights whose tile counts a CTA keeps there
constexpr int CACHED = 256;          // sequences whose lengths a CTA keeps in shared memory
constexpr int MAX_PARTS = 160;       // CTAs of a launch that splits keys
constexpr int HALVE = 3;             // blocks from which a CTA's two groups of softmax warps share a row tile
constexpr int PART_FLOATS = 128 * BQ + 2 * BQ;      // O [dim][row], then (m, l) per row
constexpr int64_t PARTS_BYTES = (int64_t)MAX_PARTS * PART_FLOATS * 4;
static_assert(PARTS_BYTES == KTIR_PROMPT_PARTS_BYTES);
constexpr int SCHED_READERS = 11;    // 8 softmax warps, two MMA, TMA
constexpr float RESCALE_THRESHOLD = 8.0f;   // log2 units
constexpr float FAR = 16777216.0f;          // 2^24: a maximum from here on is rounded to whole log2 units
constexpr int SOFTMAX_REGS = 208, OTHER_REGS = 80;
constexpr uint32_t TMEM_COLS = 512;

// TMEM has 512 columns for S (BK), P (BK / 2) and O (D) of two row tiles.
template <int D>
struct Cfg {
  static constexpr int BK = D == 128 ? 80 : 128;    // keys of a block
  static constexpr int PANELS = D / 64;             // of 64 elements, rows of 128 bytes, swizzled
  static constexpr int Q_PANEL = BQ * 128, Q_TILE = PANELS * Q_PANEL;
  static constexpr int PANEL = BK * 128, TILE = PANELS * PANEL;      // a K or V block
  static constexpr int STAGES = D == 128 ? 6 : 9;
  // a softmax warp's 32 rows of 64 output elements on their way to memory, rows
  // 16 bytes apart from a multiple of 128 (no two of eight lanes in one bank)
  static constexpr int OUT_ROW = 144, OUT_WARP = 32 * OUT_ROW;
  static constexpr int OUT = 2 * Q_TILE + STAGES * TILE;
  static constexpr int BYTES = OUT + 8 * OUT_WARP;
  // first columns of row tile 0, and from one row tile to the next
  static constexpr uint32_t S_COL = 0, S_STEP = 128, O_COL = D == 128 ? 256 : 384, O_STEP = D;
  static constexpr uint32_t P_COL = D == 128 ? 80 : 256, P_STEP = D == 128 ? 128 : 64;
};
constexpr int MAX_STAGES = 9;

struct RowTile {
  int token;      // its first token
  int tokens;     // of the sequence from there on, at most a row tile's
  int seen;       // keys that the first token sees (causal)
  int keys;       // of the sequence
  int key0;       // its first key
  int head;       // kv head
  int blocks;     // key blocks
};

struct Tile {
  int stop;
  int shared;     // both row tiles use the same K and V blocks
  int halves;     // row tile 1 is the second half of row tile 0's keys
  int splits;     // CTAs that share row tile 0, each with a stretch of its keys,
  int split;      // which of them this is
  int unit;       // and the row tile's number
  RowTile r[2];
};

struct PromptParams {
  KtirPromptDesc d;
  int group;            // query heads per kv head
  int tile_tokens;      // tokens of a row tile
  int k_head_step, v_head_step, q_head_step;   // 0 where all heads share one vector
  uint32_t token_magic;  // for divisions by tile_tokens, and by twice that
  uint32_t pair_magic;
  float* parts;          // or null: no splitting
  int* counters;         // zero between calls
};

struct Shared {
  uint64_t q_full[2], q_empty[2];
  uint64_t full[MAX_STAGES], empty[MAX_STAGES];
  uint64_t s_full[2], s_free[2], p_full[2], pv_done[2], o_free[2];
  uint64_t tail[MAX_STAGES];        // a V block with rows past the last key has arrived
  uint64_t drain[2];
  uint64_t sched_full[SCHED], sched_empty[SCHED];
  uint64_t meet, part_in, part_out;
  Tile tile[SCHED];
  int2 lengths[CACHED];             // tokens and keys of the first sequences
  int last;
  int weights[WEIGHTS];             // tiles of at least this weight
  uint32_t tmem_base;
  int abort_flag;
  int gaps;                         // offsets out of their range, or tokens outside all sequences
};


__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y,
                                            int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}

// Bounded wait for a barrier's phase: false (and the abort flag raised) when the
// limit runs out or another role has given up.  Kept from being unrolled: four
// tests in a row before the first branch cost a wait that is over 120 cycles
// (8192 tokens, 32 heads over 8: 611 -> 543 us).
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile int* abort) {
  if (mbar_try_wait(bar, parity)) return true;
#pragma unroll 1
  for (uint32_t i = 0; i < kSpinLimit; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if (*abort) return false;
  }
  *abort = 1;
  return false;
}

// One lane of the (converged) warp.  Code under this predicate may use uniform
// registers, under `lane == 0` it may not: eight tcgen05.mma then take 413
// cycles to issue instead of 129 (512 to run).
__device__ __forceinline__ bool elect() {
  uint32_t one;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(one));
  return one != 0;
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// two f32 in a 64-bit register, one instruction for both
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// A block of this thread's TMEM lane, loaded (stored) and waited for in one
// statement: the registers are the compiler's to move once it ends.
__device__ __forceinline__ void tmem_ld_block(uint32_t taddr, uint32_t (&r)[128]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, "
      "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, "
      "%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63 "
      "}, [%128];\n"
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
      "%64, %65, %66, %67, %68, %69, %70, %71, %72, %73, %74, %75, %76, %77, %78, %79, "
      "%80, %81, %82, %83, %84, %85, %86, %87, %88, %89, %90, %91, %92, %93, %94, %95, "
      "%96, %97, %98, %99, %100, %101, %102, %103, %104, %105, %106, %107, %108, %109, %110, %111, "
      "%112, %113, %114, %115, %116, %117, %118, %119, %120, %121, %122, %123, %124, %125, %126, %127 "
      "}, [%129];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
        "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
        "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
        "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
        "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63]),
        "=r"(r[64]), "=r"(r[65]), "=r"(r[66]), "=r"(r[67]), "=r"(r[68]), "=r"(r[69]), "=r"(r[70]), "=r"(r[71]),
        "=r"(r[72]), "=r"(r[73]), "=r"(r[74]), "=r"(r[75]), "=r"(r[76]), "=r"(r[77]), "=r"(r[78]), "=r"(r[79]),
        "=r"(r[80]), "=r"(r[81]), "=r"(r[82]), "=r"(r[83]), "=r"(r[84]), "=r"(r[85]), "=r"(r[86]), "=r"(r[87]),
        "=r"(r[88]), "=r"(r[89]), "=r"(r[90]), "=r"(r[91]), "=r"(r[92]), "=r"(r[93]), "=r"(r[94]), "=r"(r[95]),
        "=r"(r[96]), "=r"(r[97]), "=r"(r[98]), "=r"(r[99]), "=r"(r[100]), "=r"(r[101]), "=r"(r[102]), "=r"(r[103]),
        "=r"(r[104]), "=r"(r[105]), "=r"(r[106]), "=r"(r[107]), "=r"(r[108]), "=r"(r[109]), "=r"(r[110]), "=r"(r[111]),
        "=r"(r[112]), "=r"(r[113]), "=r"(r[114]), "=r"(r[115]), "=r"(r[116]), "=r"(r[117]), "=r"(r[118]), "=r"(r[119]),
        "=r"(r[120]), "=r"(r[121]), "=r"(r[122]), "=r"(r[123]), "=r"(r[124]), "=r"(r[125]), "=r"(r[126]), "=r"(r[127])
      : "r"(taddr), "r"(taddr + 64)
      : "memory");
}
__device__ __forceinline__ void tmem_ld_block(uint32_t taddr, uint32_t (&r)[80]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, "
      "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, "
      "%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63 "
      "}, [%80];\n"
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {"
      "%64, %65, %66, %67, %68, %69, %70, %71, %72, %73, %74, %75, %76, %77, %78, %79 "
      "}, [%81];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),
        "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),
        "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
        "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
        "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63]),
        "=r"(r[64]), "=r"(r[65]), "=r"(r[66]), "=r"(r[67]), "=r"(r[68]), "=r"(r[69]), "=r"(r[70]), "=r"(r[71]),
        "=r"(r[72]), "=r"(r[73]), "=r"(r[74]), "=r"(r[75]), "=r"(r[76]), "=r"(r[77]), "=r"(r[78]), "=r"(r[79])
      : "r"(taddr), "r"(taddr + 64)
      : "memory");
}
__device__ __forceinline__ void tmem_st_block(uint32_t taddr, const uint32_t (&r)[64]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x64.b32 [%64], {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, "
      "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, "
      "%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63 "
      "};\n"
      "tcgen05.wait::st.sync.aligned;" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
        "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
        "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]),
        "r"(r[32]), "r"(r[33]), "r"(r[34]), "r"(r[35]), "r"(r[36]), "r"(r[37]), "r"(r[38]), "r"(r[39]),
        "r"(r[40]), "r"(r[41]), "r"(r[42]), "r"(r[43]), "r"(r[44]), "r"(r[45]), "r"(r[46]), "r"(r[47]),
        "r"(r[48]), "r"(r[49]), "r"(r[50]), "r"(r[51]), "r"(r[52]), "r"(r[53]), "r"(r[54]), "r"(r[55]),
        "r"(r[56]), "r"(r[57]), "r"(r[58]), "r"(r[59]), "r"(r[60]), "r"(r[61]), "r"(r[62]), "r"(r[63]),
        "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_block(uint32_t taddr, const uint32_t (&r)[40]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%40], {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31 "
      "};\n"
      "tcgen05.st.sync.aligned.32x32b.x8.b32 [%41], {"
      "%32, %33, %34, %35, %36, %37, %38, %39 "
      "};\n"
      "tcgen05.wait::st.sync.aligned;" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
        "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
        "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]),
        "r"(r[32]), "r"(r[33]), "r"(r[34]), "r"(r[35]), "r"(r[36]), "r"(r[37]), "r"(r[38]), "r"(r[39]),
        "r"(taddr), "r"(taddr + 32)
      : "memory");
}

// registers per thread after the split of a launch's 168 x 384 between the
// softmax warps (8) and the other four: 208 x 256 + 80 x 128 = 63,488 of 64,512
template <int N>
__device__ __forceinline__ void more_registers() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void fewer_registers() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// -- the order of tiles -----------------------------------------------------------
// A tile holds T tokens of a sequence (n tokens, m keys): tile i tokens [i T, (i + 1)
// T).  Its weight is the number of key blocks that its last token sees.  Tiles are
// numbered by falling weight over all sequences, within a weight by sequence, and
// each once per kv head.
struct Seq {
  int n, m;
};

__device__ __forceinline__ Seq sequence(const KtirPromptDesc& d, long long b, bool& bad) {
  const int q0 = d.offsets[b], q1 = d.offsets[b + 1], k0 = d.kv_offsets[b], k1 = d.kv_offsets[b + 1];
  bad = q0 < 0 || q1 < q0 || q1 > d.tokens || k0 < 0 || k1 < k0 || k1 > d.kv_tokens;
  Seq s;
  s.n = bad ? 0 : q1 - q0;
  s.m = bad ? 0 : k1 - k0;
  return s;
}

__device__ __forceinline__ int warp_sum(int v) { return __reduce_add_sync(0xffffffffu, v); }

// The tiles of one size, walked from heaviest to lightest by one warp.
template <int BK>
struct Order {
  const PromptParams& p;
  const int2* cached;
  int lane, T;
  uint32_t magic;
  int weight;            // of the tile last found, at first the heaviest of all
  int above;             // tiles heavier than that
  int upto;              // and tiles of at least that weight, once one has been found
  long long from;        // sequences before this one have had all their tiles of the weight looked at,
  int passed;            // this many: a walk over all tiles looks once at every sequence for each weight
  int* table;            // tiles of at least each weight, or null

  __device__ __forceinline__ int divide(int x) const {      // x / T, x >= 0
    int q = (int)__umulhi((uint32_t)x, magic);
    q -= q * T > x;
    q += (q + 1) * T <= x;
    return q;
  }
  __device__ __forceinline__ Seq seq(long long b) const {
    if (b < CACHED) {
      const int2 v = cached[b];
      return Seq{v.x, v.y};
    }
    bool bad;
    return sequence(p.d, b, bad);
  }
  // tiles of weight at least `w`: the last ones of the sequence
  __device__ __forceinline__ int heavier(const Seq& s, int w) const {
    const int tiles = divide(s.n + T - 1);
    if (w <= 0) return tiles;
    const int need = (w - 1) * BK;             // more than this many keys seen
    if (s.m <= need) return 0;
    if (!p.d.causal) return tiles;
    const int x = need - (s.m - s.n);          // (i + 1) T > x
    return x <= 0 ? tiles : tiles - divide(x);
  }
  __device__ int count(int w) const {
    int c = 0;
    for (long long b = lane; b < p.d.batch; b += 32) c += heavier(seq(b), w);
    return warp_sum(c);
  }
  // the table: every tile counted at its weight, then summed from the heaviest down
  __device__ void tabulate(int* place, int heaviest) {
    if (heaviest >= WEIGHTS) return;
    table = place;
    for (int w = lane; w <= heaviest; w += 32) table[w] = 0;
    __syncwarp();
    for (long long b = lane; b < p.d.batch; b += 32) {
      const Seq s = seq(b);
      if (!s.n) continue;
      const int seen = p.d.causal ? min(s.m, min(s.n, T) + s.m - s.n) : s.m;        // by the first tile
      for (int w = seen > 0 ? (seen + BK - 1) / BK : 0, have = divide(s.n + T - 1); have > 0; ++w) {
        const int more = heavier(s, w + 1);                            // the others have weight w
        if (have > more) atomicAdd(table + w, have - more);
        have = more;
      }
    }
    __syncwarp();
    int sum = 0;
    for (int w0 = heaviest - (heaviest & 31); w0 >= 0; w0 -= 32) {
      int v = w0 + lane <= heaviest ? table[w0 + lane] : 0;
#pragma unroll
      for (int k = 1; k < 32; k <<= 1) {
        const int o = __shfl_down_sync(0xffffffffu, v, k);
        if (lane + k < 32) v += o;
      }
      v += sum;
      sum = __shfl_sync(0xffffffffu, v, 0);
      if (w0 + lane <= heaviest) table[w0 + lane] = v;
    }
    __syncwarp();
  }
  // tile number `x`, not below the last one found: its sequence and place there.
  // With a tile for every CTA their order does not matter (`any`): by sequence, then.
  __device__ void find(int x, bool any, long long& b_out, int& i_out) {
    if (any) {
      weight = above = 0;
    } else if (x < upto) {
      // of the weight last found
    } else if (table) {
      while (weight > 0 && table[weight] <= x) above = table[weight--];
      upto = table[weight];
      from = passed = 0;
    } else {
      int hi = weight + 1, hi_count = above;   // count(hi) <= x
      int step = 1, lo = max(0, hi - 1), c = count(lo), lo_count;
      while (c <= x && lo > 0) {
        hi = lo;
        hi_count = c;
        step <<= 1;
        lo = max(0, hi - step);
        c = count(lo);
      }
      lo_count = c;
      while (hi - lo > 1) {                    // lo_count = count(lo) > x >= count(hi)
        const int mid = (lo + hi) >> 1;
        c = count(mid);
        if (c > x) {
          lo = mid;
          lo_count = c;
        } else {
          hi = mid;
          hi_count = c;
        }
      }
      weight = lo;
      above = hi_count;
      upto = lo_count;
      from = passed = 0;
    }
    const int lo = weight;
    int r = x - above - passed;
    b_out = -1;
    i_out = 0;
    for (long long b0 = from; b0 < p.d.batch; b0 += 32) {
      const long long b = b0 + lane;
      int first = 0, mine = 0;
      if (b < p.d.batch) {
        const Seq s = seq(b);
        const int tiles = divide(s.n + T - 1), all = any ? tiles : heavier(s, lo);
        mine = any ? tiles : all - heavier(s, lo + 1);
        first = tiles - all;
      }
      int incl = mine;
#pragma unroll
      for (int w = 1; w < 32; w <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, incl, w);
        if (lane >= w) incl += o;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, r >= incl - mine && r < incl);
      if (hit) {
        const int at = __ffs(hit) - 1;
        b_out = b0 + at;
        i_out = __shfl_sync(0xffffffffu, first + r - (incl - mine), at);
        from = b0;
        passed = x - above - r;
        return;
      }
      r -= __shfl_sync(0xffffffffu, incl, 31);
    }
  }
};

// the row tile at token `at` of sequence b
template <int BK>
__device__ __forceinline__ void row_tile(const PromptParams& p, long long b, const Seq& s, int at, int head, RowTile& r) {
  const int here = max(0, min(p.tile_tokens, s.n - at));     // its tokens
  const int end = p.d.causal ? min(s.m, at + here + s.m - s.n) : s.m;
  r.token = p.d.offsets[b] + at;
  r.tokens = here;
  r.seen = at + s.m - s.n + 1;
  r.keys = s.m;
  r.key0 = p.d.kv_offsets[b];
  r.head = head;
  r.blocks = here > 0 && end > 0 ? (end + BK - 1) / BK : 0;
}

// Bad offsets: tokens of no sequence get zeros, not what the memory held before (nothing
// else writes them).  256 threads of every CTA; a function of its own, out of the way of
// the softmax's registers.
template <typename T, int D>
__device__ __noinline__ void fill_gaps(const PromptParams& p, int tid) {
  const KtirPromptDesc& d = p.d;
  for (long long at = (long long)blockIdx.x * 256 + tid; at < d.tokens; at += (long long)gridDim.x * 256) {
    auto covers = [&](long long b) -> bool {
      bool bad;
      const long long n = sequence(d, b, bad).n, from = at - d.offsets[b];
      return from >= 0 && from < n;
    };
    // by halves, which finds it where offsets rise, else among all (among all for every
    // token of 40,000 sequences of 20, the last ones in none: 57.6 ms against 7.7)
    long long low = 0, high = d.batch;
    while (high - low > 1) {
      const long long mid = (low + high) >> 1;
      if (d.offsets[mid] <= at) low = mid;
      else high = mid;
    }
    bool covered = covers(low);
    for (long long b = 0; b < d.batch && !covered; ++b) covered = covers(b);
    if (covered) continue;
    for (int h = 0; h < d.heads; ++h) {
      T* out = static_cast<T*>(d.out) + at * d.out_stride[0] + h * d.out_stride[1];
      for (int i = 0; i < D; i += 8) *reinterpret_cast<uint4*>(out + i) = make_uint4(0, 0, 0, 0);
      if (d.lse) d.lse[at * d.heads + h] = -INFINITY;
    }
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(THREADS, 1)
    k_prompt_attention(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                       const __grid_constant__ CUtensorMap tv, const __grid_constant__ PromptParams p) {
  using C = Cfg<D>;
  constexpr uint32_t TYPE = sizeof(T) == 2 && Elem<T>::BF16 ? (1u << 7) | (1u << 10) : 0u;
  constexpr int STAGES = C::STAGES, BK = C::BK;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Shared B;
  const KtirPromptDesc& d = p.d;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t sQ = base, ring = base + 2 * C::Q_TILE;
  volatile int* abort = &B.abort_flag;

  if (tid == 0) {
    B.abort_flag = 0;
    B.gaps = 0;
    for (int w = 0; w < 2; ++w) {
      mbar_init(smem_u32(&B.q_full[w]), 1);
      mbar_init(smem_u32(&B.q_empty[w]), 1);
      mbar_init(smem_u32(&B.s_full[w]), 1);
      mbar_init(smem_u32(&B.s_free[w]), 4);
      mbar_init(smem_u32(&B.p_full[w]), 4);
      mbar_init(smem_u32(&B.pv_done[w]), 1);
      mbar_init(smem_u32(&B.o_free[w]), 4);
    }
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(smem_u32(&B.full[s]), 1);
      mbar_init(smem_u32(&B.empty[s]), 2);
      mbar_init(smem_u32(&B.tail[s]), 1);
    }
    for (int w = 0; w < 2; ++w) mbar_init(smem_u32(&B.drain[w]), 1);
    mbar_init(smem_u32(&B.meet), 8);
    mbar_init(smem_u32(&B.part_in), 8);
    mbar_init(smem_u32(&B.part_out), 1);
    for (int s = 0; s < SCHED; ++s) {
      mbar_init(smem_u32(&B.sched_full[s]), 1);
      mbar_init(smem_u32(&B.sched_empty[s]), SCHED_READERS);
    }
    fence_barrier_init();
  }
  if (warp == 8) {
    tmem_alloc(smem_u32(&B.tmem_base), TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = B.tmem_base;
  pdl_launch();
  pdl_wait();

  // announced tiles, waited for by whole warps (false at the end, or on an abort) and
  // left in their place until the warp has done with them
  auto next_tile = [&](int k) -> bool {
    const int s = k % SCHED;
    return __all_sync(0xffffffffu, wait(smem_u32(&B.sched_full[s]), (k / SCHED) & 1, abort)) && !B.tile[s].stop;
  };
  auto done_tile = [&](int k) {
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&B.sched_empty[k % SCHED]));
  };

  if (warp >= 8) {
    fewer_registers<OTHER_REGS>();
    if (warp == 11) {
      // ---------------- tile finder ----------------
      // plan(): the same in every CTA
      const int half = p.tile_tokens;
      int heaviest = 0, singles = 0, pairs = 0;
      bool any_bad = false;
      const int ends = d.offsets[0] | (d.offsets[d.batch] ^ (int)d.tokens);   // 0 if they cover the tokens
      for (long long b = lane; b < d.batch; b += 32) {
        bool bad;
        const Seq s = sequence(d, b, bad);
        if (b < CACHED) B.lengths[b] = make_int2(s.n, s.m);
        any_bad |= bad;
        if (s.n) heaviest = max(heaviest, (s.m + BK - 1) / BK);
        const int tiles = (int)((unsigned)(s.n + half - 1) / (unsigned)half);
        singles += tiles;
        pairs += (tiles + 1) / 2;
      }
      __syncwarp();
      heaviest = (int)__reduce_max_sync(0xffffffffu, (unsigned)heaviest);
      const int rows = warp_sum(singles) * d.kv_heads, twos = warp_sum(pairs) * d.kv_heads;     // below 2^30
      const int G = (int)gridDim.x;
      // No more row tiles than CTAs: one each, its keys shared by the two groups of
      // softmax warps (512 tokens, 32 heads over 8, dim 128: 12.1 us against 13.5), and
      // what CTAs are left over share them too, S to a row tile.  The longest stretch
      // costs ceil(blocks / S) blocks, and joining costs about J of them for every four
      // parts (64 KiB each at dim 128, from L2 through one SM).  64 queries over 400
      // keys: whole 9.9 us, in three parts 15.6; over 2000 keys whole 21.5, in four 19.5.
      const bool parts = rows <= G;
      int splits = 1;
      if (parts && rows > 0 && p.parts) {
        constexpr int J = D == 128 ? 12 : 6;
        const int cap = min(G, MAX_PARTS) / rows;
        for (int r = 1, best = heaviest; cap > 1 && r * J < best; ++r) {
          const int S = min(4 * r, cap), cost = (heaviest + S - 1) / S + r * J;
          if (cost < best) {
            best = cost;
            splits = S;
          }
          if (4 * r >= cap) break;
        }
      }
      // Singles where a CTA has few row tiles, each then next to one of another weight
      // (7 pieces of prompts, 200 row tiles: 37 us against 44 in pairs), or where pairs
      // would leave more than a third of them empty (200 prompts of 32 tokens: 46 us
      // against 59).  Else pairs: their shared blocks save L2 traffic (8192 tokens: 30
      // us of 489).
      const bool singly = parts || rows <= 2 * G || 2 * twos - rows > (2 * twos) / 3;
      const int all = parts ? rows * splits : singly ? (rows + 1) / 2 : twos;
      Order<BK> order = {p, B.lengths, lane, singly ? half : 2 * half, singly ? p.token_magic : p.pair_magic, heaviest, 0, 0, 0, 0, nullptr};

      for (int next = 0;; ++next) {
        const int s = next % SCHED;
        if (next >= SCHED &&
            !__all_sync(0xffffffffu, wait(smem_u32(&B.sched_empty[s]), (next / SCHED - 1) & 1, abort)))
          break;
        // rounds of G (two of them at once for singles), back and forth: a heavy one here
        // is followed by a light one
        const int x = next * G + ((next & 1) ? G - 1 - blockIdx.x : blockIdx.x);
        const int first = !parts && singly ? 2 * next * G + blockIdx.x : x;
        Tile& t = B.tile[s];
        // a CTA may have a tile in the last round after having none before it
        const bool stop = next * G >= all;
        if (lane == 0) {
          t.stop = stop;
          t.shared = !singly;
          t.halves = 0;
          t.splits = 1;                       // an empty tile has no part in another's
          t.split = t.unit = 0;
          for (int w = 0; w < 2; ++w) t.r[w].tokens = t.r[w].blocks = t.r[w].keys = 0;
        }
        __syncwarp();
        if (!stop) {
          for (int w = 0; w < 2; ++w) {
            const int y = parts ? x / splits : singly && w ? first + 2 * (G - 1 - blockIdx.x) + 1 : first;
            if ((parts && (w || x >= all)) || y >= (singly ? rows : twos)) break;
            long long b = 0;
            int i;
            const int index = (int)((unsigned)y / (unsigned)d.kv_heads);
            if (d.batch == 1) i = (singly ? rows : twos) / d.kv_heads - 1 - index;    // its last tile is the heaviest
            else order.find(index, parts, b, i);
            if (lane == 0 && b >= 0) {
              const int head = y - index * d.kv_heads;
              const Seq q = order.seq(b);
              row_tile<BK>(p, b, q, i * order.T, head, t.r[w]);
              if (!singly) row_tile<BK>(p, b, q, i * order.T + half, head, t.r[1]);
              if (splits > 1) {               // this CTA's stretch of the keys
                RowTile& r = t.r[0];
                t.splits = splits;
                t.split = x - y * splits;
                t.unit = y;
                const int per = (r.blocks + splits - 1) / splits, from = min(r.blocks, t.split * per);
                r.blocks = min(per, r.blocks - from);
                r.key0 += from * BK;
                r.keys -= from * BK;
                r.seen -= from * BK;
              }
              if (parts && t.r[0].blocks >= HALVE) {      // for both groups of softmax warps
                RowTile &r = t.r[0], &o = t.r[1];
                o = r;
                r.blocks = (r.blocks + 1) / 2;
                o.blocks -= r.blocks;
                o.key0 += r.blocks * BK;
                o.keys -= r.blocks * BK;
                o.seen -= r.blocks * BK;
                t.halves = 1;
              }
            }
            if (!singly) break;
          }
        }
        if (stop) {                           // not before the first tile: its way is the short prompts' time
          any_bad = __any_sync(0xffffffffu, any_bad || ends);
          if (lane == 0) {
            B.gaps = any_bad;
            if (any_bad && blockIdx.x == 0) atomicOr(d.status, KTIR_STATUS_BAD_INDEX);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&B.sched_full[s]));
        if (stop) break;
        if (next == 0 && all > 2 * G && d.batch > 1) order.tabulate(B.weights, heaviest);    // worth it for a few more
      }
    } else if (warp == 9) {
      // ---------------- TMA ----------------
      const bool leader = elect();
      if (leader) {
        tma_prefetch_desc(&tq);
        tma_prefetch_desc(&tk);
        tma_prefetch_desc(&tv);
      }
      const uint32_t q_bytes = (uint32_t)(p.group * p.tile_tokens) * 128u * C::PANELS;
      int loads = 0, q_loads[2] = {0, 0};
      uint32_t was_tail = 0, tail_phase = 0;      // per ring stage: last load, next phase's parity
      bool ok = true;
      for (int k = 0; ok && next_tile(k); ++k) {
        const Tile& t = B.tile[k % SCHED];
        if (leader) {
          for (int w = 0; ok && w < 2; ++w) {
            const RowTile& r = t.r[w];
            if (!r.blocks) continue;
            if (q_loads[w] && !wait(smem_u32(&B.q_empty[w]), (q_loads[w] - 1) & 1, abort)) {
              ok = false;
              break;
            }
            const uint32_t bar = smem_u32(&B.q_full[w]);
            mbar_arrive_expect_tx(bar, q_bytes);
#pragma unroll
            for (int c = 0; c < C::PANELS; ++c)
              tma_load_3d(sQ + w * C::Q_TILE + c * C::Q_PANEL, &tq, bar, 64 * c, r.head * p.q_head_step, r.token);
            ++q_loads[w];
          }
          // block j for both row tiles, or for each that has one
          auto load = [&](bool kv, int j) -> bool {
            for (int w = 0; w < 2; ++w) {
              const RowTile& r = t.r[t.shared && !t.r[0].blocks ? 1 : w];
              const int has = t.shared ? max(t.r[0].blocks, t.r[1].blocks) : r.blocks;
              if (j >= has) {
                if (t.shared) break;
                continue;
              }
              const int s = loads % STAGES;
              if (loads >= STAGES && !wait(smem_u32(&B.empty[s]), (loads / STAGES - 1) & 1, abort)) return false;
              // V rows past the last key: a softmax warp passes the block on when it has cleared them
              const bool tail = kv && (j + 1) * BK > r.keys;
              const uint32_t bar = smem_u32(tail ? &B.tail[s] : &B.full[s]);
              was_tail = (was_tail & ~(1u << s)) | (tail ? 1u << s : 0u);
              if (tail) tail_phase ^= 1u << s;
              mbar_arrive_expect_tx(bar, C::TILE);
#pragma unroll
              for (int c = 0; c < C::PANELS; ++c)
                tma_load_3d(ring + s * C::TILE + c * C::PANEL, kv ? &tv : &tk, bar, 64 * c,
                            r.head * (kv ? p.v_head_step : p.k_head_step), r.key0 + j * BK);
              ++loads;
              if (t.shared) break;
            }
            return true;
          };
          // in the order of their use: K_0, K_1, then V_j and K_{j+2}
          const int blocks = max(t.r[0].blocks, t.r[1].blocks);
          for (int j = 0; ok && j < 2 && j < blocks; ++j) ok = load(false, j);
          for (int j = 0; ok && j < blocks; ++j) {
            ok = load(true, j);
            if (ok && j + 2 < blocks) ok = load(false, j + 2);
          }
        }
        ok = __all_sync(0xffffffffu, ok);
        done_tile(k);
      }
      if (leader && *abort) {
        // leave no copy in flight
        int none = 0;
        for (int s = 0; s < STAGES && s < loads; ++s) {
          if ((was_tail >> s) & 1) wait(smem_u32(&B.tail[s]), ((tail_phase >> s) & 1) ^ 1, &none);
          else wait(smem_u32(&B.full[s]), ((loads - 1 - s) / STAGES) & 1, &none);
        }
        for (int w = 0; w < 2; ++w)
          if (q_loads[w]) wait(smem_u32(&B.q_full[w]), (q_loads[w] - 1) & 1, &none);
      }
    } else {
      // ---------------- MMA, one warp per row tile ----------------
      // One thread issues a row tile's products, and its waits, one after the
      // other, are on the way of every block: so there is one for each row tile,
      // and what it does between two products is kept short.
      auto mma = [&](auto W) {
        constexpr int w = decltype(W)::value;
        constexpr uint32_t idesc_s = idesc_f16(BQ, BK, 0, 0) | TYPE;     // Q and K both K-major
        constexpr uint32_t idesc_pv = idesc_f16(BQ, D, 0, 1) | TYPE;     // P K-major, V MN-major
        const uint64_t q_desc = sdesc_sw128(sQ + w * C::Q_TILE, 16, 1024), k_desc = sdesc_sw128(ring, 16, 1024),
                       v_desc = sdesc_sw128(ring, C::PANEL, 1024);
        const uint32_t S = tmem + C::S_COL + w * C::S_STEP, P = tmem + C::P_COL + w * C::P_STEP,
                       O = tmem + C::O_COL + w * C::O_STEP;
        uint32_t stage = 0, ring_phase = 0;         // next ring load to wait for
        uint32_t p_phase = 0, q_phase = 0;
        uint32_t o_phase = 1, s_phase = 1;          // a first wait for these is over at once
        auto next_load = [&]() -> bool {
          return wait(smem_u32(&B.full[stage]), ring_phase, abort);
        };
        auto advance = [&]() {
          if (++stage == STAGES) {
            stage = 0;
            ring_phase ^= 1;
          }
        };
        const bool leader = elect();
        bool ok = true;
        for (int k = 0; ok && next_tile(k); ++k) {
          const Tile& t = B.tile[k % SCHED];
          if (leader) {
            const int mine = t.r[w].blocks, other = t.r[w ^ 1].blocks, blocks = max(mine, other);
            auto run = [&](auto SHARED) {       // the two apart: the loop of one is short
              constexpr bool shared = decltype(SHARED)::value;
              // Both row tiles see every load arrive and give its place in the ring back
              // (else one could take a phase of a barrier for another): a shared block after
              // its product, the other's at once.
              auto pass = [&]() -> bool {
                if (!next_load()) return false;
                mbar_arrive(smem_u32(&B.empty[stage]));
                advance();
                return true;
              };
              auto issue_s = [&](int j) -> bool {
                if (!shared && w == 1 && j < other && !pass()) return false;
                if (shared || j < mine) {
                  if (!next_load()) return false;
                  const uint32_t bar = smem_u32(&B.empty[stage]);
                  if (j < mine) {
                    if (j == 0) {
                      if (!wait(smem_u32(&B.q_full[w]), q_phase, abort)) return false;
                      q_phase ^= 1;
                    }
                    // the block before is in registers
                    if (!wait(smem_u32(&B.s_free[w]), s_phase, abort)) return false;
                    s_phase ^= 1;
                    tc_fence_after();
                    const uint64_t kb = k_desc + (uint64_t)(stage * (C::TILE >> 4));
#pragma unroll
                    for (int kk = 0; kk < D / 16; ++kk)
                      mma_f16(S, q_desc + (((kk >> 2) * C::Q_PANEL + (kk & 3) * 32) >> 4),
                              kb + (((kk >> 2) * C::PANEL + (kk & 3) * 32) >> 4), idesc_s, kk != 0);
                    mma_commit(smem_u32(&B.s_full[w]));
                    mma_commit(bar);
                    if (j + 1 == mine) mma_commit(smem_u32(&B.q_empty[w]));
                  } else {
                    mbar_arrive(bar);
                  }
                  advance();
                }
                if (!shared && w == 0 && j < other && !pass()) return false;
                return true;
              };
              auto issue_pv = [&](int j) -> bool {
                if (!shared && w == 1 && j < other && !pass()) return false;
                if (shared || j < mine) {
                  if (!next_load()) return false;
                  const uint32_t bar = smem_u32(&B.empty[stage]);
                  if (j < mine) {
                    if (j == 0) {                       // O of the tile before has been read
                      if (!wait(smem_u32(&B.o_free[w]), o_phase, abort)) return false;
                      o_phase ^= 1;
                    }
                    if (!wait(smem_u32(&B.p_full[w]), p_phase, abort)) return false;
                    p_phase ^= 1;
                    tc_fence_after();
                    const uint64_t v = v_desc + (uint64_t)(stage * (C::TILE >> 4));
#pragma unroll
                    for (int kk = 0; kk < BK / 16; ++kk)
                      mma_f16_ts(O, P + kk * 8, v + (uint64_t)((kk * 16 * 128) >> 4), idesc_pv,
                                 kk == 0 ? (uint32_t)(j != 0) : 1u);
                    mma_commit(smem_u32(&B.pv_done[w]));
                    mma_commit(bar);
                  } else {
                    mbar_arrive(bar);
                  }
                  advance();
                }
                if (!shared && w == 0 && j < other && !pass()) return false;
                return true;
              };
              for (int j = 0; ok && j < 2 && j < blocks; ++j) ok = issue_s(j);
              for (int j = 0; ok && j < blocks; ++j) {
                ok = issue_pv(j);
                if (ok && j + 2 < blocks) ok = issue_s(j + 2);
              }
            };
            if (t.shared) run(std::true_type());
            else run(std::false_type());
          }
          ok = __all_sync(0xffffffffu, ok);
          done_tile(k);
        }
        if (leader && *abort) {
          int none = 0;
          mma_commit(smem_u32(&B.drain[w]));
          wait(smem_u32(&B.drain[w]), 0, &none);
        }
      };
      if (warp == 8) mma(std::integral_constant<int, 0>());
      else mma(std::integral_constant<int, 1>());
    }
  } else {
    // ---------------- softmax, one row per thread ----------------
    more_registers<SOFTMAX_REGS>();
    const int w = warp >> 2;
    const int row = tid & 127;
    const uint32_t at_lane = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t S = at_lane + C::S_COL + w * C::S_STEP, P = at_lane + C::P_COL + w * C::P_STEP,
                   O = at_lane + C::O_COL + w * C::O_STEP;
    const int token = row / p.group;                 // of the row tile
    const int head_in = row - token * p.group;
    const bool real = token < p.tile_tokens;
    const float c = d.scale * LOG2E;
    uint8_t* staged = smem_raw + (base - smem_u32(smem_raw)) + C::OUT + warp * C::OUT_WARP;
    int n_s = 0;                                     // blocks so far: S, P and PV each
    int loads = 0;                                   // ring loads of the tiles before
    uint32_t tails = 0;                              // per place of the ring: the next tail's phase
    for (int k = 0; next_tile(k); ++k) {
      const Tile& t = B.tile[k % SCHED];
      const RowTile& r_t = t.r[w];
      const int splits = t.splits;
      // both groups of softmax warps join the stretches of a row tile, half of the outputs each
      const bool joined = splits > 1 || t.halves;
      const RowTile& o_t = t.r[joined ? 0 : w];
      const bool store = real && token < o_t.tokens;
      const int blocks = r_t.blocks;
      const int limit = d.causal ? r_t.seen + token : r_t.keys;      // keys this row sees
      const int least = d.causal ? r_t.seen : r_t.keys;              // and the tile's first row
      // V blocks with rows past the last key: their places in the ring, and the phases
      // of those places' barriers, counted by every warp over all of them
      int tail_stage = 0;
      uint32_t tail_phase = 0;
      bool tail = false;
      {
        const int b0 = t.r[0].blocks, b1 = t.r[1].blocks, most = max(b0, b1);
        int at[2];                 // of the row tiles' last V blocks, or -1
        if (t.shared) {
          at[0] = most && most * BK > r_t.keys ? 2 * most - 1 : -1;
          at[1] = -1;
          tail = at[0] >= 0 && w == (b0 == most ? 0 : 1);
        } else {
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            const int j = (v ? b1 : b0) - 1;
            at[v] = j >= 0 && (j + 1) * BK > t.r[v].keys
                        ? min(b0, 2) + min(b1, 2) + min(b0, j) + min(b1, j) + min(max(b0 - 2, 0), j) +
                              min(max(b1 - 2, 0), j) + (v && j < b0 ? 1 : 0)
                        : -1;
          }
          tail = at[w] >= 0;
        }
        const bool swap = at[1] >= 0 && at[1] < at[0];
#pragma unroll
        for (int u = 0; u < 2; ++u) {          // in the order of the loads
          const int v = swap ? u ^ 1 : u;
          if (at[v] >= 0) {
            const int st = (loads + at[v]) % STAGES;
            if (t.shared || v == w) {
              tail_stage = st;
              tail_phase = (tails >> st) & 1;
            }
            tails ^= 1u << st;
          }
        }
      }
      float m = -INFINITY, l = 0.f;
      float from = 0.f;                                // m as a score in S, where it is far
      bool ok = true;
      for (int j = 0; j < blocks; ++j) {
        ok = __all_sync(0xffffffffu, wait(smem_u32(&B.s_full[w]), n_s & 1, abort));
        if (!ok) break;
        tc_fence_after();
        float s[BK];
        tmem_ld_block(S, reinterpret_cast<uint32_t (&)[BK]>(s));
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&B.s_free[w]));
        if ((j + 1) * BK > least) {
          const int left = limit - j * BK;
#pragma unroll
          for (int i = 0; i < BK; ++i)
            if (i >= left) s[i] = -INFINITY;
        }
        float m4[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) m4[x] = fmaxf(s[x], s[4 + x]);
#pragma unroll
        for (int i = 8; i < BK; i += 8)
#pragma unroll
          for (int x = 0; x < 4; ++x) m4[x] = max3(m4[x], s[i + x], s[i + 4 + x]);
        const float s_top = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])), top = __fmul_rn(s_top, c);
        const bool move = top - m > RESCALE_THRESHOLD + Elem<T>::LIFT;     // also from -inf (m + 8 may round to m + 16)
        bool done = j == 0;                                // PV of the block before
        if (__any_sync(0xffffffffu, move || from != 0.f)) {
          float f = 1.f;
          if (move) {
            const bool is_far = fabsf(top) >= FAR;
            const float mn = is_far ? top : top - Elem<T>::LIFT;
            f = ex2(m - mn);
            m = mn;
            from = is_far ? -s_top : 0.f;
          }
          l *= f;
          if (j) {
            ok = __all_sync(0xffffffffu, wait(smem_u32(&B.pv_done[w]), (n_s - 1) & 1, abort));
            if (!ok) break;
            done = true;
            tc_fence_after();
#pragma unroll 1
            for (int i = 0; i < D; i += 32) {
              uint32_t r[32];
              tmem_ld32_wait(O + i, r);
#pragma unroll
              for (int x = 0; x < 32; ++x) r[x] = __float_as_uint(__uint_as_float(r[x]) * f);
              tmem_st32_wait(O + i, r);
            }
          }
          // s c - m in one rounding, below, is m's own rounding where s is the maximum, and
          // scales all weights of a row by that: by at most 2^(1/2) below FAR, out of their
          // range from 2^27 on.  There the maximum is subtracted from the scores first, here
          // and not on every block's way (prompts of 60 to 1,196 tokens: 79.1 us, there 82.3).
          if (__any_sync(0xffffffffu, from != 0.f)) {
            const uint64_t from2 = pack2(from, from);
#pragma unroll
            for (int i = 0; i < BK / 2; ++i)
              unpack2(add2(pack2(s[2 * i], s[2 * i + 1]), from2), s[2 * i], s[2 * i + 1]);
          }
        }
        const float sub = m == -INFINITY || from != 0.f ? 0.f : -m;
        const uint64_t c2 = pack2(c, c), sub2 = pack2(sub, sub);
        uint64_t l4[4] = {0, 0, 0, 0};
        uint32_t r[BK / 2];
#pragma unroll
        for (int i = 0; i < BK / 2; ++i) {
          float a, b;
          unpack2(fma2(pack2(s[2 * i], s[2 * i + 1]), c2, sub2), a, b);
          a = ex2(a);
          b = ex2(b);
          l4[i & 3] = add2(l4[i & 3], pack2(a, b));
          r[i] = Elem<T>::from2(a, b);
        }
        if (!done) {                                       // it has read P
          ok = __all_sync(0xffffffffu, wait(smem_u32(&B.pv_done[w]), (n_s - 1) & 1, abort));
          if (!ok) break;
          tc_fence_after();
        }
        tmem_st_block(P, r);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&B.p_full[w]));
        float a, b;
        unpack2(add2(add2(l4[0], l4[1]), add2(l4[2], l4[3])), a, b);
        l += a + b;
        ++n_s;
      }
      // the last block's V, cleared by one warp (of the first row tile that uses it)
      if (ok && tail && (warp & 3) == 3) {
        ok = __all_sync(0xffffffffu, wait(smem_u32(&B.tail[tail_stage]), tail_phase, abort));
        if (!ok) break;
        uint8_t* v = smem_raw + (ring + tail_stage * C::TILE - smem_u32(smem_raw));
        // whole 128-byte rows of each panel: the swizzle permutes within a row
        for (int i = (r_t.keys - (blocks - 1) * BK) * 8 + lane; i < BK * 8; i += 32)
#pragma unroll
          for (int c = 0; c < C::PANELS; ++c)
            *reinterpret_cast<uint4*>(v + c * C::PANEL + i * 16) = make_uint4(0, 0, 0, 0);
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&B.full[tail_stage]));
      }
      loads += t.shared ? 2 * max(t.r[0].blocks, t.r[1].blocks) : 2 * (t.r[0].blocks + t.r[1].blocks);
      if (!ok) break;
      const long long tok = (long long)o_t.token + token;
      const int head = o_t.head * p.group + head_in;
      const int unit = t.unit, split = t.split;
      done_tile(k);
      T* out = static_cast<T*>(d.out) + tok * d.out_stride[0] + head * d.out_stride[1];
      // 64 outputs of the warp's 32 rows: every lane's own row to shared memory, then
      // eight lanes a row from there (a row at a time from one lane, a store would
      // touch 32 rows: 4,600 cycles a tile against 3,300)
      const uint32_t keep = __ballot_sync(0xffffffffu, store);
      auto store_rows = [&](int i, const uint32_t (&v)[32]) {
        uint8_t* mine = staged + lane * C::OUT_ROW;
#pragma unroll
        for (int x = 0; x < 8; ++x)
          *reinterpret_cast<uint4*>(mine + 16 * x) = make_uint4(v[4 * x], v[4 * x + 1], v[4 * x + 2], v[4 * x + 3]);
        __syncwarp();
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const int from = 4 * x + (lane >> 3);
          T* to = reinterpret_cast<T*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(out), from));
          if ((keep >> from) & 1)
            *reinterpret_cast<uint4*>(to + i + 8 * (lane & 7)) =
                *reinterpret_cast<const uint4*>(staged + from * C::OUT_ROW + 16 * (lane & 7));
        }
        __syncwarp();
      };
      if (blocks) {
        // every PV of this row tile is complete
        if (!__all_sync(0xffffffffu, wait(smem_u32(&B.pv_done[w]), (n_s - 1) & 1, abort))) break;
        tc_fence_after();
      }
      if (joined) {
        constexpr int EACH = D / 2;                    // outputs per group
        // Every thread reads its row of both row tiles' O, with their m and l (left where
        // Q was: its products are complete, and a CTA has one tile when keys are shared).
        float2* row_ml = reinterpret_cast<float2*>(smem_raw + (sQ - smem_u32(smem_raw)));
        auto ml_at = [&](int w) -> float2& { return row_ml[w * (C::Q_TILE / 8) + row]; };
        ml_at(w) = make_float2(blocks ? m : -INFINITY, blocks ? l : 0.f);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&B.meet));
        if (!__all_sync(0xffffffffu, wait(smem_u32(&B.meet), 0, abort))) break;
        tc_fence_after();
        const float2 ml0 = ml_at(0), ml1 = ml_at(1);
        m = fmaxf(ml0.x, ml1.x);
        const float at_most = m == -INFINITY ? 0.f : m;
        const float f0 = ex2(ml0.x - at_most), f1 = ex2(ml1.x - at_most);
        l = ml0.y * f0 + ml1.y * f1;
        const uint32_t O0 = at_lane + C::O_COL;
        const bool any1 = __any_sync(0xffffffffu, ml1.x != -INFINITY);
        auto both = [&](int i, float (&o)[32]) {        // 32 columns of f0 O_0 + f1 O_1
          uint32_t r[32];
          tmem_ld32_wait(O0 + i, r);
#pragma unroll
          for (int x = 0; x < 32; ++x) o[x] = ml0.x == -INFINITY ? 0.f : __uint_as_float(r[x]) * f0;
          if (any1) {
            tmem_ld32_wait(O0 + C::O_STEP + i, r);
#pragma unroll
            for (int x = 0; x < 32; ++x) o[x] += ml1.x == -INFINITY ? 0.f : __uint_as_float(r[x]) * f1;
          }
        };
        auto store_half = [&](const uint32_t (&v)[32]) {
          if constexpr (EACH == 64) {
            store_rows(w * 64, v);
          } else if (store) {
#pragma unroll
            for (int x = 0; x < 16; x += 4)
              *reinterpret_cast<uint4*>(out + w * 32 + 2 * x) = make_uint4(v[x], v[x + 1], v[x + 2], v[x + 3]);
          }
        };
        if (splits == 1) {
          const float inv = l == 0.f ? 0.f : 1.f / l;
          uint32_t v[32];
#pragma unroll
          for (int i = 0; i < EACH; i += 32) {
            float o[32];
            both(w * EACH + i, o);
#pragma unroll
            for (int x = 0; x < 16; ++x) v[i / 2 + x] = Elem<T>::from2(o[2 * x] * inv, o[2 * x + 1] * inv);
          }
          store_half(v);
          if (store && d.lse && w == 0) d.lse[tok * d.heads + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * LN2;
          continue;
        }
        // this stretch's O [dim][row], m and l; the last CTA of the row tile joins them
        {
          float* part = p.parts + (long long)(unit * splits + split) * PART_FLOATS;
          if (__any_sync(0xffffffffu, m != -INFINITY)) {
#pragma unroll 1
            for (int i = 0; i < EACH; i += 32) {
              float o[32];
              both(w * EACH + i, o);
#pragma unroll
              for (int x = 0; x < 32; ++x) part[(w * EACH + i + x) * BQ + row] = o[x];
            }
          }
          if (w == 0) reinterpret_cast<float2*>(part + 128 * BQ)[row] = make_float2(m, l);
          __threadfence();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&B.part_in));
          if (tid == 0) {
            if (wait(smem_u32(&B.part_in), 0, abort)) {
              B.last = atomicAdd(p.counters + unit, 1) == splits - 1;
              if (B.last) p.counters[unit] = 0;
              __threadfence();
              mbar_arrive(smem_u32(&B.part_out));
            }
          }
          __syncwarp();
        }
        if (!__all_sync(0xffffffffu, wait(smem_u32(&B.part_out), 0, abort))) break;
        if (!B.last) continue;
        const float* all = p.parts + (long long)unit * splits * PART_FLOATS;
        auto ml_of = [&](int q) -> float2 {
          return __ldcg(reinterpret_cast<const float2*>(all + (long long)q * PART_FLOATS + 128 * BQ) + row);
        };
        float top = -INFINITY, sum = 0.f;
        for (int q = 0; q < splits; ++q) top = fmaxf(top, ml_of(q).x);
        const float sub = top == -INFINITY ? 0.f : top;
        for (int q = 0; q < splits; ++q) {
          const float2 ml = ml_of(q);
          sum += ml.y * ex2(ml.x - sub);
        }
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        uint32_t v[32];
#pragma unroll
        for (int i = 0; i < EACH; i += 32) {
          float o[32];
#pragma unroll
          for (int x = 0; x < 32; ++x) o[x] = 0.f;
#pragma unroll 1
          for (int q = 0; q < splits; q += 4) {        // four parts on their way at once
            float f[4], y[4][32];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
              const float mq = q + u < splits ? ml_of(q + u).x : -INFINITY;
              f[u] = ex2(mq - sub) * inv;
              const float* from = all + (long long)(q + u) * PART_FLOATS + (w * EACH + i) * BQ + row;
#pragma unroll
              for (int x = 0; x < 32; ++x)
                y[u][x] = mq == -INFINITY ? 0.f : __ldcg(from + x * BQ);     // nothing seen, perhaps nothing written
            }
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
              for (int x = 0; x < 32; ++x) o[x] += f[u] * y[u][x];
          }
#pragma unroll
          for (int x = 0; x < 16; ++x) v[(i & 32) / 2 + x] = Elem<T>::from2(o[2 * x], o[2 * x + 1]);
        }
        store_half(v);
        if (store && d.lse && w == 0) d.lse[tok * d.heads + head] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * LN2;
        continue;
      }
      if (blocks) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
        for (int i = 0; i < D; i += 64) {
          uint32_t r[64], v[32];
          tmem_ld64_wait(O + i, r);
#pragma unroll
          for (int x = 0; x < 32; ++x)
            v[x] = l == 0.f ? 0u
                            : Elem<T>::from2(__uint_as_float(r[2 * x]) * inv, __uint_as_float(r[2 * x + 1]) * inv);
          if (i + 64 == D) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&B.o_free[w]));
          }
          store_rows(i, v);
        }
      } else if (keep) {
        uint32_t v[32];
#pragma unroll
        for (int x = 0; x < 32; ++x) v[x] = 0u;
        for (int i = 0; i < D; i += 64) store_rows(i, v);
      }
      if (store && d.lse) d.lse[tok * d.heads + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * LN2;
    }
    if (B.gaps && !*abort) fill_gaps<T, D>(p, tid);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, TMEM_COLS);
  }
  if (tid == 0 && B.abort_flag) atomicOr(d.status, KTIR_STATUS_TIMEOUT);
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                  CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                  CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  if (!fn) {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(ptr);
  }
  return fn;
}

// [tokens][heads][dim] in boxes of 64 elements x box_heads x box_tokens; *head_step
// is 0 where all heads are one vector (an expanded axis has stride 0)
bool make_map(CUtensorMap* m, const void* base, bool bf16, int dim, int64_t heads, int64_t tokens,
              const int64_t stride[2], int box_heads, int box_tokens, int* head_step) {
  EncodeTiledFn enc = encode_fn();
  if (!enc) return false;
  *head_step = box_heads;
  if (heads > 1 && stride[1] == 0) {
    if (box_heads > 1) return false;
    heads = 1;
    *head_step = 0;
  }
  cuuint64_t dims[3] = {(cuuint64_t)dim, (cuuint64_t)heads, (cuuint64_t)tokens};
  // an axis with one entry has no stride of its own
  cuuint64_t strides[2] = {(cuuint64_t)(heads > 1 ? stride[1] : dim) * 2, (cuuint64_t)(tokens > 1 ? stride[0] : heads * dim) * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_tokens};
  cuuint32_t estr[3] = {1, 1, 1};
  return enc(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
             const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D>
int launch(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const PromptParams& p,
           unsigned grid, cudaStream_t stream) {
  constexpr int BYTES = Cfg<D>::BYTES + 1024;
  static bool ready[MAX_DEVICES] = {};
  const int dev = current_device();
  if (dev < 0) return ktir_set_error(KTIR_ERR_CUDA, "ktir_prompt_attention: no usable current device");
  if (!ready[dev]) {
    if (cudaFuncSetAttribute(k_prompt_attention<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, BYTES) !=
        cudaSuccess)
      return ktir_set_error(KTIR_ERR_CUDA, "ktir_prompt_attention: shared-memory attribute refused");
    // the split of registers inside the kernel draws on what it is launched with
    cudaFuncAttributes attr;
    if (cudaFuncGetAttributes(&attr, k_prompt_attention<T, D>) != cudaSuccess ||
        attr.numRegs * THREADS < SOFTMAX_REGS * 256 + OTHER_REGS * 128)
      return ktir_set_error(KTIR_ERR_CUDA, "ktir_prompt_attention: built with too few registers for its split");
    ready[dev] = true;
  }
  return launched(launch_pdl(k_prompt_attention<T, D>, grid, THREADS, BYTES, stream, tq, tk, tv, p),
                  "ktir_prompt_attention: launch failed");
}

}  // namespace

extern "C" int64_t ktir_prompt_attention_workspace(void) { return PARTS_BYTES + MAX_PARTS * 4; }

extern "C" int ktir_prompt_attention(const KtirPromptDesc* d, void* stream) {
  if (!d) return ktir_set_error(KTIR_ERR_ARG, "ktir_prompt_attention: null argument");
  if (d->tokens == 0) return KTIR_OK;
  if (!d->q || !d->out || !d->offsets || !d->kv_offsets || !d->status ||
      (d->kv_tokens > 0 && (!d->k || !d->v)))
    return ktir_set_error(KTIR_ERR_ARG, "ktir_prompt_attention: null argument");
  if (d->dtype != KTIR_F16 && d->dtype != KTIR_BF16)
    return ktir_set_error(KTIR_ERR_UNSUPPORTED, "ktir_prompt_attention: needs f16 or bf16");
  if (d->dim != 64 && d->dim != 128)
    return ktir_set_error(KTIR_ERR_UNSUPPORTED, "ktir_prompt_attention: needs dim 64 or 128");
  if (d->batch > (1 << 20))      // every CTA looks at every sequence for each weight of a tile (40,000 of 20 tokens: 2.6 ms)
    return ktir_set_error(KTIR_ERR_UNSUPPORTED, "ktir_prompt_attention: more than 2^20 sequences in a call");
  if (d->batch < 1 || d->tokens < 0 || d->tokens > 0x7fffffffLL ||
      d->kv_tokens < 0 || d->kv_tokens > 0x7fffffffLL || d->heads < 1 || d->kv_heads < 1 ||
      d->heads % d->kv_heads || d->heads > (1 << 16))
    return ktir_set_error(KTIR_ERR_ARG, "ktir_prompt_attention: extent out of range");
  if (d->heads / d->kv_heads > 128)
    return ktir_set_error(KTIR_ERR_UNSUPPORTED, "ktir_prompt_attention: heads / kv_heads above 128");
  if (!(d->scale > 0.f) || !isfinite(d->scale))
    return ktir_set_error(KTIR_ERR_UNSUPPORTED, "ktir_prompt_attention: needs a positive, finite scale");
  const int64_t qe[2] = {d->tokens, d->heads}, ke[2] = {d->kv_tokens, d->kv_heads};
  if (!vector_strides(d->q_stride, qe, 2) || !vector_strides(d->out_stride, qe, 2) ||
      !vector_strides(d->k_stride, ke, 2) || !vector_strides(d->v_stride, ke, 2) || !aligned16(d->q) ||
      !aligned16(d->k) || !aligned16(d->v) || !aligned16(d->out) || !aligned16(d->workspace))
    return ktir_set_error(KTIR_ERR_UNSUPPORTED,
                          "ktir_prompt_attention: head vectors must start on 16-byte boundaries");
  if (!apart(d->out_stride, qe, 2))
    return ktir_set_error(KTIR_ERR_ARG, "ktir_prompt_attention: rows of out share memory");
  const bool bf16 = d->dtype == KTIR_BF16;
  PromptParams p;
  p.d = *d;
  p.group = d->heads / d->kv_heads;
  p.tile_tokens = BQ / p.group;
  // without keys nothing is loaded, but the maps must be valid
  const int64_t none[2] = {d->dim, d->dim};
  const int64_t keys = d->kv_tokens > 0 ? d->kv_tokens : 1;
  const int block = d->dim == 128 ? Cfg<128>::BK : Cfg<64>::BK;
  CUtensorMap tq, tk, tv;
  if (!make_map(&tq, d->q, bf16, d->dim, d->heads, d->tokens, d->q_stride, p.group, p.tile_tokens,
                &p.q_head_step) ||
      !make_map(&tk, d->kv_tokens > 0 ? d->k : d->q, bf16, d->dim, d->kv_tokens > 0 ? d->kv_heads : 1, keys,
                d->kv_tokens > 0 ? d->k_stride : none, 1, block, &p.k_head_step) ||
      !make_map(&tv, d->kv_tokens > 0 ? d->v : d->q, bf16, d->dim, d->kv_tokens > 0 ? d->kv_heads : 1, keys,
                d->kv_tokens > 0 ? d->v_stride : none, 1, block, &p.v_head_step))
    return ktir_set_error(KTIR_ERR_UNSUPPORTED, "ktir_prompt_attention: strides that a tensor map does not take");
  const int sms = sm_count();
  if (sms < 1) return ktir_set_error(KTIR_ERR_CUDA, "ktir_prompt_attention: no usable current device");
  // at most this many row tiles: every sequence may end in a part of one
  const long long tiles = (d->tokens / p.tile_tokens + d->batch) * d->kv_heads;
  if (tiles > 0x3fffffffLL) return ktir_set_error(KTIR_ERR_UNSUPPORTED, "ktir_prompt_attention: too many tiles");
  p.token_magic = (uint32_t)(((1ULL << 32) + p.tile_tokens - 1) / p.tile_tokens - (p.tile_tokens == 1));
  p.pair_magic = (uint32_t)(((1ULL << 32) + 2 * p.tile_tokens - 1) / (2 * p.tile_tokens));
  p.parts = d->workspace && d->workspace_bytes >= ktir_prompt_attention_workspace() ? static_cast<float*>(d->workspace) : nullptr;
  p.counters = reinterpret_cast<int*>(static_cast<char*>(d->workspace) + PARTS_BYTES);
  // with a workspace the SMs left over share the keys, if there are enough of them
  const unsigned grid = (unsigned)(tiles < sms && !(p.parts && d->kv_tokens > 4 * block) ? tiles : sms);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (d->dim == 64)
    return bf16 ? launch<__nv_bfloat16, 64>(tq, tk, tv, p, grid, s) : launch<__half, 64>(tq, tk, tv, p, grid, s);
  return bf16 ? launch<__nv_bfloat16, 128>(tq, tk, tv, p, grid, s) : launch<__half, 128>(tq, tk, tv, p, grid, s);
}

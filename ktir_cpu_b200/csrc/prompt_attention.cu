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
// kv head lie side by side, 128 / g tokens per tile, so that every row of a
// tile uses the same K and V whatever g is, and a short prompt fills more of a
// tile.
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
//                   CTAs, so that the last ones to finish are the shortest; and
//                   sets V's rows past the sequence's last key to zero (they
//                   belong to another sequence; a weight of 0 does not cancel
//                   an infinity there)
// TMEM holds S, P and O of both row tiles apart, which at dim 128 leaves room for
// blocks of 80 keys (128 at dim 64).
// The running maximum moves only when a row's maximum exceeds it by more than
// 2^8; O's rows are then rescaled in TMEM, after the product before.
// Precision: S, O, m and l in f32; P is rounded to the element type for the
// second product (tcgen05 wants one type for both operands), half an ulp per
// weight; l adds the unrounded weights.
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
constexpr int SCHED_READERS = 11;    // 8 softmax warps, two MMA, TMA
constexpr float RESCALE_THRESHOLD = 8.0f;   // log2 units
constexpr int SOFTMAX_REGS = 208, OTHER_REGS = 80;
constexpr uint32_t TMEM_COLS = 512;

// TMEM has 512 columns for S (BK), P (BK / 2) and O (D) of two row tiles.
template <int D>
struct Cfg {
  static constexpr int BK = D == 128 ? 80 : 128;    // keys of a block
  static constexpr int PANELS = D / 64;             // of 64 elements, rows of 128 bytes, swizzled
  static constexpr int Q_PANEL = BQ * 128, Q_TILE = PANELS * Q_PANEL;
  static constexpr int PANEL = BK * 128, TILE = PANELS * PANEL;      // a K or V block
  static constexpr int STAGES = D == 128 ? 8 : 10;
  static constexpr int BYTES = 2 * Q_TILE + STAGES * TILE;
  // first columns of row tile 0, and from one row tile to the next
  static constexpr uint32_t S_COL = 0, S_STEP = 128, O_COL = D == 128 ? 256 : 384, O_STEP = D;
  static constexpr uint32_t P_COL = D == 128 ? 80 : 256, P_STEP = D == 128 ? 128 : 64;
};
constexpr int MAX_STAGES = 10;

struct Tile {
  int stop;
  int token;      // first token of the tile (of row tile 0)
  int tokens;     // of the sequence from there on
  int seen;       // keys that the first token sees (causal)
  int keys;       // of the sequence
  int key0;       // its first key
  int head;       // kv head
  int blocks[2];  // key blocks of each row tile
};

struct Shared {
  uint64_t q_full[2], q_empty[2];
  uint64_t full[MAX_STAGES], empty[MAX_STAGES];
  uint64_t s_full[2], s_free[2], p_full[2], pv_done[2], o_free[2];
  uint64_t tail[MAX_STAGES];        // a V block with rows past the last key has arrived
  uint64_t drain[2];
  uint64_t sched_full[SCHED], sched_empty[SCHED];
  Tile tile[SCHED];
  uint32_t tmem_base;
  int abort_flag;
};

struct PromptParams {
  KtirPromptDesc d;
  int group;            // query heads per kv head
  int tile_tokens;      // tokens of a row tile
  int k_head_step, v_head_step, q_head_step;   // 0 where all heads share one vector
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
// Tile i of a sequence (n tokens, m keys) holds tokens [i T, (i + 1) T), T = two row
// tiles; its weight is the number of key blocks that its last token sees.  Tiles
// are numbered by falling weight over all sequences; within a weight by
// sequence, and each tile once per kv head.
struct Seq {
  int n, m, tiles;
};

__device__ __forceinline__ Seq sequence(const KtirPromptDesc& d, long long b, int T, bool& bad) {
  const int q0 = d.offsets[b], q1 = d.offsets[b + 1], k0 = d.kv_offsets[b], k1 = d.kv_offsets[b + 1];
  bad = q0 < 0 || q1 < q0 || q1 > d.tokens || k0 < 0 || k1 < k0 || k1 > d.kv_tokens;
  Seq s;
  s.n = bad ? 0 : q1 - q0;
  s.m = bad ? 0 : k1 - k0;
  s.tiles = (s.n + T - 1) / T;
  return s;
}

// tiles of weight at least `w`: the last ones of the sequence
template <int BK>
__device__ __forceinline__ int heavier(const Seq& s, int w, int T, int causal) {
  if (w <= 0) return s.tiles;
  const int need = (w - 1) * BK;             // more than this many keys seen
  if (s.m <= need) return 0;
  if (!causal) return s.tiles;
  const int x = need - (s.m - s.n);          // (i + 1) T > x
  return x <= 0 ? s.tiles : s.tiles - x / T;
}

__device__ __forceinline__ int warp_sum(int v) {
#pragma unroll
  for (int w = 16; w; w >>= 1) v += __shfl_xor_sync(0xffffffffu, v, w);
  return v;
}

template <int BK>
__device__ int tiles_of_weight(const KtirPromptDesc& d, int w, int T, int lane) {
  int c = 0;
  for (long long b = lane; b < d.batch; b += 32) {
    bool bad;
    c += heavier<BK>(sequence(d, b, T, bad), w, T, d.causal);
  }
  return warp_sum(c);
}

// tile number `x` (0 = heaviest), by one warp
template <int BK>
__device__ void find_tile(const KtirPromptDesc& d, int x, int head, int T, int heaviest, int lane, Tile& t) {
  int lo = 0, hi = heaviest + 1;             // count(lo) > x >= count(hi)
  int above = 0;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    const int c = tiles_of_weight<BK>(d, mid, T, lane);
    if (c > x) {
      lo = mid;
    } else {
      hi = mid;
      above = c;
    }
  }
  int r = x - above;
  for (long long b0 = 0; b0 < d.batch; b0 += 32) {
    const long long b = b0 + lane;
    Seq s = {0, 0, 0};
    int first = 0, count = 0;
    bool bad;
    if (b < d.batch) {
      s = sequence(d, b, T, bad);
      const int c = heavier<BK>(s, lo, T, d.causal);
      count = c - heavier<BK>(s, lo + 1, T, d.causal);
      first = s.tiles - c;
    }
    int incl = count;
#pragma unroll
    for (int w = 1; w < 32; w <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, incl, w);
      if (lane >= w) incl += o;
    }
    const int all = __shfl_sync(0xffffffffu, incl, 31);
    if (r >= all) {
      r -= all;
      continue;
    }
    if (r >= incl - count && r < incl) {
      const int i = first + r - (incl - count), at = i * T, half = T / 2;
      t.stop = 0;
      t.token = d.offsets[b] + at;
      t.tokens = s.n - at;
      t.seen = at + s.m - s.n + 1;
      t.keys = s.m;
      t.key0 = d.kv_offsets[b];
      t.head = head;
      for (int w = 0; w < 2; ++w) {
        const int here = min(half, t.tokens - w * half);       // tokens of the row tile
        const int end = d.causal ? min(s.m, at + w * half + here + s.m - s.n) : s.m;
        t.blocks[w] = here > 0 && end > 0 ? (end + BK - 1) / BK : 0;
      }
    }
    break;
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

  // announced tiles, read by whole warps: false at the end (or on an abort)
  auto next_tile = [&](int k, Tile& t) -> bool {
    const int s = k % SCHED;
    if (!__all_sync(0xffffffffu, wait(smem_u32(&B.sched_full[s]), (k / SCHED) & 1, abort))) return false;
    t = B.tile[s];
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&B.sched_empty[s]));
    return !t.stop;
  };

  if (warp >= 8) {
    fewer_registers<OTHER_REGS>();
    if (warp == 11) {
      // ---------------- tile finder ----------------
      const int span = 2 * p.tile_tokens;
      int heaviest = 0, total = 0;
      bool any_bad = false;
      for (long long b = lane; b < d.batch; b += 32) {
        bool bad;
        const Seq s = sequence(d, b, span, bad);
        any_bad |= bad;
        if (s.n) heaviest = max(heaviest, (s.m + BK - 1) / BK);
        total += s.tiles;
      }
      if (blockIdx.x == 0) {
        if (lane == 0) any_bad |= d.offsets[0] != 0 || d.offsets[d.batch] != d.tokens;
        if (any_bad) atomicOr(d.status, KTIR_STATUS_BAD_INDEX);
      }
      total = warp_sum(total);
  #pragma unroll
      for (int w = 16; w; w >>= 1) heaviest = max(heaviest, __shfl_xor_sync(0xffffffffu, heaviest, w));
      const long long all = (long long)total * d.kv_heads;
      int next = 0, fix = 0, loads = 0;         // tile to announce, tile to look after, ring loads before it
      bool stop = false;
      uint32_t phase = 0;                       // of the ring stages' tail barriers
      for (uint32_t idle = 0; !stop || fix < next - 1;) {
        bool moved = false;
        const int s = next % SCHED;
        if (!stop && next < fix + SCHED &&
            (next < SCHED || __all_sync(0xffffffffu, mbar_test_wait(smem_u32(&B.sched_empty[s]),
                                                                    (next / SCHED - 1) & 1)))) {
          const long long x =
              (long long)next * gridDim.x + ((next & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
          // back and forth, a CTA may have a tile in the last round after having none before it
          stop = (long long)next * gridDim.x >= all;
          if (stop) {
            if (lane == 0) B.tile[s].stop = 1;
          } else if (x < all) {
            find_tile<BK>(d, (int)(x / d.kv_heads), (int)(x % d.kv_heads), span, heaviest, lane, B.tile[s]);
          } else if (lane == 0) {
            Tile& t = B.tile[s];
            t.stop = 0;
            t.tokens = t.blocks[0] = t.blocks[1] = t.keys = 0;
            t.token = t.key0 = t.head = 0;
            t.seen = 0;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&B.sched_full[s]));
          ++next;
          moved = true;
        }
        if (fix < next - (stop ? 1 : 0)) {
          // V rows past the last key of tile `fix`
          const Tile& t = B.tile[fix % SCHED];
          const int blocks = max(t.blocks[0], t.blocks[1]), left = t.keys - (blocks - 1) * BK;
          const int r = (loads + 2 * blocks - 1) % STAGES;
          const bool tail = blocks && left < BK;
          if (!tail || __all_sync(0xffffffffu, mbar_test_wait(smem_u32(&B.tail[r]), (phase >> r) & 1))) {
            if (tail) {
              phase ^= 1u << r;
              uint8_t* v = smem_raw + (ring + r * C::TILE - smem_u32(smem_raw));
              // whole 128-byte rows of each panel: the swizzle permutes within a row
              for (int i = left * 8 + lane; i < BK * 8; i += 32)
#pragma unroll
                for (int c = 0; c < C::PANELS; ++c)
                  *reinterpret_cast<uint4*>(v + c * C::PANEL + i * 16) = make_uint4(0, 0, 0, 0);
              fence_proxy_async();
              __syncwarp();
              if (lane == 0) mbar_arrive(smem_u32(&B.full[r]));
            }
            loads += 2 * blocks;
            ++fix;
            moved = true;
          }
        }
        if (moved) {
          idle = 0;
        } else {
          if (__any_sync(0xffffffffu, *abort != 0)) break;
          if (++idle > kSpinLimit) {
            *abort = 1;
            break;
          }
          __nanosleep(40);
        }
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
      Tile t;
      bool ok = true;
      for (int k = 0; ok && next_tile(k, t); ++k) {
          if (leader) {
          const int blocks = max(t.blocks[0], t.blocks[1]);
          for (int w = 0; ok && w < 2; ++w) {
            if (!t.blocks[w]) continue;
            if (q_loads[w] && !wait(smem_u32(&B.q_empty[w]), (q_loads[w] - 1) & 1, abort)) {
              ok = false;
              break;
            }
            const uint32_t bar = smem_u32(&B.q_full[w]);
            mbar_arrive_expect_tx(bar, q_bytes);
#pragma unroll
            for (int c = 0; c < C::PANELS; ++c)
              tma_load_3d(sQ + w * C::Q_TILE + c * C::Q_PANEL, &tq, bar, 64 * c, t.head * p.q_head_step,
                          t.token + w * p.tile_tokens);
            ++q_loads[w];
          }
          auto load = [&](bool kv, int j) -> bool {
            const int s = loads % STAGES;
            if (loads >= STAGES && !wait(smem_u32(&B.empty[s]), (loads / STAGES - 1) & 1, abort)) return false;
            // V rows past the last key: warp 11 passes the block on when it has cleared them
            const bool tail = kv && (j + 1) * BK > t.keys;
            const uint32_t bar = smem_u32(tail ? &B.tail[s] : &B.full[s]);
            was_tail = (was_tail & ~(1u << s)) | (tail ? 1u << s : 0u);
            if (tail) tail_phase ^= 1u << s;
            mbar_arrive_expect_tx(bar, C::TILE);
#pragma unroll
            for (int c = 0; c < C::PANELS; ++c)
              tma_load_3d(ring + s * C::TILE + c * C::PANEL, kv ? &tv : &tk, bar, 64 * c,
                          t.head * (kv ? p.v_head_step : p.k_head_step), t.key0 + j * BK);
            ++loads;
            return true;
          };
          // in the order of their use: K_0, K_1, then V_j and K_{j+2}
          for (int j = 0; ok && j < 2 && j < blocks; ++j) ok = load(false, j);
          for (int j = 0; ok && j < blocks; ++j) {
            ok = load(true, j);
            if (ok && j + 2 < blocks) ok = load(false, j + 2);
          }
        }
        ok = __all_sync(0xffffffffu, ok);
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
        Tile t;
        bool ok = true;
        for (int k = 0; ok && next_tile(k, t); ++k) {
          if (leader) {
            const int mine = t.blocks[w], blocks = max(mine, t.blocks[w ^ 1]);
            // S(j) from the K block just arrived, which both row tiles give back
            auto issue_s = [&](int j) -> bool {
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
              return true;
            };
            auto issue_pv = [&](int j) -> bool {
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
              return true;
            };
            for (int j = 0; ok && j < 2 && j < blocks; ++j) ok = issue_s(j);
            for (int j = 0; ok && j < blocks; ++j) {
              ok = issue_pv(j);
              if (ok && j + 2 < blocks) ok = issue_s(j + 2);
            }
          }
          ok = __all_sync(0xffffffffu, ok);
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
    int n_s = 0;                                     // blocks so far: S, P and PV each
    Tile t;
    for (int k = 0; next_tile(k, t); ++k) {
      const int at = w * p.tile_tokens + token;       // of the tile's tokens
      const bool store = real && at < t.tokens;
      const int blocks = t.blocks[w];
      const int limit = d.causal ? t.seen + at : t.keys;                           // keys this row sees
      const int least = d.causal ? t.seen + w * p.tile_tokens : t.keys;            // and the tile's first row
      float m = -INFINITY, l = 0.f;
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
        const float top = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * c;
        const bool move = top > m + RESCALE_THRESHOLD;     // also from -inf
        bool done = j == 0;                                // PV of the block before
        if (__any_sync(0xffffffffu, move)) {
          const float f = move ? ex2(m - top) : 1.f;
          if (move) m = top;
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
        }
        const float sub = m == -INFINITY ? 0.f : -m;
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
      if (!ok) break;
      const long long tok = (long long)t.token + at;
      const int head = t.head * p.group + head_in;
      T* out = static_cast<T*>(d.out) + tok * d.out_stride[0] + head * d.out_stride[1];
      if (blocks) {
        // every PV of this row tile is complete
        if (!__all_sync(0xffffffffu, wait(smem_u32(&B.pv_done[w]), (n_s - 1) & 1, abort))) break;
        tc_fence_after();
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
        for (int i = 0; i < D; i += 32) {
          uint32_t r[32];
          tmem_ld32_wait(O + i, r);
          if (store) {
#pragma unroll
            for (int x = 0; x < 32; x += 8) {
              uint32_t v[4];
#pragma unroll
              for (int y = 0; y < 4; ++y)
                v[y] = l == 0.f ? 0u
                                : Elem<T>::from2(__uint_as_float(r[x + 2 * y]) * inv,
                                                 __uint_as_float(r[x + 2 * y + 1]) * inv);
              *reinterpret_cast<uint4*>(out + i + x) = make_uint4(v[0], v[1], v[2], v[3]);
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&B.o_free[w]));
      } else if (store) {
#pragma unroll
        for (int i = 0; i < D; i += 8) *reinterpret_cast<uint4*>(out + i) = make_uint4(0, 0, 0, 0);
      }
      if (store && d.lse) d.lse[tok * d.heads + head] = l == 0.f ? -INFINITY : (m + log2f(l)) * LN2;
    }
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
  if (d->batch < 1 || d->batch > (1 << 24) || d->tokens < 0 || d->tokens > 0x7fffffffLL ||
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
      !aligned16(d->k) || !aligned16(d->v) || !aligned16(d->out))
    return ktir_set_error(KTIR_ERR_UNSUPPORTED,
                          "ktir_prompt_attention: head vectors must start on 16-byte boundaries");
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
  // at most this many tiles: every sequence may end in a part of one
  const long long tiles = (d->tokens / (2 * p.tile_tokens) + d->batch) * d->kv_heads;
  if (tiles > 0x7fffffffLL) return ktir_set_error(KTIR_ERR_UNSUPPORTED, "ktir_prompt_attention: too many tiles");
  const unsigned grid = (unsigned)(tiles < sms ? tiles : sms);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (d->dim == 64)
    return bf16 ? launch<__nv_bfloat16, 64>(tq, tk, tv, p, grid, s) : launch<__half, 64>(tq, tk, tv, p, grid, s);
  return bf16 ? launch<__nv_bfloat16, 128>(tq, tk, tv, p, grid, s) : launch<__half, 128>(tq, tk, tv, p, grid, s);
}

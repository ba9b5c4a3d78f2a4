// Attention of one new token per sequence over its paged keys and values.
//
//   o = sum_j e^(x_j - m) v_j / l,   l = sum_j e^(x_j - m),   m = max_j x_j,
//   x_j = scale q . k_j
//
// Bound by memory: every cached key and value is read once and meets the g =
// heads / kv_heads queries that share it, 2 g operations per byte.  So the
// cache streams through shared memory in 16-byte asynchronous copies, and the
// two products run on mma.sync (m16n8k16) with 16 keys, or 16 elements of the
// values, as its rows and 8 query heads as its columns: x^T = K q^T, then o^T +=
// V^T p^T (tcgen05's 64 or 128 rows would be mostly empty).  A head tile has 8
// heads, or 16 where g is above 8; a larger g takes several.  (32 sequences of 200 to
// 4000 keys, 8 kv heads, floor 34.0 us: g = 4 43.7 us, 12 50.2, 16 52.4; dim 64, floor
// 17.0: g = 8 29.5, 16 36.0, where the second tile's queries and outputs spill 80 bytes.)
//
// Split over the cache: the 64-key tiles of all sequences form one list, cut
// into equal stretches, one per group of CTAs; the CTAs of a group take the
// head tiles over the same stretch (so a page's heads, neighbours in a
// token-major cache, are read at the same time).  The work is even however the
// lengths differ.  A few sequences get groups of their own instead, whole or in
// even parts, and short ones are not cut, where that makes a stretch little
// longer.  Within a CTA each of the four warps owns 16 keys of every tile, with its
// own ring of copies in flight, its own running m, l and o: the warps meet only
// where a sequence ends.  A stretch that holds part of a sequence leaves (m, l, o)
// in the workspace, and the last of the CTAs that share the sequence joins the
// parts in the order of the list (so the result does not depend on which was last).
//
// Precision: scores, m, l and o in f32; the weights p are rounded to the
// element type for the second product (as the values are), at most one half
// ulp each (in f16 2^-32 of a row's largest where that is more).  m moves only when
// the maximum grows by more than 2^8, so the largest p of a row lies between 1 and 2^8,
// and in f16, where m is kept 2^7 lower (Elem::LIFT), between 2^7 and 2^15.
#include "serve_common.cuh"

using namespace ktir::serve;

namespace {

constexpr int WARPS = 4;
constexpr int THREADS = WARPS * 32;
constexpr int KPW = 16;                    // keys per warp and tile
constexpr int TILE = WARPS * KPW;          // keys per tile
constexpr int ROWS = 16;                   // query heads per head tile at most
constexpr int MAX_CTAS = 512;              // of a launch that splits sequences
constexpr int MIN_TILES = 2;               // per stretch: both in flight at once
constexpr int FIT_BATCH = 64;              // sequences of a launch that may get CTAs of their own,
// And tiles of an even stretch then.  8 sequences of 8.9 (and 16 of 6.5) tiles to a stretch,
// 8 kv heads of 128: CTAs of their own 21.4 (17.4) us, even stretches 23.0 (19.6).  Above
// that it goes either way: 8 sequences of 13.6 28.1 against 30.1, 32 of 13.3 29.3 against
// 28.9, 16 of 10.9 (20 heads of 64) 22.6 against 22.3.
constexpr int FIT_TILES = 10;
constexpr unsigned SNAP = 12;              // tiles of a sequence that is not cut in two
constexpr int LOOK = 3;                    // tiles between a look into the page table and the copy
constexpr float RESCALE_THRESHOLD = 8.0f;  // log2 units
constexpr int PART_STRIDE = ROWS * (128 + 2);   // floats of a part: o, then (m, l) per row
constexpr int64_t PARTS_BYTES = (int64_t)MAX_CTAS * 2 * PART_STRIDE * 4;
static_assert(PARTS_BYTES == KTIR_PAGED_DECODE_PARTS_BYTES);

struct DecodeParams {
  KtirPagedDecodeDesc d;
  int group;          // query heads per kv head
  int htiles;         // head tiles per kv head
  int ht;             // kv_heads * htiles
  int groups;         // CTA groups of the launch
  int page_shift;     // log2(page_size), or -1
  int same;           // K and V have the same strides
  float* parts;
  int* counters;      // [batch][ht], zero between calls
};

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                                 uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4],
                                                        uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// 16 bytes, or 16 zero bytes where `bytes` is 0 (nothing is read then)
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
// an 8 x 8 tile of 16-bit values transposed across the warp
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// where a stretch stands: tile t of sequence b's nt tiles (len keys)
struct Cursor {
  long long b;
  int t, nt, len;
};

template <int D>
struct Cfg {
  static constexpr int CHUNKS = D / 8;                 // 16-byte pieces of a row
  static constexpr int ROW_BYTES = D * 2;
  static constexpr int HALF_STAGE = KPW * ROW_BYTES;   // K, then V
  static constexpr int STAGE = 2 * HALF_STAGE;
  // what hides a tile's latency: copies in flight at dim 128 (24 KiB per warp), more
  // warps at dim 64, whose tiles are half as long (45 sequences of 20 heads: 26 us
  // against 32 with two CTAs of six stages; at dim 128 three CTAs leave two stages,
  // 34 us against 32 for 32 sequences)
  static constexpr int CTAS_PER_SM = D == 128 ? 2 : 3;
  static constexpr int STAGES = 3;
  static constexpr int RING = WARPS * STAGES * STAGE;
  static constexpr int JOIN = WARPS * 8 * D * 4;       // eight heads' outputs of each warp
  static constexpr int SMEM = RING + JOIN;
};

template <typename T, int D, int NT>       // NT: tiles of 8 heads
__global__ void __launch_bounds__(THREADS, Cfg<D>::CTAS_PER_SM)
    k_paged_decode(const __grid_constant__ DecodeParams p) {
  using C = Cfg<D>;
  const KtirPagedDecodeDesc& d = p.d;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long long s_scan[WARPS];
  __shared__ unsigned s_longest[WARPS];
  __shared__ long long s_start[2], s_end[2];           // sequence, its first tile
  __shared__ int s_own[2];                             // CTA groups of the sequence, where it has its own
  __shared__ float2 s_ml[WARPS][ROWS];
  __shared__ int s_last;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int grp = blockIdx.x / p.ht, ht = blockIdx.x - grp * p.ht;
  const int kvh = ht / p.htiles, head0 = kvh * p.group + (ht - kvh * p.htiles) * (8 * NT);
  const int nrows = min(8 * NT, (kvh + 1) * p.group - head0);
  const long long most = d.max_pages * d.page_size;

  // tiles of a sequence; a length outside its range counts as 0
  auto length_of = [&](long long b) -> int {
    const int len = d.lengths[b];
    return len < 0 || len > most ? 0 : len;
  };

  pdl_launch();
  pdl_wait();

  // sequences without keys give zeros
  auto zeros = [&]() {
    for (long long b = grp; b < d.batch; b += p.groups) {
      if (length_of(b) == 0) {
        for (int i = tid; i < nrows * C::CHUNKS; i += THREADS) {
          const int r = i / C::CHUNKS, c = i - r * C::CHUNKS;
          *reinterpret_cast<uint4*>(static_cast<T*>(d.out) + b * d.out_stride[0] +
                                    (head0 + r) * d.out_stride[1] + c * 8) = make_uint4(0, 0, 0, 0);
        }
        if (d.lse && tid < nrows) d.lse[b * d.heads + head0 + tid] = -INFINITY;
      }
    }
  };

  // This CTA's stretch of the list: tiles [t_begin, t_end), the first one tile `first`
  // of sequence `start`, whose tiles begin at `base`.
  long long t_begin, t_end, base, start, ng = 0, total = 0;
  int first;
  bool fits = false;
  constexpr int FREE = NT == 1 ? 4 : 6;       // tiles that one CTA takes as fast as several join their parts
  // this CTA's part of a sequence that CTA groups own0 .. own0 + own - 1 have to themselves
  auto take = [&](int tiles, int own0, int own) {
    const int least = (unsigned)tiles / (unsigned)own, left = tiles - least * own, piece = grp - own0;
    base = 0;
    first = piece * least + min(piece, left);
    t_begin = first;
    t_end = first + least + (piece < left ? 1 : 0);
    if (tid == 0) {
      s_own[0] = own0;
      s_own[1] = own0 + own - 1;
    }
  };
  if (d.batch == 1) {                         // nothing to count (77 keys: 4.5 us against 5.2, 400: 6.6 against 7.9)
    const int len = d.lengths[0];
    const bool bad = len < 0 || len > most;
    if (bad && blockIdx.x == 0 && tid == 0) atomicOr(d.status, KTIR_STATUS_BAD_INDEX);
    if (bad || len == 0) {
      zeros();
      return;
    }
    const int tiles = (int)(((unsigned)len + TILE - 1) / TILE);
    const int own = tiles <= FREE ? 1 : min(p.groups, tiles > 16 ? (tiles + 1) / 2 : tiles);
    if (grp >= own) return;
    fits = true;
    start = 0;
    take(tiles, 0, own);
  } else if (d.batch <= min(FIT_BATCH, p.groups)) {
    // Few sequences: each gets CTAs of its own if that costs at most three tiles more
    // than even stretches (ending one sequence and beginning another costs as much: 7
    // sequences of 700 keys, 5 heads of 64: 7.5 us against 10.3).  One of few tiles is
    // not split, since joining parts takes about as long as three of them.
    const int each = d.batch > 32 ? 2 : 1;
    unsigned t[2] = {0, 0};
    bool none = false, bad = false;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const long long b = lane * each + x;
      if (x < each && b < d.batch) {
        const int len = d.lengths[b];
        if (len < 0 || len > most) bad = true;
        else t[x] = ((unsigned)len + TILE - 1) / TILE;
        none |= t[x] == 0;
      }
    }
    if (bad && blockIdx.x == 0 && warp == 0) atomicOr(d.status, KTIR_STATUS_BAD_INDEX);
    if (__any_sync(0xffffffffu, none)) zeros();
    const unsigned sum = __reduce_add_sync(0xffffffffu, t[0] + t[1]);     // at most 64 x 2^25
    const unsigned longest = __reduce_max_sync(0xffffffffu, max(t[0], t[1]));
    // 16 parts are joined at once
    unsigned size = max((sum + p.groups - 1) / p.groups, longest > 16 ? 2u : 1u);
    auto pieces = [&](unsigned tiles, unsigned size, float over) -> unsigned {
      return tiles <= max(size, (unsigned)FREE) ? (tiles ? 1u : 0u)
                                                : (unsigned)(((float)(min(tiles, 8191u) + size) - 0.5f) * over);
    };
    int more = 0;
    if (size <= FIT_TILES) {
      unsigned two[2];                         // what sizes size .. size + 3 take, two to a word
#pragma unroll
      for (unsigned x = 0; x < 2; ++x) {
        const unsigned a = size + 2 * x, b = a + 1;
        const float oa = __frcp_rn((float)a), ob = __frcp_rn((float)b);
        two[x] = __reduce_add_sync(0xffffffffu, min(511u, pieces(t[0], a, oa) + pieces(t[1], a, oa)) +
                                                    (min(511u, pieces(t[0], b, ob) + pieces(t[1], b, ob)) << 16));
      }
      const unsigned limit = min(p.groups, 510);
#pragma unroll
      for (int x = 3; x >= 0; --x)
        if (((two[x >> 1] >> (16 * (x & 1))) & 0xffffu) <= limit) {
          fits = true;
          more = x;
        }
    }
    if (fits) {
      size += more;
      const float over = __frcp_rn((float)size);
      const int n0 = (int)pieces(t[0], size, over), mine = n0 + (int)pieces(t[1], size, over);
      int incl = mine;
#pragma unroll
      for (int w = 1; w < 32; w <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, incl, w);
        if (lane >= w) incl += o;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, grp >= incl - mine && grp < incl);
      if (!hit) return;
      const int from = __ffs(hit) - 1;
      const int at = incl - mine, second = grp >= at + n0 ? 1 : 0;       // of the lane's two sequences
      start = __shfl_sync(0xffffffffu, lane * each + second, from);
      const int own0 = __shfl_sync(0xffffffffu, at + (second ? n0 : 0), from);
      const int own = __shfl_sync(0xffffffffu, second ? mine - n0 : n0, from);
      const int tiles = (int)__shfl_sync(0xffffffffu, second ? t[1] : t[0], from);
      take(tiles, own0, own);
    }
  }
  if (!fits) {
    // even stretches: an exclusive scan over runs of sequences
    const long long run = (d.batch + THREADS - 1) / THREADS;
    const long long r0 = min((long long)d.batch, tid * run), r1 = min((long long)d.batch, r0 + run);
    long long mine = 0;
    unsigned longest = 0;
    for (long long b = r0; b < r1; ++b) {
      const int len = d.lengths[b];
      if (len < 0 || len > most) {
        if (blockIdx.x == 0) atomicOr(d.status, KTIR_STATUS_BAD_INDEX);
      } else {
        const unsigned nt = ((unsigned)len + TILE - 1) / TILE;
        mine += nt;
        longest = max(longest, nt);
      }
    }
    long long incl = mine;
#pragma unroll
    for (int w = 1; w < 32; w <<= 1) {
      const long long o = __shfl_up_sync(0xffffffffu, incl, w);
      if (lane >= w) incl += o;
    }
    longest = __reduce_max_sync(0xffffffffu, longest);
    if (lane == 31) s_scan[warp] = incl;
    if (lane == 0) s_longest[warp] = longest;
    __syncthreads();
    long long before = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      if (w < warp) before += s_scan[w];
      total += s_scan[w];
      longest = max(longest, s_longest[w]);
    }
    if (d.batch > min(FIT_BATCH, p.groups)) zeros();      // else done above
    const long long want = (total + MIN_TILES - 1) / MIN_TILES;
    ng = min((long long)p.groups, want);
    if (grp >= ng) return;
    t_begin = total * grp / ng;
    t_end = total * (grp + 1) / ng;
    const long long excl = before + incl - mine;
    // Short sequences stay whole: a stretch then begins and ends where the sequence
    // nearest to its cut does, if that makes it little longer (182 sequences of 75 to
    // 277 keys, 21 heads over 3, dim 64: 11.4 us against 14.4; 211 of 35 to 652, 48 over
    // 12: 38.6 against 42.4; with up to 24 tiles 300 of 500 to 1500 take 184 us against
    // 178).
    const bool snap = longest <= SNAP && longest * ng <= total + FREE * ng;
    auto place = [&](long long t, long long (&at)[2]) {      // sequence, its first tile or the one cut at
      if (t < excl || t >= excl + mine) return;
      long long from = excl;
      for (long long b = r0; b < r1; ++b) {
        const int nt = (length_of(b) + TILE - 1) / TILE;
        if (t < from + nt) {
          const bool next = snap && 2 * (t - from) >= nt;
          at[0] = next ? b + 1 : b;
          at[1] = next ? from + nt : from;
          break;
        }
        from += nt;
      }
    };
    place(t_begin, s_start);
    if (snap) place(t_end, s_end);
    __syncthreads();
    start = s_start[0];
    base = s_start[1];
    if (snap) {
      t_begin = base;
      t_end = t_end == total ? total : s_end[1];
      if (t_begin >= t_end) return;
    }
    first = (int)(t_begin - base);
  }
  const int n = (int)(t_end - t_begin);

  auto open = [&](Cursor& c, long long b) {   // the next sequence from b on that has keys
    c.b = b;
    c.t = 0;
    while (c.b < d.batch - 1 && length_of(c.b) == 0) ++c.b;
    c.len = length_of(c.b);
    c.nt = (c.len + TILE - 1) / TILE;
  };
  auto step = [&](Cursor& c) {
    if (++c.t == c.nt) open(c, c.b + 1);
  };
  Cursor get, use;
  open(get, start);
  get.t = first;
  use = get;

  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + warp * (C::STAGES * C::STAGE);
  float* join = reinterpret_cast<float*>(smem + C::RING);

  // -- copies: lane l < 16 looks up key l of the warp's 16, LOOK tiles ahead (a look
  // into the page table takes about as long as a tile) --------------------------
  int page[LOOK], place[LOOK];
  auto look = [&](int i) {                    // page and place for cursor `get`
    const int key = get.t * TILE + warp * KPW + (lane & 15);
    page[i] = -1;
    if (key < get.len) {
      const int pi = p.page_shift >= 0 ? key >> p.page_shift : key / (int)d.page_size;
      place[i] = key - pi * (int)d.page_size;
      page[i] = d.pages[get.b * d.page_row + pi];
      if (page[i] < 0) page[i] = -2;          // a bad page; -1 is no key
    }
  };
  int looked = 1, got = 0;                    // tiles looked up, tiles issued
  look(0);
#pragma unroll
  for (int i = 1; i < LOOK; ++i) {
    page[i] = -1;
    if (looked < n) {
      step(get);
      look(i);
      ++looked;
    }
  }
  auto issue = [&]() {
    if (got < n) {
      const uint32_t st = ring + (got % C::STAGES) * C::STAGE;
      const int pg = page[0];
      long long ko = -1, vo = -1;
      if (pg >= 0 && pg < d.num_pages) {
        ko = pg * d.kc_stride[0] + place[0] * d.kc_stride[1] + kvh * d.kc_stride[2];
        vo = pg * d.vc_stride[0] + place[0] * d.vc_stride[1] + kvh * d.vc_stride[2];
      } else if (pg != -1) {
        atomicOr(d.status, KTIR_STATUS_BAD_INDEX);
      }
      ++got;
#pragma unroll
      for (int i = 0; i + 1 < LOOK; ++i) {
        page[i] = page[i + 1];
        place[i] = place[i + 1];
      }
      page[LOOK - 1] = -1;
      if (looked < n) {
        step(get);
        look(LOOK - 1);
        ++looked;
      }
      const int c = lane % C::CHUNKS;
      constexpr int PER = 32 / C::CHUNKS;     // rows per instruction
#pragma unroll
      for (int i = 0; i < KPW / PER; ++i) {
        const int r = i * PER + lane / C::CHUNKS;
        const long long k = __shfl_sync(0xffffffffu, ko, r);
        const long long v = p.same ? k : __shfl_sync(0xffffffffu, vo, r);
        const uint32_t dst = st + r * C::ROW_BYTES + ((c ^ (r & 7)) << 4);
        cp16(dst, static_cast<const T*>(d.k_cache) + (k < 0 ? 0 : k + c * 8), k < 0 ? 0 : 16);
        cp16(dst + C::HALF_STAGE, static_cast<const T*>(d.v_cache) + (v < 0 ? 0 : v + c * 8), v < 0 ? 0 : 16);
      }
    }
    cp_commit();
  };
#pragma unroll
  for (int s = 0; s < C::STAGES - 1; ++s) issue();

  // q^T as the first product's second operand; o^T, and per head m and l (l over
  // this thread's keys): heads 2 (lane % 4) and the next of every tile of 8
  uint32_t qb[D / 16][NT][2];
  float o[D / 16][NT][4], m[NT][2], l[NT][2];
  const float sl = d.scale * LOG2E;
  const int at = lane >> 2, col = (lane & 3) * 2;

  auto begin = [&](long long b) {             // a sequence, or this stretch of it
    const T* q = static_cast<const T*>(d.q) + b * d.q_stride[0];
#pragma unroll
    for (int h = 0; h < NT; ++h)
#pragma unroll
      for (int k = 0; k < D / 16; ++k)
#pragma unroll
        for (int x = 0; x < 2; ++x)
          qb[k][h][x] = 8 * h + at < nrows ? *reinterpret_cast<const uint32_t*>(
                                                 q + (head0 + 8 * h + at) * d.q_stride[1] + k * 16 + x * 8 + col)
                                           : 0u;
  };
  auto clear = [&]() {
#pragma unroll
    for (int h = 0; h < NT; ++h) {
#pragma unroll
      for (int k = 0; k < D / 16; ++k) o[k][h][0] = o[k][h][1] = o[k][h][2] = o[k][h][3] = 0.f;
      m[h][0] = m[h][1] = -INFINITY;
      l[h][0] = l[h][1] = 0.f;
    }
  };
  begin(use.b);
  clear();

  for (int i = 0; i < n; ++i) {
    cp_wait<C::STAGES - 2>();
    __syncwarp();                             // every lane's copies of tile i, and its reads of tile i - 1
    issue();
    const uint32_t kt = ring + (i % C::STAGES) * C::STAGE, vt = kt + C::HALF_STAGE;

    // x^T = K q^T, in two chains
    float s[NT][4] = {}, s2[NT][4] = {};
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      uint32_t a[4];
      const int r = (lane & 7) + (((lane >> 3) & 1) << 3), c = 2 * k + (lane >> 4);
      ldsm4(a, kt + r * C::ROW_BYTES + ((c ^ (r & 7)) << 4));
#pragma unroll
      for (int h = 0; h < NT; ++h) mma16816<T>(k & 1 ? s2[h] : s[h], a, qb[k][h][0], qb[k][h][1]);
    }
    const int left = use.len - use.t * TILE - warp * KPW;      // keys of the 16 that exist
    uint32_t pb[NT][2];
#pragma unroll
    for (int h = 0; h < NT; ++h) {
      float top[2];
#pragma unroll
      for (int x = 0; x < 4; ++x)
        s[h][x] = at + 8 * (x >> 1) < left ? __fmul_rn(s[h][x] + s2[h][x], sl) : -INFINITY;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        top[x] = fmaxf(s[h][x], s[h][x + 2]);
        top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 4));
        top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 8));
        top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 16));
      }
      if (__any_sync(0xffffffffu,
                     top[0] - m[h][0] > RESCALE_THRESHOLD + Elem<T>::LIFT ||
                         top[1] - m[h][1] > RESCALE_THRESHOLD + Elem<T>::LIFT)) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float mn = fmaxf(m[h][x], top[x] - Elem<T>::LIFT);
          const float f = mn == -INFINITY ? 1.f : ex2(m[h][x] - mn);
          m[h][x] = mn;
          l[h][x] *= f;
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            o[k][h][x] *= f;
            o[k][h][x + 2] *= f;
          }
        }
      }
      const float sub0 = m[h][0] == -INFINITY ? 0.f : m[h][0], sub1 = m[h][1] == -INFINITY ? 0.f : m[h][1];
#pragma unroll
      for (int x = 0; x < 2; ++x) {           // keys `at` and `at` + 8
        const float a = ex2(s[h][2 * x] - sub0), b = ex2(s[h][2 * x + 1] - sub1);
        l[h][0] += a;
        l[h][1] += b;
        pb[h][x] = transpose8(Elem<T>::from2(a, b));
      }
    }
    // o^T += V^T p^T
#pragma unroll
    for (int k = 0; k < D / 16; ++k) {
      uint32_t a[4];
      const int r = (lane & 7) + ((lane >> 4) << 3), c = 2 * k + ((lane >> 3) & 1);
      ldsm4t(a, vt + r * C::ROW_BYTES + ((c ^ (r & 7)) << 4));
#pragma unroll
      for (int h = 0; h < NT; ++h) mma16816<T>(o[k][h], a, pb[h][0], pb[h][1]);
    }

    if (use.t + 1 < use.nt && i + 1 < n) {
      ++use.t;
      continue;
    }
    // -- the sequence, or this stretch of it, ends: join the warps ---------------
    const long long b = use.b, end = base + use.nt;
    const bool whole = base >= t_begin && end <= t_end;
    const bool more = i + 1 < n;
    if (more) {                               // the next one's queries are on their way meanwhile
      open(use, b + 1);
      begin(use.b);
    }
#pragma unroll
    for (int h = 0; h < NT; ++h)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) l[h][x] += __shfl_xor_sync(0xffffffffu, l[h][x], w);
        if (lane < 4) s_ml[warp][8 * h + col + x] = make_float2(m[h][x], l[h][x]);
      }
    T* out = static_cast<T*>(d.out) + b * d.out_stride[0];
    float* part = p.parts + ((long long)blockIdx.x * 2 + (base >= t_begin ? 1 : 0)) * PART_STRIDE;
    // eight heads at a time: [warp][head][D] in shared memory, eight floats of a
    // head moved by its number (the heads would lie in one bank), then each thread
    // four outputs
#pragma unroll
    for (int h = 0; h < NT; ++h) {
      if (8 * h < nrows) {
        float* to = join + (warp * 8 + col) * D;
        const int move = (lane & 3) * 8;       // of heads `col` and `col` + 1
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
#pragma unroll
          for (int x = 0; x < 4; ++x) to[(x & 1) * D + ((16 * k + 8 * (x >> 1)) ^ move) + at] = o[k][h][x];
        __syncthreads();
        for (int e = tid; e < min(8, nrows - 8 * h) * (D / 4); e += THREADS) {
          const int r = e / (D / 4), c = (e - r * (D / 4)) * 4;
          float mt = -INFINITY, lt = 0.f;
#pragma unroll
          for (int w = 0; w < WARPS; ++w) mt = fmaxf(mt, s_ml[w][8 * h + r].x);
          const float sub = mt == -INFINITY ? 0.f : mt;
          float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < WARPS; ++w) {
            const float2 ml = s_ml[w][8 * h + r];
            const float f = ex2(ml.x - sub);
            const float4 y = *reinterpret_cast<const float4*>(join + (w * 8 + r) * D + (c ^ ((r >> 1) * 8)));
            lt += ml.y * f;
            x.x += y.x * f;
            x.y += y.y * f;
            x.z += y.z * f;
            x.w += y.w * f;
          }
          if (whole) {
            const float inv = lt == 0.f ? 0.f : 1.f / lt;     // every score -inf: nothing to weigh
            uint2 v;
            v.x = Elem<T>::from2(x.x * inv, x.y * inv);
            v.y = Elem<T>::from2(x.z * inv, x.w * inv);
            *reinterpret_cast<uint2*>(out + (head0 + 8 * h + r) * d.out_stride[1] + c) = v;
            if (d.lse && c == 0) d.lse[b * d.heads + head0 + 8 * h + r] = (mt + log2f(lt)) * LN2;
          } else {
            *reinterpret_cast<float4*>(part + (8 * h + r) * D + c) = x;
            if (c == 0) reinterpret_cast<float2*>(part + ROWS * D)[8 * h + r] = make_float2(mt, lt);
          }
        }
        if (!whole) __threadfence();
        __syncthreads();
      }
    }
    clear();
    if (!whole) {
      // stretches that share the sequence: those of its first to its last tile
      const long long g0 = fits ? s_own[0] : ((base + 1) * ng - 1) / total, g1 = fits ? s_own[1] : (end * ng - 1) / total;
      if (tid == 0) {
        int* counter = p.counters + b * p.ht + ht;
        const int before = atomicAdd(counter, 1);
        s_last = before == (int)(g1 - g0);
        if (s_last) *counter = 0;
        __threadfence();
      }
      __syncthreads();
      if (s_last) {
        for (int e = tid; e < nrows * (D / 4); e += THREADS) {
          const int r = e / (D / 4), c = (e - r * (D / 4)) * 4;
          float mm = -INFINITY, ll = 0.f;
          float4 oo = make_float4(0.f, 0.f, 0.f, 0.f);
          // sixteen parts on their way at once
          for (long long g = g0; g <= g1; g += 16) {
            float2 ml[16];
            float4 x[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              ml[i] = make_float2(-INFINITY, 0.f);
              x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
              if (g + i <= g1) {
                // the first part ends its stretch, the others begin theirs
                const bool begins = g + i == g0;
                const float* part = p.parts + (((g + i) * p.ht + ht) * 2 + (begins ? 1 : 0)) * PART_STRIDE;
                ml[i] = __ldcg(reinterpret_cast<const float2*>(part + ROWS * D) + r);
                x[i] = __ldcg(reinterpret_cast<const float4*>(part + r * D + c));
              }
            }
            float mn = mm;
#pragma unroll
            for (int i = 0; i < 16; ++i) mn = fmaxf(mn, ml[i].x);
            const float sub = mn == -INFINITY ? 0.f : mn;
            const float f = ex2(mm - sub);
            mm = mn;
            ll *= f;
            oo.x *= f;
            oo.y *= f;
            oo.z *= f;
            oo.w *= f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float w = ex2(ml[i].x - sub);
              ll += ml[i].y * w;
              oo.x += x[i].x * w;
              oo.y += x[i].y * w;
              oo.z += x[i].z * w;
              oo.w += x[i].w * w;
            }
          }
          const float inv = ll == 0.f ? 0.f : 1.f / ll;
          uint2 v;
          v.x = Elem<T>::from2(oo.x * inv, oo.y * inv);
          v.y = Elem<T>::from2(oo.z * inv, oo.w * inv);
          *reinterpret_cast<uint2*>(static_cast<T*>(d.out) + b * d.out_stride[0] +
                                    (head0 + r) * d.out_stride[1] + c) = v;
          if (d.lse && c == 0) d.lse[b * d.heads + head0 + r] = (mm + log2f(ll)) * LN2;
        }
      }
    }
    base = end;
  }
}

template <typename T, int D, int NT>
int launch(const DecodeParams& p, unsigned grid, cudaStream_t stream) {
  // the attribute is per device
  static bool ready[MAX_DEVICES] = {};
  const int dev = current_device();
  if (dev < 0) return ktir_set_error(KTIR_ERR_CUDA, "ktir_paged_decode: no usable current device");
  if (!ready[dev]) {
    if (cudaFuncSetAttribute(k_paged_decode<T, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             Cfg<D>::SMEM) != cudaSuccess)
      return ktir_set_error(KTIR_ERR_CUDA, "ktir_paged_decode: shared-memory attribute refused");
    ready[dev] = true;
  }
  return launched(launch_pdl(k_paged_decode<T, D, NT>, grid, THREADS, Cfg<D>::SMEM, stream, p),
                  "ktir_paged_decode: launch failed");
}

// head tiles of a kv head: 8 query heads each, 16 where there are more than 8
int head_tiles(int group) { return group <= 8 ? 1 : (group + 15) / 16; }

}  // namespace

extern "C" int64_t ktir_paged_decode_workspace(int64_t batch, int32_t heads, int32_t kv_heads,
                                               int32_t dim) {
  if (batch < 1 || heads < 1 || kv_heads < 1 || dim < 1) return 0;
  const int64_t htiles = head_tiles(heads / kv_heads);
  // the parts first, at a size of their own: the counters keep their places
  // (and their zeros) between calls of different batches
  return PARTS_BYTES + batch * kv_heads * htiles * 4;
}

extern "C" int ktir_paged_decode(const KtirPagedDecodeDesc* d, void* stream) {
  if (!d) return ktir_set_error(KTIR_ERR_ARG, "ktir_paged_decode: null argument");
  if (d->batch == 0) return KTIR_OK;
  if (!d->q || !d->k_cache || !d->v_cache || !d->out || !d->pages || !d->lengths || !d->status ||
      !d->workspace)
    return ktir_set_error(KTIR_ERR_ARG, "ktir_paged_decode: null argument");
  if (d->dtype != KTIR_F16 && d->dtype != KTIR_BF16)
    return ktir_set_error(KTIR_ERR_UNSUPPORTED, "ktir_paged_decode: needs f16 or bf16");
  if (d->dim != 64 && d->dim != 128)
    return ktir_set_error(KTIR_ERR_UNSUPPORTED, "ktir_paged_decode: needs dim 64 or 128");
  if (d->batch < 0 || d->heads < 1 || d->kv_heads < 1 || d->heads % d->kv_heads ||
      d->heads > (1 << 16) || d->batch > (1 << 24) || d->num_pages < 1 || d->page_size < 1 ||
      d->max_pages < 1 || d->num_pages > 0x7fffffffLL || d->page_size > 0x7fffffffLL ||
      d->max_pages > 0x7fffffffLL || d->max_pages * d->page_size > 0x7fffff00LL)
    return ktir_set_error(KTIR_ERR_ARG, "ktir_paged_decode: extent out of range");
  if (!(d->scale > 0.f) || !isfinite(d->scale))
    return ktir_set_error(KTIR_ERR_UNSUPPORTED, "ktir_paged_decode: needs a positive, finite scale");
  const int64_t qe[2] = {d->batch, d->heads};
  const int64_t ce[3] = {d->num_pages, d->page_size, d->kv_heads};
  if (!vector_strides(d->q_stride, qe, 2) || !vector_strides(d->out_stride, qe, 2) ||
      !vector_strides(d->kc_stride, ce, 3) || !vector_strides(d->vc_stride, ce, 3) || !aligned16(d->q) ||
      !aligned16(d->k_cache) || !aligned16(d->v_cache) || !aligned16(d->out) || !aligned16(d->workspace))
    return ktir_set_error(KTIR_ERR_UNSUPPORTED,
                          "ktir_paged_decode: head vectors must start on 16-byte boundaries");
  if (!apart(d->out_stride, qe, 2))
    return ktir_set_error(KTIR_ERR_ARG, "ktir_paged_decode: rows of out share memory");
  if (d->workspace_bytes < ktir_paged_decode_workspace(d->batch, d->heads, d->kv_heads, d->dim))
    return ktir_set_error(KTIR_ERR_ARG, "ktir_paged_decode: workspace too small");
  const int sms = sm_count();
  if (sms < 1) return ktir_set_error(KTIR_ERR_CUDA, "ktir_paged_decode: no usable current device");
  DecodeParams p;
  p.d = *d;
  p.group = d->heads / d->kv_heads;
  p.htiles = head_tiles(p.group);
  p.same = 1;
  for (int i = 0; i < 3; ++i) p.same &= d->kc_stride[i] == d->vc_stride[i];
  p.ht = d->kv_heads * p.htiles;
  p.parts = static_cast<float*>(d->workspace);
  p.counters = reinterpret_cast<int*>(static_cast<char*>(d->workspace) + PARTS_BYTES);
  p.page_shift = -1;
  if ((d->page_size & (d->page_size - 1)) == 0)
    for (p.page_shift = 0; (1LL << p.page_shift) < d->page_size; ++p.page_shift) {}
  // one resident wave of CTAs, no more groups than the cache could have stretches
  int slots = sms * (d->dim == 128 ? Cfg<128>::CTAS_PER_SM : Cfg<64>::CTAS_PER_SM);
  if (slots > MAX_CTAS) slots = MAX_CTAS;
  long long groups = slots / p.ht;
  const __int128 tiles = (__int128)d->batch * ((d->max_pages * d->page_size + TILE - 1) / TILE);
  if (groups > tiles) groups = (long long)tiles;
  if (groups < 1) groups = 1;
  p.groups = (int)groups;
  const unsigned grid = (unsigned)(groups * p.ht);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool f16 = d->dtype == KTIR_F16;
  if (p.group <= 8) {
    if (d->dim == 64) return f16 ? launch<__half, 64, 1>(p, grid, s) : launch<__nv_bfloat16, 64, 1>(p, grid, s);
    return f16 ? launch<__half, 128, 1>(p, grid, s) : launch<__nv_bfloat16, 128, 1>(p, grid, s);
  }
  if (d->dim == 64) return f16 ? launch<__half, 64, 2>(p, grid, s) : launch<__nv_bfloat16, 64, 2>(p, grid, s);
  return f16 ? launch<__half, 128, 2>(p, grid, s) : launch<__nv_bfloat16, 128, 2>(p, grid, s);
}

// New tokens into a paged key-value cache, rotated by position on the way.
//
// A pair (a, b) of a head vector becomes (a c - b s, b c + a s), c and s the
// cosine and sine of the position times the pair's frequency, read from an f32
// table and applied in f32; one rounding to the element type at the end.
//
// Bound by memory: each of q, k, v is read once and written once.  One block per
// token (or several short ones, see below); dim / 16 threads share a head vector, each with two 16-byte vectors
// that hold whole pairs: vectors j and j + rot/16 of the rotated part when pairs
// are (i, i + rot/2), vectors 2j and 2j+1 when they are (2i, 2i+1).  A thread
// keeps its cosines and sines in registers and walks over the token's heads,
// three vectors on their way at once, the first ones asked for before the
// position, the slot and the table's row are there.  Blocks of 64 threads, 12 of
// them on an SM at once, keep the most copies in flight: 24576 tokens of 32 + 8 + 8
// heads of 128 take 93 to 97 us = 6.6 to 6.4 TB/s (128 threads: 106 us, one vector at a time: 98).
// Where a token has less than three vectors for each thread of a block, and there
// are more tokens than blocks fit at once, a block takes as many tokens as it has
// threads for: 20344 tokens of 6 + 1 + 1 heads of 64 11.8 us against 28.9, of 15 +
// 3 + 3 heads 25.3 against 34.1.
#include "serve_common.cuh"

using namespace ktir::serve;

namespace {

constexpr int UNROLL = 3;      // head vectors of a thread on their way at once
constexpr int RESIDENT = 12;   // blocks of 64 threads on an SM at once, by their registers

struct AppendParams {
  KtirKvAppendDesc d;
  long long slots_total;
  int vector_table;      // rows of the table start on 16-byte boundaries
  int lanes;             // head vectors of a token in flight at once
  int each;              // tokens of a block
};

template <typename T>
__device__ __forceinline__ uint4 rotate_first(const uint4& a, const uint4& b, const float (&c)[8],
                                              const float (&s)[8]) {
  const uint32_t* x = reinterpret_cast<const uint32_t*>(&a);
  const uint32_t* y = reinterpret_cast<const uint32_t*>(&b);
  uint4 r;
  uint32_t* o = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 u = Elem<T>::to2(x[i]), v = Elem<T>::to2(y[i]);
    o[i] = Elem<T>::from2(u.x * c[2 * i] - v.x * s[2 * i], u.y * c[2 * i + 1] - v.y * s[2 * i + 1]);
  }
  return r;
}

template <typename T>
__device__ __forceinline__ uint4 rotate_second(const uint4& a, const uint4& b, const float (&c)[8],
                                               const float (&s)[8]) {
  const uint32_t* x = reinterpret_cast<const uint32_t*>(&a);
  const uint32_t* y = reinterpret_cast<const uint32_t*>(&b);
  uint4 r;
  uint32_t* o = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 u = Elem<T>::to2(x[i]), v = Elem<T>::to2(y[i]);
    o[i] = Elem<T>::from2(v.x * c[2 * i] + u.x * s[2 * i], v.y * c[2 * i + 1] + u.y * s[2 * i + 1]);
  }
  return r;
}

// four interleaved pairs of one vector, cosines and sines from `at` on
template <typename T>
__device__ __forceinline__ uint4 rotate_pairs(const uint4& a, const float (&c)[8], const float (&s)[8],
                                              int at) {
  const uint32_t* x = reinterpret_cast<const uint32_t*>(&a);
  uint4 r;
  uint32_t* o = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 u = Elem<T>::to2(x[i]);
    const float cc = c[at + i], ss = s[at + i];
    o[i] = Elem<T>::from2(u.x * cc - u.y * ss, u.y * cc + u.x * ss);
  }
  return r;
}

template <typename T, int THREADS, bool SEVERAL>
__global__ void __launch_bounds__(THREADS, SEVERAL ? RESIDENT : 0) k_kv_append(const __grid_constant__ AppendParams p) {
  const KtirKvAppendDesc& d = p.d;
  const int parts = d.dim >> 4;                 // threads per head vector
  const int lanes = SEVERAL ? p.lanes : THREADS / parts;     // head vectors of a token in flight
  const int vec = threadIdx.x / parts, j = threadIdx.x - vec * parts;
  const int sub = SEVERAL ? vec / lanes : 0, hl = SEVERAL ? vec - sub * lanes : vec;
  const long long t = SEVERAL ? (long long)blockIdx.x * p.each + sub : blockIdx.x;
  if (SEVERAL ? sub >= p.each || t >= d.tokens : hl >= lanes) return;
  const int rparts = d.rot >> 4;
  const bool turn = j < rparts;
  // this thread's two vectors of a head vector, rotated or copied
  const int first = d.interleaved ? 16 * j : turn ? 8 * j : d.rot + 16 * (j - rparts);
  const int second = !d.interleaved && turn ? first + (d.rot >> 1) : first + 8;
  const int hq = d.q ? d.heads : 0, hk = hq + d.kv_heads, n = hk + d.kv_heads;

  pdl_launch();
  pdl_wait();
  const int slot = d.slots[t];
  const int pos = rparts ? d.positions[t] : 0;
  // A bad slot leaves the token's key and value out, a bad position makes its query
  // zeros as well (never what the memory held before).
  const bool lost = rparts && (pos < 0 || pos >= d.table_rows);
  const bool kept = slot >= 0 && slot < p.slots_total && !lost;
  float c[8], s[8];
  const long long page = kept ? slot / d.page_size : 0;
  const long long place = kept ? slot - page * d.page_size : 0;
  for (int h0 = hl; h0 < n; h0 += UNROLL * lanes) {
    uint4 a[UNROLL], b[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int h = h0 + u * lanes;
      if (h < n) {
        const T* src = h < hq   ? static_cast<const T*>(d.q) + t * d.q_stride[0] + h * d.q_stride[1]
                       : h < hk ? static_cast<const T*>(d.k) + t * d.k_stride[0] + (h - hq) * d.k_stride[1]
                                : static_cast<const T*>(d.v) + t * d.v_stride[0] + (h - hk) * d.v_stride[1];
        a[u] = *reinterpret_cast<const uint4*>(src + first);
        b[u] = *reinterpret_cast<const uint4*>(src + second);
      }
    }
    if (h0 == hl) {                             // the vectors are on their way meanwhile
      if (!kept && slot >= 0 && hl == 0 && j == 0) atomicOr(d.status, KTIR_STATUS_BAD_INDEX);
      if (turn && !lost) {
        const float* row = d.table + (long long)pos * d.table_stride + 8 * j;
        if (p.vector_table) {
#pragma unroll
          for (int i = 0; i < 8; i += 4) {
            *reinterpret_cast<float4*>(c + i) = __ldg(reinterpret_cast<const float4*>(row + i));
            *reinterpret_cast<float4*>(s + i) = __ldg(reinterpret_cast<const float4*>(row + (d.rot >> 1) + i));
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            c[i] = row[i];
            s[i] = row[(d.rot >> 1) + i];
          }
        }
      }
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int h = h0 + u * lanes;
      if (h >= n || (h >= hq && !kept)) continue;
      uint4 x = a[u], y = b[u];
      if (lost) {
        x = y = make_uint4(0, 0, 0, 0);
      } else if (turn && h < hk) {
        if (d.interleaved) {
          x = rotate_pairs<T>(a[u], c, s, 0);
          y = rotate_pairs<T>(b[u], c, s, 4);
        } else {
          x = rotate_first<T>(a[u], b[u], c, s);
          y = rotate_second<T>(a[u], b[u], c, s);
        }
      }
      T* dst;
      if (h < hq)
        dst = static_cast<T*>(d.q_out) + t * d.qo_stride[0] + h * d.qo_stride[1];
      else if (h < hk)
        dst = static_cast<T*>(d.k_cache) + page * d.kc_stride[0] + place * d.kc_stride[1] + (h - hq) * d.kc_stride[2];
      else
        dst = static_cast<T*>(d.v_cache) + page * d.vc_stride[0] + place * d.vc_stride[1] + (h - hk) * d.vc_stride[2];
      *reinterpret_cast<uint4*>(dst + first) = x;
      *reinterpret_cast<uint4*>(dst + second) = y;
    }
  }
}

}  // namespace

extern "C" int ktir_kv_append(const KtirKvAppendDesc* d, void* stream) {
  if (!d) return ktir_set_error(KTIR_ERR_ARG, "ktir_kv_append: null argument");
  if (d->tokens == 0) return KTIR_OK;
  if (!d->k || !d->v || !d->k_cache || !d->v_cache || !d->slots || !d->status || (d->q && !d->q_out) ||
      (d->rot && (!d->positions || !d->table)))
    return ktir_set_error(KTIR_ERR_ARG, "ktir_kv_append: null argument");
  if (d->dtype != KTIR_F16 && d->dtype != KTIR_BF16)
    return ktir_set_error(KTIR_ERR_UNSUPPORTED, "ktir_kv_append: needs f16 or bf16");
  if (d->dim < 16 || d->dim > 256 || (d->dim & 15) || d->rot < 0 || d->rot > d->dim || (d->rot & 15))
    return ktir_set_error(KTIR_ERR_UNSUPPORTED,
                          "ktir_kv_append: dim a multiple of 16 up to 256, rot a multiple of 16 up to dim");
  if (d->tokens < 0 || d->tokens > 0x7fffffffLL || d->kv_heads < 1 || d->heads < 1 ||
      d->heads > (1 << 20) || d->kv_heads > (1 << 20) || d->num_pages < 1 || d->page_size < 1 ||
      (d->rot && d->table_rows < 1))
    return ktir_set_error(KTIR_ERR_ARG, "ktir_kv_append: extent out of range");
  const int64_t te[2] = {d->tokens, d->heads}, ke[2] = {d->tokens, d->kv_heads};
  const int64_t ce[3] = {d->num_pages, d->page_size, d->kv_heads};
  if ((d->q && (!vector_strides(d->q_stride, te, 2) || !vector_strides(d->qo_stride, te, 2))) ||
      !vector_strides(d->k_stride, ke, 2) || !vector_strides(d->v_stride, ke, 2) ||
      !vector_strides(d->kc_stride, ce, 3) || !vector_strides(d->vc_stride, ce, 3) || !aligned16(d->q) ||
      !aligned16(d->k) || !aligned16(d->v) || !aligned16(d->q_out) || !aligned16(d->k_cache) ||
      !aligned16(d->v_cache))
    return ktir_set_error(KTIR_ERR_UNSUPPORTED,
                          "ktir_kv_append: head vectors must start on 16-byte boundaries");
  if ((d->q && !apart(d->qo_stride, te, 2)) || !apart(d->kc_stride, ce, 3) || !apart(d->vc_stride, ce, 3))
    return ktir_set_error(KTIR_ERR_ARG, "ktir_kv_append: places of a cache, or rows of q_out, share memory");
  AppendParams p;
  p.d = *d;
  const __int128 total = (__int128)d->num_pages * d->page_size;
  p.slots_total = total > 0x7fffffffLL ? 0x80000000LL : (long long)total;
  p.vector_table = aligned16(d->table) && !(d->table_stride & 3);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int vectors = (d->q ? d->heads : 0) + 2 * d->kv_heads, across = 64 / (d->dim >> 4);
  const int sms = sm_count();
  const bool few = d->tokens <= sms, several = d->tokens > (int64_t)RESIDENT * sms && vectors < UNROLL * across;
  p.lanes = (vectors + UNROLL - 1) / UNROLL;
  p.each = several ? across / p.lanes : 1;
  const unsigned grid = (unsigned)((d->tokens + p.each - 1) / p.each);
  const bool f16 = d->dtype == KTIR_F16;
  const cudaError_t e =
      few ? (f16 ? launch_pdl(k_kv_append<__half, 128, false>, grid, 128, 0, s, p)
                 : launch_pdl(k_kv_append<__nv_bfloat16, 128, false>, grid, 128, 0, s, p))
      : several ? (f16 ? launch_pdl(k_kv_append<__half, 64, true>, grid, 64, 0, s, p)
                       : launch_pdl(k_kv_append<__nv_bfloat16, 64, true>, grid, 64, 0, s, p))
                : (f16 ? launch_pdl(k_kv_append<__half, 64, false>, grid, 64, 0, s, p)
                       : launch_pdl(k_kv_append<__nv_bfloat16, 64, false>, grid, 64, 0, s, p));
  return launched(e, "ktir_kv_append: launch failed");
}

// New tokens into a paged key-value cache, rotated by position on the way.
//
// A pair (a, b) of a head vector becomes (a c - b s, b c + a s), c and s the
// cosine and sine of the position times the pair's frequency, read from an f32
// table and applied in f32; one rounding to the element type at the end.
//
// Bound by memory: each of q, k, v is read once and written once.  dim / 16
// threads share a head vector, each with two 16-byte vectors that hold whole
// pairs: vectors j and j + rot/16 of the rotated part when pairs are (i, i +
// rot/2), vectors 2j and 2j+1 when they are (2i, 2i+1).  A thread keeps its
// cosines and sines in registers and walks over the token's heads.
#include "serve_common.cuh"

using namespace ktir::serve;

namespace {

constexpr int THREADS = 128;

struct AppendParams {
  KtirKvAppendDesc d;
  long long slots_total;
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

template <typename T>
__global__ void __launch_bounds__(THREADS) k_kv_append(const __grid_constant__ AppendParams p) {
  const KtirKvAppendDesc& d = p.d;
  const long long t = blockIdx.x;
  const int parts = d.dim >> 4;                 // threads per head vector
  const int j = threadIdx.x % parts;
  const int lanes = THREADS / parts;            // head vectors in flight per block
  int hl = threadIdx.x / parts;
  if (hl >= lanes) return;
  const int rparts = d.rot >> 4;
  const bool turn = j < rparts;

  pdl_launch();
  pdl_wait();
  const int slot = d.slots[t];
  bool bad = slot >= p.slots_total;
  float c[8], s[8];
  if (rparts) {
    const int pos = d.positions[t];
    if (pos < 0 || pos >= d.table_rows) {
      bad = true;
    } else if (turn) {
      const float* row = d.table + (long long)pos * d.table_stride + 8 * j;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        c[i] = row[i];
        s[i] = row[(d.rot >> 1) + i];
      }
    }
  }
  if (bad) {
    if (threadIdx.x == 0) atomicOr(d.status, KTIR_STATUS_BAD_INDEX);
    return;
  }
  // this thread's two vectors of a head vector, rotated (r) or copied
  const int first = d.interleaved ? 16 * j : turn ? 8 * j : d.rot + 16 * (j - rparts);
  const int second = !d.interleaved && turn ? first + (d.rot >> 1) : first + 8;
  const T* q = static_cast<const T*>(d.q);
  const int hq = q ? d.heads : 0;
  const int n = hq + (slot >= 0 ? 2 * d.kv_heads : 0);
  const long long page = slot >= 0 ? slot / d.page_size : 0;
  const long long place = slot >= 0 ? slot - page * d.page_size : 0;
  for (int h = hl; h < n; h += lanes) {
    const T* src;
    T* dst;
    bool r = turn;
    if (h < hq) {
      src = q + t * d.q_stride[0] + h * d.q_stride[1];
      dst = static_cast<T*>(d.q_out) + t * d.qo_stride[0] + h * d.qo_stride[1];
    } else if (h < hq + d.kv_heads) {
      const int g = h - hq;
      src = static_cast<const T*>(d.k) + t * d.k_stride[0] + g * d.k_stride[1];
      dst = static_cast<T*>(d.k_cache) + page * d.kc_stride[0] + place * d.kc_stride[1] +
            g * d.kc_stride[2];
    } else {
      const int g = h - hq - d.kv_heads;
      src = static_cast<const T*>(d.v) + t * d.v_stride[0] + g * d.v_stride[1];
      dst = static_cast<T*>(d.v_cache) + page * d.vc_stride[0] + place * d.vc_stride[1] +
            g * d.vc_stride[2];
      r = false;
    }
    const uint4 a = *reinterpret_cast<const uint4*>(src + first);
    const uint4 b = *reinterpret_cast<const uint4*>(src + second);
    uint4 x = a, y = b;
    if (r) {
      if (d.interleaved) {
        x = rotate_pairs<T>(a, c, s, 0);
        y = rotate_pairs<T>(b, c, s, 4);
      } else {
        x = rotate_first<T>(a, b, c, s);
        y = rotate_second<T>(a, b, c, s);
      }
    }
    *reinterpret_cast<uint4*>(dst + first) = x;
    *reinterpret_cast<uint4*>(dst + second) = y;
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
  AppendParams p;
  p.d = *d;
  const __int128 total = (__int128)d->num_pages * d->page_size;
  p.slots_total = total > 0x7fffffffLL ? 0x80000000LL : (long long)total;
  const unsigned grid = (unsigned)d->tokens;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = d->dtype == KTIR_F16
                            ? launch_pdl(k_kv_append<__half>, grid, THREADS, 0, s, p)
                            : launch_pdl(k_kv_append<__nv_bfloat16>, grid, THREADS, 0, s, p);
  return launched(e, "ktir_kv_append: launch failed");
}

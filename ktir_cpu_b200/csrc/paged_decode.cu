// Attention of one new token per sequence over its paged keys and values.
//
//   o = sum_j e^(x_j - m) v_j / l,   l = sum_j e^(x_j - m),   m = max_j x_j,
//   x_j = scale q . k_j
//
// One warp per (sequence, head): the keys one after the other, m, l and o in
// f32 registers (o scaled by e^(m - m') when the maximum moves to m').
#include "serve_common.cuh"

using namespace ktir::serve;

namespace {

constexpr int WARPS = 4;

template <typename T, int D>
__global__ void __launch_bounds__(WARPS * 32)
    k_paged_decode(const __grid_constant__ KtirPagedDecodeDesc d) {
  constexpr int E = D / 32;            // elements per lane
  const long long item = (long long)blockIdx.x * WARPS + (threadIdx.x >> 5);
  if (item >= d.batch * d.heads) return;
  const int lane = threadIdx.x & 31;
  const long long b = item / d.heads;
  const int h = (int)(item - b * d.heads);
  const int g = h / (d.heads / d.kv_heads);
  const float sl = d.scale * LOG2E;
  int len = d.lengths[b];
  if (len < 0 || len > d.max_pages * d.page_size) {
    if (lane == 0) atomicOr(d.status, KTIR_STATUS_BAD_INDEX);
    len = 0;
  }
  float q[E], o[E], m = -INFINITY, l = 0.f;
  const T* qp = static_cast<const T*>(d.q) + b * d.q_stride[0] + h * d.q_stride[1] + lane * E;
#pragma unroll
  for (int i = 0; i < E; i += 2) {
    const float2 x = Elem<T>::to2(*reinterpret_cast<const uint32_t*>(qp + i));
    q[i] = x.x * sl;
    q[i + 1] = x.y * sl;
    o[i] = o[i + 1] = 0.f;
  }
  for (int j = 0; j < len; ++j) {
    const int page = d.pages[b * d.page_row + j / d.page_size];
    if (page < 0 || page >= d.num_pages) {
      if (lane == 0) atomicOr(d.status, KTIR_STATUS_BAD_INDEX);
      continue;
    }
    const long long place = j % d.page_size;
    const T* k = static_cast<const T*>(d.k_cache) + page * d.kc_stride[0] + place * d.kc_stride[1] +
                 g * d.kc_stride[2] + lane * E;
    const T* v = static_cast<const T*>(d.v_cache) + page * d.vc_stride[0] + place * d.vc_stride[1] +
                 g * d.vc_stride[2] + lane * E;
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      const float2 kk = Elem<T>::to2(*reinterpret_cast<const uint32_t*>(k + i));
      x += q[i] * kk.x + q[i + 1] * kk.y;
    }
#pragma unroll
    for (int w = 16; w; w >>= 1) x += __shfl_xor_sync(0xffffffffu, x, w);
    const float mn = fmaxf(m, x);
    const float f = mn == -INFINITY ? 1.f : ex2(m - mn), e = mn == -INFINITY ? 0.f : ex2(x - mn);
    m = mn;
    l = l * f + e;
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      const float2 vv = Elem<T>::to2(*reinterpret_cast<const uint32_t*>(v + i));
      o[i] = o[i] * f + e * vv.x;
      o[i + 1] = o[i + 1] * f + e * vv.y;
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  T* out = static_cast<T*>(d.out) + b * d.out_stride[0] + h * d.out_stride[1] + lane * E;
#pragma unroll
  for (int i = 0; i < E; i += 2)
    *reinterpret_cast<uint32_t*>(out + i) = Elem<T>::from2(o[i] * inv, o[i + 1] * inv);
  if (d.lse && lane == 0) d.lse[b * d.heads + h] = l > 0.f ? (m + log2f(l)) * LN2 : -INFINITY;
}

}  // namespace

extern "C" int64_t ktir_paged_decode_workspace(int64_t batch, int32_t heads, int32_t kv_heads,
                                               int32_t dim) {
  return batch > 0 && heads > 0 && kv_heads > 0 && dim > 0 ? 256 : 0;
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
      d->max_pages > 0x7fffffffLL)
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
  if (d->workspace_bytes < ktir_paged_decode_workspace(d->batch, d->heads, d->kv_heads, d->dim))
    return ktir_set_error(KTIR_ERR_ARG, "ktir_paged_decode: workspace too small");
  const unsigned grid = (unsigned)((d->batch * d->heads + WARPS - 1) / WARPS);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool f16 = d->dtype == KTIR_F16;
  if (d->dim == 64) {
    if (f16) k_paged_decode<__half, 64><<<grid, WARPS * 32, 0, s>>>(*d);
    else k_paged_decode<__nv_bfloat16, 64><<<grid, WARPS * 32, 0, s>>>(*d);
  } else {
    if (f16) k_paged_decode<__half, 128><<<grid, WARPS * 32, 0, s>>>(*d);
    else k_paged_decode<__nv_bfloat16, 128><<<grid, WARPS * 32, 0, s>>>(*d);
  }
  return launched("ktir_paged_decode: launch failed");
}

// Attention over packed prompts with grouped heads.
//
// Query i of a sequence's n sees keys j <= i + m - n of its m when causal, all
// of them otherwise; o = softmax(scale q K^T) V over those.  One warp per
// (token, head): the keys one after the other, running maximum, sum and output
// in f32 registers.
#include "serve_common.cuh"

using namespace ktir::serve;

namespace {

constexpr int WARPS = 4;

template <typename T, int D>
__global__ void __launch_bounds__(WARPS * 32)
    k_prompt_attention(const __grid_constant__ KtirPromptDesc d) {
  constexpr int E = D / 32;            // elements per lane
  const long long item = (long long)blockIdx.x * WARPS + (threadIdx.x >> 5);
  if (item >= d.tokens * d.heads) return;
  const int lane = threadIdx.x & 31;
  const long long t = item / d.heads;
  const int h = (int)(item - t * d.heads);
  const int g = h / (d.heads / d.kv_heads);
  const float sl = d.scale * LOG2E;
  // the sequence whose stretch of tokens holds t
  long long lo = 0, hi = d.batch;
  while (hi - lo > 1) {
    const long long mid = (lo + hi) >> 1;
    if (d.offsets[mid] <= t) lo = mid;
    else hi = mid;
  }
  const long long q0 = d.offsets[lo], q1 = d.offsets[lo + 1];
  const long long k0 = d.kv_offsets[lo], k1 = d.kv_offsets[lo + 1];
  long long seen = 0;
  if (t >= q0 && t < q1) {
    if (k0 < 0 || k1 < k0 || k1 > d.kv_tokens) {
      if (lane == 0) atomicOr(d.status, KTIR_STATUS_BAD_INDEX);
    } else {
      seen = k1 - k0;
      if (d.causal) seen = min(seen, max(0LL, t - q0 + 1 + (k1 - k0) - (q1 - q0)));
    }
  } else if (lane == 0) {
    atomicOr(d.status, KTIR_STATUS_BAD_INDEX);
  }
  float q[E], o[E], m = -INFINITY, l = 0.f;
  const T* qp = static_cast<const T*>(d.q) + t * d.q_stride[0] + h * d.q_stride[1] + lane * E;
#pragma unroll
  for (int i = 0; i < E; i += 2) {
    const float2 x = Elem<T>::to2(*reinterpret_cast<const uint32_t*>(qp + i));
    q[i] = x.x * sl;
    q[i + 1] = x.y * sl;
    o[i] = o[i + 1] = 0.f;
  }
  const T* kp = static_cast<const T*>(d.k) + k0 * d.k_stride[0] + g * d.k_stride[1] + lane * E;
  const T* vp = static_cast<const T*>(d.v) + k0 * d.v_stride[0] + g * d.v_stride[1] + lane * E;
  for (long long j = 0; j < seen; ++j) {
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < E; i += 2) {
      const float2 kk = Elem<T>::to2(*reinterpret_cast<const uint32_t*>(kp + j * d.k_stride[0] + i));
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
      const float2 vv = Elem<T>::to2(*reinterpret_cast<const uint32_t*>(vp + j * d.v_stride[0] + i));
      o[i] = o[i] * f + e * vv.x;
      o[i + 1] = o[i + 1] * f + e * vv.y;
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  T* out = static_cast<T*>(d.out) + t * d.out_stride[0] + h * d.out_stride[1] + lane * E;
#pragma unroll
  for (int i = 0; i < E; i += 2)
    *reinterpret_cast<uint32_t*>(out + i) = Elem<T>::from2(o[i] * inv, o[i + 1] * inv);
  if (d.lse && lane == 0) d.lse[t * d.heads + h] = l > 0.f ? (m + log2f(l)) * LN2 : -INFINITY;
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
  const long long blocks = (d->tokens * d->heads + WARPS - 1) / WARPS;
  if (blocks > 0x7fffffffLL)
    return ktir_set_error(KTIR_ERR_UNSUPPORTED, "ktir_prompt_attention: too many rows");
  const unsigned grid = (unsigned)blocks;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool f16 = d->dtype == KTIR_F16;
  if (d->dim == 64) {
    if (f16) k_prompt_attention<__half, 64><<<grid, WARPS * 32, 0, s>>>(*d);
    else k_prompt_attention<__nv_bfloat16, 64><<<grid, WARPS * 32, 0, s>>>(*d);
  } else {
    if (f16) k_prompt_attention<__half, 128><<<grid, WARPS * 32, 0, s>>>(*d);
    else k_prompt_attention<__nv_bfloat16, 128><<<grid, WARPS * 32, 0, s>>>(*d);
  }
  return launched("ktir_prompt_attention: launch failed");
}

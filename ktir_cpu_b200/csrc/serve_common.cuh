// Shared by the serving operators (kv_append.cu, paged_decode.cu,
// prompt_attention.cu): element types, conversions and host-side checks.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "../../include/ktir_b200.h"

int ktir_set_error(int code, const char* msg);

namespace ktir {
namespace serve {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

template <typename T> struct Elem;
template <> struct Elem<__half> {
  static constexpr bool BF16 = false;
  // log2 of what softmax weights are scaled up by (and their sum with them): f16 has no
  // more than 2^-24 below 1, and many small weights of a long row count.  From 1 to 2^8
  // of themselves, the largest of a row's weights are then 2^7 to 2^15, and one is lost
  // from 2^-32 of the largest down (131,072 keys: 2^-15 of the sum, unscaled 2^-8).
  static constexpr float LIFT = 7.0f;
  static __device__ __forceinline__ float2 to2(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2*>(&v));
  }
  static __device__ __forceinline__ uint32_t from2(float a, float b) {   // round to nearest even
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <> struct Elem<__nv_bfloat16> {
  static constexpr bool BF16 = true;
  static constexpr float LIFT = 0.0f;         // as much range as f32
  static __device__ __forceinline__ float2 to2(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t from2(float a, float b) {   // round to nearest even
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

// 2^x on the special-function unit (relative error about 2^-22; -inf gives 0)
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Programmatic dependent launch: the kernels are launched while the one before
// them on the stream still runs, and touch no memory before it has completed
// (pdl_wait); pdl_launch lets the next one come as early.
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename... Params, typename... Args>
inline cudaError_t launch_pdl(void (*kernel)(Params...), unsigned grid, unsigned threads, size_t smem,
                              cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t c = {};
  c.gridDim = dim3(grid);
  c.blockDim = dim3(threads);
  c.dynamicSmemBytes = smem;
  c.stream = stream;
  cudaLaunchAttribute a[1];
  a[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  a[0].val.programmaticStreamSerializationAllowed = 1;
  c.attrs = a;
  c.numAttrs = 1;
  return cudaLaunchKernelEx(&c, kernel, args...);
}

// -- host-side checks ---------------------------------------------------------
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// strides (elements) of axes with more than one entry keep head vectors on 16-byte boundaries
inline bool vector_strides(const int64_t* stride, const int64_t* extent, int n) {
  for (int i = 0; i < n; ++i)
    if (extent[i] > 1 && ((stride[i] & 7) || stride[i] < 0)) return false;
  return true;
}

// a written tensor's entries lie apart (an expanded axis has stride 0)
inline bool apart(const int64_t* stride, const int64_t* extent, int n) {
  for (int i = 0; i < n; ++i)
    if (extent[i] > 1 && stride[i] == 0) return false;
  return true;
}

constexpr int MAX_DEVICES = 64;

// the current device, or -1
inline int current_device() {
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < MAX_DEVICES ? dev : -1;
}

inline int sm_count() {   // of the current device, 0 if there is none
  static int count[MAX_DEVICES] = {};
  const int dev = current_device();
  if (dev < 0) return 0;
  if (!count[dev] && cudaDeviceGetAttribute(&count[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 0;
  return count[dev];
}

inline int launched(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return KTIR_OK;
  cudaGetLastError();      // the error is this call's, not the next one's
  return ktir_set_error(KTIR_ERR_CUDA, what);
}

}  // namespace serve
}  // namespace ktir

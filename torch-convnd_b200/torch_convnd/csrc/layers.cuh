// Shared by the layer kernels (norm.cu, recurrence.cu, linear.cu): element conversion,
// 16-byte vectors and launch checks.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "convnd_b200_layers.h"
#include "internal.h"

namespace cnd {
namespace layers {

// The type a value is computed and summed in.
template <typename T>
struct Wide {
  using type = float;
};
template <>
struct Wide<double> {
  using type = double;
};

template <typename T>
__device__ __forceinline__ typename Wide<T>::type widen(T v) {
  return v;
}
template <>
__device__ __forceinline__ float widen(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <>
__device__ __forceinline__ float widen(__half v) {
  return __half2float(v);
}

template <typename T>
__device__ __forceinline__ T narrow(typename Wide<T>::type v) {
  return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 narrow(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half narrow(float v) {
  return __float2half_rn(v);
}

// V consecutive elements, moved by one load or store of V * sizeof(T) bytes.
template <typename T, int V>
struct alignas(V * sizeof(T)) Pack {
  T v[V];
};

// Vector parameter element i of `type` T or float32 (uniform flag), 0-d when absent.
template <typename T>
__device__ __forceinline__ typename Wide<T>::type load_param(const void* p, bool is_f32, int64_t i) {
  if (is_f32) return static_cast<const float*>(p)[i];
  return widen(static_cast<const T*>(p)[i]);
}

template <typename T>
__device__ __forceinline__ void store_param(void* p, bool is_f32, int64_t i,
                                            typename Wide<T>::type v) {
  if (is_f32) {
    static_cast<float*>(p)[i] = static_cast<float>(v);
  } else {
    static_cast<T*>(p)[i] = narrow<T>(v);
  }
}

inline int element_size(int dtype) { return dtype == CND_F64 ? 8 : dtype == CND_F32 ? 4 : 2; }
inline bool known_dtype(int dtype) { return dtype >= CND_F16 && dtype <= CND_F64; }

// a * b for nonnegative sizes, or -1 when the product passes 2^62.
inline int64_t product(int64_t a, int64_t b) {
  if (a < 0 || b < 0) return -1;
  if (a != 0 && b > (int64_t{1} << 62) / a) return -1;
  return a * b;
}

inline bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Status of the launches made so far on this thread.
inline int launch_status(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(CND_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  return CND_OK;
}

// SMs of the current device.
int sm_count();

// Limit of every wait inside a kernel (CND_WAIT_TIMEOUT_MS, 2 s).
uint64_t wait_timeout_ns();

}  // namespace layers
}  // namespace cnd

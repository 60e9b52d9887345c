// Shared by the layer kernels (norm.cu, recurrence.cu, linear.cu): element conversion,
// 16-byte vectors and launch checks.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <initializer_list>
#include <type_traits>

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

// Two float32 values in one 64-bit register pair: sm_100 multiplies and adds them with one
// instruction.
struct Two {
  unsigned long long bits;
};

__device__ __forceinline__ Two two(float lo, float hi) {
  Two t;
  asm("mov.b64 %0, {%1, %2};" : "=l"(t.bits) : "f"(lo), "f"(hi));
  return t;
}
__device__ __forceinline__ void unpack(Two t, float* lo, float* hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(*lo), "=f"(*hi) : "l"(t.bits));
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  Two d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.bits) : "l"(a.bits), "l"(b.bits), "l"(c.bits));
  return d;
}
__device__ __forceinline__ Two mul2(Two a, Two b) {
  Two d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.bits) : "l"(a.bits), "l"(b.bits));
  return d;
}
__device__ __forceinline__ Two add2(Two a, Two b) {
  Two d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.bits) : "l"(a.bits), "l"(b.bits));
  return d;
}
__device__ __forceinline__ Two same(float v) { return two(v, v); }

// 2^v and 1 / v to a few units in the last place, results below 2^-126 as zero.
__device__ __forceinline__ float exp2_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float reciprocal_fast(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// V elements at a 16-byte aligned address as pairs, and back (rounded once).
template <typename T, int V>
__device__ __forceinline__ void load_twos(const void* p, Two (&v)[V / 2]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      const ulonglong2 q = static_cast<const ulonglong2*>(p)[i];
      v[2 * i] = Two{q.x};
      v[2 * i + 1] = Two{q.y};
    }
  } else {
    uint32_t q[V / 2];
    *reinterpret_cast<uint4*>(q) = *static_cast<const uint4*>(p);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      if constexpr (std::is_same_v<T, __nv_bfloat16>) {
        v[i] = two(__uint_as_float(q[i] << 16), __uint_as_float(q[i] & 0xffff0000u));
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&q[i]));
        v[i] = two(f.x, f.y);
      }
    }
  }
}

template <typename T>
__device__ __forceinline__ uint32_t narrow2(Two v) {
  float lo, hi;
  unpack(v, &lo, &hi);
  uint32_t bits = 0;
  if constexpr (std::is_same_v<T, __nv_bfloat16>) {
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(bits) : "f"(hi), "f"(lo));
  } else if constexpr (std::is_same_v<T, __half>) {
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(bits) : "f"(hi), "f"(lo));
  }
  return bits;
}

template <typename T, int V>
__device__ __forceinline__ void store_twos(void* p, const Two (&v)[V / 2]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      static_cast<ulonglong2*>(p)[i] = make_ulonglong2(v[2 * i].bits, v[2 * i + 1].bits);
    }
  } else {
    *static_cast<uint4*>(p) =
        make_uint4(narrow2<T>(v[0]), narrow2<T>(v[1]), narrow2<T>(v[2]), narrow2<T>(v[3]));
  }
}

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

// Whether buffers (some may be NULL) start on multiples of `size` bytes, their elements' or, for a
// workspace, 16. An address in between would be a fault on the device.
inline bool aligned_to(size_t size, std::initializer_list<const void*> buffers) {
  for (const void* p : buffers) {
    if (reinterpret_cast<uintptr_t>(p) % size != 0) return false;
  }
  return true;
}
inline int wide_size(int dtype) { return dtype == CND_F64 ? 8 : 4; }  // of statistics and states
inline int misaligned(const char* who) {
  return fail(CND_ERR_INVALID, "%s: a buffer is not aligned to its elements", who);
}

// Status of the launches made so far on this thread.
inline int launch_status(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return fail(CND_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
  return CND_OK;
}

// SMs of the current device, which launches go by; and of a B200, which plans and workspace sizes
// go by: they are the same on a machine without a GPU.
int sm_count();
constexpr int kSms = 148;

}  // namespace layers
}  // namespace cnd

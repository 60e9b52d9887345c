// GELU (exact), SiLU and their slopes.
//   GELU(v) = v Phi(v), GELU'(v) = Phi(v) + v phi(v);
//   SiLU(v) = v s, SiLU'(v) = s (1 + v (1 - s)), s = 1 / (1 + exp(-v)).
#pragma once

#include "layers.cuh"

namespace cnd {
namespace layers {

// Phi(v) and exp(-v^2 / 2) by Abramowitz and Stegun, Handbook of Mathematical Functions,
// formula 7.1.26: erfc(x) = (a1 t + ... + a5 t^5) exp(-x^2), t = 1 / (1 + p x), off by at most
// 1.5e-7. Used where the result is rounded to 16 bits: it costs half of erff and shares
// its exponential with phi.
__device__ __forceinline__ float normal_cdf_16(float v, float* gauss) {
  const float x = fabsf(v) * 0.70710678f;
  const float t = __fdividef(1.0f, fmaf(0.3275911f, x, 1.0f));
  const float e = __expf(-x * x);
  float p = fmaf(1.061405429f, t, -1.453152027f);
  p = fmaf(p, t, 1.421413741f);
  p = fmaf(p, t, -0.284496736f);
  p = fmaf(p, t, 0.254829592f);
  const float tail = 0.5f * p * t * e;  // Phi(-|v|)
  *gauss = e;
  return v < 0.0f ? tail : 1.0f - tail;
}

// kExact: results of float32 or float64 accuracy; else good to well below 16-bit rounding.
template <bool kExact, typename A>
__device__ __forceinline__ A activate(A v, int act) {
  if (act == CND_ACT_GELU) {
    if constexpr (kExact) {
      return A(0.5) * v * (A(1) + erf(v * A(0.70710678118654752440)));
    } else {
      float gauss;
      const float cdf = normal_cdf_16(v, &gauss);
      return v == -INFINITY ? 0.0f * v : v * cdf;
    }
  }
  if (act == CND_ACT_SILU) {
    if constexpr (kExact) return v / (A(1) + exp(-v));
    return __fdividef(v, 1.0f + __expf(-v));
  }
  return v;
}

template <bool kExact, typename A>
__device__ __forceinline__ A activation_slope(A v, int act) {
  if (act == CND_ACT_GELU) {
    if constexpr (kExact) {
      const A cdf = A(0.5) * (A(1) + erf(v * A(0.70710678118654752440)));
      return cdf + v * exp(A(-0.5) * v * v) * A(0.39894228040143267794);
    } else {
      float gauss;
      const float cdf = normal_cdf_16(v, &gauss);
      return fmaf(v * gauss, 0.39894228f, cdf);
    }
  }
  if (act == CND_ACT_SILU) {
    A s;
    if constexpr (kExact) {
      s = A(1) / (A(1) + exp(-v));
    } else {
      s = __fdividef(1.0f, 1.0f + __expf(-v));
    }
    return s * (A(1) + v * (A(1) - s));
  }
  return A(1);
}

}  // namespace layers
}  // namespace cnd

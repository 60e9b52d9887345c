// GELU (exact), SiLU and their slopes.
//   GELU(v) = v Phi(v), GELU'(v) = Phi(v) + v phi(v);
//   SiLU(v) = v s, SiLU'(v) = s (1 + v (1 - s)), s = 1 / (1 + exp(-v)).
#pragma once

#include "layers.cuh"

namespace cnd {
namespace layers {

// Phi(-|v|) and exp(-v^2 / 2) of two values, with |v| cut at 6 in `size`:
//   Phi(-a) = Q(a) exp(-a^2 / 2),
// where Q(a) = erfcx(a / sqrt 2) / 2 is smooth and falls from 0.5 to 0.066 on [0, 6]. Q is the
// polynomial of degree 9 in a - 3 with the least relative error there, 9.0e-5 (fitted to
// double-precision erfc by iteratively reweighted least squares at Chebyshev points); beyond
// 6, Phi(-a) is below 1e-9. Used where the result is rounded to 16 bits (2^-11 and more):
// half an instruction a value and step and one exponential, shared with phi. A
// reciprocal beside the exponential costs 3 % more (1M x 64 -> 256 GELU 319 us against 310,
// where no activation took 192).
__device__ __forceinline__ Two normal_tail(Two v, Two* size, Two* gauss) {
  float lo, hi;
  unpack(v, &lo, &hi);
  *size = two(fminf(fabsf(lo), 6.0f), fminf(fabsf(hi), 6.0f));
  // exp(-v^2 / 2) = 2^(-v^2 / (2 ln 2))
  float e0, e1;
  unpack(mul2(mul2(v, v), same(-0.72134752044f)), &e0, &e1);
  *gauss = two(exp2_fast(e0), exp2_fast(e1));
  const Two t = add2(*size, same(-3.0f));
  Two q = fma2(t, same(-5.601578436653654e-07f), same(3.234303903809632e-06f));
  q = fma2(q, t, same(-4.0969457586470526e-06f));
  q = fma2(q, t, same(1.1100694791821297e-05f));
  q = fma2(q, t, same(-0.0001310931402258575f));
  q = fma2(q, t, same(0.0006133195711299777f));
  q = fma2(q, t, same(-0.0023177030961960554f));
  q = fma2(q, t, same(0.009094280190765858f));
  q = fma2(q, t, same(-0.03439052030444145f));
  q = fma2(q, t, same(0.12152419984340668f));
  return mul2(q, *gauss);
}

// act(v) of two values, good to well below 16-bit rounding. GELU(v) = max(v, 0) - |v| Phi(-|v|)
// for either sign; its value at -infinity is the limit, 0.
__device__ __forceinline__ Two activate2(Two v, int act) {
  if (act == CND_ACT_GELU) {
    Two size, gauss;
    const Two tail = normal_tail(v, &size, &gauss);
    float lo, hi;
    unpack(v, &lo, &hi);
    return fma2(mul2(size, same(-1.0f)), tail, two(fmaxf(lo, 0.0f), fmaxf(hi, 0.0f)));
  }
  if (act == CND_ACT_SILU) {
    float lo, hi, e0, e1;
    unpack(v, &lo, &hi);
    unpack(mul2(v, same(-1.44269504089f)), &e0, &e1);
    return two(__fdividef(lo, 1.0f + exp2_fast(e0)), __fdividef(hi, 1.0f + exp2_fast(e1)));
  }
  return v;
}

// act'(v) of two values, likewise.
__device__ __forceinline__ Two slope2(Two v, int act) {
  float lo, hi;
  unpack(v, &lo, &hi);
  if (act == CND_ACT_GELU) {
    Two size, gauss;
    // Phi(v) = 1/2 + copysign(1/2 - Phi(-|v|), v)
    float s0, s1;
    unpack(fma2(normal_tail(v, &size, &gauss), same(-1.0f), same(0.5f)), &s0, &s1);
    const Two cdf = add2(two(copysignf(s0, lo), copysignf(s1, hi)), same(0.5f));
    return fma2(mul2(two(copysignf(1.0f, lo), copysignf(1.0f, hi)), mul2(size, gauss)),
                same(0.39894228040f), cdf);
  }
  if (act == CND_ACT_SILU) {
    float e0, e1;
    unpack(mul2(v, same(-1.44269504089f)), &e0, &e1);
    const Two s = two(reciprocal_fast(1.0f + exp2_fast(e0)), reciprocal_fast(1.0f + exp2_fast(e1)));
    return mul2(s, fma2(v, fma2(s, same(-1.0f), same(1.0f)), same(1.0f)));
  }
  return same(1.0f);
}

// To the accuracy of float32 and float64.
template <typename A>
__device__ __forceinline__ A activate(A v, int act) {
  if (act == CND_ACT_GELU) return A(0.5) * v * (A(1) + erf(v * A(0.70710678118654752440)));
  if (act == CND_ACT_SILU) return v / (A(1) + exp(-v));
  return v;
}

template <typename A>
__device__ __forceinline__ A activation_slope(A v, int act) {
  if (act == CND_ACT_GELU) {
    const A cdf = A(0.5) * (A(1) + erf(v * A(0.70710678118654752440)));
    return cdf + v * exp(A(-0.5) * v * v) * A(0.39894228040143267794);
  }
  if (act == CND_ACT_SILU) {
    const A s = A(1) / (A(1) + exp(-v));
    return s * (A(1) + v * (A(1) - s));
  }
  return A(1);
}

}  // namespace layers
}  // namespace cnd

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
// double-precision erfc by iteratively reweighted least squares at Chebyshev points). Beyond
// 6, Phi(-a) is below 1e-9, and a Q(a) and a phi(a) are taken with the a of 6: GELU there, below
// 6e-9, is 1 to 3 % off, and its slope, below 4e-8, too small by up to 6 / a. Used where the result
// is rounded to 16 bits (2^-11 and more): half an instruction a value and step and one
// exponential, shared with phi. A reciprocal beside the exponential costs 3 % more (1M x 64 ->
// 256 GELU 319 us against 310, where no activation took 192).
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

// act(v) of two values, good to well below 16-bit rounding for |v| < 6. GELU(v) = max(v, 0) - |v| Phi(-|v|)
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

// Phi(-|v|) and exp(-v^2 / 2) to the accuracy of float32 and float64, also where the result is far
// smaller than v (0.5 (1 + erf(v / sqrt 2)) loses a quarter of a thousandth at v = -4 in float32 and
// everything at -5.6). `size` is |v|, cut at 40: from there on phi(v) is zero in float64 too, and
// at the infinities 40 * 0 is GELU's limit.
// float32: Phi(-a) = t R(t) exp(-a^2 / 2) with t = 1 / (1 + 0.35 a), the form of Hastings
// (Approximations for Digital Computers, 1955). R is the polynomial of degree 8 with the least
// relative error for a in [0, 14.5], 3.2e-8 (fitted to double-precision erfcx by iteratively
// reweighted least squares at Chebyshev points; the best of 0.15 ... 0.6 in the denominator);
// with float32 roundings 5.4 units of 2^-24. erfc takes half again the time (262144 x 64 -> 256
// GELU 448 us against 286; with erf, 278).
__device__ __forceinline__ float normal_tail(float v, float* size, float* gauss) {
  *size = fminf(fabsf(v), 40.0f);
  *gauss = expf(-0.5f * v * v);
  const float d = fmaf(0.35f, *size, 1.0f);
  float t = reciprocal_fast(d);
  t = fmaf(t, fmaf(-d, t, 1.0f), t);  // one Newton step
  float r = fmaf(t, -0.029158029705286026f, 0.1440316140651703f);
  r = fmaf(r, t, -0.25584039092063904f);
  r = fmaf(r, t, 0.15932124853134155f);
  r = fmaf(r, t, -0.02321339212357998f);
  r = fmaf(r, t, 0.10555292665958405f);
  r = fmaf(r, t, 0.11982118338346481f);
  r = fmaf(r, t, 0.1398635357618332f);
  r = fmaf(r, t, 0.139621302485466f);
  return r * t * *gauss;
}

__device__ __forceinline__ double normal_tail(double v, double* size, double* gauss) {
  *size = fmin(fabs(v), 40.0);
  *gauss = exp(-0.5 * v * v);
  return 0.5 * erfc(*size * 0.70710678118654752440);
}

// SiLU below -88 (float32) is zero.
template <typename A>
__device__ __forceinline__ A activate(A v, int act) {
  if (act == CND_ACT_GELU) {
    A size, gauss;
    const A tail = normal_tail(v, &size, &gauss);
    return v < A(0) ? -size * tail : v * (A(1) - tail);
  }
  if (act == CND_ACT_SILU) return v / (A(1) + exp(-v));
  return v;
}

template <typename A>
__device__ __forceinline__ A activation_slope(A v, int act) {
  if (act == CND_ACT_GELU) {
    A size, gauss;
    const A tail = normal_tail(v, &size, &gauss);
    return (v < A(0) ? tail : A(1) - tail) +
           copysign(size, v) * gauss * A(0.39894228040143267794);
  }
  if (act == CND_ACT_SILU) {
    const A s = A(1) / (A(1) + exp(-v));
    return s * (A(1) + v * (A(1) - s));
  }
  return A(1);
}

}  // namespace layers
}  // namespace cnd

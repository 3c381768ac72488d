// Activations of tsc_linear_act on f32 values.
#pragma once

#include "common.hpp"

namespace tsc {

// 2^x and 1/x by the hardware's one-instruction forms (within a few ulp of f32).
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float rcp_fast(float x) { return __builtin_amdgcn_rcpf(x); }

// x * sigmoid(y): x / (1 + e^-y).  e^-y is infinite for y below about -89,
// where 1/inf = 0 gives the limit.
__device__ __forceinline__ float times_sigmoid(float x, float y) {
  return x * rcp_fast(1.f + exp2_fast(-1.442695041f * y));
}

// x * Phi(x), Phi the normal distribution function, for results of type T.  With
// u = |x| and Q(u) = 1 - Phi(u) = R(u) e^(-u^2 / 2),
//   x Phi(x) = max(x, 0) - u Q(u):
// nothing cancels where x is negative, and there is no branch.  R falls from 1/2
// like 0.4 / u, so it is t times a polynomial in t = 1 / (1 + c u); both
// polynomials are least-maximum fits over u from 0 to 14.5, from where on u Q(u)
// is 0 in f32.  The library's erff takes several times as many operations, and
// loses the negative tail, where 1 + erf cancels (relative errors, fit / 1 + erf in
// f32: -3 4e-7 / 1e-5, -5 4e-7 / 5e-2, -8 4e-7 / 1).
// 60,013 x 192 -> 768 f16 48.3 us, with a polynomial of one degree less that is
// right to 1.5e-7 of 1 only (2e-3 relative at -5, 4e-2 at -13) 47.7.
template <typename T>
__device__ __forceinline__ float gelu(float x) {
  constexpr bool F32 = sizeof(T) == 4;
  // (the limit keeps inf * 0 from being formed; NaN passes in f32)
  const float a = __builtin_fabsf(x), u = F32 ? (a > 16.f ? 16.f : a) : __builtin_amdgcn_fmed3f(a, 0.f, 16.f);
  const float t = rcp_fast(__builtin_fmaf(F32 ? 0.345f : 0.29f, u, 1.f));
  float p, e;
  if constexpr (F32) {
    // 2.3e-8 relative
    p = __builtin_fmaf(-0.02815178409f, t, 0.1442335248f);
    p = __builtin_fmaf(p, t, -0.2691534162f);
    p = __builtin_fmaf(p, t, 0.185054481f);
    p = __builtin_fmaf(p, t, -0.03623782471f);
    p = __builtin_fmaf(p, t, 0.1112676784f);
    p = __builtin_fmaf(p, t, 0.117362f);
    p = __builtin_fmaf(p, t, 0.1380052418f);
    p = __builtin_fmaf(p, t, 0.1376201063f);
    // e^(-u^2 / 2) = 2^(-k u^2), the exponent in two parts: rounded to one, it is off by
    // up to 4e-6 where u is 13
    constexpr float k = 0.72134752f, k_low = 0x1.4ae0bfp-27f;
    const float s = u * u, h = -k * s;
    float low = __builtin_fmaf(-k, s, -h);
    low = __builtin_fmaf(-k, __builtin_fmaf(u, u, -s), low);
    low = __builtin_fmaf(-k_low, s, low);
    e = exp2_fast(h);
    e = __builtin_fmaf(e * low, 0.69314718f, e);
  } else {
    // 8e-8 of 1 and 9e-5 relative, 15 operations in all: a fifth of f16's rounding
    // at most
    p = __builtin_fmaf(-0.08813589066f, t, 0.2824412286f);
    p = __builtin_fmaf(p, t, -0.0898046419f);
    p = __builtin_fmaf(p, t, 0.1772846878f);
    p = __builtin_fmaf(p, t, 0.1014221385f);
    p = __builtin_fmaf(p, t, 0.1167925596f);
    e = exp2_fast(-0.72134752f * x * x);  // NaN for NaN
  }
  return __builtin_fmaf(-u, p * t * e, __builtin_amdgcn_fmed3f(x, 0.f, __builtin_inff()));
}

// The activation of a value that leaves as T.
template <int ACT, typename T>
__device__ __forceinline__ float activate(float v) {
  if constexpr (ACT == TSC_ACT_RELU) return v < 0.f ? 0.f : v;  // NaN stays NaN
  if constexpr (ACT == TSC_ACT_GELU) return gelu<T>(v);
  if constexpr (ACT == TSC_ACT_GELU_TANH) {
    // 0.5 v (1 + tanh u) = v sigmoid(2u), u = sqrt(2/pi) (v + 0.044715 v^3)
    const float y = 1.5957691216f * v * __builtin_fmaf(0.044715f * v, v, 1.f);
    return v == -__builtin_inff() ? 0.f : times_sigmoid(v, y);
  }
  if constexpr (ACT == TSC_ACT_SILU) return v == -__builtin_inff() ? 0.f : times_sigmoid(v, v);
  return v;
}

}  // namespace tsc

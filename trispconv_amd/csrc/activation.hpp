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

// x * Phi(x), Phi the normal distribution function.  With z = |x| / sqrt(2)
// and t = 1 / (1 + 0.3275911 z), erfc(z) = t (a1 + t (a2 + ...)) e^(-z^2) to
// 1.5e-7 (Abramowitz and Stegun, Handbook of Mathematical Functions, 7.1.26).
// Phi(x) is 1 - erfc / 2 for x >= 0 and erfc / 2 below, so
//   x Phi(x) = max(x, 0) - |x| erfc(z) / 2:
// nothing cancels in the negative tail, and there is no branch.  14 operations
// for every output; the library's erff takes several times as many.
__device__ __forceinline__ float gelu(float x) {
  // erfc is 0 in f32 long before 16: the limit keeps inf * 0 from being formed
  const float u = __builtin_amdgcn_fmed3f(__builtin_fabsf(x), 0.f, 16.f);
  const float t = rcp_fast(__builtin_fmaf(0.3275911f * 0.70710678f, u, 1.f));
  // the coefficients, halved
  float p = __builtin_fmaf(0.5307027145f, t, -0.7265760135f);
  p = __builtin_fmaf(p, t, 0.7107068705f);
  p = __builtin_fmaf(p, t, -0.142248368f);
  p = __builtin_fmaf(p, t, 0.127414796f);
  // e^(-z^2) = 2^(-x^2 / (2 ln 2)); NaN for NaN
  const float e = exp2_fast(-0.72134752f * x * x);
  return __builtin_fmaf(-u, p * t * e, __builtin_amdgcn_fmed3f(x, 0.f, __builtin_inff()));
}

template <int ACT>
__device__ __forceinline__ float activate(float v) {
  if constexpr (ACT == TSC_ACT_RELU) return v < 0.f ? 0.f : v;  // NaN stays NaN
  if constexpr (ACT == TSC_ACT_GELU) return gelu(v);
  if constexpr (ACT == TSC_ACT_GELU_TANH) {
    // 0.5 v (1 + tanh u) = v sigmoid(2u), u = sqrt(2/pi) (v + 0.044715 v^3)
    const float y = 1.5957691216f * v * __builtin_fmaf(0.044715f * v, v, 1.f);
    return v == -__builtin_inff() ? 0.f : times_sigmoid(v, y);
  }
  if constexpr (ACT == TSC_ACT_SILU) return v == -__builtin_inff() ? 0.f : times_sigmoid(v, v);
  return v;
}

}  // namespace tsc

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
// 1.5e-7 (Abramowitz and Stegun, Handbook of Mathematical Functions, 7.1.26);
// x Phi(x) is x - x erfc / 2 for x >= 0 and x erfc / 2 below, so the negative
// tail keeps its relative accuracy instead of cancelling against 1.  A dozen
// operations; the library's erff takes several times as many, and this
// epilogue runs once for every output of products that are bound by memory.
__device__ __forceinline__ float gelu(float x) {
  const float z = __builtin_fabsf(x) * 0.70710678f;
  const float t = rcp_fast(__builtin_fmaf(0.3275911f, z, 1.f));
  float p = __builtin_fmaf(1.061405429f, t, -1.453152027f);
  p = __builtin_fmaf(p, t, 1.421413741f);
  p = __builtin_fmaf(p, t, -0.284496736f);
  p = __builtin_fmaf(p, t, 0.254829592f);
  // e^(-z^2) = 2^(-x^2 / (2 ln 2))
  const float e = exp2_fast(-0.72134752f * x * x);
  const float half_erfc = 0.5f * p * t * e;
  // x = +-inf: t = 0 and e = 0, so half_erfc = 0 and inf * 0 must not be formed
  if (x >= 0.f) return half_erfc == 0.f ? x : __builtin_fmaf(-x, half_erfc, x);
  return half_erfc == 0.f ? 0.f : x * half_erfc;
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

// y = act(x W^T + bias) + residual for the rows of a feature tensor.
//
//   v[r][o] = sum_i x[r][i] w[o][i]  (f32 sums),  v += bias[o],
//   v = act(v),  v += residual[r][o],  one rounding to the rows' type.
#include "common.hpp"

#include "activation.hpp"

namespace tsc {
namespace {

struct LinearArgs {
  const void* x;
  int64_t x_stride;
  const void* w;
  int64_t w_stride;
  const void* bias;
  int bias_dtype;
  const void* residual;
  int64_t r_stride;
  void* out;
  int64_t n;
  int c_in, c_out;
};

__device__ __forceinline__ float load_any(const void* p, int dtype, int64_t i) {
  if (dtype == TSC_F32) return static_cast<const float*>(p)[i];
  if (dtype == TSC_F16) return to_f32(static_cast<const __half*>(p)[i]);
  return to_f32(static_cast<const __hip_bfloat16*>(p)[i]);
}

// 64 rows x 64 columns for a workgroup, 4 x 4 of them for a thread, operands
// widened to f32 in LDS sixteen input channels at a time.  Any size, stride
// and alignment.
template <typename T, int ACT>
__global__ void __launch_bounds__(256) linear_any_kernel(LinearArgs a) {
  __shared__ float xs[16][65], ws[16][65];
  const int64_t r0 = blockIdx.x * (int64_t)64;
  const int o0 = blockIdx.y * 64;
  const T* x = static_cast<const T*>(a.x);
  const T* w = static_cast<const T*>(a.w);
  const int tr = threadIdx.x / 16, tc = threadIdx.x % 16;
  float acc[4][4] = {};
  for (int i0 = 0; i0 < a.c_in; i0 += 16) {
    for (int e = threadIdx.x; e < 1024; e += 256) {
      const int m = e / 16, i = e % 16;
      const bool in = i0 + i < a.c_in;
      xs[i][m] = in && r0 + m < a.n ? to_f32(x[(r0 + m) * a.x_stride + i0 + i]) : 0.f;
      ws[i][m] = in && o0 + m < a.c_out ? to_f32(w[(o0 + m) * a.w_stride + i0 + i]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 16; ++i)
#pragma unroll
      for (int p = 0; p < 4; ++p)
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[p][q] += xs[i][tr + 16 * p] * ws[i][tc + 16 * q];
    __syncthreads();
  }
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const int64_t r = r0 + tr + 16 * p;
    if (r >= a.n) continue;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int o = o0 + tc + 16 * q;
      if (o >= a.c_out) continue;
      float v = acc[p][q];
      if (a.bias) v += load_any(a.bias, a.bias_dtype, o);
      v = activate<ACT>(v);
      if (a.residual) v += to_f32(static_cast<const T*>(a.residual)[r * a.r_stride + o]);
      static_cast<T*>(a.out)[r * a.c_out + o] = from_f32<T>(v);
    }
  }
}

template <typename T, int ACT>
int launch_linear(const LinearArgs& a, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(ceil_div(a.n, 64)), static_cast<unsigned>(ceil_div(a.c_out, 64)));
  linear_any_kernel<T, ACT><<<grid, 256, 0, s>>>(a);
  TSC_LAUNCH_CHECK("linear_act");
  return 0;
}

template <typename T>
int launch_linear(int act, const LinearArgs& a, hipStream_t s) {
  switch (act) {
    case TSC_ACT_NONE: return launch_linear<T, TSC_ACT_NONE>(a, s);
    case TSC_ACT_RELU: return launch_linear<T, TSC_ACT_RELU>(a, s);
    case TSC_ACT_GELU: return launch_linear<T, TSC_ACT_GELU>(a, s);
    case TSC_ACT_GELU_TANH: return launch_linear<T, TSC_ACT_GELU_TANH>(a, s);
    default: return launch_linear<T, TSC_ACT_SILU>(a, s);
  }
}

}  // namespace
}  // namespace tsc

using namespace tsc;

extern "C" int tsc_linear_act(const void* x, int64_t x_stride, const void* weight,
                              int64_t w_stride, const void* bias, int32_t bias_dtype,
                              const void* residual, int64_t r_stride, int32_t dtype, int64_t n,
                              int32_t c_in, int32_t c_out, int32_t act, void* out,
                              tsc_stream_t stream) {
  TSC_REQUIRE(dtype_ok(dtype) && dtype_ok(bias_dtype), "linear_act: unknown dtype");
  TSC_REQUIRE(n >= 0 && n < (1ll << 31) && c_in >= 0 && c_out >= 0, "linear_act: invalid sizes");
  TSC_REQUIRE(act >= TSC_ACT_NONE && act <= TSC_ACT_SILU, "linear_act: unknown activation");
  if (n == 0 || c_out == 0) return 0;
  TSC_REQUIRE(out && (c_in == 0 || (x && weight)), "linear_act: null pointer");
  TSC_REQUIRE(x_stride >= 0 && w_stride >= 0 && r_stride >= 0, "linear_act: negative stride");
  const LinearArgs a{x, x_stride, weight, w_stride, bias, bias_dtype, residual, r_stride, out, n, c_in, c_out};
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case TSC_F32: return launch_linear<float>(act, a, s);
    case TSC_F16: return launch_linear<__half>(act, a, s);
    default: return launch_linear<__hip_bfloat16>(act, a, s);
  }
}

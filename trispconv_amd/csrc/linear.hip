// Entry point of act(x W^T + bias) + residual.
#include "linear.hpp"

namespace tsc {
extern template int launch_linear<float>(const LinearArgs&, hipStream_t);
extern template int launch_linear<__half>(const LinearArgs&, hipStream_t);
extern template int launch_linear<__hip_bfloat16>(const LinearArgs&, hipStream_t);
}  // namespace tsc

using namespace tsc;

extern "C" int tsc_linear_act(const void* x, int64_t x_stride, const void* weight,
                              int64_t w_stride, const void* bias, int32_t bias_dtype,
                              const void* residual, int64_t r_stride, int32_t dtype, int64_t n,
                              int32_t c_in, int32_t c_out, int32_t act, void* out,
                              tsc_stream_t stream) {
  TSC_REQUIRE(dtype_ok(dtype) && dtype_ok(bias_dtype), "linear_act: unknown dtype");
  TSC_REQUIRE(n >= 0 && n < (1ll << 31) && c_in >= 0 && c_out >= 0 && c_out < (1 << 24),
              "linear_act: invalid sizes");
  TSC_REQUIRE(act >= TSC_ACT_NONE && act <= TSC_ACT_SILU, "linear_act: unknown activation");
  if (n == 0 || c_out == 0) return 0;
  TSC_REQUIRE(out && (c_in == 0 || (x && weight)), "linear_act: null pointer");
  TSC_REQUIRE(x_stride >= 0 && w_stride >= 0 && r_stride >= 0, "linear_act: negative stride");
  const LinearArgs a{x, x_stride, weight, w_stride, bias, bias_dtype, residual, r_stride, act, out, n, c_in, c_out};
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case TSC_F32: return launch_linear<float>(a, s);
    case TSC_F16: return launch_linear<__half>(a, s);
    default: return launch_linear<__hip_bfloat16>(a, s);
  }
}

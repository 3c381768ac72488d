// The product kernels on bf16 tensors.
#include "linear.hpp"

namespace tsc {
template int launch_linear<__hip_bfloat16>(const LinearArgs&, hipStream_t);
}  // namespace tsc

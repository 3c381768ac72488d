// The product kernels on f32 tensors.
#include "linear.hpp"

namespace tsc {
template int launch_linear<float>(const LinearArgs&, hipStream_t);
}  // namespace tsc

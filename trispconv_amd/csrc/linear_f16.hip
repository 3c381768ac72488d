// The product kernels on f16 tensors.
#include "linear.hpp"

namespace tsc {
template int launch_linear<__half>(const LinearArgs&, hipStream_t);
}  // namespace tsc

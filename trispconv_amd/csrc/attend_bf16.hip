// The attention kernels on bf16 tensors.
#include "attend.hpp"

namespace tsc {
template int launch_attend<__hip_bfloat16>(const AttendArgs&, const Cut&, hipStream_t);
}  // namespace tsc

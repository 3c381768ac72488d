// The attention kernels on f32 tensors.
#include "attend.hpp"

namespace tsc {
template int launch_attend<float>(const AttendArgs&, const Cut&, hipStream_t);
}  // namespace tsc

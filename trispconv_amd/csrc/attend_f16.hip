// The attention kernels on f16 tensors.
#include "attend.hpp"

namespace tsc {
template int launch_attend<__half>(const AttendArgs&, const Cut&, hipStream_t);
}  // namespace tsc

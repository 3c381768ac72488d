// The paged attention kernels on bf16 tensors.
#include "cache.hpp"

namespace tsc {
template int launch_cache<__hip_bfloat16>(const CacheArgs&, const CachePlan&, hipStream_t);
}  // namespace tsc

// The paged attention kernels on f32 tensors.
#include "cache.hpp"

namespace tsc {
template int launch_cache<float>(const CacheArgs&, const CachePlan&, hipStream_t);
}  // namespace tsc

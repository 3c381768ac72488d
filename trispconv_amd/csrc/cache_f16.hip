// The paged attention kernels on f16 tensors.
#include "cache.hpp"

namespace tsc {
template int launch_cache<__half>(const CacheArgs&, const CachePlan&, hipStream_t);
}  // namespace tsc

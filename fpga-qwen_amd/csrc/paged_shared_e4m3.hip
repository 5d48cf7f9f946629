// Attention behind shared prefixes over E4M3 caches.
#include "paged_shared.hpp"

namespace qwen_hip {
template void shared_launch<kPagedE4M3>(int, const PagedView&, const SharedArgs&, const SharedPlan&, hipStream_t);
}  // namespace qwen_hip

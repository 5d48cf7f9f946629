// Attention behind shared prefixes over F16 caches.
#include "paged_shared.hpp"

namespace qwen_hip {
template void shared_launch<kPagedF16>(int, const PagedView&, const SharedArgs&, const SharedPlan&, hipStream_t);
}  // namespace qwen_hip

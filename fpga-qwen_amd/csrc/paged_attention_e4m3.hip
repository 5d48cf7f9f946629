// Paged attention over E4M3 caches.
#include "paged_attention.hpp"

namespace qwen_hip {
template void attention_launch<kPagedE4M3>(int, const PagedView&, const AttentionArgs&, const AttentionPlan&,
                                         hipStream_t);
}  // namespace qwen_hip

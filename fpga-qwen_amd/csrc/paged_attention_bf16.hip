// Paged attention over BF16 caches.
#include "paged_attention.hpp"

namespace qwen_hip {
template void attention_launch<kPagedBF16>(int, const PagedView&, const AttentionArgs&, const AttentionPlan&,
                                         hipStream_t);
}  // namespace qwen_hip

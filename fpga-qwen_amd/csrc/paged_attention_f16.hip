// Paged attention over F16 caches.
#include "paged_attention.hpp"

namespace qwen_hip {
template void attention_launch<kPagedF16>(int, const PagedView&, const AttentionArgs&, const AttentionPlan&,
                                        hipStream_t);
}  // namespace qwen_hip

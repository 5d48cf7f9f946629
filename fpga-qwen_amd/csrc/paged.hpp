// Paged key-value cache: append, attention of new tokens, eviction.
#pragma once
#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "qwen_gpu.h"

namespace qwen_hip {

// Each checks its arguments (std::runtime_error) before it launches anything
// and runs on the device that holds the cache.
void launch_paged_append(const qwen_gpu_paged_cache& cache, const qwen_gpu_paged_batch& batch, const float* keys,
                         int64_t key_stride, const float* values, int64_t value_stride, hipStream_t stream);
void launch_paged_attention(const qwen_gpu_paged_cache& cache, const qwen_gpu_paged_batch& batch, const float* queries,
                            int64_t query_stride, int query_heads, float scale, float* out, int64_t out_stride,
                            void* workspace, size_t workspace_bytes, hipStream_t stream);
void launch_paged_evict(const qwen_gpu_paged_cache& cache, const qwen_gpu_paged_batch& batch, int keep, int sinks,
                        int recent, int32_t* new_lengths, float* new_weights, int32_t* new_positions, void* workspace,
                        size_t workspace_bytes, hipStream_t stream);
void launch_paged_attention_shared(const qwen_gpu_paged_cache& cache, const qwen_gpu_paged_batch& batch,
                                   const qwen_gpu_paged_prefix& prefix, const float* queries, int64_t query_stride,
                                   int query_heads, float scale, float* out, int64_t out_stride, void* workspace,
                                   size_t workspace_bytes, hipStream_t stream);
size_t paged_shared_workspace_bytes(const qwen_gpu_paged_cache& cache, const qwen_gpu_paged_batch& batch,
                                    const qwen_gpu_paged_prefix& prefix, int query_heads);
// Bytes of workspace that serve both the attention and the eviction, without query heads the eviction alone.
size_t paged_workspace_bytes(const qwen_gpu_paged_cache& cache, const qwen_gpu_paged_batch& batch, int query_heads);

}  // namespace qwen_hip

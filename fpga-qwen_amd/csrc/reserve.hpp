// Pages and rows of a step over a paged cache.
#pragma once
#include <hip/hip_runtime.h>

#include "qwen_gpu.h"

namespace qwen_hip {

// Checks its arguments (std::runtime_error) before it launches anything.
void launch_paged_reserve(const qwen_gpu_paged_pool& pool, const qwen_gpu_paged_growth& growth, hipStream_t stream);

}  // namespace qwen_hip

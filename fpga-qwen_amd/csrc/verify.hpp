// Verification of drafted tokens against the target's probabilities.
#pragma once
#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

#include "qwen_gpu.h"

namespace qwen_hip {

// Each checks its arguments first (std::runtime_error).
size_t verify_workspace_bytes(const qwen_gpu_draft& draft);
void launch_verify_draft(const qwen_gpu_draft& draft, int32_t* accepted, int32_t* next, int32_t* back, void* workspace,
                         size_t workspace_bytes, hipStream_t stream);

}  // namespace qwen_hip

// Norm of queries' and keys' heads and their rotation by position.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "qwen_gpu.h"

namespace qwen_hip {

// Each checks its arguments first (std::runtime_error).
void rotary_frequencies(int scaling, int dims, double base, double factor, double trained, double slow, double fast,
                        double* frequencies, float* magnitude);
void launch_rotate(const qwen_gpu_rotary& rotary, const qwen_gpu_rotary_heads& queries,
                   const qwen_gpu_rotary_heads* keys, const int32_t* positions, int rows, hipStream_t stream);

}  // namespace qwen_hip

// What the kernels of the paged key-value cache share: the view of cache and
// batch that a launch gets by value, and where its rows lie.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "half_split.hpp"
#include "op_device.hpp"
#include "qwen_gpu.h"

namespace qwen_hip {

constexpr int kPagedF16 = QWEN_GPU_PAGED_F16, kPagedBF16 = QWEN_GPU_PAGED_BF16, kPagedE4M3 = QWEN_GPU_PAGED_E4M3;
constexpr int kPagedMaxLength = 1 << 24;
// The front of a workspace, zero between calls; the rest is any call's own.
constexpr size_t kPagedCounterBytes = QWEN_GPU_PAGED_COUNTER_BYTES;

// Slot j of a sequence is slot j % page_size of its page j / page_size. With
// magic = floor((2^32 - 1) / page_size) the upper half of j * magic is the
// quotient or one less for every j < 2^32.
struct PageSlot {
    int page, slot;
};
__host__ __device__ __forceinline__ PageSlot page_slot(unsigned j, unsigned page_size, unsigned magic) {
    unsigned q = static_cast<unsigned>((static_cast<unsigned long long>(j) * magic) >> 32);
    unsigned r = j - q * page_size;
    if (r >= page_size) ++q, r -= page_size;
    return {static_cast<int>(q), static_cast<int>(r)};
}

// Strides in bytes.
struct PagedView {
    char* keys;
    char* values;
    uint8_t* exponents;
    int64_t page_stride, head_stride, slot_stride;
    const int32_t* table;
    const int32_t* lengths;
    const int32_t* offsets;
    const int32_t* seen;
    float* weights;
    int32_t* positions;
    int64_t track_stride;
    int pages, page_size, kv_heads;
    unsigned magic;
    int sequences, table_stride, max_length, rows, total_rows;

    __device__ int length(int s) const { return min(max(lengths[s], 0), max_length); }
    // First new row of a sequence and their number.
    __device__ int new_rows(int s, int& first) const {
        if (!offsets) {
            first = s * rows;
            return rows;
        }
        first = offsets[s];
        const int64_t n = int64_t(offsets[s + 1]) - first;
        return n < 0 ? 0 : n > rows ? rows : int(n);
    }
    // Which of a sequence's n new rows exist: from .. to - 1 (0 .. n - 1 unless offsets pass total_rows).
    __device__ void existing(int first, int n, int& from, int& to) const {
        to = int(max(int64_t(0), min(int64_t(n), int64_t(total_rows) - first)));
        from = int(min(int64_t(to), max(int64_t(0), -int64_t(first))));
    }
    // Sequence of a new row, -1 where it has none: the number of offsets up to
    // `row`, less one. The lanes of a wave probe 64 of them at a time.
    __device__ int sequence_of(int row, int lane) const {
        if (!offsets) return row / rows;
        int low = 0, high = sequences + 1;  // the number lies in low .. high
        while (high > low) {
            const int step = (high - low + 63) / 64;
            const int at = low + lane * step;
            const unsigned long long upto = __ballot(at < high && offsets[min(at, sequences)] <= row);
            const int n = __popcll(upto);  // offsets rise, so these are the first lanes
            if (n == 0) {
                high = low;
            } else {
                const int last = low + (n - 1) * step;  // offsets[last] <= row
                high = min(high, last + step);
                low = last + 1;
            }
        }
        return low - 1 < sequences ? low - 1 : -1;
    }
    // Page of the table's entry, -1 where it holds none.
    __device__ int page_of(int s, int entry) const {
        const int page = table[int64_t(s) * table_stride + entry];
        return page >= 0 && page < pages ? page : -1;
    }
    __device__ int64_t row_at(int page, int head, int slot) const {
        return page * page_stride + head * head_stride + slot * slot_stride;
    }
    __device__ int64_t exponents_at(int page, int head, int slot) const {
        return 2 * ((int64_t(page) * kv_heads + head) * page_size + slot);
    }
    __device__ int64_t track_at(int s, int head) const { return (int64_t(s) * kv_heads + head) * track_stride; }
};

// 2^(byte - 127); a byte of 0 stands for 2^-127, which is no normal number,
// and is taken as 0: no row is written with it.
__device__ __forceinline__ float byte_pow2(unsigned byte) { return __builtin_bit_cast(float, byte << 23); }

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned uint4_t __attribute__((ext_vector_type(4)));
// Eight floats at any 4-byte address: global loads need no more alignment.
typedef float float4_a4 __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ unsigned pack_bf16(float a, float b) {
    const bf16x2 v = {static_cast<__bf16>(a), static_cast<__bf16>(b)};  // v_cvt_pk_bf16_f32, to nearest even
    return __builtin_bit_cast(unsigned, v);
}
__device__ __forceinline__ unsigned pack_half(float a, float b) {
    return to_half_bits(a) | unsigned(to_half_bits(b)) << 16;
}

// Sum of the lanes up to this one, through DPP row shifts and broadcasts.
__device__ __forceinline__ int scan_lanes(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, true);   // row_shr:1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2 and 3
    return x;
}

// Host side: checks (std::runtime_error), the view, the device.
PagedView paged_view(const qwen_gpu_paged_cache& cache, const qwen_gpu_paged_batch& batch);
void paged_check_rows(const qwen_gpu_paged_batch& batch);
void paged_check_heads(const qwen_gpu_paged_cache& cache, int query_heads);

// Workspace of an eviction that moves at most `room` rows of a head.
size_t paged_moves_bytes(const qwen_gpu_paged_cache& cache, const qwen_gpu_paged_batch& batch, int64_t room);

// The device that holds the cache; all of a call's arrays are checked.
class PagedDevice : public OpDevice {
public:
    PagedDevice(const qwen_gpu_paged_cache& cache, const qwen_gpu_paged_batch& batch, hipStream_t stream);
};

}  // namespace qwen_hip

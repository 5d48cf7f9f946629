// Pages and rows of a step over a paged cache.
#include "reserve.hpp"

#include <cstdint>
#include <string>

#include "op_device.hpp"
#include "paged_dev.hpp"
#include "qwen_common.hpp"

namespace qwen_hip {

namespace {

constexpr int kThreads = 1024, kEach = 4, kMost = kThreads * kEach;  // sequences of a thread, of a call
constexpr int kMaxRow = 1 << 30;

struct ReserveView {
    int32_t* table;
    int32_t* free_pages;
    const int32_t *held, *free_count, *shared, *lengths, *seen, *changes;
    int32_t *new_lengths, *new_seen, *new_held, *new_free_count, *offsets, *row_sequences, *row_positions;
    int64_t* row_slots;
    int pages, page_size, sequences, table_stride, total_rows, most;  // most positions of a sequence
    unsigned magic;
};

// What a scan has to hold: pages are at most 2^24 a sequence, rows 2^30.
__device__ __forceinline__ int64_t scan_wave(int64_t x, int lane) {
#pragma unroll
    for (int off = 1; off < 64; off *= 2) {
        const int64_t other = __shfl_up(x, off);
        if (lane >= off) x += other;
    }
    return x;
}

// The sum over all threads before this one; `total` of all.
__device__ __forceinline__ int64_t scan_block(int64_t x, int64_t* waves, int64_t& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t upto = scan_wave(x, lane);
    if (lane == 63) waves[wave] = upto;
    __syncthreads();
    const int64_t of_lane = scan_wave(lane < kThreads / 64 ? waves[lane] : 0, lane);
    total = __shfl(of_lane, kThreads / 64 - 1);
    const int64_t before = __shfl(of_lane, max(wave - 1, 0));
    __syncthreads();
    return (wave ? before : 0) + upto - x;
}

// The first of n rising sums that is above k; the last one is.
__device__ __forceinline__ int owner(const int* upto, int n, int k) {
    int low = 0, high = n - 1;
    while (low < high) {
        const int middle = (low + high) / 2;
        if (upto[middle] > k)
            high = middle;
        else
            low = middle + 1;
    }
    return low;
}

__device__ __forceinline__ int clipped(int64_t x) { return int(min(x, int64_t(0x7fffffff))); }

// One workgroup: three sums over the sequences (pages given back, pages
// needed, rows granted), and after each the pages or rows themselves, a thread each,
// whose sequences are found in the sums. Latency bounds it.
__global__ __launch_bounds__(kThreads) void reserve_kernel(ReserveView v) {
    __shared__ int64_t waves[kThreads / 64];
    __shared__ int upto[kMost], start[kMost];
    const int tid = threadIdx.x, n = v.sequences;
    const int free_count = min(max(v.free_count[0], 0), v.pages);
    int length[kEach], change[kEach], held[kEach], needed[kEach], keep[kEach], need[kEach];
    int64_t surplus_sum = 0, need_sum = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int s = kEach * tid + i;
        length[i] = change[i] = held[i] = needed[i] = keep[i] = need[i] = 0;
        if (s >= n) continue;
        length[i] = min(max(v.lengths[s], 0), v.most);
        held[i] = min(max(v.held[s], 0), v.table_stride);
        change[i] = max(v.changes[s], -length[i]);
        if (int64_t(length[i]) + change[i] > v.most) change[i] = 0;
        const PageSlot end = page_slot(unsigned(length[i] + change[i]), v.page_size, v.magic);
        needed[i] = end.page + (end.slot > 0);
        const int fixed = v.shared ? min(max(v.shared[s], 0), held[i]) : 0;
        keep[i] = min(held[i], max(needed[i], fixed));
        need[i] = max(0, needed[i] - held[i]);
        surplus_sum += held[i] - keep[i];
        need_sum += need[i];
    }
    int64_t surplus_all, need_all, rows_all;
    int64_t surplus_before = scan_block(surplus_sum, waves, surplus_all);
    int64_t need_before = scan_block(need_sum, waves, need_all);
    const int available = int(min(int64_t(v.pages), free_count + surplus_all));

    if (surplus_all) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int s = kEach * tid + i;
            if (s >= n) continue;
            // A place k of the pages given back is entry start + k.
            start[s] = keep[i] - clipped(surplus_before);
            surplus_before += held[i] - keep[i];
            upto[s] = clipped(surplus_before);
        }
        __syncthreads();
        for (int k = tid; k < available - free_count; k += kThreads) {
            const int s = owner(upto, n, k);
            v.free_pages[free_count + k] = v.table[int64_t(s) * v.table_stride + start[s] + k];
        }
        __syncthreads();
    }

    // Rows of the sequences that have their pages.
    int64_t rows_sum = 0, upto_need = need_before;
    int rows[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        upto_need += need[i];
        rows[i] = need[i] == 0 || upto_need <= available ? max(change[i], 0) : 0;
        rows_sum += rows[i];
    }
    int64_t rows_before = scan_block(rows_sum, waves, rows_all);
    // How many pages are taken, and rows granted: the sums at the last sequence that gets any.
    int64_t pages_taken = 0, rows_granted = 0;
    upto_need = need_before;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int s = kEach * tid + i;
        upto_need += need[i];
        rows_before += rows[i];
        const bool granted = rows[i] > 0 && rows_before <= v.total_rows;
        if (granted) {
            rows_granted = rows_before;
            if (need[i]) pages_taken = upto_need;
        }
        const bool keeps = change[i] > 0 && !granted;  // its length, for want of pages or room
        if (s < n) {
            // A place k of the pages taken is entry start + k.
            start[s] = held[i] - clipped(upto_need - need[i]);
            upto[s] = clipped(upto_need);
            const int delta = keeps ? 0 : change[i];
            v.new_lengths[s] = length[i] + delta;
            if (v.new_seen) v.new_seen[s] = v.seen[s] + delta;
            v.new_held[s] = granted && need[i] ? needed[i] : keep[i];
        }
    }
    // The largest of all threads: they rise with the sequences.
    auto largest = [&](int64_t x) {
#pragma unroll
        for (int off = 1; off < 64; off *= 2) x = max(x, __shfl_xor(x, off));
        if ((tid & 63) == 0) waves[tid >> 6] = x;
        __syncthreads();
        int64_t all = 0;
        for (int w = 0; w < kThreads / 64; ++w) all = max(all, waves[w]);
        __syncthreads();
        return all;
    };
    const int taken = int(largest(pages_taken)), granted_rows = int(largest(rows_granted));
    if (tid == 0) {
        v.new_free_count[0] = available - taken;
        v.offsets[0] = 0;
    }
    for (int k = tid; k < taken; k += kThreads) {
        const int s = owner(upto, n, k);
        v.table[int64_t(s) * v.table_stride + start[s] + k] = v.free_pages[available - 1 - k];
    }
    __syncthreads();
    rows_before -= rows_sum;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int s = kEach * tid + i;
        rows_before += rows[i];
        if (s < n) v.offsets[s + 1] = int(min(rows_before, int64_t(granted_rows)));
    }
}

// The rows' maps, a thread a row: the sequence from the offsets, which every
// workgroup brings into LDS first.
constexpr int kMapThreads = 256, kMapRows = 4;
__global__ __launch_bounds__(kMapThreads) void reserve_rows_kernel(ReserveView v) {
    __shared__ int upto[kMost];
    const int n = v.sequences;
    for (int s = threadIdx.x; s < n; s += kMapThreads) upto[s] = v.offsets[s + 1];
    __syncthreads();
    const int all = upto[n - 1];
#pragma unroll
    for (int i = 0; i < kMapRows; ++i) {
        const int row = (blockIdx.x * kMapRows + i) * kMapThreads + threadIdx.x;
        if (row >= v.total_rows) return;
        int sequence = -1, position = -1;
        int64_t slot = -1;
        if (row < all) {
            sequence = owner(upto, n, row);
            const int back = upto[sequence] - row, length = v.new_lengths[sequence];
            position = (v.new_seen ? v.new_seen[sequence] : length) - back;
            const PageSlot at = page_slot(unsigned(length - back), v.page_size, v.magic);
            const int page = v.table[int64_t(sequence) * v.table_stride + at.page];
            if (page >= 0 && page < v.pages) slot = int64_t(page) * v.page_size + at.slot;
        }
        if (v.row_sequences) v.row_sequences[row] = sequence;
        if (v.row_positions) v.row_positions[row] = position;
        if (v.row_slots) v.row_slots[row] = slot;
    }
}

}  // namespace

void launch_paged_reserve(const qwen_gpu_paged_pool& p, const qwen_gpu_paged_growth& g, hipStream_t stream) {
    require(p.pages >= 1 && p.pages <= kMaxRow, "Pool pages must be in 1..2^30");
    require(p.page_size >= 1 && p.page_size <= 65536, "Page size must be in 1..65536");
    require(p.sequences >= 1 && p.sequences <= kMost, "Pool sequences must be in 1..4096");
    require(p.table_stride >= 1 && p.table_stride <= 1 << 24, "Pool table_stride must be in 1..2^24");
    require(g.total_rows >= 0 && g.total_rows <= 1 << 24, "Room for rows must be in 0..2^24");
    require(!g.seen == !g.new_seen, "seen and new_seen come together");
    const size_t n = size_t(p.sequences) * 4, room = size_t(g.total_rows) * 4;
    struct Array {
        const char* name;
        const void* at;
        size_t bytes;
        bool needed, written;
        const void* before;  // the array whose place it may take
        unsigned align = 4;
    };
    const Array arrays[] = {
        {"table", p.table, n * p.table_stride, true, true, nullptr},
        {"free_pages", p.free_pages, size_t(p.pages) * 4, true, true, nullptr},
        {"held", p.held, n, true, false, nullptr},
        {"free_count", p.free_count, 4, true, false, nullptr},
        {"shared", p.shared, n, false, false, nullptr},
        {"lengths", g.lengths, n, true, false, nullptr},
        {"seen", g.seen, n, false, false, nullptr},
        {"changes", g.changes, n, true, false, nullptr},
        {"new_lengths", g.new_lengths, n, true, true, g.lengths},
        {"new_seen", g.new_seen, n, false, true, g.seen},
        {"new_held", g.new_held, n, true, true, p.held},
        {"new_free_count", g.new_free_count, 4, true, true, p.free_count},
        {"offsets", g.offsets, n + 4, true, true, nullptr},
        {"row_sequences", g.row_sequences, room, false, true, nullptr},
        {"row_positions", g.row_positions, room, false, true, nullptr},
        {"row_slots", g.row_slots, 2 * room, false, true, nullptr, 8},
    };
    for (const Array& a : arrays) require(a.at || !a.needed, std::string("Null argument: ") + a.name);
    for (const Array& a : arrays)
        for (const Array& b : arrays)
            if (&a != &b && a.at && b.at && a.written && !(a.before == b.at && a.at == b.at))
                require((b.before == a.at && a.at == b.at) || apart(a.at, a.bytes, b.at, b.bytes),
                        std::string(a.name) + " overlaps " + b.name);
    const OpDevice device(p.table, "table", "the table", stream);
    for (const Array& a : arrays)
        if (a.at) device.check(a.at, a.name, a.align);
    ReserveView v{p.table,        p.free_pages,      p.held,         p.free_count,   p.shared,    g.lengths,
                  g.seen,         g.changes,         g.new_lengths,  g.new_seen,     g.new_held,  g.new_free_count,
                  g.offsets,      g.row_sequences,   g.row_positions, g.row_slots,   p.pages,     p.page_size,
                  p.sequences,    p.table_stride,    g.total_rows,   0,              0xffffffffu / unsigned(p.page_size)};
    const int64_t most = int64_t(p.table_stride) * p.page_size;
    v.most = int(most < kMaxRow ? most : kMaxRow);
    reserve_kernel<<<1, kThreads, 0, stream>>>(v);
    if (!g.total_rows || !(g.row_sequences || g.row_positions || g.row_slots)) return;
    constexpr int kOf = kMapThreads * kMapRows;
    reserve_rows_kernel<<<unsigned((g.total_rows + kOf - 1) / kOf), kMapThreads, 0, stream>>>(v);
}

}  // namespace qwen_hip

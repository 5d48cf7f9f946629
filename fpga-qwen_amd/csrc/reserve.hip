// Pages and rows of a step over a paged cache.
#include "reserve.hpp"

#include <algorithm>
#include <cstdint>
#include <iterator>

#include "decode_dev.hpp"
#include "op_device.hpp"
#include "paged_dev.hpp"
#include "qwen_common.hpp"

namespace qwen_hip {

namespace {

constexpr int kMost = 4096;  // sequences of a call
constexpr int kMaxRow = 1 << 30;
// Rows up to which they are mapped without a launch of their own: 64 sequences' 480 take 4.7 us, 5.7 with one, 960 of them
// 6.2 and 6.0.
constexpr int kFewRows = 768;

struct ReserveView {
    int32_t* table;
    int32_t* free_pages;
    const int32_t *held, *free_count, *shared, *lengths, *seen, *changes;
    int32_t *new_lengths, *new_seen, *new_held, *new_free_count, *offsets, *row_sequences, *row_positions;
    int64_t* row_slots;
    int pages, page_size, sequences, table_stride, total_rows, most;  // most positions of a sequence
    unsigned magic;
};

// Sums are 32 bits and stop at a limit above all pages and rows there can be,
// which two of them do not carry past 32 bits: nothing behind the place where a sum of pages passes
// those there are, or a sum of rows the room, is granted whatever the sum is.
constexpr unsigned kLimit = (1u << 30) + 1;
__device__ __forceinline__ unsigned limited(unsigned a, unsigned b) { return min(a + b, kLimit); }

// Sums of the lanes up to each, through DPP row shifts and broadcasts.
__device__ __forceinline__ unsigned scan_wave(unsigned x) {
    auto step = [&](int from) { x = limited(x, unsigned(from)); };
    step(__builtin_amdgcn_update_dpp(0, int(x), 0x111, 0xF, 0xF, true));  // row_shr:1, 2, 4, 8
    step(__builtin_amdgcn_update_dpp(0, int(x), 0x112, 0xF, 0xF, true));
    step(__builtin_amdgcn_update_dpp(0, int(x), 0x114, 0xF, 0xF, true));
    step(__builtin_amdgcn_update_dpp(0, int(x), 0x118, 0xF, 0xF, true));
    step(__builtin_amdgcn_update_dpp(0, int(x), 0x142, 0xA, 0xF, false));  // row_bcast:15 into rows 1 and 3
    step(__builtin_amdgcn_update_dpp(0, int(x), 0x143, 0xC, 0xF, false));  // row_bcast:31 into rows 2 and 3
    return x;
}

// N sums at once over the threads: `before` each thread, and `all`.
template <int THREADS, int N>
__device__ __forceinline__ void scan_block(const unsigned (&x)[N], unsigned (*waves)[16], unsigned (&before)[N],
                                           unsigned (&all)[N]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    unsigned upto[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        upto[i] = scan_wave(x[i]);
        if (lane == 63) waves[i][wave] = upto[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const unsigned of_lane = scan_wave(lane < THREADS / 64 ? waves[i][lane] : 0u);
        all[i] = __builtin_amdgcn_readlane(of_lane, 63);
        const int wave_before = __builtin_amdgcn_readfirstlane(max(wave - 1, 0));
        const unsigned base = wave ? __builtin_amdgcn_readlane(of_lane, wave_before) : 0u;
        // The sum up to the lane before, which the limit keeps from being a difference.
        const unsigned one_less = __shfl_up(upto[i], 1);
        before[i] = limited(base, lane ? one_less : 0u);
    }
    __syncthreads();
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

// Pages k below `count`, whose sequences' sums are `upto`: f(s, k) gives a
// place to read and one to write. Of many, a thread has four in a row, so it
// looks for the first one's sequence alone, and all its loads are in flight
// (1000 sequences with 21600 pages to move, maps and all, 21.3 us; two in a row
// 23.3, eight 25.9, four that lie 64 apart with a search each 30.2).
template <int THREADS, class F>
__device__ __forceinline__ void move_pages(const int* upto, int n, int count, F f) {
    if (count <= THREADS) {
        const int k = threadIdx.x;
        if (k >= count) return;
        const int32_t* from;
        int32_t* to;
        f(owner(upto, n, k), k, from, to);
        *to = *from;
        return;
    }
    constexpr int kRow = 4;
    for (int k0 = kRow * threadIdx.x; k0 < count; k0 += kRow * THREADS) {
        int s = owner(upto, n, k0), page[kRow];
        int32_t* to[kRow];
#pragma unroll
        for (int j = 0; j < kRow; ++j) {
            const int k = min(k0 + j, count - 1);
            while (upto[s] <= k) ++s;  // ends: the last sum is `count` or more
            const int32_t* from;
            f(s, k, from, to[j]);
            page[j] = *from;
        }
#pragma unroll
        for (int j = 0; j < kRow; ++j)
            if (k0 + j < count) *to[j] = page[j];
    }
}

// The maps of a row.
__device__ __forceinline__ void map_row(const ReserveView& v, const int* upto, int all, int row) {
    int sequence = -1, position = -1;
    int64_t slot = -1;
    if (row < all) {
        sequence = owner(upto, v.sequences, row);
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

// One workgroup: sums over the sequences (pages given back and needed, then
// rows granted), and after each the pages themselves, a thread each, whose
// sequences are found in the sums. Few rows are mapped here too. Latency
// bounds it: a thread has EACH sequences, one where there are few, and there
// are no more threads than they need. A step of 64 sequences takes 3.8 us (4.7
// with 1024 threads, 6.3 with four sequences a thread as well), of 1000 6.2
// (8.0 with four each); 1000 sequences with prompts of up to 1000 tokens among
// them, 12000 pages given back and 9600 taken, 17 us, and their 150000 rows' maps
// another 4.6.
template <int THREADS, int EACH>
__global__ __launch_bounds__(THREADS) void reserve_kernel(ReserveView v, bool maps) {
    __shared__ unsigned waves[2][16];
    __shared__ int upto[THREADS * EACH], start[THREADS * EACH];
    const int tid = threadIdx.x, n = v.sequences;
    const int free_count = min(max(v.free_count[0], 0), v.pages);
    int length[EACH], seen[EACH], change[EACH], held[EACH], needed[EACH], keep[EACH];
    unsigned need[EACH], surplus[EACH], sums[2] = {0, 0}, before[2], all[2];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {  // all loads first; sequences that are not there count as empty ones
        const int s = min(EACH * tid + i, n - 1);
        length[i] = v.lengths[s];
        seen[i] = v.seen ? v.seen[s] : 0;
        held[i] = v.held[s];
        change[i] = v.changes[s];
        keep[i] = v.shared ? v.shared[s] : 0;
    }
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const bool there = EACH * tid + i < n;
        length[i] = there ? min(max(length[i], 0), v.most) : 0;
        held[i] = there ? min(max(held[i], 0), v.table_stride) : 0;
        change[i] = there ? max(change[i], -length[i]) : 0;
        if (int64_t(length[i]) + change[i] > v.most) change[i] = 0;
        const PageSlot end = page_slot(unsigned(length[i] + change[i]), v.page_size, v.magic);
        needed[i] = end.page + (end.slot > 0);
        keep[i] = min(held[i], max(needed[i], keep[i]));
        need[i] = change[i] > 0 ? max(0, needed[i] - held[i]) : 0;
        surplus[i] = held[i] - keep[i];
        sums[0] = limited(sums[0], surplus[i]);
        sums[1] = limited(sums[1], need[i]);
    }
    scan_block<THREADS>(sums, waves, before, all);
    const int available = int(min(unsigned(v.pages), limited(free_count, all[0])));

    if (all[0]) {
        unsigned given = before[0];
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int s = EACH * tid + i;
            // A place k of the pages given back is entry start + k.
            start[s] = keep[i] - int(given);
            given = limited(given, surplus[i]);
            upto[s] = int(given);
        }
        __syncthreads();
        move_pages<THREADS>(upto, n, available - free_count, [&](int s, int k, const int32_t*& from, int32_t*& to) {
            from = v.table + (int64_t(s) * v.table_stride + start[s] + k);
            to = v.free_pages + (free_count + k);
        });
        __syncthreads();
    }

    // Rows of the sequences that have their pages.
    unsigned rows[EACH], pages = before[1], of_rows[1] = {0}, rows_before[1], rows_all[1];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        pages = limited(pages, need[i]);
        rows[i] = need[i] == 0 || pages <= unsigned(available) ? max(change[i], 0) : 0;
        of_rows[0] = limited(of_rows[0], rows[i]);
    }
    scan_block<THREADS>(of_rows, waves, rows_before, rows_all);
    // How many pages are taken, and rows granted: the sums at the last sequence that gets any.
    unsigned taken = 0, granted_rows = 0, row = rows_before[0];
    pages = before[1];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int s = EACH * tid + i;
        // A place k of the pages taken is entry start + k.
        start[s] = held[i] - int(pages);
        pages = limited(pages, need[i]);
        upto[s] = int(pages);
        row = limited(row, rows[i]);
        const bool granted = rows[i] > 0 && row <= unsigned(v.total_rows);
        if (granted) {
            granted_rows = row;
            if (need[i]) taken = pages;
        }
        if (s < n) {
            const int delta = change[i] > 0 && !granted ? 0 : change[i];
            v.new_lengths[s] = length[i] + delta;
            if (v.new_seen) v.new_seen[s] = seen[i] + delta;
            v.new_held[s] = granted && need[i] ? needed[i] : keep[i];
        }
    }
    // The largest of all threads.
    auto largest = [&](unsigned x) {
        x = max(x, unsigned(dev::xor_lanes<1>(int(x))));
        x = max(x, unsigned(dev::xor_lanes<2>(int(x))));
        x = max(x, unsigned(dev::xor_lanes<4>(int(x))));
        x = max(x, unsigned(dev::xor_lanes<8>(int(x))));
        x = max(x, unsigned(dev::xor_lanes<16>(int(x))));
        return max(x, unsigned(dev::xor_lanes<32>(int(x))));
    };
    taken = largest(taken), granted_rows = largest(granted_rows);
    if ((tid & 63) == 0) waves[0][tid >> 6] = taken, waves[1][tid >> 6] = granted_rows;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) taken = max(taken, waves[0][w]), granted_rows = max(granted_rows, waves[1][w]);
    if (tid == 0) {
        v.new_free_count[0] = available - int(taken);
        v.offsets[0] = 0;
    }
    row = rows_before[0];
    int offset[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        const int s = EACH * tid + i;
        row = limited(row, rows[i]);
        offset[i] = int(min(row, granted_rows));
        if (s < n) v.offsets[s + 1] = offset[i];
    }
    move_pages<THREADS>(upto, n, int(taken), [&](int s, int k, const int32_t*& from, int32_t*& to) {
        from = v.free_pages + (available - 1 - k);
        to = v.table + (int64_t(s) * v.table_stride + start[s] + k);
    });
    if (!maps) return;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < EACH; ++i) upto[EACH * tid + i] = offset[i];
    __syncthreads();
    for (int r = tid; r < v.total_rows; r += THREADS) map_row(v, upto, int(granted_rows), r);
}

// The maps of many rows, a thread a row; every workgroup brings the offsets into LDS first.
constexpr int kMapThreads = 256;
__global__ __launch_bounds__(kMapThreads) void reserve_rows_kernel(ReserveView v) {
    __shared__ int upto[kMost];
    for (int s = threadIdx.x; s < v.sequences; s += kMapThreads) upto[s] = v.offsets[s + 1];
    __syncthreads();
    const int all = upto[v.sequences - 1];
    for (int row = blockIdx.x * kMapThreads + threadIdx.x; row < v.total_rows; row += gridDim.x * kMapThreads)
        map_row(v, upto, all, row);
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
    const OpArray arrays[] = {
        {"table", p.table, n * p.table_stride, true, true},
        {"free_pages", p.free_pages, size_t(p.pages) * 4, true, true},
        {"held", p.held, n, true, false},
        {"free_count", p.free_count, 4, true, false},
        {"shared", p.shared, n, false, false},
        {"lengths", g.lengths, n, true, false},
        {"seen", g.seen, n, false, false},
        {"changes", g.changes, n, true, false},
        {"new_lengths", g.new_lengths, n, true, true, 4, g.lengths},
        {"new_seen", g.new_seen, n, false, true, 4, g.seen},
        {"new_held", g.new_held, n, true, true, 4, p.held},
        {"new_free_count", g.new_free_count, 4, true, true, 4, p.free_count},
        {"offsets", g.offsets, n + 4, true, true},
        {"row_sequences", g.row_sequences, room, false, true},
        {"row_positions", g.row_positions, room, false, true},
        {"row_slots", g.row_slots, 2 * room, false, true, 8},
    };
    check_arrays(arrays, std::size(arrays));
    const OpDevice device(p.table, "table", "the table", stream);
    for (const OpArray& a : arrays)
        if (a.at) device.check(a.at, a.name, a.alignment);
    ReserveView v{p.table,        p.free_pages,      p.held,         p.free_count,   p.shared,    g.lengths,
                  g.seen,         g.changes,         g.new_lengths,  g.new_seen,     g.new_held,  g.new_free_count,
                  g.offsets,      g.row_sequences,   g.row_positions, g.row_slots,   p.pages,     p.page_size,
                  p.sequences,    p.table_stride,    g.total_rows,   0,              0xffffffffu / unsigned(p.page_size)};
    const int64_t most = int64_t(p.table_stride) * p.page_size;
    v.most = int(most < kMaxRow ? most : kMaxRow);
    const bool maps = g.total_rows && (g.row_sequences || g.row_positions || g.row_slots);
    const bool few = g.total_rows <= kFewRows;
    if (p.sequences <= 256)
        reserve_kernel<256, 1><<<1, 256, 0, stream>>>(v, maps && few);
    else if (p.sequences <= 1024)
        reserve_kernel<1024, 1><<<1, 1024, 0, stream>>>(v, maps && few);
    else
        reserve_kernel<1024, 4><<<1, 1024, 0, stream>>>(v, maps && few);
    if (!maps || few) return;
    const int grid = std::min((g.total_rows + kMapThreads - 1) / kMapThreads, 2048);
    reserve_rows_kernel<<<unsigned(grid), kMapThreads, 0, stream>>>(v);
}

}  // namespace qwen_hip

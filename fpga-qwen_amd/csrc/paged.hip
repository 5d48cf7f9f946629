// Paged key-value cache: argument checks, append, eviction.
#include "paged.hpp"

#include <algorithm>
#include <string>

#include "decode_dev.hpp"
#include "paged_dev.hpp"
#include "qwen_common.hpp"

namespace qwen_hip {

namespace {
constexpr int kEvictHead = 4;  // ints of a unit's moves before its lists

void hip_check(hipError_t e) {
    if (e != hipSuccess) throw std::runtime_error(std::string("HIP error: ") + hipGetErrorString(e));
}
void need(const void* p, const char* what) {
    if (!p) throw std::runtime_error(std::string("Null argument: ") + what);
}
}  // namespace

// ---- arguments ----

PagedView paged_view(const qwen_gpu_paged_cache& c, const qwen_gpu_paged_batch& b) {
    need(c.keys, "keys");
    need(c.values, "values");
    need(b.table, "table");
    need(b.lengths, "lengths");
    require(c.type == kPagedF16 || c.type == kPagedBF16 || c.type == kPagedE4M3, "Unknown paged cache type");
    if (c.type == kPagedE4M3) need(c.exponents, "exponents");
    require(c.head_dim == 64 || c.head_dim == 128 || c.head_dim == 256, "Paged head_dim must be 64, 128 or 256");
    require(c.page_size >= 1 && c.page_size <= 65536, "Page size must be in 1..65536");
    require(c.pages >= 1, "A paged cache needs pages");
    require(c.kv_heads >= 1 && c.kv_heads <= 1024, "Paged kv_heads must be in 1..1024");
    const int size = c.type == kPagedE4M3 ? 1 : 2;
    // Rows may lie in any order of the three axes, but apart from each other.
    struct Axis {
        int64_t stride, count;
    } axes[3] = {{c.page_stride, c.pages}, {c.head_stride, c.kv_heads}, {c.slot_stride, c.page_size}};
    std::sort(axes, axes + 3, [](const Axis& x, const Axis& y) { return x.stride < y.stride; });
    int64_t span = c.head_dim;
    for (const Axis& a : axes) {
        if (a.count == 1) continue;  // its stride is never taken
        require(a.stride >= span && a.stride <= (int64_t(1) << 40), "Paged strides let rows overlap or run too far");
        require(a.stride * size % 16 == 0, "Paged strides must be multiples of 16 bytes");
        require(a.count - 1 <= ((int64_t(1) << 44) - span) / a.stride, "Paged strides let rows overlap or run too far");
        span += a.stride * (a.count - 1);
    }
    require(b.sequences >= 1 && b.sequences <= 4096, "Paged sequences must be in 1..4096");
    require(b.sequences * c.kv_heads < 1 << 21, "Too many sequences for that many KV heads");
    require(b.table_stride >= 1, "A paged table needs entries");
    require(b.max_length >= 1 && b.max_length <= kPagedMaxLength &&
                b.max_length <= int64_t(b.table_stride) * c.page_size,
            "Paged max_length must be in 1..table_stride * page_size, at most 2^24");
    require(!(b.weights || b.positions) || b.track_stride >= b.max_length, "track_stride is below max_length");
    require(b.track_stride <= (int64_t(1) << 32), "track_stride is too large");
    PagedView v{};
    v.keys = static_cast<char*>(c.keys);
    v.values = static_cast<char*>(c.values);
    v.exponents = c.exponents;
    // The stride of an axis of one is never taken, whatever it holds.
    v.page_stride = c.pages > 1 ? c.page_stride * size : 0;
    v.head_stride = c.kv_heads > 1 ? c.head_stride * size : 0;
    v.slot_stride = c.page_size > 1 ? c.slot_stride * size : 0;
    v.table = b.table;
    v.lengths = b.lengths;
    v.offsets = b.offsets;
    v.seen = b.seen;
    v.weights = b.weights;
    v.positions = b.positions;
    v.track_stride = b.track_stride;
    v.pages = c.pages;
    v.page_size = c.page_size;
    v.kv_heads = c.kv_heads;
    v.magic = 0xffffffffu / unsigned(c.page_size);
    v.sequences = b.sequences;
    v.table_stride = b.table_stride;
    v.max_length = b.max_length;
    v.rows = b.rows;
    v.total_rows = b.total_rows;
    return v;
}

void paged_check_rows(const qwen_gpu_paged_batch& b) {
    require(b.rows >= 1 && b.rows <= kPagedMaxLength, "Paged rows must be in 1..2^24");
    require(b.total_rows >= 0 && b.total_rows <= kPagedMaxLength, "Paged total_rows must be in 0..2^24");
    require(b.offsets || int64_t(b.sequences) * b.rows == b.total_rows,
            "Paged total_rows must be sequences * rows without offsets");
}

PagedDevice::PagedDevice(const qwen_gpu_paged_cache& c, const qwen_gpu_paged_batch& b, hipStream_t stream) {
    // The runtime's handles 1 and 2 stand for streams and point to none: asked for the device of 1, it ends the
    // process.
    require(stream != hipStreamLegacy && stream != hipStreamPerThread,
            "The stream must be NULL or a stream that was created");
    hipPointerAttribute_t a{};
    if (hipPointerGetAttributes(&a, c.keys) != hipSuccess || a.type == hipMemoryTypeUnregistered) {
        (void)hipGetLastError();
        throw std::runtime_error("Not device memory: keys");
    }
    device_ = a.device;
    check(c.keys, "keys", 16);
    check(c.values, "values", 16);
    if (c.type == kPagedE4M3) check(c.exponents, "exponents", 2);
    check(b.table, "table");
    check(b.lengths, "lengths");
    if (b.offsets) check(b.offsets, "offsets");
    if (b.seen) check(b.seen, "seen");
    if (b.weights) check(b.weights, "weights");
    if (b.positions) check(b.positions, "positions");
    hip_check(hipGetDevice(&before_));
    if (stream) {
        hipDevice_t of = 0;
        hip_check(hipStreamGetDevice(stream, &of));
        require(of == device_, "The stream belongs to another device than the cache");
    }
    if (before_ != device_) hip_check(hipSetDevice(device_));
}

PagedDevice::~PagedDevice() {
    if (before_ != device_) (void)hipSetDevice(before_);
}

void PagedDevice::check(const void* p, const char* what, unsigned alignment) const {
    need(p, what);
    require(reinterpret_cast<uintptr_t>(p) % alignment == 0,
            std::string("Not aligned to ") + std::to_string(alignment) + " bytes: " + what);
    hipPointerAttribute_t a{};
    if (hipPointerGetAttributes(&a, p) != hipSuccess || a.type == hipMemoryTypeUnregistered) {
        (void)hipGetLastError();
        throw std::runtime_error(std::string("Not device memory: ") + what);
    }
    require(a.type != hipMemoryTypeDevice || a.device == device_,
            std::string("On another device than the cache: ") + what);
}

size_t paged_moves_bytes(const qwen_gpu_paged_cache& c, const qwen_gpu_paged_batch& b, int64_t room) {
    return size_t(b.sequences) * c.kv_heads * (2 * room + kEvictHead) * sizeof(int32_t);
}

// ---- append ----

namespace {

// Sequence of a new row, -1 where it has none: the number of offsets up to
// `row`, less one. The lanes of a wave probe 64 of them at a time.
__device__ int sequence_of(const PagedView& v, int row, int lane) {
    if (!v.offsets) return row / v.rows;
    int low = 0, high = v.sequences + 1;  // the number lies in low .. high
    while (high > low) {
        const int step = (high - low + 63) / 64;
        const int at = low + lane * step;
        const unsigned long long upto = __ballot(at < high && v.offsets[min(at, v.sequences)] <= row);
        const int n = __popcll(upto);  // offsets rise, so these are the first lanes
        if (n == 0) {
            high = low;
        } else {
            const int last = low + (n - 1) * step;  // offsets[last] <= row
            high = min(high, last + step);
            low = last + 1;
        }
    }
    return low - 1 < v.sequences ? low - 1 : -1;
}

// The smallest exponent byte whose power of two brings `top` to 448 = 1.75 * 2^8
// or below, and what the row's values are multiplied by. A power of two keeps
// every rounding where it would be without it, and both sides exact.
__device__ __forceinline__ int e4m3_byte(float top) {
    const unsigned bits = __builtin_bit_cast(unsigned, top);
    const int byte = int(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u);
    return min(max(byte, 1), 254);
}

// One wave writes 512 elements of a new row's keys and the same of its
// values: lane l the elements 8 l .. 8 l + 7 of both, so a lane's four loads
// of 16 bytes are all in flight at once, and the row's sequence and slot are
// found meanwhile. Memory bounds it: 82,600 rows of 8 heads of 128 (BF16, 1.02
// GB) take 201 us, 5.1 TB/s, the rate of a copy; 24 ragged prompts (E4M3, 208
// MB) 50 us, 4.2 TB/s. A row alone takes a launch (2.5 us).
template <int TYPE, int DIM>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedView v, const float* keys, int64_t key_stride,
                                                           const float* values, int64_t value_stride, int parts) {
    const int lane = threadIdx.x & 63, item = blockIdx.x * 4 + (threadIdx.x >> 6);
    const int row = item / parts, part = item - row * parts;
    if (row >= v.total_rows) return;
    const int at = part * 512 + lane * 8, head = at / DIM;
    const bool live = head < v.kv_heads;
    float x[2][8];
    if (live) {
        const float* from[2] = {keys + row * key_stride + at, values + row * value_stride + at};
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            const float4_a4 a = *reinterpret_cast<const float4_a4*>(from[side]);
            const float4_a4 b = *reinterpret_cast<const float4_a4*>(from[side] + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) x[side][i] = a[i], x[side][4 + i] = b[i];
        }
    }
    const int s = sequence_of(v, row, lane);
    if (s < 0) return;
    int first;
    const int n = v.new_rows(s, first), rank = row - first;
    const int j = v.length(s) - n + rank;
    if (rank < 0 || rank >= n || j < 0 || !live) return;
    const PageSlot where = page_slot(j, v.page_size, v.magic);
    const int page = v.page_of(s, where.page);
    const bool leader = at % DIM == 0;
    if (leader) {
        if (v.weights) v.weights[v.track_at(s, head) + j] = 0.f;
        if (v.positions) v.positions[v.track_at(s, head) + j] = (v.seen ? v.seen[s] : v.length(s)) - n + rank;
    }
    if (page < 0) return;
    const int64_t to = v.row_at(page, head, where.slot) + (at % DIM) * (TYPE == kPagedE4M3 ? 1 : 2);
    char* const pools[2] = {v.keys, v.values};
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        float* const e = x[side];
        if constexpr (TYPE == kPagedF16) {
            *reinterpret_cast<uint4_t*>(pools[side] + to) = uint4_t{pack_half(e[0], e[1]), pack_half(e[2], e[3]),
                                                                    pack_half(e[4], e[5]), pack_half(e[6], e[7])};
        } else if constexpr (TYPE == kPagedBF16) {
            *reinterpret_cast<uint4_t*>(pools[side] + to) = uint4_t{pack_bf16(e[0], e[1]), pack_bf16(e[2], e[3]),
                                                                    pack_bf16(e[4], e[5]), pack_bf16(e[6], e[7])};
        } else {
            float top = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float a = __builtin_fabsf(e[i]);
                if (a < __builtin_huge_valf()) top = fmaxf(top, a);  // neither infinite nor NaN
            }
#pragma unroll
            for (int off = 1; off < DIM / 8; off *= 2) top = fmaxf(top, __shfl_xor(top, off));
            const int byte = e4m3_byte(top);
            const float down = byte_pow2(254 - byte);
            unsigned words[2];
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                int packed = 0;
                packed = __builtin_amdgcn_cvt_pk_fp8_f32(e[4 * w] * down, e[4 * w + 1] * down, packed, false);
                packed = __builtin_amdgcn_cvt_pk_fp8_f32(e[4 * w + 2] * down, e[4 * w + 3] * down, packed, true);
                words[w] = unsigned(packed);
            }
            *reinterpret_cast<u32x2*>(pools[side] + to) = u32x2{words[0], words[1]};
            if (leader) v.exponents[v.exponents_at(page, head, where.slot) + side] = uint8_t(byte);
        }
    }
}

template <int TYPE>
void append_of(int dim, const PagedView& v, const float* keys, int64_t key_stride, const float* values,
               int64_t value_stride, hipStream_t stream) {
    const int parts = (v.kv_heads * dim + 511) / 512;
    const dim3 grid(unsigned((int64_t(v.total_rows) * parts + 3) / 4));
    if (dim == 64)
        paged_append_kernel<TYPE, 64><<<grid, 256, 0, stream>>>(v, keys, key_stride, values, value_stride, parts);
    else if (dim == 128)
        paged_append_kernel<TYPE, 128><<<grid, 256, 0, stream>>>(v, keys, key_stride, values, value_stride, parts);
    else
        paged_append_kernel<TYPE, 256><<<grid, 256, 0, stream>>>(v, keys, key_stride, values, value_stride, parts);
}

}  // namespace

void launch_paged_append(const qwen_gpu_paged_cache& cache, const qwen_gpu_paged_batch& batch, const float* keys,
                         int64_t key_stride, const float* values, int64_t value_stride, hipStream_t stream) {
    const PagedView v = paged_view(cache, batch);
    paged_check_rows(batch);
    need(keys, "new keys");
    need(values, "new values");
    const int64_t row = int64_t(cache.kv_heads) * cache.head_dim;
    require(key_stride >= row && value_stride >= row, "Paged rows overlap: stride below kv_heads * head_dim");
    require(key_stride <= (int64_t(1) << 32) && value_stride <= (int64_t(1) << 32), "Paged row stride is too large");
    require(int64_t(batch.total_rows) * ((row + 511) / 512) < (int64_t(1) << 26), "Too many new rows for one call");
    const PagedDevice device(cache, batch, stream);
    device.check(keys, "new keys");
    device.check(values, "new values");
    if (!batch.total_rows) return;
    if (cache.type == kPagedF16)
        append_of<kPagedF16>(cache.head_dim, v, keys, key_stride, values, value_stride, stream);
    else if (cache.type == kPagedBF16)
        append_of<kPagedBF16>(cache.head_dim, v, keys, key_stride, values, value_stride, stream);
    else
        append_of<kPagedE4M3>(cache.head_dim, v, keys, key_stride, values, value_stride, stream);
}

// ---- eviction ----

namespace {

constexpr int kEvictThreads = 1024, kEvictWaves = kEvictThreads / 64, kEvictBins = 2048;
constexpr unsigned kEvictFixed = 0xffffffffu;
constexpr int kEvictFew = 4, kEvictHeld = 8, kMoveRows = 64;

// Weights as whole numbers of the same order; NaN is the lowest, -0 is 0.
__device__ __forceinline__ unsigned weight_key(float w) {
    if (w != w) return 0u;
    const unsigned bits = __builtin_bit_cast(unsigned, w + 0.f);
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

// The lanes' lowest value, in every lane.
__device__ __forceinline__ uint64_t lowest_of_wave(uint64_t x) {
    auto with = [&](double other) { x = min(x, __builtin_bit_cast(uint64_t, other)); };
    with(dev::xor_lanes<32>(__builtin_bit_cast(double, x)));
    with(dev::xor_lanes<16>(__builtin_bit_cast(double, x)));
    with(dev::xor_lanes<8>(__builtin_bit_cast(double, x)));
    with(dev::xor_lanes<4>(__builtin_bit_cast(double, x)));
    with(dev::xor_lanes<2>(__builtin_bit_cast(double, x)));
    with(dev::xor_lanes<1>(__builtin_bit_cast(double, x)));
    return x;
}

struct EvictArgs {
    int keep, sinks, recent;
    int32_t* new_lengths;
    float* new_weights;
    int32_t* new_positions;
    int32_t* moves;  // workspace, a unit: their number, padding, holes[room], sources[room] from the last
    int64_t room;
    int size;        // bytes of a row
    bool scaled;     // rows have exponents
};

// Moves one 16-byte piece of a row (keys, then values, of 2 * size bytes), and
// with the first piece the row's exponents.
__device__ __forceinline__ void move_piece(const PagedView& v, const EvictArgs& a, int s, int head, int from, int to,
                                           int piece) {
    const int half = a.size / 16;
    const PageSlot to_at = page_slot(to, v.page_size, v.magic), from_at = page_slot(from, v.page_size, v.magic);
    const int to_page = v.page_of(s, to_at.page), from_page = v.page_of(s, from_at.page);
    if (to_page < 0 || from_page < 0) return;
    char* const pool = piece < half ? v.keys : v.values;
    const int64_t at = 16 * (piece < half ? piece : piece - half);
    *reinterpret_cast<uint4_t*>(pool + v.row_at(to_page, head, to_at.slot) + at) =
        *reinterpret_cast<const uint4_t*>(pool + v.row_at(from_page, head, from_at.slot) + at);
    if (piece == 0 && a.scaled)
        *reinterpret_cast<uint16_t*>(v.exponents + v.exponents_at(to_page, head, to_at.slot)) =
            *reinterpret_cast<const uint16_t*>(v.exponents + v.exponents_at(from_page, head, from_at.slot));
}

// One workgroup per sequence and KV head chooses what stays, and moves it where
// `MOVE` (few rows at most); else the next kernel does.
//
// A few rows too many (kEvictFew; every step of a cache of fixed length): the
// lowest weight, of equal ones the last slot, is found that many times. More:
// the threshold weight (the keep-th largest) is found digit by digit, 11 + 11
// + 10 bits from the top: a histogram of the digit among the slots that share
// the digits so far, and the digit at which the count from above reaches what
// is still wanted. Of the slots at the threshold the first ones are kept. A
// hole's rank among holes is its slot less the kept slots before it, and a
// kept slot's rank needs the same count, so one running count gives both
// lists. Up to kEvictHeld slots a thread's keys stay in registers. Latency
// bounds it: 1025 slots of 64 heads take 5.5 us with one row too many (10.4
// digit by digit), 4001 slots of 8 heads 9.3, up to 8192 of 256 13.3 (a barrier
// for each 1024 slots, and weights moved here, took 22).
template <bool MOVE>
__global__ __launch_bounds__(kEvictThreads) void paged_evict_kernel(PagedView v, EvictArgs a) {
    __shared__ int bins[kEvictBins];
    __shared__ int2 wave_counts[kEvictHeld][kEvictWaves];
    __shared__ uint64_t lowest[2][kEvictWaves];
    __shared__ int found[2];
    __shared__ int few_holes[kEvictFew], few_sources[kEvictFew];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int s = blockIdx.x / v.kv_heads, head = blockIdx.x - s * v.kv_heads;
    const int n = v.length(s), keep = a.keep;
    const int64_t track = v.track_at(s, head);
    const float* weights = v.weights + track;
    const int32_t* positions = v.positions + track;
    float* new_weights = a.new_weights + track;
    int32_t* new_positions = a.new_positions + track;
    const bool copies = new_weights != weights || new_positions != positions;
    int32_t* const moves = a.moves + int64_t(blockIdx.x) * (2 * a.room + kEvictHead);
    if (head == 0 && tid == 0) a.new_lengths[s] = min(n, keep);
    if (!MOVE && tid == 0 && n <= keep) moves[0] = 0;
    if (n <= keep) {
        for (int j = tid; copies && j < n; j += kEvictThreads) {
            new_weights[j] = weights[j];
            new_positions[j] = positions[j];
        }
        return;
    }
    const int64_t late = int64_t(v.seen ? v.seen[s] : n) - a.recent;
    auto key_of = [&](int j) {
        const int p = positions[j];
        const float w = weights[j];
        return p < a.sinks || p >= late ? kEvictFixed : weight_key(w);
    };
    unsigned held[kEvictHeld];
    const bool holds = n <= kEvictHeld * kEvictThreads;
    if (holds) {
        float w[kEvictHeld];
        int p[kEvictHeld];
#pragma unroll
        for (int i = 0; i < kEvictHeld; ++i) {
            const int j = min(i * kEvictThreads + tid, n - 1);
            w[i] = weights[j];
            p[i] = positions[j];
        }
#pragma unroll
        for (int i = 0; i < kEvictHeld; ++i) {
            const int j = i * kEvictThreads + tid;
            held[i] = p[i] < a.sinks || p[i] >= late ? kEvictFixed : weight_key(w[i]);
            if (copies && j < keep) {
                new_weights[j] = w[i];
                new_positions[j] = p[i];
            }
        }
    } else if (copies) {
        for (int j = tid; j < keep; j += kEvictThreads) {
            new_weights[j] = weights[j];
            new_positions[j] = positions[j];
        }
    }
    // f(slot, key) for all slots, this thread's among each 1024 in turn.
    auto each = [&](auto f) {
        if (holds) {
#pragma unroll
            for (int i = 0; i < kEvictHeld; ++i)
                if (i * kEvictThreads + tid < n) f(i * kEvictThreads + tid, held[i]);
        } else {
            for (int j = tid; j < n; j += kEvictThreads) f(j, key_of(j));
        }
    };
    int32_t *holes = moves + kEvictHead, *sources = holes + a.room;
    int moved;

    if (n - keep <= kEvictFew && holds) {
        holes = few_holes;
        sources = few_sources;
        int gone[kEvictFew];
#pragma unroll
        for (int e = 0; e < kEvictFew; ++e) {
            gone[e] = -1;
            if (e >= n - keep) continue;
            uint64_t low = ~0ull;
            each([&](int j, unsigned key) {
                bool out = false;
#pragma unroll
                for (int f = 0; f < e; ++f) out |= gone[f] == j;
                const uint64_t x = uint64_t(key) << 32 | unsigned(~j);
                if (!out && x < low) low = x;
            });
            low = lowest_of_wave(low);
            if (lane == 0) lowest[e & 1][wave] = low;
            __syncthreads();
            low = lowest_of_wave(lowest[e & 1][lane % kEvictWaves]);
            gone[e] = ~int(unsigned(low));
        }
        // The evicted slots before `keep` are the holes, the others' complement the sources, both in order.
        moved = 0;
        int behind = 0;
#pragma unroll
        for (int e = 0; e < kEvictFew; ++e) {
            if (e >= n - keep) continue;
            bool out = false;  // of slot keep + e
            int rank = 0;      // holes before gone[e]
#pragma unroll
            for (int f = 0; f < kEvictFew; ++f) {
                out |= gone[f] == keep + e;
                rank += gone[f] >= 0 && gone[f] < gone[e];
            }
            if (gone[e] < keep) {
                if (tid == 0) holes[rank] = gone[e];
                ++moved;
            }
            if (!out) {
                if (tid == 0) sources[behind] = keep + e;
                ++behind;
            }
        }
        __syncthreads();
    } else {
        unsigned prefix = 0, known = 0;  // the threshold's digits so far, and which bits they are
        int wanted = keep;               // slots still to be taken among those that share them
        for (int digit = 0; digit < 3; ++digit) {
            const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0, width = digit == 2 ? 1024 : 2048;
            bins[tid] = bins[tid + kEvictThreads] = 0;
            __syncthreads();
            each([&](int, unsigned key) {
                if ((key & known) == prefix) atomicAdd(&bins[(key >> shift) & (width - 1)], 1);
            });
            __syncthreads();
            // Thread t holds the t-th pair of bins from the top; counts from above.
            const int2 pair = reinterpret_cast<const int2*>(bins)[kEvictThreads - 1 - tid];
            const int upper = pair.y, lower = pair.x, sum = scan_lanes(upper + lower);
            if (lane == 63) wave_counts[0][wave].x = sum;
            __syncthreads();
            const int of_wave = lane < kEvictWaves && lane < wave ? wave_counts[0][lane].x : 0;
            const int above = sum - upper - lower + __builtin_amdgcn_readlane(scan_lanes(of_wave), 63);
            if (above < wanted && above + upper + lower >= wanted) {
                const bool second = above + upper < wanted;
                found[0] = kEvictBins - 1 - 2 * tid - second;
                found[1] = wanted - above - (second ? upper : 0);
            }
            __syncthreads();
            prefix |= unsigned(found[0]) << shift;
            known |= unsigned(width - 1) << shift;
            wanted = found[1];
        }
        // Slot j, with the slots before it above and at the threshold.
        auto place = [&](int j, unsigned key, int above_rank, int at_rank) {
            const bool kept = key > prefix || (key == prefix && at_rank < wanted);
            const int rank = above_rank + min(at_rank, wanted);  // kept slots before this one
            if (j == keep) found[0] = keep - rank;               // the rest of them have to move
            if (j >= keep) {
                if (kept && keep - 1 - rank < a.room) sources[keep - 1 - rank] = j;  // from the last
            } else if (!kept) {
                if (j - rank < a.room) holes[j - rank] = j;
            }
        };
        const unsigned long long before = (1ull << lane) - 1;
        __syncthreads();
        if (holds) {
            // The counts of every wave's part of every 1024 slots, then their running sums.
#pragma unroll
            for (int i = 0; i < kEvictHeld; ++i) {
                const bool in = i * kEvictThreads + tid < n;
                const int above = __popcll(__ballot(in && held[i] > prefix));
                const int at = __popcll(__ballot(in && held[i] == prefix));
                if (lane == 0) wave_counts[i][wave] = int2{above, at};
            }
            __syncthreads();
            static_assert(kEvictHeld * kEvictWaves == 128, "two counts for each lane");
            const int2 c0 = wave_counts[0][2 * lane], c1 = wave_counts[0][2 * lane + 1];
            const int above_upto = scan_lanes(c0.x + c1.x), at_upto = scan_lanes(c0.y + c1.y);
#pragma unroll
            for (int i = 0; i < kEvictHeld; ++i) {
                const int of = (i * kEvictWaves + wave) / 2;
                int above_rank = __builtin_amdgcn_readlane(above_upto - c1.x - (wave & 1 ? 0 : c0.x), of);
                int at_rank = __builtin_amdgcn_readlane(at_upto - c1.y - (wave & 1 ? 0 : c0.y), of);
                const bool in = i * kEvictThreads + tid < n;
                above_rank += __popcll(__ballot(in && held[i] > prefix) & before);
                at_rank += __popcll(__ballot(in && held[i] == prefix) & before);
                if (in) place(i * kEvictThreads + tid, held[i], above_rank, at_rank);
            }
        } else {
            int above_before = 0, at_before = 0, turn = 0;
            for (int begin = 0; begin < n; begin += kEvictThreads, turn ^= 1) {
                const int j = begin + tid;
                const unsigned key = j < n ? key_of(j) : 0u;
                const unsigned long long above = __ballot(j < n && key > prefix), at = __ballot(j < n && key == prefix);
                if (lane == 0) wave_counts[turn][wave] = int2{__popcll(above), __popcll(at)};
                __syncthreads();
                const int2 c = lane < kEvictWaves ? wave_counts[turn][lane] : int2{0, 0};
                const int above_upto = scan_lanes(c.x), at_upto = scan_lanes(c.y);
                const int above_rank = above_before + (wave ? __builtin_amdgcn_readlane(above_upto, wave - 1) : 0);
                const int at_rank = at_before + (wave ? __builtin_amdgcn_readlane(at_upto, wave - 1) : 0);
                if (j < n) place(j, key, above_rank + __popcll(above & before), at_rank + __popcll(at & before));
                above_before += __builtin_amdgcn_readlane(above_upto, 63);
                at_before += __builtin_amdgcn_readlane(at_upto, 63);
            }
        }
        __syncthreads();
        moved = int(min(int64_t(found[0]), a.room));
        sources += moved - 1;
    }
    if constexpr (MOVE) {
        const int order = sources == few_sources ? 1 : -1;  // the long list begins with the last source
        for (int i = tid; i < moved; i += kEvictThreads) {
            const int to = holes[i], from = sources[order * i];
            new_weights[to] = weights[from];
            new_positions[to] = positions[from];
        }
        const int pieces = a.size / 8;
        for (int i = tid; i < moved * pieces; i += kEvictThreads) {
            const int m = i / pieces;
            move_piece(v, a, s, head, sources[order * m], holes[m], i - m * pieces);
        }
    } else {
        if (tid == 0) moves[0] = moved;
        if (sources == few_sources && tid < moved) {
            moves[kEvictHead + tid] = few_holes[tid];
            moves[kEvictHead + a.room + moved - 1 - tid] = few_sources[tid];
        }
    }
}

// The moves that the choice left, 64 rows a workgroup's turn: a lane of the
// first wave finds where one row goes from and to, and moves its weight,
// position and exponents; then all threads move the rows' pieces, four loads in
// flight each. Memory bounds it: 70 MB read and 66 written in rows of 128 bytes
// take 31 us, 4.3 TB/s (every thread finding its own rows 41).
__global__ __launch_bounds__(256) void paged_move_kernel(PagedView v, EvictArgs a) {
    __shared__ int64_t from_at[kMoveRows], to_at[kMoveRows];
    const int tid = threadIdx.x, s = blockIdx.x / v.kv_heads, head = blockIdx.x - s * v.kv_heads;
    const int32_t* const moves = a.moves + int64_t(blockIdx.x) * (2 * a.room + kEvictHead);
    const int64_t track = v.track_at(s, head);
    const int moved = moves[0];
    const int32_t *const holes = moves + kEvictHead, *const sources = holes + a.room + moved - 1;
    const int pieces = a.size / 8, shift = 31 - __builtin_clz(unsigned(pieces)), half = pieces / 2;  // powers of two
    const int piece = tid & (pieces - 1), together = 256 >> shift;
    char* const pool = (piece < half ? v.keys : v.values) + 16 * (piece & (half - 1));
    for (int m0 = blockIdx.y * kMoveRows; m0 < moved; m0 += int(gridDim.y) * kMoveRows) {
        const int rows = min(kMoveRows, moved - m0);
        if (tid < rows) {
            const int hole = holes[m0 + tid], source = sources[-m0 - tid];
            const PageSlot to = page_slot(hole, v.page_size, v.magic);
            const PageSlot from = page_slot(source, v.page_size, v.magic);
            const int to_page = v.page_of(s, to.page), from_page = v.page_of(s, from.page);
            const bool both = to_page >= 0 && from_page >= 0;
            from_at[tid] = both ? v.row_at(from_page, head, from.slot) : -1;
            to_at[tid] = v.row_at(to_page, head, to.slot);
            a.new_weights[track + hole] = v.weights[track + source];
            a.new_positions[track + hole] = v.positions[track + source];
            if (a.scaled && both)
                *reinterpret_cast<uint16_t*>(v.exponents + v.exponents_at(to_page, head, to.slot)) =
                    *reinterpret_cast<const uint16_t*>(v.exponents + v.exponents_at(from_page, head, from.slot));
        }
        __syncthreads();
        for (int r0 = tid >> shift; r0 < rows; r0 += 4 * together) {
            int64_t from[4], to[4];
            uint4_t data[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = min(r0 + i * together, rows - 1);
                from[i] = from_at[r];
                to[i] = to_at[r];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) data[i] = *reinterpret_cast<const uint4_t*>(pool + max(from[i], int64_t(0)));
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (from[i] >= 0 && r0 + i * together < rows) *reinterpret_cast<uint4_t*>(pool + to[i]) = data[i];
        }
        __syncthreads();
    }
}

bool apart(const void* p, const void* q, size_t bytes) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(p), y = reinterpret_cast<uintptr_t>(q);
    return x < y ? y - x >= bytes : x - y >= bytes;
}

}  // namespace

void launch_paged_evict(const qwen_gpu_paged_cache& cache, const qwen_gpu_paged_batch& batch, int keep, int sinks,
                        int recent, int32_t* new_lengths, float* new_weights, int32_t* new_positions, void* workspace,
                        size_t workspace_bytes, hipStream_t stream) {
    const PagedView v = paged_view(cache, batch);
    need(batch.weights, "weights");
    need(batch.positions, "positions");
    need(new_lengths, "new_lengths");
    need(new_weights, "new_weights");
    need(new_positions, "new_positions");
    require(keep >= 1, "keep must be at least 1");
    require(sinks >= 0 && recent >= 0 && int64_t(sinks) + recent <= keep,
            "Need 0 <= sinks, 0 <= recent and sinks + recent <= keep");
    const size_t tracked = size_t(batch.sequences) * cache.kv_heads * batch.track_stride * 4;
    require(apart(new_lengths, batch.lengths, size_t(batch.sequences) * 4), "new_lengths overlaps lengths");
    require(!batch.seen || apart(new_lengths, batch.seen, size_t(batch.sequences) * 4), "new_lengths overlaps seen");
    require(new_weights == batch.weights || apart(new_weights, batch.weights, tracked), "new_weights overlaps weights");
    require(new_positions == batch.positions || apart(new_positions, batch.positions, tracked),
            "new_positions overlaps positions");
    const PagedDevice device(cache, batch, stream);
    device.check(new_lengths, "new_lengths");
    device.check(new_weights, "new_weights");
    device.check(new_positions, "new_positions");
    keep = std::min(keep, batch.max_length);
    const EvictArgs a{keep,        sinks,
                      recent,      new_lengths,
                      new_weights, new_positions,
                      reinterpret_cast<int32_t*>(static_cast<char*>(workspace) + kPagedCounterBytes),
                      std::min(keep, batch.max_length - keep),
                      cache.head_dim * (cache.type == kPagedE4M3 ? 1 : 2),
                      cache.type == kPagedE4M3};
    const size_t bytes = paged_moves_bytes(cache, batch, a.room);
    if (a.room) {
        device.check(workspace, "workspace", 16);
        require(workspace_bytes >= kPagedCounterBytes + bytes, "Workspace is too small");
    }
    const unsigned units = unsigned(batch.sequences) * cache.kv_heads;
    if (a.room <= kEvictFew) {
        paged_evict_kernel<true><<<units, kEvictThreads, 0, stream>>>(v, a);
    } else {
        paged_evict_kernel<false><<<units, kEvictThreads, 0, stream>>>(v, a);
        const int64_t most = (a.room + kMoveRows - 1) / kMoveRows;
        const unsigned share = unsigned(std::min<int64_t>(most, std::max(1u, 8192 / units)));
        paged_move_kernel<<<dim3(units, share), 256, 0, stream>>>(v, a);
    }
}

}  // namespace qwen_hip

// Paged key-value cache: argument checks, append, eviction.
#include "paged.hpp"

#include <algorithm>
#include <string>

#include "paged_dev.hpp"
#include "qwen_common.hpp"

namespace qwen_hip {

namespace {
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
        span += a.stride * (a.count - 1);
        require(span <= (int64_t(1) << 44), "Paged strides let rows overlap or run too far");
    }
    require(b.sequences >= 1 && b.sequences <= 65536, "Paged sequences must be in 1..65536");
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
    require(b.rows >= 1 && b.rows <= b.max_length, "Paged rows must be in 1..max_length");
    require(b.total_rows >= 0 && b.total_rows <= kPagedMaxLength, "Paged total_rows must be in 0..2^24");
    require(b.offsets || int64_t(b.sequences) * b.rows == b.total_rows,
            "Paged total_rows must be sequences * rows without offsets");
}

PagedDevice::PagedDevice(const qwen_gpu_paged_cache& c, const qwen_gpu_paged_batch& b, hipStream_t stream) {
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
// of 16 bytes are all in flight at once.
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
    require(int64_t(batch.total_rows) * ((row + 511) / 512) < (int64_t(1) << 32), "Too many new rows for one call");
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

// Weights as whole numbers of the same order; NaN is the lowest, -0 is 0.
__device__ __forceinline__ unsigned weight_key(float w) {
    if (w != w) return 0u;
    const unsigned bits = __builtin_bit_cast(unsigned, w + 0.f);
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

struct EvictArgs {
    int keep, sinks, recent;
    int32_t* new_lengths;
    float* new_weights;
    int32_t* new_positions;
    int32_t* moves;  // workspace: [sequences * kv_heads][2][room], holes then (from the last) sources
    int64_t room;
    int size;        // bytes of a row
    bool scaled;     // rows have exponents
};

// One workgroup per sequence and KV head. The threshold weight (the keep-th
// largest) is found digit by digit, 11 + 11 + 10 bits from the top: a
// histogram of the digit among the slots that share the digits so far, and
// the digit at which the count from above reaches what is still wanted. Of
// the slots at the threshold the first ones are kept. A hole's rank among
// holes is its slot less the kept slots before it, and a kept slot's rank
// needs the same count, so one running count gives both lists.
__global__ __launch_bounds__(kEvictThreads) void paged_evict_kernel(PagedView v, EvictArgs a) {
    __shared__ int bins[kEvictBins];
    __shared__ int2 wave_counts[2][kEvictWaves];
    __shared__ int found[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int s = blockIdx.x / v.kv_heads, head = blockIdx.x - s * v.kv_heads;
    const int n = v.length(s), keep = a.keep;
    const int64_t track = v.track_at(s, head);
    const float* weights = v.weights + track;
    const int32_t* positions = v.positions + track;
    float* new_weights = a.new_weights + track;
    int32_t* new_positions = a.new_positions + track;
    if (head == 0 && tid == 0) a.new_lengths[s] = min(n, keep);
    if (n <= keep) {
        for (int j = tid; j < n; j += kEvictThreads) {
            new_weights[j] = weights[j];
            new_positions[j] = positions[j];
        }
        return;
    }
    const int64_t late = int64_t(v.seen ? v.seen[s] : v.length(s)) - a.recent;
    auto key_of = [&](int j) {
        const int p = positions[j];
        return p < a.sinks || p >= late ? kEvictFixed : weight_key(weights[j]);
    };

    unsigned prefix = 0, known = 0;  // the threshold's digits so far, and which bits they are
    int wanted = keep;               // slots still to be taken among those that share them
    for (int digit = 0; digit < 3; ++digit) {
        const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0, width = digit == 2 ? 1024 : 2048;
        for (int b = tid; b < kEvictBins; b += kEvictThreads) bins[b] = 0;
        __syncthreads();
        for (int j = tid; j < n; j += kEvictThreads) {
            const unsigned key = key_of(j);
            if ((key & known) == prefix) atomicAdd(&bins[(key >> shift) & (width - 1)], 1);
        }
        __syncthreads();
        // Thread t holds bins top - 2 t and the one below; counts from above.
        const int upper = bins[kEvictBins - 1 - 2 * tid], lower = bins[kEvictBins - 2 - 2 * tid];
        int sum = upper + lower;
        for (int off = 1; off < 64; off *= 2) {
            const int other = __shfl_up(sum, off);
            if (lane >= off) sum += other;
        }
        if (lane == 63) wave_counts[0][wave].x = sum;
        __syncthreads();
        int above = sum - upper - lower;
        for (int w = 0; w < wave; ++w) above += wave_counts[0][w].x;
        if (above < wanted && above + upper + lower >= wanted) {
            const bool second = above + upper < wanted;
            found[0] = kEvictBins - 1 - 2 * tid - second;
            found[1] = wanted - above - (second ? upper : 0);
        }
        __syncthreads();
        prefix |= unsigned(found[0]) << shift;
        known |= unsigned(width - 1) << shift;
        wanted = found[1];
        __syncthreads();
    }

    int32_t* const holes = a.moves + int64_t(blockIdx.x) * 2 * a.room;
    int32_t* const sources = holes + a.room;
    int above_before = 0, at_before = 0;
    for (int begin = 0, turn = 0; begin < n; begin += kEvictThreads, turn ^= 1) {
        const int j = begin + tid;
        const unsigned key = j < n ? key_of(j) : 0u;
        const bool above = j < n && key > prefix, at = j < n && key == prefix;
        const unsigned long long above_mask = __ballot(above), at_mask = __ballot(at);
        if (lane == 0) wave_counts[turn][wave] = int2{__popcll(above_mask), __popcll(at_mask)};
        __syncthreads();
        const unsigned long long before = (1ull << lane) - 1;
        int above_rank = above_before + __popcll(above_mask & before), at_rank = at_before + __popcll(at_mask & before);
        for (int w = 0; w < kEvictWaves; ++w) {
            const int2 c = wave_counts[turn][w];
            if (w < wave) above_rank += c.x, at_rank += c.y;
            above_before += c.x;
            at_before += c.y;
        }
        const bool kept = above || (at && at_rank < wanted);
        const int rank = above_rank + min(at_rank, wanted);  // kept slots before this one
        if (j == keep) found[0] = keep - rank;               // the rest of them have to move
        if (j >= n) continue;
        if (j >= keep) {
            if (kept && keep - 1 - rank < a.room) sources[keep - 1 - rank] = j;
        } else if (!kept) {
            if (j - rank < a.room) holes[j - rank] = j;
        } else {
            new_weights[j] = weights[j];
            new_positions[j] = positions[j];
        }
    }
    __syncthreads();
    const int moved = int(min(int64_t(found[0]), a.room));
    for (int i = tid; i < moved; i += kEvictThreads) {
        const int to = holes[i], from = sources[moved - 1 - i];
        new_weights[to] = weights[from];
        new_positions[to] = positions[from];
    }
    // Rows move in pieces of 16 bytes: keys, then values.
    const int pieces = a.size / 16, all = 2 * pieces;
    for (int64_t i = tid; i < int64_t(moved) * all; i += kEvictThreads) {
        const int m = int(i / all), piece = int(i - int64_t(m) * all);
        const PageSlot to = page_slot(holes[m], v.page_size, v.magic);
        const PageSlot from = page_slot(sources[moved - 1 - m], v.page_size, v.magic);
        const int to_page = v.page_of(s, to.page), from_page = v.page_of(s, from.page);
        if (to_page < 0 || from_page < 0) continue;
        char* const pool = piece < pieces ? v.keys : v.values;
        const int64_t at = 16 * (piece < pieces ? piece : piece - pieces);
        *reinterpret_cast<uint4_t*>(pool + v.row_at(to_page, head, to.slot) + at) =
            *reinterpret_cast<const uint4_t*>(pool + v.row_at(from_page, head, from.slot) + at);
        if (piece == 0 && a.scaled)
            *reinterpret_cast<uint16_t*>(v.exponents + v.exponents_at(to_page, head, to.slot)) =
                *reinterpret_cast<const uint16_t*>(v.exponents + v.exponents_at(from_page, head, from.slot));
    }
}

int64_t evict_room(const qwen_gpu_paged_batch& b, int keep) { return std::min(keep, b.max_length - keep); }
size_t evict_bytes(const qwen_gpu_paged_cache& c, const qwen_gpu_paged_batch& b, int64_t room) {
    return size_t(b.sequences) * c.kv_heads * 2 * room * sizeof(int32_t);
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
                      evict_room(batch, keep),
                      cache.head_dim * (cache.type == kPagedE4M3 ? 1 : 2),
                      cache.type == kPagedE4M3};
    const size_t bytes = evict_bytes(cache, batch, a.room);
    if (bytes) {
        device.check(workspace, "workspace", 16);
        require(workspace_bytes >= kPagedCounterBytes + bytes, "Workspace is too small");
    }
    paged_evict_kernel<<<batch.sequences * cache.kv_heads, kEvictThreads, 0, stream>>>(v, a);
}

}  // namespace qwen_hip

// Attention of new rows over a paged key-value cache whose sequences share
// prefixes: the kernel and its launch, included by one source for each type of
// cache (they compile side by side).
#pragma once
#include <algorithm>

#include "paged_attention.hpp"

namespace qwen_hip {

struct SharedArgs {
    const float* queries;
    int64_t query_stride;
    float* out;
    int64_t out_stride;
    int group, query_heads;
    unsigned magic;             // of the group
    float scale;                // times log2(e)
    const int32_t* lengths;     // of the prefixes
    const int32_t* offsets;     // NULL: one group of all sequences
    int groups;
    int rest_tiles;             // of a sequence's query rows
    int parts, rest_parts;      // of a prefix, of what is behind it, at most
    int part, rest_part;        // positions of each
    int jobs, rest_jobs;        // workgroups of the prefixes (a multiple of 8), of what is behind them
    bool compact;               // behind the prefixes only those with work come first
    float* sums;                // [parts + rest_parts][total_rows][query_heads][DIM]
    float2* states;             // [parts + rest_parts][total_rows][query_heads]: reference, sum

    __device__ __forceinline__ int new_row(int r) const { return page_slot(r, group, magic).page; }
    __device__ __forceinline__ int64_t place(const PagedView& v, int slot, int row, int head) const {
        return (int64_t(slot) * v.total_rows + row) * query_heads + head;
    }
    // Sequences of a group.
    __device__ __forceinline__ int first_of(const PagedView& v, int g) const {
        return offsets ? min(max(offsets[g], 0), v.sequences) : g ? v.sequences : 0;
    }
    // First new row of a sequence, which is the end of the one before.
    __device__ __forceinline__ int row_of(const PagedView& v, int s) const {
        return v.offsets ? min(max(v.offsets[s], 0), v.total_rows) : s * v.rows;
    }
    __device__ __forceinline__ static int parts_of(int positions, int part, int most) {
        return min(most, (positions + part - 1) / part);
    }
};

// The groups, as a wave knows them: of up to 63, lane g has group g's first
// sequence and prefix, so that a job is found in two or three loads one behind
// the other instead of five.
struct SharedGroups {
    const PagedView& v;
    const SharedArgs& a;
    const int lane;
    const bool few;
    int start = 0, length = 0;

    __device__ __forceinline__ SharedGroups(const PagedView& view, const SharedArgs& args)
        : v(view), a(args), lane(threadIdx.x & 63), few(args.groups < 64) {
        if (few) {
            start = a.first_of(v, min(lane, a.groups));
            length = a.lengths[min(lane, a.groups - 1)];
        }
    }
    __device__ __forceinline__ int first(int g) const {
        return few ? __builtin_amdgcn_readlane(start, g) : a.first_of(v, g);
    }
    // Query rows of a KV head in group g0 + lane, and the parts of its prefix at most.
    __device__ __forceinline__ void of_lane(int g0, int& rows, int& parts) const {
        const int g = g0 + lane;
        const bool there = g < a.groups;
        const int from = few ? start : a.first_of(v, min(g, a.groups));
        const int row = a.row_of(v, from);
        int next;
        if (few)
            next = __shfl_down(row, 1);
        else
            next = a.row_of(v, a.first_of(v, min(g + 1, a.groups)));
        rows = there ? max(0, next - row) * a.group : 0;
        parts = there ? a.parts_of(max(0, min(few ? length : a.lengths[g], v.max_length)), a.part, a.parts) : 0;
    }
    // Group of a sequence, -1 where it has none; the same in all lanes.
    __device__ __forceinline__ int of(int s) const {
        if (few) {
            const int n = __popcll(__ballot(lane < a.groups && start <= s));
            return n > 0 && s < __builtin_amdgcn_readlane(start, n) ? n - 1 : -1;
        }
        int low = 0, high = a.groups;  // the number of groups that begin at s or before lies in low .. high
        while (high > low) {
            const int step = (high - low + 63) / 64, at = low + lane * step;
            const int n = __popcll(__ballot(at < high && a.offsets[min(at, a.groups)] <= s));
            if (n == 0) {
                high = low;
            } else {
                const int last = low + (n - 1) * step;
                high = min(high, last + step);
                low = last + 1;
            }
        }
        return low > 0 && s < a.offsets[low] ? low - 1 : -1;
    }
    // Positions that a group's sequences share, no more than any of them has before its new rows, and its first
    // sequence with new rows, through whose table they are read.
    __device__ __forceinline__ int prefix(int g, int& reads) const {
        if (g < 0 || !a.jobs) return 0;  // no group, or none that has workgroups
        const int from = first(g), to = first(g + 1);
        int least = few ? __builtin_amdgcn_readlane(length, g) : a.lengths[g];
        reads = to;
        for (int s = from + lane; s < to; s += 64) {
            int row;
            const int n = v.new_rows(s, row), positions = v.length(s);
            if (n > 0) least = min(least, positions - n), reads = min(reads, s);
        }
        each_half([&](auto off) {
            constexpr int kOff = decltype(off)::value;
            least = min(least, dev::xor_lanes<kOff>(least));
            reads = min(reads, dev::xor_lanes<kOff>(reads));
        });
        reads = __builtin_amdgcn_readfirstlane(reads);
        return max(0, __builtin_amdgcn_readfirstlane(least));
    }
    // Positions that a group's prefix has, whatever its sequences have of it; 0 without a group.
    __device__ __forceinline__ int nominal(int g) const {
        if (g < 0 || !a.jobs) return 0;
        return few ? __builtin_amdgcn_readlane(length, g) : a.lengths[g];
    }
    // Of each lane's sequence (few groups).
    __device__ __forceinline__ int nominal_of_lane(int s) const {
        int of = 0;
        if (a.jobs)
            for (int g = 0; g < a.groups; ++g)
                if (s >= __builtin_amdgcn_readlane(start, g) && s < __builtin_amdgcn_readlane(start, g + 1))
                    of = __builtin_amdgcn_readlane(length, g);
        return of;
    }
    // Parts of what a sequence has behind a prefix of that many positions, its own new rows at least.
    __device__ __forceinline__ int rest_parts(int positions, int n, int of_group) const {
        return a.parts_of(positions - max(0, min(of_group, positions - n)), a.rest_part, a.rest_parts);
    }
    template <class F>
    static __device__ __forceinline__ void each_half(F f) {
        f(std::integral_constant<int, 32>{}), f(std::integral_constant<int, 16>{}), f(std::integral_constant<int, 8>{});
        f(std::integral_constant<int, 4>{}), f(std::integral_constant<int, 2>{}), f(std::integral_constant<int, 1>{});
    }
};

// What a workgroup does: a tile of query rows of a KV head against a range of
// a sequence's positions.
struct SharedJob {
    int head, s;              // whose table
    int first;                // new row of query row 0
    int row0, rows;           // query rows: the tile's first one, the end
    int from, to;             // positions
    int sees;                 // behind a prefix: positions that the first new row attends, one more each row
    int slot;                 // of its sums
};

// LDS of a workgroup: a wave's values, then its sums.
template <int DIM>
struct SharedSpace {
    static constexpr int kPitch = DIM * 2 + 32;  // bytes of a value row
    __attribute__((aligned(16))) char rows[kWaves][kTile * kPitch];
    float2 states[kWaves][16];
};

// Query rows of a job as their terms: row r is head r % group of new row
// r / group. Scores' factor is above 0, so that minus infinity stays that: a scale's
// sign goes into the queries.
template <int DIM>
__device__ __forceinline__ const float* query_at(const PagedView& v, const SharedArgs& a, const SharedJob& job, int query_row,
                                                 bool& live) {
    const int new_row = a.new_row(query_row);
    const int64_t row = int64_t(job.first) + new_row;
    live = query_row < job.rows && row >= 0 && row < v.total_rows;
    return a.queries + (live ? row * a.query_stride + (job.head * a.group + query_row - new_row * a.group) * DIM : 0);
}
// PER: 16-bit products of a lane's 16 bytes of a stored row, whose channels it holds.
template <int DIM, int PER>
__device__ __forceinline__ void load_query(const float* from, bool live, int part, float (&x)[DIM / 32][8]) {
#pragma unroll
    for (int k = 0; k < DIM / 32; ++k) {
        const int channel = PER == 1 ? 32 * k + 8 * part : 64 * (k / 2) + 16 * part + 8 * (k % 2);
        const float4_a4 lo = *reinterpret_cast<const float4_a4*>(from + channel);
        const float4_a4 hi = *reinterpret_cast<const float4_a4*>(from + channel + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[k][e] = live ? lo[e] : 0.f, x[k][4 + e] = live ? hi[e] : 0.f;
    }
}
template <int TYPE, int DIM, int TERMS>
__device__ __forceinline__ float split_query(float (&x)[DIM / 32][8], float scale, uint4_t (&query)[DIM / 32][TERMS]) {
    float to_score = fmaxf(__builtin_fabsf(scale), 1e-37f), times = scale == 0.f ? 0.f : __builtin_copysignf(1.f, scale);
    if constexpr (TYPE == kPagedF16) {
        // An exact power of two brings a row's largest query to [2^14, 2^15), so that neither term leaves
        // FP16's range; non-finite ones stay so.
        float top = 0.f;
#pragma unroll
        for (int k = 0; k < DIM / 32; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) top = fmaxf(top, __builtin_fabsf(x[k][e]));
        top = fmaxf(top, dev::xor_lanes<16>(top));
        top = fmaxf(top, dev::xor_lanes<32>(top));
        const int up = 14 - max(int(__builtin_bit_cast(unsigned, top) >> 23) - 127, -100);
        times *= pow2(up);
        to_score = fmaxf(to_score * pow2(-up), 0x1p-149f);
    }
#pragma unroll
    for (int k = 0; k < DIM / 32; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            unsigned words[TERMS];
            Terms<TYPE, false>::split(x[k][2 * e] * times, x[k][2 * e + 1] * times, false, words);
#pragma unroll
            for (int p = 0; p < TERMS; ++p) query[k][p][e] = words[p];
        }
    return to_score;
}

// A step of a row's online softmax: 8 scores of a lane (minus infinity where
// hidden) times factor(u, r) become weights relative to the row's reference,
// which moves, and the sums so far with it, only when a score passes it by 2^8.
template <int TYPE, int OUT, class F>
__device__ __forceinline__ void soften(const float4_t (&s)[2], F factor, float high, float& reference, float& sum,
                                       float4_t (&acc)[OUT], float (&weights)[2][4]) {
    constexpr float kHead = TYPE == kPagedF16 ? 6.f : 0.f;  // FP16 weights are kept up to 2^14, far from subnormals
    constexpr float kGrow = 8.f;
    if (__any(high > reference + (kHead + kGrow))) {
        high = fmaxf(high, dev::xor_lanes<16>(high));
        high = fmaxf(high, dev::xor_lanes<32>(high));
        const float moved = fmaxf(reference, high - kHead);
        const float shrink = reference == moved ? 1.f : exp2_fast(reference - moved);
        reference = moved;
        sum *= shrink;
#pragma unroll
        for (int o = 0; o < OUT; ++o) acc[o] *= shrink;
    }
    const float from = reference == -kInf ? 0.f : reference;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            weights[u][r] = exp2_fast(__builtin_fmaf(s[u][r], factor(u, r), -from));
            sum += weights[u][r];
        }
}
template <int TYPE, int TERMS>
__device__ __forceinline__ void split_weights(const float (&weights)[2][4], uint4_t (&terms)[TERMS]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        unsigned words[TERMS];
        Terms<TYPE, false>::split(weights[e / 2][2 * (e % 2)], weights[e / 2][2 * (e % 2) + 1], false, words);
#pragma unroll
        for (int p = 0; p < TERMS; ++p) terms[p][e] = words[p];
    }
}

// Up to 16 query rows: S^T = K Q^T and O^T = V^T P^T on the matrix cores as
// paged_attention_kernel has them, 32 positions a wave's step, FP32 queries and
// weights as two FP16 or three BF16 terms, each wave every fourth step, the
// next one's loads in flight. CAUSAL: positions behind a prefix, which end at
// each new row's own. Memory bounds it where there are many positions; a
// workgroup spends 8 us besides (2 to find its job, 3 for the first rows, 3
// for the waves' sums and to make place for the next).
template <int TYPE, int DIM, bool CAUSAL>
__device__ __forceinline__ void shared_attend(const PagedView& v, const SharedArgs& a, const SharedJob& job,
                                              SharedSpace<DIM>& space) {
    constexpr int kSize = TYPE == kPagedE4M3 ? 1 : 2, kLoads = DIM * kSize / 64, kSteps = DIM / 32, kOut = DIM / 16;
    constexpr int kPer = kSteps / kLoads;         // products per load: 1, or 2 for E4M3
    constexpr int kProducts = Terms<TYPE, false>::kProducts, kPitch = SharedSpace<DIM>::kPitch;
    constexpr std::integral_constant<int, TYPE> kType{};
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int column = lane & 15, part = lane >> 4;
    // Positions from shared_end on are seen by some of the tile's new rows only, from `end` on by none.
    const int last_row = min(job.rows, job.row0 + 16) - 1;
    const int shared_end = CAUSAL ? min(job.to, job.sees + a.new_row(job.row0)) : job.to;
    const int end = CAUSAL ? min(job.to, job.sees + a.new_row(last_row)) : job.to;
    const int32_t* const table = v.table + int64_t(job.s) * v.table_stride;

    // A step's rows: page entries, then offsets, then 16-byte pieces.
    int pages[2], slots[2];
    int64_t at[2];
    bool there[2];
    uint4_t keys[2][kLoads], values[2][kLoads];
    unsigned bytes[2] = {0, 0};
    auto find = [&](int base) {  // entries; positions past the end take the last one's
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const PageSlot where = page_slot(max(0, min(base + 16 * u + column, end - 1)), v.page_size, v.magic);
            slots[u] = where.slot;
            pages[u] = table[where.page];
        }
    };
    auto place = [&](int base) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const bool known = pages[u] >= 0 && pages[u] < v.pages;
            there[u] = known && base + 16 * u + column < end;
            const int page = known ? pages[u] : 0;
            at[u] = v.row_at(page, job.head, slots[u]) + 16 * part;
            if constexpr (TYPE == kPagedE4M3)
                bytes[u] = *reinterpret_cast<const uint16_t*>(v.exponents + v.exponents_at(page, job.head, slots[u]));
        }
    };
    auto load = [&](const char* pool, uint4_t (&to)[2][kLoads]) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < kLoads; ++i) to[u][i] = *reinterpret_cast<const uint4_t*>(pool + at[u] + 64 * i);
    };
    char* const mine = space.rows[wave];
    const char* const transposed = mine + (4 * part + (column >> 2)) * kPitch + (column & 3) * 8;

    // The table's entries first, then queries, keys and values in one flight.
    int base = job.from + kTile * wave;
    if (base < end) find(base);
    bool live;
    const float* const from = query_at<DIM>(v, a, job, job.row0 + column, live);
    const int sees = !live ? 0 : CAUSAL ? job.sees + a.new_row(job.row0 + column) : job.to;  // of the lane's row
    float x[kSteps][8];
    load_query<DIM, kPer>(from, live, part, x);
    if (base < end) {
        place(base);
        load(v.keys, keys);
        if (base + kBlock < end) find(base + kBlock);
        load(v.values, values);
    }
    uint4_t query[kSteps][kProducts];
    const float to_score = split_query<TYPE, DIM>(x, a.scale, query);
    float4_t acc[kOut];
    float reference = -kInf, sum = 0.f;
#pragma unroll
    for (int o = 0; o < kOut; ++o) acc[o] = float4_t{0.f, 0.f, 0.f, 0.f};

    for (; base < end; base += kBlock) {
        float4_t s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                uint4_t k[kPer];
                widen<TYPE>(keys[u][i], byte_pow2(bytes[u] & 255), k);
#pragma unroll
                for (int j = 0; j < kPer; ++j)
#pragma unroll
                    for (int p = 0; p < kProducts; ++p) s[u] = multiply(k[j], query[kPer * i + j][p], s[u], kType);
            }
        // What the rest of this step needs of its rows, before the next one's take their place.
        const bool was[2] = {there[0], there[1]};
        const int64_t row_at[2] = {at[0] - 16 * part, at[1] - 16 * part};
        const float value_up[2] = {byte_pow2(bytes[0] >> 8), byte_pow2(bytes[1] >> 8)};
        const unsigned exist = (unsigned(__ballot(was[0])) & 0xffffu) | unsigned(__ballot(was[1])) << 16;
        const bool more_steps = base + kBlock < end;
        if (more_steps) {
            place(base + kBlock);
            load(v.keys, keys);
        }
        const bool whole = exist == 0xffffffffu && base + kTile <= shared_end;

        // Values into LDS, 0 for those that are not there. A weight of 0 does not keep infinities and NaN
        // out, so those in rows that only some new rows see are 0 here as well, and added below. They are found
        // in the 16-bit words: an E4M3 row's power of two may carry finite codes past what these hold.
        const bool triangle = CAUSAL && base + kTile > shared_end;
        unsigned spoilt_bits = 0;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const unsigned partly = base + 16 * u + column >= shared_end ? ~0u : 0u;
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                uint4_t w[kPer];
                widen<TYPE>(values[u][i], value_up[u], w);
#pragma unroll
                for (int j = 0; j < kPer; ++j) {
                    if (!whole && !was[u]) w[j] = uint4_t{0u, 0u, 0u, 0u};
                    if (triangle)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const unsigned bad = not_finite<TYPE == kPagedF16>(w[j][e]) & partly;
                            spoilt_bits |= bad;
                            w[j][e] &= ~((bad >> 15) * 0xffffu);
                        }
                    char* const to = mine + (16 * u + column) * kPitch + 64 * kPer * i + 16 * kPer * part + 16 * j;
                    *reinterpret_cast<uint4_t*>(to) = w[j];
                }
            }
        }
        const bool spoilt = triangle && __any(spoilt_bits != 0);
        if (more_steps) {
            if (base + 2 * kBlock < end) find(base + 2 * kBlock);
            load(v.values, values);
        }

        if (!whole)
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int j = 16 * u + 4 * part + r;
                    if (!(exist >> j & 1) || (CAUSAL && base + j >= sees)) s[u][r] = -kInf;
                }
        float high = s[0][0], weights[2][4];
#pragma unroll
        for (int i = 1; i < 8; ++i) high = fmaxf(high, s[i / 4][i % 4]);
        soften<TYPE>(s, [&](int, int) { return to_score; }, high * to_score, reference, sum, acc, weights);
        uint4_t weight[kProducts];
        split_weights<TYPE>(weights, weight);
#pragma unroll
        for (int o = 0; o < kOut; ++o) {
            const short4_t low = read_transposed(transposed + 32 * o);
            const short4_t top = read_transposed(transposed + 16 * kPitch + 32 * o);
            const uint4_t w = {__builtin_bit_cast(u32x2, low)[0], __builtin_bit_cast(u32x2, low)[1],
                               __builtin_bit_cast(u32x2, top)[0], __builtin_bit_cast(u32x2, top)[1]};
#pragma unroll
            for (int p = 0; p < kProducts; ++p) acc[o] = multiply(w, weight[p], acc[o], kType);
        }

        // One row at a time, for the new rows that see it; the wave's weights pass through its part of LDS, whose
        // values have been read.
        if (CAUSAL && spoilt) {
            float* const passed = reinterpret_cast<float*>(mine);
#pragma unroll
            for (int u = 0; u < 2; ++u)
                *reinterpret_cast<float4_t*>(passed + column * kTile + 16 * u + 4 * part) =
                    float4_t{weights[u][0], weights[u][1], weights[u][2], weights[u][3]};
            for (int j = max(0, shared_end - base); j < kTile; ++j) {
                if (!(exist >> j & 1)) continue;
                const int64_t row = __shfl(j < 16 ? row_at[0] : row_at[1], j & 15);
                const float up = __shfl(j < 16 ? value_up[0] : value_up[1], j & 15);
                const float p = passed[column * kTile + j];
                if (base + j >= sees) continue;
#pragma unroll
                for (int o = 0; o < kOut; ++o)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float value = stored<TYPE>(v.values + row, 16 * o + 4 * part + e, up);
                        if (value - value != 0.f) acc[o][e] = __builtin_fmaf(p, value, acc[o][e]);
                    }
            }
        }
    }

    // The four waves' sums, brought to their largest reference.
    float* const sums = reinterpret_cast<float*>(space.rows);  // [kWaves][16][DIM]
    __syncthreads();
    sum += dev::xor_lanes<16>(sum);
    sum += dev::xor_lanes<32>(sum);
    if (lane < 16) space.states[wave][lane] = float2{reference, sum};
#pragma unroll
    for (int o = 0; o < kOut; ++o)
        *reinterpret_cast<float4_t*>(sums + (wave * 16 + column) * DIM + 16 * o + 4 * part) = acc[o];
    __syncthreads();
    for (int item = threadIdx.x; item < 16 * DIM / 4; item += kWaves * 64) {
        const int local = item / (DIM / 4), channel = 4 * (item - local * (DIM / 4));
        const int query_row = job.row0 + local, new_row = a.new_row(query_row);
        const int64_t row = int64_t(job.first) + new_row;
        if (query_row >= job.rows || row < 0 || row >= v.total_rows) continue;
        float top = -kInf, all = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) top = fmaxf(top, space.states[w][local].x);
        float4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float2 state = space.states[w][local];
            const float shrink = state.x == top ? 1.f : exp2_fast(state.x - top);
            all = __builtin_fmaf(state.y, shrink, all);
            const float4_t y = *reinterpret_cast<const float4_t*>(sums + (w * 16 + local) * DIM + channel);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(y[e], shrink, o[e]);
        }
        const int64_t to = a.place(v, job.slot, int(row), job.head * a.group + query_row - new_row * a.group);
        *reinterpret_cast<float4_t*>(a.sums + to * DIM + channel) = o;
        if (channel == 0) a.states[to] = float2{top, all};
    }
}

// 16 E4M3 values as FP16, exact.
__device__ __forceinline__ void widen_f16(uint4_t raw, uint4_t (&out)[2]) {
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const auto low = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(raw[w], 1.f, false);
        const auto high = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(raw[w], 1.f, true);
        out[w / 2][2 * (w % 2)] = __builtin_bit_cast(unsigned, low);
        out[w / 2][2 * (w % 2) + 1] = __builtin_bit_cast(unsigned, high);
    }
}

// LDS of a workgroup whose waves share its positions: two steps' keys and
// values, 16-bit whatever the cache's type, and which of them exist. (64
// positions a step instead of 32 took 46 us, not 42, for 8192 F16 positions,
// and 132, not 120, for 4 times 24 BF16 sequences.)
template <int DIM>
struct WideSpace {
    static constexpr int kPositions = DIM == 64 ? 64 : 32, kPitch = DIM * 2 + 32;
    __attribute__((aligned(16))) char keys[2][kPositions * kPitch];
    __attribute__((aligned(16))) char values[2][kPositions * kPitch];
    __attribute__((aligned(16))) int there[2][kPositions];
    __attribute__((aligned(16))) float powers[2][kPositions];  // E4M3: of the keys
    __attribute__((aligned(16))) int all[2][kWaves];
};

// A prefix against more query rows: each wave has TILES times 16 rows of its
// own and all waves go over the same positions, which the workgroup brings
// into LDS together, a step ahead, widened to 16 bits once. A wave's part of the loads
// takes a quarter of the registers, so that two workgroups fit a CU and one's
// products run beside the other's exponentials.
//
// A prefix is read once from memory, but multiplied with every query row, in
// two or three terms: 65000 E4M3 positions of 8 heads by 128 rows are 30 us of
// products at the rate of a large matrix product, 74 in terms (a score's two
// and a weight's three), 26 of their bytes. The kernel takes 105 to 111, a call
// of both kernels among others 103, as LDS, exponentials and products wait for
// each other at two waves a SIMD; tiles that every wave reads for itself,
// without LDS, took 1020. Of 64 rows (TILES 1) 8192 positions and what 64 users
// have behind them took 48 us a call in a graph, of 128 40; heads of 256 have
// registers for 64.
template <int TYPE, int DIM, int TILES>
__device__ __forceinline__ void shared_attend_wide(const PagedView& v, const SharedArgs& a, const SharedJob& job,
                                                   WideSpace<DIM>& space) {
    typedef WideSpace<DIM> Space;
    constexpr int kSize = TYPE == kPagedE4M3 ? 1 : 2, kSteps = DIM / 32, kOut = DIM / 16;
    constexpr int kPositions = Space::kPositions, kPitch = Space::kPitch;
    // E4M3 keys are FP16 in LDS, which holds them all, and their rows' powers of two go to the scores: two terms
    // of a query instead of three. Values' powers belong to the sums over positions, so values become BF16.
    constexpr bool kScaled = TYPE == kPagedE4M3;
    constexpr int kKeyType = kScaled ? kPagedF16 : TYPE;
    constexpr int kProducts = Terms<TYPE, false>::kProducts, kTerms = Terms<kKeyType, false>::kProducts;
    constexpr int kChunks = DIM * kSize / 16;     // threads of a stored row, 16 bytes each
    constexpr int kAtOnce = kWaves * 64 / kChunks, kLoads = kPositions / kAtOnce;  // rows of a load; loads
    constexpr int kWords = TYPE == kPagedE4M3 ? 2 : 1;
    constexpr std::integral_constant<int, TYPE> kType{};
    constexpr std::integral_constant<int, kKeyType> kKeys{};
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int column = lane & 15, part = lane >> 4;
    const int my_row = threadIdx.x / kChunks, chunk = threadIdx.x % kChunks, end = job.to;
    const int32_t* const table = v.table + int64_t(job.s) * v.table_stride;

    int pages[kLoads], slots[kLoads];
    bool there[kLoads];
    uint4_t keys[kLoads], values[kLoads];
    unsigned bytes[kLoads] = {};
    auto find = [&](int base) {  // entries; positions past the end take the last one's
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const PageSlot where = page_slot(min(base + i * kAtOnce + my_row, end - 1), v.page_size, v.magic);
            slots[i] = where.slot;
            pages[i] = table[where.page];
        }
    };
    auto load = [&](int base) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const bool known = pages[i] >= 0 && pages[i] < v.pages;
            there[i] = known && base + i * kAtOnce + my_row < end;
            const int page = known ? pages[i] : 0;
            const int64_t at = v.row_at(page, job.head, slots[i]) + 16 * chunk;
            if constexpr (TYPE == kPagedE4M3)
                bytes[i] = *reinterpret_cast<const uint16_t*>(v.exponents + v.exponents_at(page, job.head, slots[i]));
            keys[i] = *reinterpret_cast<const uint4_t*>(v.keys + at);
            values[i] = *reinterpret_cast<const uint4_t*>(v.values + at);
        }
    };
    int base = job.from, buffer = 0;
    find(base);

    // A wave's tiles are four apart, so that fewer than 4 * TILES of them are shared out evenly.
    const int first_row = job.row0 + 16 * wave;
    const int live_tiles = first_row < job.rows ? min(TILES, (job.rows - first_row + 63) / 64) : 0;
    uint4_t query[TILES][kSteps][kTerms];
    float to_score[TILES], reference[TILES], sum[TILES];
    float4_t acc[TILES][kOut];
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
        reference[t] = -kInf, sum[t] = 0.f;
#pragma unroll
        for (int o = 0; o < kOut; ++o) acc[t][o] = float4_t{0.f, 0.f, 0.f, 0.f};
        float x[kSteps][8];
        if (t < live_tiles) {
            bool live;
            const float* const from = query_at<DIM>(v, a, job, first_row + 64 * t + column, live);
            load_query<DIM, 1>(from, live, part, x);
        }
        if (t == 0) {  // in one flight with the first queries
            load(base);
            if (base + kPositions < end) find(base + kPositions);
        }
        if (t < live_tiles) to_score[t] = split_query<kKeyType, DIM>(x, a.scale, query[t]);
        __builtin_amdgcn_sched_barrier(0);  // a tile's queries at a time, for the registers
    }

    // The loop has no branches around a tile's products, which would wait for every piece of LDS by itself.
    auto go = [&](auto live) {
        constexpr int LIVE = decltype(live)::value;
        for (; base < end; base += kPositions, buffer ^= 1) {
            bool whole_here = true;
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                uint4_t k[kWords], w[kWords];
                if constexpr (kScaled)
                    widen_f16(keys[i], k);
                else
                    widen<TYPE>(keys[i], 1.f, k);
                widen<TYPE>(values[i], byte_pow2(bytes[i] >> 8), w);
                const int row = i * kAtOnce + my_row, to = row * kPitch + 16 * kWords * chunk;
#pragma unroll
                for (int j = 0; j < kWords; ++j) {
                    if (!there[i]) w[j] = uint4_t{0u, 0u, 0u, 0u};  // a weight of 0 does not keep NaN out
                    *reinterpret_cast<uint4_t*>(space.keys[buffer] + to + 16 * j) = k[j];
                    *reinterpret_cast<uint4_t*>(space.values[buffer] + to + 16 * j) = w[j];
                }
                if (chunk == 0) {
                    space.there[buffer][row] = there[i];
                    if constexpr (kScaled) space.powers[buffer][row] = byte_pow2(bytes[i] & 255);
                }
                whole_here = whole_here && there[i];
            }
            const bool whole_wave = __all(whole_here);
            if (lane == 0) space.all[buffer][wave] = whole_wave;
            if (base + kPositions < end) {
                load(base + kPositions);
                if (base + 2 * kPositions < end) find(base + 2 * kPositions);
            }
            // Nobody writes a buffer again before all have passed the next barrier, and so have read it.
            __syncthreads();
            if constexpr (!LIVE) continue;
            bool whole = true;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) whole = whole && space.all[buffer][w];

            // 32 positions at a time, for the registers.
#pragma unroll 1
            for (int h = 0; h < kPositions / 32; ++h) {
                const char* const key = space.keys[buffer] + (32 * h + column) * kPitch + 16 * part;
                const char* const transposed =
                    space.values[buffer] + (32 * h + 4 * part + (column >> 2)) * kPitch + (column & 3) * 8;
                float4_t s[LIVE ? LIVE : 1][2];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
#pragma unroll
                    for (int t = 0; t < LIVE; ++t) s[t][u] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int k = 0; k < kSteps; ++k) {
                        const uint4_t x = *reinterpret_cast<const uint4_t*>(key + 16 * u * kPitch + 64 * k);
#pragma unroll
                        for (int t = 0; t < LIVE; ++t) {
#pragma unroll
                            for (int p = 0; p < kTerms; ++p) s[t][u] = multiply(x, query[t][k][p], s[t][u], kKeys);
                        }
                    }
                }
                float4_t powers[2];
                if constexpr (kScaled)
#pragma unroll
                    for (int u = 0; u < 2; ++u)
                        powers[u] = *reinterpret_cast<const float4_t*>(space.powers[buffer] + 32 * h + 16 * u + 4 * part);
                unsigned hidden = 0;  // bit 4 u + r
                if (!whole)
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (!space.there[buffer][32 * h + 16 * u + 4 * part + r]) hidden |= 1u << (4 * u + r);
                uint4_t weight[LIVE ? LIVE : 1][kProducts];
#pragma unroll
                for (int t = 0; t < LIVE; ++t) {
                    if (!whole)
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (hidden >> i & 1) s[t][i / 4][i % 4] = -kInf;
                    float weights[2][4], high = -kInf;
                    if constexpr (kScaled) {
                        float factor[2][4];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            factor[i / 4][i % 4] = fmaxf(to_score[t] * powers[i / 4][i % 4], 0x1p-149f);
                            high = fmaxf(high, s[t][i / 4][i % 4] * factor[i / 4][i % 4]);
                        }
                        soften<TYPE>(s[t], [&](int u, int r) { return factor[u][r]; }, high, reference[t], sum[t], acc[t],
                                     weights);
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i) high = fmaxf(high, s[t][i / 4][i % 4]);
                        soften<TYPE>(s[t], [&](int, int) { return to_score[t]; }, high * to_score[t], reference[t], sum[t],
                                     acc[t], weights);
                    }
                    split_weights<TYPE>(weights, weight[t]);
                }
#pragma unroll
                for (int o = 0; o < kOut; ++o) {
                    const short4_t low = read_transposed(transposed + 32 * o);
                    const short4_t high = read_transposed(transposed + 16 * kPitch + 32 * o);
                    const uint4_t w = {__builtin_bit_cast(u32x2, low)[0], __builtin_bit_cast(u32x2, low)[1],
                                       __builtin_bit_cast(u32x2, high)[0], __builtin_bit_cast(u32x2, high)[1]};
#pragma unroll
                    for (int t = 0; t < LIVE; ++t) {
#pragma unroll
                        for (int p = 0; p < kProducts; ++p) acc[t][o] = multiply(w, weight[t][p], acc[t][o], kType);
                    }
                }
            }
        }
    };
    if (live_tiles == TILES)
        go(std::integral_constant<int, TILES>{});
    else if (TILES > 1 && live_tiles)
        go(std::integral_constant<int, 1>{});
    else
        go(std::integral_constant<int, 0>{});

#pragma unroll
    for (int t = 0; t < TILES; ++t) {
        if (t >= live_tiles) continue;
        float all = sum[t];
        all += dev::xor_lanes<16>(all);
        all += dev::xor_lanes<32>(all);
        const int query_row = first_row + 64 * t + column, new_row = a.new_row(query_row);
        if (query_row >= job.rows) continue;
        const int64_t to = a.place(v, job.slot, job.first + new_row, job.head * a.group + query_row - new_row * a.group);
#pragma unroll
        for (int o = 0; o < kOut; ++o) *reinterpret_cast<float4_t*>(a.sums + to * DIM + 16 * o + 4 * part) = acc[t][o];
        if (part == 0) a.states[to] = float2{reference[t], all};
    }
}

// Query rows of a workgroup of the prefixes, by how wide it is: 16 that its
// waves split the positions of, or 64 or 128 dealt to the waves.
__host__ __device__ constexpr int rows_of_wide(int wide) { return wide ? 64 * wide : 16; }

// Workgroups of the prefixes come first, then those of what is behind them.
template <int TYPE, int DIM, int WIDE>
__global__ __launch_bounds__(kWaves * 64, DIM == 256 ? 1 : 2) void shared_attention_kernel(PagedView v, SharedArgs a) {
    constexpr int kRows = rows_of_wide(WIDE);
    __shared__ union Space {
        SharedSpace<DIM> narrow;
        WideSpace<DIM> wide;
    } space;
    const SharedGroups groups(v, a);
    int block = blockIdx.x;
    const bool of_prefix = block < a.jobs;
    SharedJob job;
    if (of_prefix) {
        // Each group has its tiles for each head and part of its prefix. Those of one head and part are 8 workgroups
        // apart, on one XCD, whose L2 reads its positions once for all; workgroups without work come behind all
        // others (between them, they left half of the CUs with twice the work: 65000 positions took 205 us, not 110).
        int before = 0, g = -1, tiles = 0, index = 0, group_rows = 0, most = 0;
        for (int g0 = 0; g0 < a.groups; g0 += 64) {
            int rows, parts;
            groups.of_lane(g0, rows, parts);
            const int of_lane = (rows + kRows - 1) / kRows;
            const int count = (parts * v.kv_heads + 7) / 8 * 8 * of_lane, upto = before + scan_lanes(count);
            const unsigned long long hit = __ballot(upto > block);
            if (hit) {
                const int at = __ffsll(hit) - 1;
                g = g0 + at;
                tiles = __builtin_amdgcn_readlane(of_lane, at);
                index = block - __builtin_amdgcn_readlane(upto - count, at);
                most = __builtin_amdgcn_readlane(parts, at);
                group_rows = __builtin_amdgcn_readlane(rows, at);
                break;
            }
            before = __builtin_amdgcn_readlane(upto, 63);
        }
        if (g < 0 || index < 0 || tiles <= 0 || most <= 0) return;  // (the last three only where offsets fall)
        const int of_eight = index / (8 * tiles), within = index - of_eight * 8 * tiles;
        const int pair = of_eight * 8 + (within & 7);
        // Tiles of equal size, of whole 16 rows.
        const int tile_rows = (group_rows + 16 * tiles - 1) / (16 * tiles) * 16;
        job.row0 = (within >> 3) * tile_rows;
        job.head = pair / most;
        index = pair - job.head * most;
        if (job.head >= v.kv_heads) return;
        const int prefix = groups.prefix(g, job.s);
        if (job.s >= v.sequences) return;
        job.first = a.row_of(v, groups.first(g));
        job.rows = min(group_rows, job.row0 + tile_rows);
        if (job.row0 >= job.rows) return;
        job.from = index * a.part;
        if (job.from >= prefix) return;
        job.to = index == a.parts - 1 ? prefix : min(prefix, job.from + a.part);
        job.sees = 0;
        job.slot = index;
        if constexpr (WIDE)
            shared_attend_wide<TYPE, DIM, WIDE>(v, a, job, space.wide);
        else
            shared_attend<TYPE, DIM, false>(v, a, job, space.narrow);
    } else {
        block -= a.jobs;
        if (block >= a.rest_jobs) return;
        int at = block, parts = 0, index = 0, of_head = 0;
        if (a.compact) {
            // A head's tiles and parts, one sequence after the other, so that no workgroup between others is without
            // work: up to 256 sequences' are counted by every wave, 64 at a time, for the head and then the place.
            int counts[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                counts[c] = 0;
                const int s = 64 * c + groups.lane;
                if (64 * c >= v.sequences) continue;
                int row;
                const int n = v.new_rows(min(s, v.sequences - 1), row), positions = v.length(min(s, v.sequences - 1));
                const int of = groups.rest_parts(positions, n, groups.nominal_of_lane(s));
                // (The launch has workgroups for no more sequences than there are rows.)
                int there, past;
                v.existing(row, n, there, past);
                if (s < v.sequences && there < past) counts[c] = of * ((n * a.group + 15) / 16);
                of_head += __builtin_amdgcn_readlane(scan_lanes(counts[c]), 63);
            }
            if (!of_head) return;
            job.head = at / of_head;
            if (job.head >= v.kv_heads) return;
            at -= job.head * of_head;
            job.s = -1;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int upto = scan_lanes(counts[c]);
                const unsigned long long hit = __ballot(upto > at);
                if (job.s < 0 && hit) {
                    const int lane = __ffsll(hit) - 1;
                    job.s = 64 * c + lane;
                    at -= __builtin_amdgcn_readlane(upto - counts[c], lane);
                } else if (job.s < 0) {
                    at -= __builtin_amdgcn_readlane(upto, 63);
                }
            }
        } else {
            // First parts first: of ragged lengths, the last parts are those that some sequences do not have.
            job.row0 = at % a.rest_tiles * 16;
            at /= a.rest_tiles;
            job.s = at % v.sequences;
            at /= v.sequences;
            job.head = at % v.kv_heads;
            index = at / v.kv_heads;
        }
        const int n = v.new_rows(job.s, job.first), length = v.length(job.s), g = groups.of(job.s);
        parts = groups.rest_parts(length, n, groups.nominal(g));
        job.rows = n * a.group;
        if (a.compact) {
            index = at % parts;
            job.row0 = at / parts * 16;
        }
        if (job.row0 >= job.rows || index >= parts) return;
        int reads;
        const int prefix = groups.prefix(g, reads);
        job.from = prefix + index * a.rest_part;
        job.to = index == parts - 1 ? length : min(length, job.from + a.rest_part);
        job.sees = length - n + 1;
        job.slot = a.parts + index;
        shared_attend<TYPE, DIM, true>(v, a, job, space.narrow);
    }
}

// A new row's parts: those of its group's prefix, then those behind it, by
// their references. A workgroup has 256 channels of a row, a lane four of
// them, and each of its waves every fourth part: 4.2 us for 8 rows, 7 for 64
// rows of 33 parts (17 MB), 10.5 for 240 of up to seven.
constexpr int kJoinItems = 64;  // of four channels
template <int DIM>
__global__ __launch_bounds__(kWaves * 64) void shared_join_kernel(PagedView v, SharedArgs a) {
    __shared__ float4_t sums[kWaves][kJoinItems];
    __shared__ float2 states[kWaves][kJoinItems];
    const SharedGroups groups(v, a);
    const int row = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int s = v.sequence_of(row, lane);
    if (s < 0) return;
    int first, reads;
    const int n = v.new_rows(s, first);
    // (first may be as low as -2^31, and above the row where offsets fall)
    if (const int64_t rank = int64_t(row) - first; rank < 0 || rank >= n) return;
    const int g = groups.of(s), shared = a.parts_of(groups.prefix(g, reads), a.part, a.parts);
    const int count = shared + groups.rest_parts(v.length(s), n, groups.nominal(g));
    for (int piece = blockIdx.y; piece * kJoinItems < a.query_heads * (DIM / 4); piece += gridDim.y) {
        const int item = piece * kJoinItems + lane, head = min(item / (DIM / 4), a.query_heads - 1);
        const int channel = 4 * (item % (DIM / 4));
        float top = -kInf, all = 0.f;
        float4_t o = {0.f, 0.f, 0.f, 0.f};
        constexpr int kFlight = 8;  // parts whose sums are loaded at a time
        for (int p0 = wave; p0 < count; p0 += kFlight * kWaves) {
            float2 state[kFlight];
            float4_t x[kFlight];
#pragma unroll
            for (int p = 0; p < kFlight; ++p) {
                const int index = min(p0 + p * kWaves, count - 1);
                const int64_t from = a.place(v, index < shared ? index : a.parts + index - shared, row, head);
                state[p] = a.states[from];
                x[p] = *reinterpret_cast<const float4_t*>(a.sums + from * DIM + channel);
            }
            float grown = top;
#pragma unroll
            for (int p = 0; p < kFlight; ++p) grown = fmaxf(grown, state[p].x);
            const float shrink = top == grown ? 1.f : exp2_fast(top - grown);
            top = grown;
            all *= shrink;
            o *= shrink;
#pragma unroll
            for (int p = 0; p < kFlight; ++p) {
                if (p0 + p * kWaves >= count) continue;
                const float by = state[p].x == top ? 1.f : exp2_fast(state[p].x - top);
                all = __builtin_fmaf(state[p].y, by, all);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(x[p][e], by, o[e]);
            }
        }
        states[wave][lane] = float2{top, all};
        sums[wave][lane] = o;
        __syncthreads();
        if (wave == 0 && item < a.query_heads * (DIM / 4)) {
#pragma unroll
            for (int w = 1; w < kWaves; ++w) top = fmaxf(top, states[w][lane].x);
            all = 0.f;
            o = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const float2 state = states[w][lane];
                const float by = state.x == top ? 1.f : exp2_fast(state.x - top);
                all = __builtin_fmaf(state.y, by, all);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(sums[w][lane][e], by, o[e]);
            }
            o = all == 0.f ? float4_t{0.f, 0.f, 0.f, 0.f} : o * (1.f / all);
            *reinterpret_cast<float4_a4*>(a.out + row * a.out_stride + item * 4) = o;
        }
        __syncthreads();  // LDS is written anew
    }
}

// The sums behind the prefixes take 256 MiB at most, which the last level of
// the caches holds, or one part's. 2048 new rows of 32 heads of 128 that may
// have 32768 positions behind their prefix take 827 us with 260 MiB in all,
// 1457 with parts of 640 and 1.7 GB; 64 sequences of 4 rows that may have 131072
// 430 us with 252 MiB, 426 with 837.
constexpr int64_t kRestBytes = int64_t(1) << 28;

// Sizes of a call: how its work is split, and what its workspace holds.
struct SharedPlan {
    int wide;
    bool compact;
    int64_t tiles, rest_tiles, parts, rest_parts, part, rest_part, jobs, rest_jobs, slots;
    size_t sum_bytes, state_bytes;
    SharedPlan(const qwen_gpu_paged_cache& c, const qwen_gpu_paged_batch& b, const qwen_gpu_paged_prefix& p,
               int query_heads) {
        const int64_t group = query_heads / c.kv_heads, rows = group * b.total_rows;
        const int64_t of_group = rows / p.groups;  // a group has as many of them if all have the same
        // (16 query rows behind 8192 positions: 20.3 us, or 21 as a wide tile; 24 of them 26.4, or 21.5; E4M3 17.7 or 20.5,
        // and 23.5 or 21.5.)
        wide = of_group <= 16 ? 0 : c.head_dim == 256 ? 1 : 2;
        const int64_t tile = rows_of_wide(wide);
        tiles = (rows + p.groups * (tile - 1)) / tile;  // however the groups share them
        rest_tiles = (group * b.rows + 15) / 16;
        // Parts for as many workgroups as the GPU holds at once, half of that where each has 16 query rows, which is one a
        // CU (8 sequences behind 512 positions 19.4 us, 20.3 with two, 4 with up to 3000 more 25.1 and 29.7), of 256
        // positions or more (two sequences behind 4000 14.2 us, of 128 16.1, of 512 17.5), and of 640 at most behind the
        // prefixes, where ragged lengths would keep a few workgroups long (64 sequences of up to 3000 90 us, with 1024 98,
        // without 122; 4 times 24 of up to 1500 100, 99 and 114).
        const int64_t held = c.head_dim == 256 ? 256 : 512;
        auto split = [&](int64_t units, int64_t places, int64_t positions, int64_t shortest, int64_t longest, int64_t step,
                         int64_t& count, int64_t& size) {
            const int64_t most = std::max<int64_t>(1, (positions + shortest - 1) / shortest);
            const int64_t least = std::max<int64_t>(1, (positions + longest - 1) / longest);
            count = std::clamp<int64_t>(places / std::max<int64_t>(1, units), least, most);
            size = (positions + count - 1) / count;
            size = std::max<int64_t>(step, (size + step - 1) / step * step);
            count = std::max<int64_t>(1, (positions + size - 1) / size);
        };
        // (A sequence has a row at least where it has work.)
        const int64_t working = std::min<int64_t>(b.sequences, b.total_rows), units = rest_tiles * working * c.kv_heads;
        // Parts of 640 only while their sums, which every row has for every part, fit kRestBytes.
        const int64_t row_bytes = int64_t(query_heads) * (c.head_dim * 4 + 8);
        const int64_t room = std::max<int64_t>(1, kRestBytes / std::max<int64_t>(1, b.total_rows * row_bytes));
        const int64_t longest = std::max<int64_t>(640, (p.max_rest + room - 1) / room);
        split(units, 256, p.max_rest, 256, longest, kBlock, rest_parts, rest_part);
        // The prefixes have as many of the places as their share of the work, and a third more, so that none of their
        // workgroups is the last one: 85 ns a position of theirs, 65 (E4M3 45) behind them, where half of the most are
        // taken for ragged ones' mean. (All places, as if there were nothing behind them: 4 times 24 sequences 120 us,
        // not 98, as each workgroup of theirs has its start and its sums.)
        const int64_t of_prefixes = std::max<int64_t>(1, tiles) * c.kv_heads;
        const double ahead = double(of_prefixes) * p.max_length * (c.type == kPagedE4M3 ? 85. / 45 : 85. / 65);
        const double share = ahead / (ahead + double(units) * p.max_rest / 2 + 1);
        const int64_t places = std::min(held, int64_t(held * 4 / 3 * share) + of_prefixes - 1);
        // Wide tiles' workgroups go 32 positions a step (64 with heads of 64) and may be short, up to 128 parts: 14
        // sequences of 16 query heads on one KV head behind 3616 positions 18 us, of 256 positions at least 25; with 503
        // parts of 60000 positions instead of 235 44 us, not 36.
        if (wide)
            split(of_prefixes, places, p.max_length, std::clamp<int64_t>(p.max_length / 128, 64, 256), kPagedMaxLength,
                  c.head_dim == 64 ? 64 : 32, parts, part);
        else  // a workgroup a CU: 8 sequences behind 16000 positions 22.8 us, with two 27.8, behind 60000 54 and 56
            split(of_prefixes, std::min<int64_t>(places, 256), p.max_length, 256, kPagedMaxLength, kBlock, parts, part);
        jobs = p.max_length ? (parts * c.kv_heads + 7) / 8 * 8 * tiles : 0;
        rest_jobs = rest_parts * rest_tiles * b.sequences * c.kv_heads;
        // Where all workgroups start at once, those without work cost nothing; where they do not, 4 times 24 ragged
        // sequences take 127 us with them, 116 without.
        compact = b.sequences <= 256 && p.groups < 64 && rest_jobs > held;
        if (compact) rest_jobs = rest_parts * units;
        slots = parts + rest_parts;
        state_bytes = (size_t(slots) * b.total_rows * query_heads * 8 + 15) / 16 * 16;
        sum_bytes = size_t(slots) * b.total_rows * query_heads * c.head_dim * 4;
    }
    int64_t groups() const { return jobs + (rest_jobs + 7) / 8 * 8; }
    size_t bytes() const { return sum_bytes + state_bytes; }
};

template <int TYPE, int DIM, int WIDE>
void shared_run(const PagedView& v, const SharedArgs& a, const SharedPlan& plan, hipStream_t stream) {
    shared_attention_kernel<TYPE, DIM, WIDE>
        <<<unsigned(plan.groups()), kWaves * 64, 0, stream>>>(v, a);
}

template <int TYPE>
void shared_launch(int dim, const PagedView& v, const SharedArgs& a, const SharedPlan& plan, hipStream_t stream) {
    auto run = [&](auto of_dim) {
        constexpr int kDim = decltype(of_dim)::value;
        if (plan.wide == 0) return shared_run<TYPE, kDim, 0>(v, a, plan, stream);
        shared_run<TYPE, kDim, kDim == 256 ? 1 : 2>(v, a, plan, stream);
    };
    if (dim == 64) return run(std::integral_constant<int, 64>{});
    if (dim == 128) return run(std::integral_constant<int, 128>{});
    run(std::integral_constant<int, 256>{});
}

}  // namespace qwen_hip

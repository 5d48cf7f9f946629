// Attention of new rows over a paged key-value cache: the kernel and its launch,
// included by one source for each type of cache (they compile side by side).
#pragma once
#include <algorithm>
#include <type_traits>

#include "decode_dev.hpp"
#include "paged_dev.hpp"

namespace qwen_hip {

constexpr int kTile = 32;                       // positions of a wave's step
constexpr int kWaves = 4;                       // of a workgroup
constexpr int kBlock = kTile * kWaves;          // positions of a workgroup's step
// Workgroups that the positions are dealt to: as many as the GPU holds at once, two for each CU, one where heads of
// 256 take the registers of two.
__host__ __device__ constexpr int shares_of(int dim) { return dim == 256 ? 256 : 512; }
constexpr int kStream = 4;                      // blocks a share from which on workgroups cross units
constexpr int kAdds = 2;                        // turns that a unit's last workgroup takes to add to the weights
constexpr int kCounterStep = 16;                // ints: a counter has a line of its own
constexpr float kInf = __builtin_huge_valf();
// More grid rows than shares split no unit, up to there a row has shares / rows + 1 counters.
static_assert(2 * shares_of(64) * kCounterStep * sizeof(int) <= kPagedCounterBytes, "counters");

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef short short4_t __attribute__((ext_vector_type(4)));

struct AttentionArgs {
    const float* queries;
    int64_t query_stride;
    float* out;
    int64_t out_stride;
    int group;          // query heads of a KV head
    unsigned magic;     // of the group, as page_slot takes it
    int extra, pitch;   // counters and partials of a row of the grid
    int tiles;          // of a KV head's query rows: grid row y has head y / tiles, tile y % tiles
    float scale;        // times log2(e)
    float* partials;    // [parts][rows of a tile][DIM + 4]: output, reference, sum, the same of a group of parts
    int* counters;      // kCounterStep apart, 0 between launches
    bool adds;          // tracked: the attention adds to the weights itself
    float2* states;     // tracked, not so: [kv_heads][total_rows * group]: reference, 1 / sum
    float* scores;      // tracked: [kv_heads][total_rows * group][score_stride]
    int64_t score_stride;

    // Of a KV head's query row, the new row that it belongs to.
    __device__ __forceinline__ int new_row(int r) const { return page_slot(r, group, magic).page; }
    // Where query row 0 of a KV head and a sequence whose new rows begin at `first` has its state and scores. They
    // lie by new rows, not by sequences: those of a batch may have very different numbers of them.
    __device__ __forceinline__ int64_t tracked(const PagedView& v, int head, int first) const {
        return (int64_t(head) * v.total_rows + first) * group;
    }
};

// How the positions are dealt. A unit is a sequence, a KV head and a tile of its
// query rows; it has `blocks` blocks of 128 positions (one at least, so that
// rows without positions are written too). Row blockIdx.y of the grid has a head
// and a tile, so the tiles of a head's rows take the same positions at the same
// time. Workgroups find their shares from the lengths on the device, every wave
// by itself, so the host needs no lengths and a captured launch follows them.
// With up to 4 blocks a share, a workgroup has one part of one unit, of 1, 2 or
// 4 blocks, whichever spreads all over as many workgroups as the GPU holds at
// once. With more, that many workgroups take equal runs of blocks
// in the order of a grid row's units, across their borders: with parts of units
// the last round of workgroups left CUs idle (5% for 64 sequences of 1 to 4096
// positions, BF16). With 768, 1024 and 1536 runs these take 120, 114 and 116 us
// where 512 take 110, and 64 equal ones of 2048 (FP16) 118, 104 and 111 where
// 512 take 96.
// Ragged new rows leave a head's later tiles fewer units, so that some rows of a
// grid may take runs and others parts: a row's counters and partials lie at the
// same place for both.
struct Deal {
    int length, n, first, blocks;  // of a sequence: positions, new rows, the first of them, blocks (0: no unit)
};
struct Share {
    Deal d;
    int s;
    int from, to;             // blocks of the unit
    int parts, part;          // of the unit; part p's sums lie at part0 (p = 0), part1 + (p - 1) * step
    int part0, part1, step;
    int counter;              // the first of parts - 1 that are the unit's own

    __device__ __forceinline__ int64_t slot(int p) const { return p == 0 ? part0 : part1 + (p - 1) * step; }
};
template <int ROWS>
__device__ __forceinline__ Deal deal_one(const PagedView& v, int group, int tile, int s) {
    Deal d;
    d.length = v.length(s);
    d.n = v.new_rows(s, d.first);
    d.blocks = tile * ROWS < group * d.n ? max(1, (d.length + kBlock - 1) / kBlock) : 0;
    return d;
}
__device__ __forceinline__ Deal deal_of_lane(const Deal& d, int lane) {
    return {__builtin_amdgcn_readlane(d.length, lane), __builtin_amdgcn_readlane(d.n, lane),
            __builtin_amdgcn_readlane(d.first, lane), __builtin_amdgcn_readlane(d.blocks, lane)};
}
// Runs of a row of the grid.
__host__ __device__ __forceinline__ int runs_of_row(int shares, int grid_rows) {
    return shares > grid_rows ? shares / grid_rows : 1;
}

// Of 64 sequences' units in a row of the grid: their parts of 1, 2 and 4 blocks
// (the first are their blocks as well), and their number.
struct ChunkSums {
    int of[4][64];
};

// The host has checked that all units' blocks together fit 31 bits.
template <int ROWS, int SHARES>
struct Dealer {
    const PagedView& v;
    const AttentionArgs& a;
    const ChunkSums& chunks;
    const int lane, w, tile;
    Deal own;     // up to 64 sequences: of sequence `lane`
    int total;    // blocks of the grid row's units
    int runs;     // of the grid row
    int shift;    // parts have 2^shift blocks
    int at, end;  // blocks of this workgroup's run
    bool streams;

    static __device__ __forceinline__ int parts_of(int blocks, int shift) {
        return (blocks + (1 << shift) - 1) >> shift;
    }

    __device__ __forceinline__ Dealer(const PagedView& view, const AttentionArgs& args, ChunkSums& shared,
                                      int rows_tile)
        : v(view), a(args), chunks(shared), lane(threadIdx.x & 63), w(blockIdx.z * gridDim.x + blockIdx.x),
          tile(rows_tile), own{}, runs(runs_of_row(SHARES, gridDim.y)) {
        if (v.sequences <= 64) {
            if (lane < v.sequences) own = deal_one<ROWS>(v, a.group, tile, lane);
            total = v.sequences == 1 ? __builtin_amdgcn_readfirstlane(own.blocks)
                                     : __builtin_amdgcn_readlane(scan_lanes(own.blocks), 63);
        } else {
            // The waves sum 64 sequences each in turn, with four turns' loads in flight.
            for (int c0 = threadIdx.x >> 6; c0 < 64; c0 += 4 * kWaves) {
                Deal d[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int s = (c0 + i * kWaves) * 64 + lane;
                    d[i] = deal_one<ROWS>(v, a.group, tile, min(s, v.sequences - 1));
                    if (s >= v.sequences) d[i].blocks = 0;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int sum = scan_lanes(k < 3 ? parts_of(d[i].blocks, k) : d[i].blocks > 0);
                        if (lane == 63) shared.of[k][c0 + i * kWaves] = sum;
                    }
                if ((c0 + 4 * kWaves) * 64 >= v.sequences) {  // the rest of the wave's sums are 0
                    for (int c = c0 + 4 * kWaves + kWaves * lane; c < 64; c += 64 * kWaves)
                        for (int k = 0; k < 4; ++k) shared.of[k][c] = 0;
                    break;
                }
            }
            __syncthreads();
            total = __builtin_amdgcn_readlane(scan_lanes(chunks.of[0][lane]), 63);
        }
        const int all = total * int(gridDim.y);
        streams = all > kStream * SHARES;
        shift = all <= SHARES ? 0 : all <= 2 * SHARES ? 1 : 2;
        static_assert(kStream == 4, "parts of 1, 2 or 4 blocks");
        at = end = 0;
        if (streams) {
            at = start(w);
            end = start(w + 1);
        }
    }
    __device__ __forceinline__ int start(int run) const {
        const int even = total / runs;
        return run >= runs ? total : run * even + min(run, total - runs * even);
    }
    __device__ __forceinline__ int owner(int block) const {
        const int even = total / runs, more = total - runs * even;
        const int longer = more * (even + 1);
        return block < longer ? block / (even + 1) : more + (block - longer) / even;
    }
    // This workgroup's next share, if it has one.
    __device__ __forceinline__ bool next(Share& share) {
        if (streams && at >= end) return false;
        const int wanted = streams ? at : w, row = blockIdx.y, split_shift = streams ? 0 : shift;
        int begin = 0, before = 0, known = 0;  // sequences, blocks or workgroups, and units, of the chunks before
        Deal d = own;
        if (v.sequences > 64) {
            const int count = chunks.of[split_shift][lane], upto = scan_lanes(count);
            const unsigned long long hit = __ballot(upto > wanted);
            if (!hit) return false;
            const int chunk = __ffsll(hit) - 1, units = chunks.of[3][lane];
            begin = 64 * chunk;
            before = __builtin_amdgcn_readlane(upto - count, chunk);
            known = __builtin_amdgcn_readlane(scan_lanes(units) - units, chunk);
            d = deal_one<ROWS>(v, a.group, tile, min(begin + lane, v.sequences - 1));
            if (begin + lane >= v.sequences) d.blocks = 0;
        }
        const int count = parts_of(d.blocks, split_shift), upto = v.sequences == 1 ? count : scan_lanes(count);
        const unsigned long long hit = __ballot(before + upto > wanted);
        if (!hit) return false;
        const int from = __ffsll(hit) - 1;
        // Units before the sequence's: all sequences where each has the same new rows.
        const int units =
            v.offsets ? known + __popcll(__ballot(d.blocks > 0) & ((1ull << from) - 1)) : begin + from;
        share.s = begin + from;
        share.d = d = deal_of_lane(d, from);
        const int within = wanted - before - __builtin_amdgcn_readlane(upto - count, from);
        if (streams) {
            share.from = within;
            share.to = min(d.blocks, share.from + end - at);
            const int first = owner(at - share.from), last = owner(at - share.from + d.blocks - 1);
            share.parts = last - first + 1;
            // A run's last share comes second; its first one is the end of another unit.
            share.part0 = row * a.pitch + 2 * first + 1;
            share.part1 = row * a.pitch + 2 * (first + 1);
            share.step = 2;
            share.part = w - first;
            // No other unit starts in these runs, but for the last, and ends behind its own first.
            share.counter = row * a.extra + first;
            at += share.to - share.from;
        } else {
            share.from = within << shift;
            share.to = min(d.blocks, (within + 1) << shift);
            share.parts = __builtin_amdgcn_readlane(count, from);
            share.part = within;
            share.part0 = row * a.pitch + w - within;
            share.part1 = share.part0 + 1;
            share.step = 1;
            // A grid row's units have fewer than shares / rows parts beyond one each: these are counted.
            share.counter = row * a.extra + w - within - units;
        }
        return true;
    }
};

// Values that other workgroups of the launch read, on other XCDs too: stores
// and loads that pass by the caches of one XCD.
__device__ __forceinline__ void post(float* p, float a, float b) {
    const uint64_t w = __builtin_bit_cast(unsigned, a) | uint64_t(__builtin_bit_cast(unsigned, b)) << 32;
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void posted_stores_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ float2 posted(const float* p) {
    const uint64_t w =
        __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return float2{__builtin_bit_cast(float, unsigned(w)), __builtin_bit_cast(float, unsigned(w >> 32))};
}

// ds_read_b64_tr_b16: within each 16-lane group, lane 4a + b receives element
// b of the 8-byte chunks addressed by lanes a, a + 4, a + 8 and a + 12.
__device__ __forceinline__ short4_t read_transposed(const char* p) {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef __attribute__((address_space(3))) short4_t lds_short4;
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(__attribute__((address_space(3))) char*)(p));
#else
    (void)p;
    return short4_t{};
#endif
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ float4_t multiply(uint4_t a, uint4_t b, float4_t c, std::integral_constant<int, kPagedF16>) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0,
                                                  0);
}
template <int TYPE>
__device__ __forceinline__ float4_t multiply(uint4_t a, uint4_t b, float4_t c, std::integral_constant<int, TYPE>) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
}

// FP32 values as sums of 16-bit ones, for products on the matrix cores: three
// BF16 terms hold them (two, 2^-17 off, would lose ten times what the sums do),
// two FP16 terms all but a quarter of them, which are one unit of FP32's last
// place off, as after one addition (with a third one 8 sequences of 2048 are as
// far from 64 bits, 4.6e-7, and take 18.4 us instead of 17.8). A product has 16 columns. Up to 8 query rows are
// packed: columns 0-7 take the first term and 8-15 the second, the halves of
// the result are added, and a third term takes a second product with columns
// 8-15 empty. More rows take a column each and a product for every term (16
// rows as two packed tiles took 132 us for 16 sequences of 8192, so 105; BF16
// 172 and 105). E4M3 rows become BF16 as they are read, with their power of
// two: exact, but that of what lies below 2^-126 multiples of 2^-133 are left.
template <int TYPE, bool PACKED>
struct Terms {
    static constexpr int kTerms = TYPE == kPagedF16 ? 2 : 3, kProducts = PACKED ? kTerms - 1 : kTerms;
    // Two values; `second`: this lane's column is one of 8-15.
    static __device__ __forceinline__ void split(float a, float b, bool second, unsigned (&out)[kProducts]) {
        unsigned term[kTerms];
        if constexpr (TYPE == kPagedF16) {
            _Float16 ha, la, hb, lb;
            split_half(a, ha, la);
            split_half(b, hb, lb);
            if constexpr (PACKED) {
                const _Float16 x = second ? la : ha, y = second ? lb : hb;
                out[0] = __builtin_bit_cast(uint16_t, x) | unsigned(__builtin_bit_cast(uint16_t, y)) << 16;
                return;
            }
            term[0] = __builtin_bit_cast(uint16_t, ha) | unsigned(__builtin_bit_cast(uint16_t, hb)) << 16;
            term[1] = __builtin_bit_cast(uint16_t, la) | unsigned(__builtin_bit_cast(uint16_t, lb)) << 16;
        } else {
#pragma unroll
            for (int t = 0; t < 3; ++t) {
                a = fp32_fixed(a);
                b = fp32_fixed(b);
                term[t] = pack_bf16(a, b);
                a -= __builtin_bit_cast(float, term[t] << 16);
                b -= __builtin_bit_cast(float, term[t] & 0xffff0000u);
            }
        }
        if constexpr (PACKED) {
            out[0] = second ? term[1] : term[0];
            if constexpr (kProducts == 2) out[1] = second ? 0u : term[2];
        } else {
#pragma unroll
            for (int t = 0; t < kTerms; ++t) out[t] = term[t];
        }
    }
};

// 16 bytes of a stored row as 16-bit operands: one of 8, or two (E4M3).
template <int TYPE>
__device__ __forceinline__ void widen(uint4_t raw, float up, uint4_t (&out)[TYPE == kPagedE4M3 ? 2 : 1]) {
    if constexpr (TYPE != kPagedE4M3) {
        out[0] = raw;
    } else {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            out[w / 2][2 * (w % 2)] =
                __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(raw[w], up, false));
            out[w / 2][2 * (w % 2) + 1] =
                __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(raw[w], up, true));
        }
    }
}

// The sign bits of those of a word's two 16-bit values that are infinite or NaN.
template <bool HALF>
__device__ __forceinline__ unsigned not_finite(unsigned w) {
    if constexpr (HALF) return ((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
    return ((w & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
}

template <int TYPE>
__device__ __forceinline__ float stored(const char* row, int i, float up) {
    if constexpr (TYPE == kPagedF16) {
        return float(reinterpret_cast<const _Float16*>(row)[i]);
    } else if constexpr (TYPE == kPagedBF16) {
        return __builtin_bit_cast(float, unsigned(reinterpret_cast<const uint16_t*>(row)[i]) << 16);
    } else {
        return float(__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(reinterpret_cast<const uint8_t*>(row)[i], up, false)[0]);
    }
}

// Lanes l and l ^ 8 of each 16: the sum of both halves in both.
__device__ __forceinline__ float add_halves(float x) {
    const int other = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), 0x128, 0xF, 0xF, true);  // row_ror:8
    return x + __builtin_bit_cast(float, other);
}

// S^T = K Q^T and O^T = V^T P^T on the matrix cores, 32 positions a step, each
// wave with its own online softmax over every fourth step of the workgroup's
// positions; the waves are added at the end. A lane holds row l % 16 of each
// 16 positions, pieces l / 16, l / 16 + 4, ... of 16 bytes: the A operand of
// S^T as it comes from memory. S^T leaves lane l with column l % 16 and
// positions 4 (l / 16) .. + 3 of each 16, which is the B operand of O^T when
// V^T's columns are taken in that order, so weights never change lanes. V
// goes through LDS (each wave its own 32 rows) and comes back transposed; a
// row's pitch is 32 bytes more than its values, so that the 16 rows of a read
// fall on all banks twice.
//
// Memory bounds long calls (a step's products take a tenth of the time in which
// HBM delivers its 16 KiB), so the loads of the next step are in flight all the
// time: keys are loaded again as soon as the scores have been multiplied, values
// as soon as they are in LDS, and a step's table entries ahead of the values
// before it, so that no wait for one covers the other. 64 sequences of 2048
// positions (FP16, 537 MB) take 96 us, 5.6 TB/s, where a copy of 1 GiB runs at
// 5.1; 200 VGPRs and more leave two waves a SIMD (three, with 107 spilled
// registers and 768 runs, take 201 us for 64 ragged BF16 sequences instead of 110).
// Latency bounds short ones: 300 positions take 9 us in the kernel, 1.3 to find
// the share, 2.2 for the table and the first rows behind it, 1.2 for a step, 1.7
// for the waves' sums, 2 for the last workgroup to add the parts.
template <int TYPE, int DIM, bool PACKED, bool TRACK>
__global__ __launch_bounds__(kWaves * 64, DIM == 256 ? 1 : 2) void paged_attention_kernel(PagedView v,
                                                                                          AttentionArgs a) {
    constexpr int kSize = TYPE == kPagedE4M3 ? 1 : 2, kLoads = DIM * kSize / 64, kSteps = DIM / 32, kOut = DIM / 16;
    constexpr int kPer = kSteps / kLoads;         // products per load: 1, or 2 for E4M3
    constexpr int kRows = PACKED ? 8 : 16, kProducts = Terms<TYPE, PACKED>::kProducts;
    constexpr int kPitch = DIM * 2 + 32;          // bytes of a value row in LDS
    constexpr float kHead = TYPE == kPagedF16 ? 6.f : 0.f;  // FP16 weights are kept up to 2^14, far from subnormals
    constexpr int kJoin = PACKED ? 16 : 8;        // parts whose sums are loaded at a time, as registers allow
    constexpr int kFlat = PACKED ? 32 : 16;       // parts that are added at once, beyond in groups of kJoin
    constexpr float kGrow = 8.f;                  // a reference is moved once a score passes it by 2^8
    constexpr std::integral_constant<int, TYPE> kType{};
    __shared__ __attribute__((aligned(16))) char lds[kWaves][kTile * kPitch];
    __shared__ float2 wave_state[kWaves][kRows], row_state[TRACK ? kRows : 1];
    __shared__ ChunkSums chunks;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int column = lane & 15, part = lane >> 4;
    const bool second = PACKED && column >= 8;
    const int row_of_lane = PACKED ? column & 7 : column;

    const int head = a.tiles == 1 ? blockIdx.y : blockIdx.y / unsigned(a.tiles), tile = blockIdx.y - head * a.tiles;
    const int row0 = tile * kRows;
    Dealer<kRows, shares_of(DIM)> dealer(v, a, chunks, tile);
    Share share;
    while (dealer.next(share)) {
        const Deal& d = share.d;
        const int begin = kBlock * share.from, query_rows = a.group * d.n;
        // Positions from shared_end on are seen by some of the tile's new rows only, from `end` on by none.
        const int shared_end = d.length - d.n + a.new_row(row0) + 1;
        const int seen_end = d.length - d.n + min(d.n - 1, a.new_row(row0 + kRows - 1)) + 1;
        const int end = min(seen_end, kBlock * share.to);
        const int32_t* const table = v.table + int64_t(share.s) * v.table_stride;

        float4_t acc[kOut];
        float reference = -kInf, sum = 0.f;
#pragma unroll
        for (int o = 0; o < kOut; ++o) acc[o] = float4_t{0.f, 0.f, 0.f, 0.f};

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
                at[u] = v.row_at(page, head, slots[u]) + 16 * part;
                if constexpr (TYPE == kPagedE4M3)
                    bytes[u] = *reinterpret_cast<const uint16_t*>(v.exponents + v.exponents_at(page, head, slots[u]));
            }
        };
        auto load = [&](const char* pool, uint4_t (&to)[2][kLoads]) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < kLoads; ++i) to[u][i] = *reinterpret_cast<const uint4_t*>(pool + at[u] + 64 * i);
        };
        char* const mine = lds[wave];
        const char* const transposed = mine + (4 * part + (column >> 2)) * kPitch + (column & 3) * 8;

        // The table's entries first, queries next, keys and values behind them.
        int base = begin + kTile * wave;
        if (base < end) find(base);
        // Queries: row r of the tile is head r % group of new row r / group.
        uint4_t query[kSteps][kProducts];
        float x[kSteps][8];
        const int query_row = row0 + row_of_lane, new_row = a.new_row(query_row);
        const int64_t row = int64_t(d.first) + new_row;
        const bool live = query_row < query_rows && row >= 0 && row < v.total_rows;
        const int sees = live ? d.length - d.n + new_row + 1 : 0;  // positions the lane's row attends
        {
            const float* const from =
                a.queries + (live ? row * a.query_stride + (head * a.group + query_row - new_row * a.group) * DIM : 0);
#pragma unroll
            for (int k = 0; k < kSteps; ++k) {
                // The channels that this lane's part of a stored row holds in step k.
                const int from_channel = kPer == 1 ? 32 * k + 8 * part : 64 * (k / 2) + 16 * part + 8 * (k % 2);
                const float4_a4 lo = *reinterpret_cast<const float4_a4*>(from + from_channel);
                const float4_a4 hi = *reinterpret_cast<const float4_a4*>(from + from_channel + 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[k][e] = live ? lo[e] : 0.f, x[k][4 + e] = live ? hi[e] : 0.f;
            }
        }
        if (base < end) {
            place(base);
            load(v.keys, keys);
            if (base + kBlock < end) find(base + kBlock);
            load(v.values, values);
        }
        float to_score = a.scale;  // what a product's sum is multiplied by
        if constexpr (TYPE == kPagedF16) {
            // An exact power of two brings a row's largest query to [2^14, 2^15), so
            // that neither term leaves FP16's range. 2^-100 is far below any query that a score depends on;
            // non-finite ones stay so.
            float top = 0.f;
#pragma unroll
            for (int k = 0; k < kSteps; ++k)
#pragma unroll
                for (int e = 0; e < 8; ++e) top = fmaxf(top, __builtin_fabsf(x[k][e]));
            top = fmaxf(top, dev::xor_lanes<16>(top));
            top = fmaxf(top, dev::xor_lanes<32>(top));
            const int up = 14 - max(int(__builtin_bit_cast(unsigned, top) >> 23) - 127, -100);
#pragma unroll
            for (int k = 0; k < kSteps; ++k)
#pragma unroll
                for (int e = 0; e < 8; ++e) x[k][e] *= pow2(up);
            to_score *= pow2(-up);
        }
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                unsigned words[kProducts];
                Terms<TYPE, PACKED>::split(x[k][2 * e], x[k][2 * e + 1], second, words);
#pragma unroll
                for (int p = 0; p < kProducts; ++p) query[k][p][e] = words[p];
            }

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

            float scores[2][4], weights[2][4], high = -kInf;
            unsigned hidden = 0;  // bit 4 u + r
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    scores[u][r] = PACKED ? add_halves(s[u][r]) : s[u][r];
                    high = fmaxf(high, scores[u][r] * to_score);
                }
            if (!whole) {
                high = -kInf;
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int j = 16 * u + 4 * part + r;
                        if (!(exist >> j & 1) || base + j >= sees)
                            hidden |= 1u << (4 * u + r);
                        else
                            high = fmaxf(high, scores[u][r] * to_score);
                    }
            }
            if (__any(high > reference + (kHead + kGrow))) {
                high = fmaxf(high, dev::xor_lanes<16>(high));
                high = fmaxf(high, dev::xor_lanes<32>(high));
                const float moved = fmaxf(reference, high - kHead);
                const float shrink = reference == moved ? 1.f : exp2_fast(reference - moved);
                reference = moved;
                sum *= shrink;
#pragma unroll
                for (int o = 0; o < kOut; ++o) acc[o] *= shrink;
            }
            {
                const float from = reference == -kInf ? 0.f : reference;
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        float p = exp2_fast(__builtin_fmaf(scores[u][r], to_score, -from));
                        if (!whole && (hidden >> (4 * u + r) & 1)) p = 0.f;
                        weights[u][r] = p;
                        sum += p;
                    }
            }
            if constexpr (TRACK) {
                if (!second && live) {
                    const int64_t at_row = a.tracked(v, head, d.first) + query_row;
                    float* const to = a.scores + at_row * a.score_stride + base + 4 * part;
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        float4_t w;
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            w[e] = !whole && (hidden >> (4 * u + e) & 1) ? -kInf : scores[u][e] * to_score;
                        if (a.adds) {
                            post(to + 16 * u, w[0], w[1]);
                            post(to + 16 * u + 2, w[2], w[3]);
                        } else {
                            *reinterpret_cast<float4_t*>(to + 16 * u) = w;
                        }
                    }
                }
            }
            uint4_t weight[kProducts];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                unsigned words[kProducts];
                Terms<TYPE, PACKED>::split(weights[e / 2][2 * (e % 2)], weights[e / 2][2 * (e % 2) + 1], second, words);
#pragma unroll
                for (int p = 0; p < kProducts; ++p) weight[p][e] = words[p];
            }

            // Values into LDS, 0 for those that are not there. A weight of 0 does not keep infinities and NaN
            // out, so those in rows that only some new rows see are 0 here as well, and added below. They are found
            // in the 16-bit words: an E4M3 row's power of two may carry finite codes past what these hold.
            const bool triangle = base + kTile > shared_end;
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
#pragma unroll
            for (int o = 0; o < kOut; ++o) {
                const short4_t low = read_transposed(transposed + 32 * o);
                const short4_t high = read_transposed(transposed + 16 * kPitch + 32 * o);
                const uint4_t w = {__builtin_bit_cast(u32x2, low)[0], __builtin_bit_cast(u32x2, low)[1],
                                   __builtin_bit_cast(u32x2, high)[0], __builtin_bit_cast(u32x2, high)[1]};
#pragma unroll
                for (int p = 0; p < kProducts; ++p) acc[o] = multiply(w, weight[p], acc[o], kType);
            }

            // One row at a time, for the new rows that see it.
            if (spoilt) {
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        for (int q = 0; q < 4; ++q) {
                            const int j = 16 * u + 4 * q + r;
                            if (base + j < shared_end || !(exist >> j & 1)) continue;
                            const int64_t from = __shfl(row_at[u], 4 * q + r);
                            const float up = __shfl(value_up[u], 4 * q + r);
                            const float p = __shfl(weights[u][r], 16 * q + column);
                            if (second || base + j >= sees) continue;
#pragma unroll
                            for (int o = 0; o < kOut; ++o)
#pragma unroll
                                for (int e = 0; e < 4; ++e) {
                                    const float x = stored<TYPE>(v.values + from, 16 * o + 4 * part + e, up);
                                    if (x - x != 0.f) acc[o][e] = __builtin_fmaf(p, x, acc[o][e]);
                                }
                        }
            }
        }

        // The four waves' sums, brought to their largest reference.
        __syncthreads();
        float* const sums = reinterpret_cast<float*>(lds);  // [kWaves][kRows][DIM]
        sum += dev::xor_lanes<16>(sum);
        sum += dev::xor_lanes<32>(sum);
        if (lane < kRows) wave_state[wave][lane] = float2{reference, sum};
#pragma unroll
        for (int o = 0; o < kOut; ++o) {
            float4_t w = acc[o];
            if constexpr (PACKED)
#pragma unroll
                for (int e = 0; e < 4; ++e) w[e] = add_halves(acc[o][e]);
            float* const to = sums + (wave * kRows + row_of_lane) * DIM + 16 * o + 4 * part;
            if (!second) *reinterpret_cast<float4_t*>(to) = w;
        }
        if (TRACK && int(threadIdx.x) < kRows) row_state[threadIdx.x] = float2{0.f, 0.f};
        __syncthreads();
        auto finish = [&](int local, int channel, float4_t o, float top, float all) {
            const int r = row0 + local, i = a.new_row(r);
            const int64_t to = int64_t(d.first) + i;
            if (to < 0 || to >= v.total_rows) return;
            if (all == 0.f) o = float4_t{0.f, 0.f, 0.f, 0.f};
            const float by = all == 0.f ? 0.f : 1.f / all;
            const int64_t at = to * a.out_stride + (head * a.group + r - i * a.group) * DIM + channel;
            *reinterpret_cast<float4_a4*>(a.out + at) = o * by;
            if (TRACK && channel == 0) {
                const float2 state = {top == -kInf ? 0.f : top, by};
                if (a.adds)
                    row_state[local] = state;
                else
                    a.states[a.tracked(v, head, d.first) + r] = state;
            }
        };
        for (int item = threadIdx.x; item < kRows * DIM / 4; item += kWaves * 64) {
            const int local = item / (DIM / 4), channel = 4 * (item - local * (DIM / 4));
            if (row0 + local >= query_rows) continue;
            float top = -kInf, all = 0.f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) top = fmaxf(top, wave_state[w][local].x);
            float4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const float2 state = wave_state[w][local];
                const float shrink = state.x == top ? 1.f : exp2_fast(state.x - top);
                all = __builtin_fmaf(state.y, shrink, all);
                const float4_t x = *reinterpret_cast<const float4_t*>(sums + (w * kRows + local) * DIM + channel);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(x[e], shrink, o[e]);
            }
            if (share.parts > 1) {
                float* const partial = a.partials + (share.slot(share.part) * kRows + local) * (DIM + 4);
                post(partial + channel, o[0], o[1]);
                post(partial + channel + 2, o[2], o[3]);
                if (channel == 0) post(partial + DIM, top, all);
            } else {
                finish(local, channel, o, top, all);
            }
        }
        bool ends = share.parts == 1;  // this is the workgroup that completes the unit
        if (share.parts > 1) {
            // The last of the unit's workgroups to get here adds their parts, in the order of the positions; of more
            // than kFlat parts the last of each kJoin adds those, and the last of these the groups (115 parts of 16
            // rows by one workgroup took 40 us). Posted values have reached memory once their stores are done, and
            // are read past the caches, so no fence of the device's scope is needed: with one in every workgroup (it
            // writes back and drops a whole L2) eight sequences of 2048 took 42 us instead of 16.
            int* const flag = reinterpret_cast<int*>(wave_state);
            auto last_of = [&](int index, int count) {
                posted_stores_done();
                __syncthreads();
                if (threadIdx.x == 0) {
                    int* const counter = a.counters + (share.counter + index) * kCounterStep;
                    const int done = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    if (done == count - 1) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    *flag = done == count - 1;
                }
                __syncthreads();
                return *flag != 0;
            };
            // f(row, channel, sums, reference, sum) of parts first, first + every, ...; their references and sums lie
            // `beside` their sums.
            auto join = [&](int first, int count, int every, int beside, auto f) {
#pragma unroll 1
                for (int item = threadIdx.x; item < kRows * DIM / 4; item += kWaves * 64) {
                    const int local = item / (DIM / 4), channel = 4 * (item - local * (DIM / 4));
                    if (row0 + local >= query_rows) continue;
                    float top = -kInf, all = 0.f;
                    float4_t o = {0.f, 0.f, 0.f, 0.f};
                    for (int p0 = 0; p0 < count; p0 += kJoin) {  // that many parts' loads in flight
                        float2 state[kJoin], low[kJoin], high[kJoin];
#pragma unroll
                        for (int p = 0; p < kJoin; ++p) {
                            const float* const from =
                                a.partials +
                                (share.slot(first + min(p0 + p, count - 1) * every) * kRows + local) * (DIM + 4);
                            state[p] = posted(from + beside);
                            low[p] = posted(from + channel);
                            high[p] = posted(from + channel + 2);
                        }
                        float grown = top;
#pragma unroll
                        for (int p = 0; p < kJoin; ++p) grown = fmaxf(grown, state[p].x);
                        const float shrink = top == grown ? 1.f : exp2_fast(top - grown);
                        top = grown;
                        all *= shrink;
                        o *= shrink;
#pragma unroll
                        for (int p = 0; p < kJoin; ++p) {
                            const float by = state[p].x == top ? 1.f : exp2_fast(state[p].x - top);
                            if (p0 + p < count) {
                                all = __builtin_fmaf(state[p].y, by, all);
                                o[0] = __builtin_fmaf(low[p].x, by, o[0]);
                                o[1] = __builtin_fmaf(low[p].y, by, o[1]);
                                o[2] = __builtin_fmaf(high[p].x, by, o[2]);
                                o[3] = __builtin_fmaf(high[p].y, by, o[3]);
                            }
                        }
                    }
                    f(local, channel, o, top, all);
                }
            };
            if (share.parts <= kFlat) {
                ends = last_of(0, share.parts);
                if (ends) join(0, share.parts, 1, DIM, finish);
            } else {
                const int group = share.part / kJoin, first = group * kJoin;
                const int of_group = min(kJoin, share.parts - first), groups = (share.parts + kJoin - 1) / kJoin;
                ends = last_of(1 + group, of_group);
                if (ends) {
                    // The group's sums take the place of its first part's, which nobody else reads any more; its
                    // reference and sum, which all threads of a row have still to read, go beside those.
                    join(first, of_group, 1, DIM, [&](int local, int channel, float4_t o, float top, float all) {
                        float* const partial = a.partials + (share.slot(first) * kRows + local) * (DIM + 4);
                        post(partial + channel, o[0], o[1]);
                        post(partial + channel + 2, o[2], o[3]);
                        if (channel == 0) post(partial + DIM + 2, top, all);
                    });
                    ends = last_of(0, groups);
                    if (ends) join(0, groups, kJoin, DIM + 2, finish);
                }
            }
        }
        if (TRACK && a.adds && ends) {
            // The unit, which has all of the head's query rows, is done, and all its scores are posted: its slots'
            // weights grow by the rows' softmax, summed in the rows' order.
            if (share.parts == 1) posted_stores_done();
            __syncthreads();
            float* const slots = v.weights + v.track_at(share.s, head);
            const int64_t unit = a.tracked(v, head, d.first);
            int from_row, to_row;
            v.existing(d.first, d.n, from_row, to_row);
            from_row *= a.group, to_row *= a.group;
            for (int j = 4 * int(threadIdx.x); j < d.length; j += 4 * kWaves * 64) {
                float4_t grown = {0.f, 0.f, 0.f, 0.f};
                for (int r0 = from_row; r0 < to_row; r0 += 4) {
                    float2 low[4], high[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const float* const from = a.scores + (unit + min(r0 + q, to_row - 1)) * a.score_stride + j;
                        low[q] = posted(from);
                        high[q] = posted(from + 2);
                    }
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        if (r0 + q >= to_row) continue;
                        const float2 state = row_state[r0 + q];
                        const int seen = state.y == 0.f ? 0 : d.length - d.n + a.new_row(r0 + q) + 1 - j;
                        if (seen > 0) grown[0] += exp2_fast(low[q].x - state.x) * state.y;
                        if (seen > 1) grown[1] += exp2_fast(low[q].y - state.x) * state.y;
                        if (seen > 2) grown[2] += exp2_fast(high[q].x - state.x) * state.y;
                        if (seen > 3) grown[3] += exp2_fast(high[q].y - state.x) * state.y;
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (j + e < d.length) slots[j + e] += grown[e];
            }
        }
        if (!dealer.streams) return;
        __syncthreads();  // LDS is written anew
    }
}

// Sizes of a call: the grid, and what its workspace holds.
struct AttentionPlan {
    bool packed, adds;
    int64_t tiles, grid_rows, blocks, score_stride, score_rows;
    int64_t columns, first, pitch;  // of a grid row: workgroups, those of the first layer, places for partials
    size_t partial_bytes, state_bytes, score_bytes;
    AttentionPlan(const qwen_gpu_paged_cache& c, const qwen_gpu_paged_batch& b, int query_heads) {
        const int64_t rows = int64_t(query_heads / c.kv_heads) * b.rows;
        packed = rows <= 8;
        const int64_t tile_rows = packed ? 8 : 16, most = (b.max_length + kBlock - 1) / kBlock;
        const int64_t row_blocks = b.sequences * most;
        tiles = (rows + tile_rows - 1) / tile_rows;
        grid_rows = tiles * c.kv_heads;
        blocks = row_blocks * grid_rows;
        const int64_t shares = shares_of(c.head_dim), runs = shares > grid_rows ? shares / grid_rows : 1;
        columns = std::min(row_blocks, b.sequences + shares / grid_rows);
        if (blocks > kStream * shares) columns = std::max(columns, runs);
        // Every sequence with new rows has a block, so beyond that many they are dealt in runs.
        if (!b.offsets && b.sequences * c.kv_heads > kStream * shares) columns = runs;
        first = std::min(columns, 2 * runs);
        // Dealt in runs, a grid row has two places for each; dealt in parts, one for each part, and no more parts
        // than blocks, which are then kStream * shares / grid_rows at most. With a share or less for a grid row
        // every unit is one part, which takes none.
        pitch = std::max(columns, blocks > kStream * shares ? 2 * runs : 0);
        pitch = grid_rows < shares ? std::min(pitch, kStream * shares / grid_rows) : 0;
        static_assert(kStream >= 2, "room for two places a run");
        partial_bytes = size_t(pitch) * grid_rows * tile_rows * (c.head_dim + 4) * 4;
        score_stride = (b.max_length + kTile - 1) / kTile * kTile;
        score_rows = int64_t(b.total_rows) * query_heads;
        // The workgroup that completes a unit adds to the weights, four positions a thread and four rows at a time,
        // while that takes it a few turns: 12.2 us for 300 positions against 14.2 with a kernel for it, 19.5 and
        // 20.6 for eight sequences of 1025, but 37.2 and 32.9 for eight of 4096. Where several units share the
        // weights, that kernel adds to them.
        adds = tiles == 1 && (b.max_length + 1023) / 1024 * ((rows + 3) / 4) <= kAdds;
        state_bytes = b.weights ? (size_t(score_rows) * 8 + 15) / 16 * 16 : 0;
        score_bytes = b.weights ? size_t(score_rows) * score_stride * 4 : 0;
    }
    size_t bytes() const { return kPagedCounterBytes + partial_bytes + state_bytes + score_bytes; }
};

template <int TYPE, int DIM, bool PACKED>
void attention_run(const PagedView& v, const AttentionArgs& a, const AttentionPlan& plan, hipStream_t stream) {
    // Heads vary slowest, and some of each head's workgroups that find no work come behind its others (the rest
    // behind all), so that the heads start one after the other: 64 sequences of 2048 in pages of [slot][head] took
    // 109 us with all heads at once (heads fastest, or no idle workgroups between them), so 100; in pages of
    // [head][slot] 96 and 97.
    const unsigned layers = unsigned((plan.columns + plan.first - 1) / plan.first);
    const dim3 grid{unsigned(plan.first), unsigned(plan.grid_rows), layers};
    const dim3 block{kWaves * 64};
    if (v.weights)
        paged_attention_kernel<TYPE, DIM, PACKED, true><<<grid, block, 0, stream>>>(v, a);
    else
        paged_attention_kernel<TYPE, DIM, PACKED, false><<<grid, block, 0, stream>>>(v, a);
}

template <int TYPE>
void attention_launch(int dim, const PagedView& v, const AttentionArgs& a, const AttentionPlan& plan,
                      hipStream_t stream) {
    auto run = [&](auto packed) {
        if (dim == 64) return attention_run<TYPE, 64, packed.value>(v, a, plan, stream);
        if (dim == 128) return attention_run<TYPE, 128, packed.value>(v, a, plan, stream);
        attention_run<TYPE, 256, packed.value>(v, a, plan, stream);
    };
    plan.packed ? run(std::true_type{}) : run(std::false_type{});
}

}  // namespace qwen_hip

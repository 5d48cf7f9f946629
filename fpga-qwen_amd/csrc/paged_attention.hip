// Attention of new rows over a paged key-value cache.
#include <algorithm>
#include <string>

#include "decode_dev.hpp"
#include "paged.hpp"
#include "paged_dev.hpp"
#include "qwen_common.hpp"

namespace qwen_hip {
namespace {

constexpr int kTile = 32;                       // positions of a wave's step
constexpr int kWaves = 4;                       // of a workgroup
constexpr int kBlock = kTile * kWaves;          // positions of a workgroup's step
constexpr int kShares = 512;                    // workgroups that the positions are dealt to
constexpr float kInf = __builtin_huge_valf();

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef short short4_t __attribute__((ext_vector_type(4)));

struct AttentionArgs {
    const float* queries;
    int64_t query_stride;
    float* out;
    int64_t out_stride;
    int group;
    int row_tiles;      // of 8 * TILES query rows, at most, of a KV head
    float scale;        // times log2(e)
    float* partials;    // [workgroups][8 * TILES][DIM + 2]: output, reference, sum
    float* scores;      // tracked: [sequences * kv_heads][rows * group][score_stride]
    int64_t score_stride;
};

// How the positions are dealt. A unit is a sequence, a KV head and a tile of
// its query rows; it has `blocks` blocks of 128 positions (one at least, so
// that rows without positions are written too). All units' blocks together,
// over kShares, is the most that one workgroup takes: units that have more
// are split evenly, so a long sequence among short ones does not hold up the
// launch, and the host needs no lengths. Every wave finds this from the
// lengths by itself: a sum over the sequences, then a running count of
// workgroups.
struct Deal {
    int s, length, n, first, tiles, blocks, splits;
    int offset;  // first workgroup of the sequence
};
template <int ROWS>
__device__ __forceinline__ void deal_one(const PagedView& v, int group, int s, Deal& d) {
    d.s = s;
    d.length = v.length(s);
    d.n = v.new_rows(s, d.first);
    d.tiles = (group * d.n + ROWS - 1) / ROWS;
    d.blocks = max(1, (d.length + kBlock - 1) / kBlock);
}
// The sequence that workgroup `w` belongs to (BY_SEQUENCE: sequence `w`); false: none.
template <int ROWS, bool BY_SEQUENCE>
__device__ __forceinline__ bool deal(const PagedView& v, int group, int w, Deal& found) {
    const int lane = threadIdx.x & 63;
    Deal d{};
    int64_t total = 0;
    for (int s = lane; s < v.sequences; s += 64) {
        deal_one<ROWS>(v, group, s, d);
        total += int64_t(d.blocks) * d.tiles;
    }
#pragma unroll
    for (int off = 1; off < 64; off *= 2) total += __shfl_xor(total, off);
    total *= v.kv_heads;
    const int most = int(min(max((total + kShares - 1) / kShares, int64_t(1)), int64_t(1) << 30));
    int before = 0;
    for (int begin = 0; begin < v.sequences; begin += 64) {
        const int s = begin + lane;
        int count = 0;
        if (s < v.sequences) {
            if (v.sequences > 64) deal_one<ROWS>(v, group, s, d);
            d.splits = (d.blocks + most - 1) / most;
            count = d.splits * d.tiles * v.kv_heads;
        }
        int upto = count;
#pragma unroll
        for (int off = 1; off < 64; off *= 2) {
            const int other = __shfl_up(upto, off);
            if (lane >= off) upto += other;
        }
        const unsigned long long hit = __ballot(BY_SEQUENCE ? s == w : before + upto > w);
        if (hit) {
            const int from = __ffsll(hit) - 1;
            found.s = begin + from;
            found.length = __shfl(d.length, from);
            found.n = __shfl(d.n, from);
            found.first = __shfl(d.first, from);
            found.tiles = __shfl(d.tiles, from);
            found.blocks = __shfl(d.blocks, from);
            found.splits = __shfl(d.splits, from);
            found.offset = before + __shfl(upto - count, from);
            // The same in every lane, and known to be.
            found.s = __builtin_amdgcn_readfirstlane(found.s);
            found.length = __builtin_amdgcn_readfirstlane(found.length);
            found.n = __builtin_amdgcn_readfirstlane(found.n);
            found.first = __builtin_amdgcn_readfirstlane(found.first);
            found.tiles = __builtin_amdgcn_readfirstlane(found.tiles);
            found.blocks = __builtin_amdgcn_readfirstlane(found.blocks);
            found.splits = __builtin_amdgcn_readfirstlane(found.splits);
            found.offset = __builtin_amdgcn_readfirstlane(found.offset);
            return true;
        }
        before += __shfl(upto, 63);
    }
    return false;
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
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0, 0);
}
template <int TYPE>
__device__ __forceinline__ float4_t multiply(uint4_t a, uint4_t b, float4_t c, std::integral_constant<int, TYPE>) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                   0);
}

// FP32 values as sums of 16-bit ones, for products on the matrix cores. The
// eight query rows of a tile take the 16 columns of a 16x16x32 product twice:
// columns 0-7 hold the first term, 8-15 the second, and the two halves of the
// result are added. FP16: two terms hold 22 bits. BF16 (8 bits a term) takes
// a second product whose columns 0-7 hold a third term, 24 bits together:
// two terms alone would be off by 2^-17, ten times what the sums lose.
// E4M3 rows become BF16 as they are read, with their power of two: exact.
template <int TYPE>
struct Terms {
    static constexpr int kProducts = TYPE == kPagedF16 ? 1 : 2;
    // Two values; `second`: this lane's column is one of 8-15.
    static __device__ __forceinline__ void split(float a, float b, bool second, unsigned (&out)[kProducts]) {
        if constexpr (TYPE == kPagedF16) {
            _Float16 ha, la, hb, lb;
            split_half(a, ha, la);
            split_half(b, hb, lb);
            const _Float16 x = second ? la : ha, y = second ? lb : hb;
            out[0] = __builtin_bit_cast(uint16_t, x) | unsigned(__builtin_bit_cast(uint16_t, y)) << 16;
        } else {
            a = fp32_fixed(a);
            b = fp32_fixed(b);
            const unsigned high = pack_bf16(a, b);
            const float ra = a - __builtin_bit_cast(float, high << 16);
            const float rb = b - __builtin_bit_cast(float, high & 0xffff0000u);
            const unsigned mid = pack_bf16(ra, rb);
            const unsigned low = pack_bf16(ra - __builtin_bit_cast(float, mid << 16),
                                           rb - __builtin_bit_cast(float, mid & 0xffff0000u));
            out[0] = second ? mid : high;
            out[1] = second ? 0u : low;
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
// goes through LDS (each wave its own 32 rows) and comes back transposed;
// rows are 32 bytes apart from a multiple of 256 so that the 16 rows of a
// read fall on all banks twice.
//
// Memory is what bounds it (two products of 16 x 16 x 32 per 1 KiB of keys
// take a tenth of the time that HBM needs for them), so the loads of the next step
// are always in flight: keys are loaded again as soon as the scores have
// been multiplied, values as soon as they are in LDS, and the table entries
// of a step ahead of the values before it, so that no wait for one covers the other.
template <int TYPE, int DIM, int TILES, bool TRACK>
__global__ __launch_bounds__(kWaves * 64, DIM == 256 ? 1 : 2) void paged_attention_kernel(PagedView v, AttentionArgs a) {
    constexpr int kSize = TYPE == kPagedE4M3 ? 1 : 2, kLoads = DIM * kSize / 64, kSteps = DIM / 32, kOut = DIM / 16;
    constexpr int kPer = kSteps / kLoads;         // products per load: 1, or 2 for E4M3
    constexpr int kRows = 8 * TILES, kProducts = Terms<TYPE>::kProducts;
    constexpr int kPitch = DIM * 2 + 32;          // bytes of a value row in LDS
    constexpr float kHead = TYPE == kPagedF16 ? 6.f : 0.f;  // FP16 weights are kept up to 2^14, far from subnormals
    constexpr float kGrow = 8.f;                  // a reference is moved once a score passes it by 2^8
    constexpr std::integral_constant<int, TYPE> kType{};
    __shared__ __attribute__((aligned(16))) char lds[kWaves][kTile * kPitch];
    __shared__ float2 wave_state[kWaves][kRows];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int column = lane & 15, part = lane >> 4;
    const bool second = column >= 8;

    Deal d;
    if (!deal<kRows, false>(v, a.group, blockIdx.x, d)) return;
    const int of_tile = v.kv_heads * d.splits, within = int(blockIdx.x) - d.offset;
    const int tile = within / of_tile, rest = within - tile * of_tile;
    const int split = rest / v.kv_heads, head = rest - split * v.kv_heads;
    const int even = d.blocks / d.splits, more = d.blocks - even * d.splits;
    const int begin = kBlock * (split * even + min(split, more));
    const int query_rows = a.group * d.n;
    // Positions from shared_end on are seen by some of the tile's new rows only, from `end` on by none.
    const int shared_end = d.length - d.n + tile * kRows / a.group + 1;
    const int seen_end = d.length - d.n + min(d.n - 1, (tile * kRows + kRows - 1) / a.group) + 1;
    const int end = min(seen_end, begin + kBlock * (even + (split < more ? 1 : 0)));

    // Queries: row r of the tile is head r % group of new row r / group, split
    // into terms after an exact power of two has brought the largest to [2^14, 2^15) (FP16).
    uint4_t query[TILES][kSteps][kProducts];
    float to_score[TILES];  // what a product's sum is multiplied by
    int sees[TILES];        // positions the lane's row attends
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
        const int r = tile * kRows + 8 * t + (column & 7), i = r / a.group;
        const int64_t row = int64_t(d.first) + i;
        const bool live = r < query_rows && row >= 0 && row < v.total_rows;
        sees[t] = live ? d.length - d.n + i + 1 : 0;
        const float* from = a.queries + (live ? row * a.query_stride + (head * a.group + r - i * a.group) * DIM : 0);
        float x[kSteps][8];
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            // The channels that this lane's part of a stored row holds in step k.
            const int at = kPer == 1 ? 32 * k + 8 * part : 64 * (k / 2) + 16 * part + 8 * (k % 2);
            const float4_a4 lo = *reinterpret_cast<const float4_a4*>(from + at);
            const float4_a4 hi = *reinterpret_cast<const float4_a4*>(from + at + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[k][e] = live ? lo[e] : 0.f, x[k][4 + e] = live ? hi[e] : 0.f;
        }
        to_score[t] = a.scale;
        if constexpr (TYPE == kPagedF16) {
            float top = 0.f;
#pragma unroll
            for (int k = 0; k < kSteps; ++k)
#pragma unroll
                for (int e = 0; e < 8; ++e) top = fmaxf(top, __builtin_fabsf(x[k][e]));
            top = fmaxf(top, dev::xor_lanes<16>(top));
            top = fmaxf(top, dev::xor_lanes<32>(top));
            // 2^-100 is far below any query that a score depends on; non-finite ones stay so.
            const int up = 14 - max(int(__builtin_bit_cast(unsigned, top) >> 23) - 127, -100);
#pragma unroll
            for (int k = 0; k < kSteps; ++k)
#pragma unroll
                for (int e = 0; e < 8; ++e) x[k][e] *= pow2(up);
            to_score[t] *= pow2(-up);
        }
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                unsigned words[kProducts];
                Terms<TYPE>::split(x[k][2 * e], x[k][2 * e + 1], second, words);
#pragma unroll
                for (int p = 0; p < kProducts; ++p) query[t][k][p][e] = words[p];
            }
    }

    float4_t acc[TILES][kOut];
    float reference[TILES], sum[TILES];
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
        reference[t] = -kInf;
        sum[t] = 0.f;
#pragma unroll
        for (int o = 0; o < kOut; ++o) acc[t][o] = float4_t{0.f, 0.f, 0.f, 0.f};
    }

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
            pages[u] = v.table[int64_t(d.s) * v.table_stride + where.page];
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

    int base = begin + kTile * wave;
    if (base < end) {
        find(base);
        place(base);
        load(v.keys, keys);
        if (base + kBlock < end) find(base + kBlock);
        load(v.values, values);
    }
    for (; base < end; base += kBlock) {
        float4_t s[TILES][2];
#pragma unroll
        for (int t = 0; t < TILES; ++t)
#pragma unroll
            for (int u = 0; u < 2; ++u) s[t][u] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                uint4_t k[kPer];
                widen<TYPE>(keys[u][i], byte_pow2(bytes[u] & 255), k);
#pragma unroll
                for (int j = 0; j < kPer; ++j)
#pragma unroll
                    for (int t = 0; t < TILES; ++t)
#pragma unroll
                        for (int p = 0; p < kProducts; ++p)
                            s[t][u] = multiply(k[j], query[t][kPer * i + j][p], s[t][u], kType);
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

        uint4_t weight[TILES][kProducts];
        float plain[TILES][2][4];
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
            float x[2][4], high = -kInf;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    x[u][r] = add_halves(s[t][u][r]);
                    high = fmaxf(high, x[u][r] * to_score[t]);
                }
            unsigned hidden = 0;  // bit 4 u + r
            if (!whole) {
                high = -kInf;
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int j = 16 * u + 4 * part + r;
                        if (!(exist >> j & 1) || base + j >= sees[t])
                            hidden |= 1u << (4 * u + r);
                        else
                            high = fmaxf(high, x[u][r] * to_score[t]);
                    }
            }
            if (__any(high > reference[t] + (kHead + kGrow))) {
                high = fmaxf(high, dev::xor_lanes<16>(high));
                high = fmaxf(high, dev::xor_lanes<32>(high));
                const float moved = fmaxf(reference[t], high - kHead);
                const float shrink = reference[t] == moved ? 1.f : exp2_fast(reference[t] - moved);
                reference[t] = moved;
                sum[t] *= shrink;
#pragma unroll
                for (int o = 0; o < kOut; ++o) acc[t][o] *= shrink;
            }
            const float from = reference[t] == -kInf ? 0.f : reference[t];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float p = exp2_fast(__builtin_fmaf(x[u][r], to_score[t], -from));
                    if (!whole && (hidden >> (4 * u + r) & 1)) p = 0.f;
                    plain[t][u][r] = p;
                    sum[t] += p;
                }
            if constexpr (TRACK) {
                const int r = tile * kRows + 8 * t + (column & 7);
                if (!second && r < query_rows) {
                    float* const to = a.scores + ((int64_t(d.s) * v.kv_heads + head) * (int64_t(v.rows) * a.group) + r) *
                                                     a.score_stride + base + 4 * part;
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        float4_t w;
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            w[e] = !whole && (hidden >> (4 * u + e) & 1) ? -kInf : x[u][e] * to_score[t];
                        *reinterpret_cast<float4_t*>(to + 16 * u) = w;
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                // Rows that only some new rows see are added below, by those alone.
                float p0 = plain[t][e / 2][2 * (e % 2)], p1 = plain[t][e / 2][2 * (e % 2) + 1];
                unsigned words[kProducts];
                Terms<TYPE>::split(p0, p1, second, words);
#pragma unroll
                for (int p = 0; p < kProducts; ++p) weight[t][p][e] = words[p];
            }
        }

        // Values into LDS. What is not there, or not seen by all rows, is 0 here:
        // a weight of 0 would not keep its infinities and NaN out.
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const bool clean = whole || (was[u] && base + 16 * u + column < shared_end);
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                uint4_t w[kPer];
                widen<TYPE>(values[u][i], value_up[u], w);
#pragma unroll
                for (int j = 0; j < kPer; ++j) {
                    if (!whole && !clean) w[j] = uint4_t{0u, 0u, 0u, 0u};
                    *reinterpret_cast<uint4_t*>(mine + (16 * u + column) * kPitch + 64 * kPer * i + 16 * kPer * part +
                                                16 * j) = w[j];
                }
            }
        }
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
            for (int t = 0; t < TILES; ++t)
#pragma unroll
                for (int p = 0; p < kProducts; ++p) acc[t][o] = multiply(w, weight[t][p], acc[t][o], kType);
        }

        // The last rows of a sequence with several new ones, one at a time.
        if (base + kTile > shared_end) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    for (int q = 0; q < 4; ++q) {
                        const int j = 16 * u + 4 * q + r;
                        if (base + j < shared_end || !(exist >> j & 1)) continue;
                        const int64_t from = __shfl(row_at[u], 4 * q + r);
                        const float up = __shfl(value_up[u], 4 * q + r);
#pragma unroll
                        for (int t = 0; t < TILES; ++t) {
                            const float p = __shfl(plain[t][u][r], 16 * q + column);
                            if (second || base + j >= sees[t]) continue;
#pragma unroll
                            for (int o = 0; o < kOut; ++o)
#pragma unroll
                                for (int e = 0; e < 4; ++e)
                                    acc[t][o][e] = __builtin_fmaf(
                                        p, stored<TYPE>(v.values + from, 16 * o + 4 * part + e, up), acc[t][o][e]);
                        }
                    }
        }
    }

    // The four waves' sums, brought to their largest reference.
    __syncthreads();
    float* const sums = reinterpret_cast<float*>(lds);  // [kWaves][kRows][DIM]
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
        sum[t] += dev::xor_lanes<16>(sum[t]);
        sum[t] += dev::xor_lanes<32>(sum[t]);
        if (lane < 8) wave_state[wave][8 * t + lane] = float2{reference[t], sum[t]};
#pragma unroll
        for (int o = 0; o < kOut; ++o) {
            float4_t w;
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = add_halves(acc[t][o][e]);
            if (!second)
                *reinterpret_cast<float4_t*>(sums + (wave * kRows + 8 * t + column) * DIM + 16 * o + 4 * part) = w;
        }
    }
    __syncthreads();
    for (int item = threadIdx.x; item < kRows * DIM / 4; item += kWaves * 64) {
        const int row = item / (DIM / 4), channel = 4 * (item - row * (DIM / 4));
        float top = -kInf, all = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) top = fmaxf(top, wave_state[w][row].x);
        float4_t o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float2 state = wave_state[w][row];
            const float shrink = state.x == top ? 1.f : exp2_fast(state.x - top);
            all = __builtin_fmaf(state.y, shrink, all);
            const float4_t x = *reinterpret_cast<const float4_t*>(sums + (w * kRows + row) * DIM + channel);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(x[e], shrink, o[e]);
        }
        const int r = tile * kRows + row, i = r / a.group;
        const int64_t to = int64_t(d.first) + i;
        if (r >= query_rows || to < 0 || to >= v.total_rows) continue;
        if (TRACK || d.splits > 1) {
            float* const partial = a.partials + (int64_t(blockIdx.x) * kRows + row) * (DIM + 4);
            *reinterpret_cast<float4_t*>(partial + channel) = o;
            if (channel == 0) *reinterpret_cast<float2*>(partial + DIM) = float2{top, all};
        } else {
            const float by = all == 0.f ? 0.f : 1.f / all;
            if (all == 0.f) o = float4_t{0.f, 0.f, 0.f, 0.f};
            *reinterpret_cast<float4_a4*>(a.out + to * a.out_stride + (head * a.group + r - i * a.group) * DIM + channel) =
                o * by;
        }
    }
}

// Adds the parts of units that were split (all, where weights are tracked) and divides. Tracked: workgroup z of a
// unit's adds its share of positions to the weights, from the scores that the attention left.
template <int DIM, int TILES, bool TRACK>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedView v, AttentionArgs a) {
    constexpr int kRows = 8 * TILES;
    const int heads = v.kv_heads, s = blockIdx.x / heads, head = blockIdx.x - s * heads;
    Deal d;
    if (!deal<kRows, true>(v, a.group, s, d)) return;
    if (!TRACK && d.splits == 1) return;
    const int query_rows = a.group * d.n;
    auto partial = [&](int r, int split) {
        const int tile = r / kRows, w = d.offset + tile * heads * d.splits + split * heads + head;
        return a.partials + (int64_t(w) * kRows + r - tile * kRows) * (DIM + 4);
    };
    auto real = [&](int r, int64_t& row) {
        row = int64_t(d.first) + r / a.group;
        return row >= 0 && row < v.total_rows;
    };
    if (blockIdx.y == 0) {
        for (int64_t item = threadIdx.x; item < int64_t(query_rows) * (DIM / 4); item += 256) {
            const int r = int(item / (DIM / 4)), channel = 4 * int(item - int64_t(r) * (DIM / 4));
            int64_t row;
            if (!real(r, row)) continue;
            float top = -kInf, all = 0.f;
            for (int p = 0; p < d.splits; ++p) top = fmaxf(top, partial(r, p)[DIM]);
            float4_t o = {0.f, 0.f, 0.f, 0.f};
            for (int p = 0; p < d.splits; ++p) {
                const float* const from = partial(r, p);
                const float shrink = from[DIM] == top ? 1.f : exp2_fast(from[DIM] - top);
                all = __builtin_fmaf(from[DIM + 1], shrink, all);
                const float4_t x = *reinterpret_cast<const float4_t*>(from + channel);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(x[e], shrink, o[e]);
            }
            if (all == 0.f) o = float4_t{0.f, 0.f, 0.f, 0.f};
            *reinterpret_cast<float4_a4*>(a.out + row * a.out_stride + (head * a.group + r % a.group) * DIM + channel) =
                o * (all == 0.f ? 0.f : 1.f / all);
        }
    }
    if constexpr (TRACK) {
        __shared__ float2 state[256];
        __shared__ int sees[256];
        float* const weights = v.weights + v.track_at(s, head);
        const float* const scores = a.scores + int64_t(blockIdx.x) * (int64_t(v.rows) * a.group) * a.score_stride;
        const int step = int(gridDim.y) * 256;
        for (int r0 = 0; r0 < query_rows; r0 += 256) {
            __syncthreads();
            const int r = r0 + threadIdx.x;
            int64_t row;
            float2 mine = {0.f, 0.f};
            sees[threadIdx.x] = d.length - d.n + r / a.group + 1;
            if (r < query_rows && real(r, row)) {
                float top = -kInf, all = 0.f;
                for (int p = 0; p < d.splits; ++p) top = fmaxf(top, partial(r, p)[DIM]);
                for (int p = 0; p < d.splits; ++p) {
                    const float* const from = partial(r, p);
                    all = __builtin_fmaf(from[DIM + 1], from[DIM] == top ? 1.f : exp2_fast(from[DIM] - top), all);
                }
                mine = {top == -kInf ? 0.f : top, all == 0.f ? 0.f : 1.f / all};
            }
            state[threadIdx.x] = mine;
            __syncthreads();
            const int count = min(256, query_rows - r0);
            for (int j = blockIdx.y * 256 + threadIdx.x; j < d.length; j += step) {
                float w = 0.f;
                for (int q = 0; q < count; ++q)
                    if (state[q].y != 0.f && j < sees[q])
                        w += exp2_fast(scores[(r0 + q) * a.score_stride + j] - state[q].x) * state[q].y;
                weights[j] += w;
            }
        }
    }
}

void check_heads(const qwen_gpu_paged_cache& cache, int query_heads) {
    require(query_heads >= cache.kv_heads && query_heads % cache.kv_heads == 0 && query_heads / cache.kv_heads <= 1024,
            "query_heads must be a multiple of kv_heads, at most 1024 times");
}

// Sizes of a call: the grid, and what its workspace holds.
struct Plan {
    int tiles, row_tiles;  // TILES, and tiles of 8 * TILES rows at most per KV head
    int64_t groups, score_stride, score_rows;
    size_t partial_bytes, score_bytes;
    Plan(const qwen_gpu_paged_cache& c, const qwen_gpu_paged_batch& b, int query_heads) {
        const int64_t rows = int64_t(query_heads / c.kv_heads) * b.rows;
        // Two tiles of eight rows per workgroup where there are as many rows: the cache is then read half as often.
        // Heads of 256 have no registers for it.
        tiles = rows > 8 && c.head_dim < 256 ? 2 : 1;
        row_tiles = int((rows + 8 * tiles - 1) / (8 * tiles));
        const int64_t units = int64_t(b.sequences) * c.kv_heads * row_tiles;
        const int64_t blocks = units * ((b.max_length + kBlock - 1) / kBlock);
        groups = std::min(blocks, units + kShares);
        partial_bytes = size_t(groups) * 8 * tiles * (c.head_dim + 4) * 4;
        score_stride = (b.max_length + kTile - 1) / kTile * kTile;
        score_rows = int64_t(b.sequences) * c.kv_heads * rows;
        score_bytes = b.weights ? size_t(score_rows) * score_stride * 4 : 0;
    }
    size_t bytes() const { return kPagedCounterBytes + partial_bytes + score_bytes; }
};

template <int TYPE, int DIM, int TILES>
void attention_run(const PagedView& v, const AttentionArgs& a, const Plan& plan, hipStream_t stream) {
    const dim3 grid{unsigned(plan.groups)}, block{kWaves * 64};
    const unsigned units = unsigned(v.sequences) * v.kv_heads;
    if (v.weights) {
        // Enough workgroups for the positions of few units.
        const unsigned share = unsigned(std::max(1, std::min((v.max_length + 255) / 256, int(1024 / units) + 1)));
        paged_attention_kernel<TYPE, DIM, TILES, true><<<grid, block, 0, stream>>>(v, a);
        paged_join_kernel<DIM, TILES, true><<<dim3(units, share), 256, 0, stream>>>(v, a);
    } else {
        paged_attention_kernel<TYPE, DIM, TILES, false><<<grid, block, 0, stream>>>(v, a);
        if (v.max_length > kBlock) paged_join_kernel<DIM, TILES, false><<<units, 256, 0, stream>>>(v, a);
    }
}

template <int TYPE>
void attention_of(int dim, const PagedView& v, const AttentionArgs& a, const Plan& plan, hipStream_t stream) {
    if (dim == 256) return attention_run<TYPE, 256, 1>(v, a, plan, stream);
    if (dim == 128)
        return plan.tiles == 1 ? attention_run<TYPE, 128, 1>(v, a, plan, stream)
                               : attention_run<TYPE, 128, 2>(v, a, plan, stream);
    return plan.tiles == 1 ? attention_run<TYPE, 64, 1>(v, a, plan, stream)
                           : attention_run<TYPE, 64, 2>(v, a, plan, stream);
}

}  // namespace

size_t paged_workspace_bytes(const qwen_gpu_paged_cache& cache, const qwen_gpu_paged_batch& batch, int query_heads) {
    (void)paged_view(cache, batch);
    check_heads(cache, query_heads);
    paged_check_rows(batch);
    const Plan plan(cache, batch, query_heads);
    // Eviction: two lists of the rows that move, at most half of the longest.
    const size_t lists = size_t(batch.sequences) * cache.kv_heads * 2 * (size_t(batch.max_length) / 2) * 4;
    return std::max(plan.bytes(), kPagedCounterBytes + lists) + 16;
}

void launch_paged_attention(const qwen_gpu_paged_cache& cache, const qwen_gpu_paged_batch& batch, const float* queries,
                            int64_t query_stride, int query_heads, float scale, float* out, int64_t out_stride,
                            void* workspace, size_t workspace_bytes, hipStream_t stream) {
    const PagedView v = paged_view(cache, batch);
    paged_check_rows(batch);
    require(queries, "Null argument: queries");
    require(out, "Null argument: out");
    check_heads(cache, query_heads);
    const int64_t row = int64_t(query_heads) * cache.head_dim;
    require(query_stride >= row && out_stride >= row, "Paged rows overlap: stride below query_heads * head_dim");
    require(query_stride <= (int64_t(1) << 32) && out_stride <= (int64_t(1) << 32), "Paged row stride is too large");
    const Plan plan(cache, batch, query_heads);
    require(plan.groups < (int64_t(1) << 24) && plan.score_rows < (int64_t(1) << 31), "Too many new rows for one call");
    const PagedDevice device(cache, batch, stream);
    device.check(queries, "queries");
    device.check(out, "out");
    if (!batch.total_rows) return;
    device.check(workspace, "workspace", 16);
    require(workspace_bytes >= plan.bytes(), "Workspace is too small");
    char* const space = static_cast<char*>(workspace) + kPagedCounterBytes;
    const AttentionArgs a{queries,
                          query_stride,
                          out,
                          out_stride,
                          query_heads / cache.kv_heads,
                          plan.row_tiles,
                          scale * 1.44269504088896340736f,
                          reinterpret_cast<float*>(space),
                          reinterpret_cast<float*>(space + plan.partial_bytes),
                          plan.score_stride};
    if (cache.type == kPagedF16)
        attention_of<kPagedF16>(cache.head_dim, v, a, plan, stream);
    else if (cache.type == kPagedBF16)
        attention_of<kPagedBF16>(cache.head_dim, v, a, plan, stream);
    else
        attention_of<kPagedE4M3>(cache.head_dim, v, a, plan, stream);
}

}  // namespace qwen_hip

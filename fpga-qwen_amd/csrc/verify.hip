// Verification of drafted tokens against the target's probabilities.
//
// With w_i = 2^(z_i), z_i = (x_i - m) log2(e) / T and m a row's largest logit,
// p = w / Z, Z = sum w. Which token a number falls on is decided at borders
// between sums over the vocabulary, so weights and sums are FP64: with 32
// bits about one drawn token in a hundred of a peaked row's tail would be
// another one.
#include "verify.hpp"

#include <algorithm>
#include <iterator>

#include "decode_dev.hpp"
#include "op_device.hpp"
#include "qwen_common.hpp"

namespace qwen_hip {

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64, kEach = 16;
constexpr int kChunk = kThreads * kEach;  // tokens of a workgroup's step
constexpr int kMostChunks = 8;            // of a workgroup that draws
constexpr float kInf = __builtin_huge_valf();

// Of a range of a row: its largest logit, the lowest token that has it (where
// the largest wins), and the sum of the weights relative to it.
struct Part {
    double sum;
    float top;
    int best;
};

// What the rows of a sequence come to.
struct Outcome {
    double z;        // of the row that the token is drawn from
    float top;
    int best;        // lowest token of the largest logit
    int row;         // -1: there is none
    int token;       // the drafted one that the row decides on, -1: none
    int accepted, drafted;
};

struct VerifyArgs {
    const char* logits;
    const float* draft;
    const int32_t *tokens, *offsets;
    const float *temperature, *accept, *sample;
    int64_t logit_stride, draft_stride;
    int vocabulary, chunks, sequences, rows, total_rows;
    int ranges, draw_chunks;    // ranges that a row's sums are made of; chunks of a workgroup that draws
    Part* parts;        // [total_rows][ranges]
    double* rest;       // [sequences][chunks]: sums of the weights that a token is drawn from
    int* done;          // [sequences]: workgroups that have added up their chunks, 0 before the second kernel
    int32_t *accepted, *next, *back;

    // First row of a sequence and how many of them there are.
    __device__ int rows_of(int s, int& first) const {
        if (!offsets) {
            first = s * rows;
            return rows;
        }
        first = offsets[s];
        if (first < 0 || first >= total_rows) return 0;
        const int64_t n = min(int64_t(offsets[s + 1]) - first, int64_t(total_rows) - first);
        return n < 0 ? 0 : int(min(n, int64_t(rows)));
    }
    // 64 log2(e) / T; 0 for an infinite T, where all tokens are equal, and where the largest logit alone counts.
    __device__ double heat(int s) const {
        const float t = temperature ? temperature[s] : 1.f;
        return t > 0.f ? 64 * 1.44269504088896340736 / t : 0.;
    }
    __device__ bool greedy(int s) const { return temperature && !(temperature[s] > 0.f); }
};

// 2^z for z <= 0 through the exponential series of its part behind the whole
// number (at most ln(2) / 2 from 0, where the first term left out is 6e-15 of
// the whole).
__device__ __forceinline__ double series(double z) {
    const double whole = rint(z), x = (z - whole) * 0.693147180559945309417;
    double p = 1. / 39916800;
    p = __builtin_fma(p, x, 1. / 3628800);
    p = __builtin_fma(p, x, 1. / 362880);
    p = __builtin_fma(p, x, 1. / 40320);
    p = __builtin_fma(p, x, 1. / 5040);
    p = __builtin_fma(p, x, 1. / 720);
    p = __builtin_fma(p, x, 1. / 120);
    p = __builtin_fma(p, x, 1. / 24);
    p = __builtin_fma(p, x, 1. / 6);
    p = __builtin_fma(p, x, 0.5);
    p = __builtin_fma(p, x, 1.);
    p = __builtin_fma(p, x, 1.);
    return __builtin_amdgcn_ldexp(p, int(whole));
}

// Weights of tokens. 2^z as 2^n * 2^(j / 64) * 2^r with the 64 powers in LDS
// and |r| <= 1 / 128, where four terms of the series are 4e-14 off: a token
// takes 13 FP64 operations, and 21 with the series alone (260 rows of 151936
// BF16 logits took 47 us with that).
struct Powers {
    double at[64];

    __device__ __forceinline__ void make() {  // by all threads of a workgroup, before a barrier
        if (threadIdx.x < 64) at[threadIdx.x] = series(threadIdx.x / 64. - 1.) * 2.;
    }
    // 2^(z / 64) for -64000 <= z <= 0.
    __device__ __forceinline__ double within(double z) const {
        constexpr double kRound = 6755399441055744.;  // 1.5 * 2^52: adding it leaves the nearest whole number in the low bits
        constexpr double kLn = 0.693147180559945309417 / 64;
        const double shifted = z + kRound, x = z - (shifted - kRound);
        const int whole = int(__builtin_bit_cast(uint64_t, shifted));
        double p = kLn * kLn * kLn * kLn / 24;
        p = __builtin_fma(p, x, kLn * kLn * kLn / 6);
        p = __builtin_fma(p, x, kLn * kLn / 2);
        p = __builtin_fma(p, x, kLn);
        p = __builtin_fma(p, x, 1.);
        const uint64_t bits = __builtin_bit_cast(uint64_t, p * at[whole & 63]);
        const unsigned high = unsigned(bits >> 32) + (unsigned(whole & ~63) << 14);
        return __builtin_bit_cast(double, (bits & 0xffffffffu) | uint64_t(high) << 32);
    }
    // The same for z <= 0; 0 for NaN and below 2^-1000.
    __device__ __forceinline__ double of(double z) const {
        const bool tiny = !(z >= -64000.);
        const double w = within(tiny ? 0. : z);
        return tiny ? 0. : w;
    }
    // Of finite tops, with 2^-1000 for what weighs nothing: for sums, which it does not change.
    __device__ __forceinline__ double summand(float x, float top, double heat) const {
        return within(fmax((double(x) - double(top)) * heat, -64000.));
    }
    // Weight of a logit in a row (or chunk) whose largest is `top`, heat 64 log2(e) / T. Minus infinity and NaN weigh
    // nothing; with a top of infinity (FINITE: it is known to be none) only equal logits do.
    template <bool FINITE = false>
    __device__ __forceinline__ double weight(float x, float top, double heat) const {
        if (!FINITE && (top == kInf || top == -kInf)) return x == kInf ? 1. : 0.;
        return of((double(x) - double(top)) * heat);
    }
};

template <typename T>
__device__ __forceinline__ float logit(const char* logits, int64_t at) {
    return float(reinterpret_cast<const T*>(logits)[at]);
}

// A thread's 16 tokens of a chunk. `together`: 16 in a row, otherwise the
// pieces of 16 bytes that make a wave's load one range. The loads of a chunk
// have no branches of their own, so that all are in flight at once.
template <typename T>
struct Tokens {
    static constexpr int kPiece = 16 / sizeof(T), kPieces = kEach / kPiece;
    typedef T piece_t __attribute__((ext_vector_type(kPiece), aligned(sizeof(T))));
    piece_t raw[kPieces];

    static __device__ __forceinline__ int at(int i, bool together) {
        const int piece = i / kPiece;
        return i % kPiece + (together ? threadIdx.x * kEach + piece * kPiece : (piece * kThreads + threadIdx.x) * kPiece);
    }
    // `behind` stands for tokens past the end.
    __device__ __forceinline__ void load(const T* row, int from, int vocabulary, bool together, T behind) {
        if (from + kChunk <= vocabulary) {
#pragma unroll
            for (int i = 0; i < kPieces; ++i)
                raw[i] = *reinterpret_cast<const piece_t*>(row + from + at(i * kPiece, together));
        } else {
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const int token = from + at(i, together);
                const T x = row[min(token, vocabulary - 1)];
                raw[i / kPiece][i % kPiece] = token < vocabulary ? x : behind;
            }
        }
    }
    __device__ __forceinline__ float value(int i) const { return float(raw[i / kPiece][i % kPiece]); }
    // NaN counts as minus infinity.
    __device__ __forceinline__ float logit(int i) const {
        const float x = value(i);
        return x == x ? x : -kInf;
    }
};

__device__ __forceinline__ float uniform(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x)));
}
__device__ __forceinline__ int wave_min(int x) {
    x = min(x, dev::xor_lanes<32>(x));
    x = min(x, dev::xor_lanes<16>(x));
    x = min(x, dev::xor_lanes<8>(x));
    x = min(x, dev::xor_lanes<4>(x));
    x = min(x, dev::xor_lanes<2>(x));
    return min(x, dev::xor_lanes<1>(x));
}

// A range of a row, of whole chunks: its largest logit and the sum of its
// weights, each lane by itself until the end, with the next chunk's logits on
// their way. The largest is wanted as a token where it wins. Memory bounds it
// where rows are many and filtered (263 rows of 151936 BF16 logits, 80 MB, 21
// us, 3.8 TB/s), latency where they are few (two rows 4.6 us, of which the
// launch has most; 40 FP32 rows, 24 MB, 10 us). Unfiltered, those 263 rows take
// 45 us as BF16 and as FP32, twice the bytes, so memory does not: 27 vector
// instructions a token, the 13 of FP64 among them, keep a SIMD busy for 67 of
// the 82 thousand cycles that its CU has work, of 115 that the kernel takes
// (starts and ends of five workgroups a CU are the rest); the table's reads
// from LDS take 10.
template <typename T>
__global__ __launch_bounds__(kThreads) void verify_parts_kernel(VerifyArgs a) {
    __shared__ Powers powers;
    __shared__ double sums[kWaves];
    __shared__ float tops[kWaves];
    __shared__ int bests[kWaves];
    const int row = blockIdx.x / a.ranges, range = blockIdx.x - row * a.ranges;
    const int first = int(int64_t(a.chunks) * range / a.ranges), end = int(int64_t(a.chunks) * (range + 1) / a.ranges);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const T* const logits = reinterpret_cast<const T*>(a.logits) + row * a.logit_stride;
    Tokens<T> tokens;
    tokens.load(logits, first * kChunk, a.vocabulary, false, T(-kInf));
    powers.make();
    for (int s = blockIdx.x * kThreads + threadIdx.x; s < a.sequences; s += gridDim.x * kThreads) a.done[s] = 0;
    // The row's sequence: the last one that does not start behind it.
    int s;
    if (a.offsets) {
        int low = 0, high = a.sequences - 1;
        while (low < high) {
            const int middle = (low + high + 1) / 2;
            if (a.offsets[middle] <= row)
                low = middle;
            else
                high = middle - 1;
        }
        s = low;
    } else {
        s = row / a.rows;
    }
    const double heat = a.heat(s);
    const bool greedy = a.greedy(s);
    // Weights below 2^-90 of a lane's largest would not change its sum: what a filter has left out costs nothing.
    const float span = heat > 0. ? float(64 * 90 / heat) : kInf;
    __syncthreads();
    float top = -kInf;
    double sum = 0.;
    int best = a.vocabulary;
    for (int chunk = first; chunk < end; ++chunk) {
        const int from = chunk * kChunk;
        float x[kEach];
#pragma unroll
        for (int i = 0; i < kEach; ++i) x[i] = tokens.value(i);
        if (chunk + 1 < end) tokens.load(logits, from + kChunk, a.vocabulary, false, T(-kInf));
        float high = x[0];
#pragma unroll
        for (int i = 1; i < kEach; ++i) high = fmaxf(high, x[i]);  // NaN is passed over
        if (greedy) {
            if (__any(high > top)) {
#pragma unroll
                for (int i = kEach - 1; i >= 0; --i)
                    if (high > top && x[i] == high) best = from + Tokens<T>::at(i, false);
                top = fmaxf(top, high);
            }
            continue;
        }
        if (high > top) {
            // Infinities: all of the weight, counted below.
            sum = high == kInf || top == -kInf ? 0. : sum * powers.weight<true>(top, high, heat);
            top = high;
        }
        // (Not `high >= top - span`: with an infinite span an infinite top leaves no number there, and counts.)
        if (!__any(high > -kInf && !(high < top - span))) continue;
        if (__any(top == kInf)) {
#pragma unroll
            for (int i = 0; i < kEach; ++i) sum += powers.weight(x[i], top, heat);
            continue;
        }
#pragma unroll
        for (int i = 0; i < kEach; i += 4)
            if (const float four = fmaxf(fmaxf(x[i], x[i + 1]), fmaxf(x[i + 2], x[i + 3]));
                __any(four > -kInf && four >= top - span))
#pragma unroll
                for (int j = 0; j < 4; ++j) sum += powers.summand(x[i + j], top, heat);
    }
    // All lanes' by the largest of all (a lane without tokens has added 2^-1000 up at most); where the largest wins, the sum
    // is 1 and the token the lowest that has it.
    auto weigh = [&](float of, float whole) { return of == whole ? 1. : powers.weight(of, whole, heat); };
    float whole = dev::wave_max(top);
    if (lane == 0) tops[wave] = whole;
    __syncthreads();
    whole = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    best = wave_min(top == whole ? best : a.vocabulary);
    sum = dev::wave_sum(top == -kInf ? 0. : sum * weigh(top, whole));
    if (lane == 0) {
        sums[wave] = sum;
        bests[wave] = best;
    }
    __syncthreads();
    if (threadIdx.x == 0)
        a.parts[int64_t(row) * a.ranges + range] = {
            greedy ? double(whole > -kInf) : (sums[0] + sums[1]) + (sums[2] + sums[3]), whole,
            min(min(bests[0], bests[1]), min(bests[2], bests[3]))};
}

// A row's parts together, by a wave; the same in all lanes.
__device__ __forceinline__ Part whole_row(const VerifyArgs& a, const Powers& powers, int row, double heat, int lane) {
    const Part* const parts = a.parts + int64_t(row) * a.ranges;
    const Part none{0., -kInf, a.vocabulary};
    const Part first = lane < a.ranges ? parts[lane] : none;
    float top = first.top;
    for (int c = lane + 64; c < a.ranges; c += 64) top = fmaxf(top, parts[c].top);
    top = dev::wave_max(top);
    double sum = 0.;
    int best = a.vocabulary;
    for (int c = lane; c < a.ranges; c += 64) {
        const Part part = c == lane ? first : parts[c];
        sum = __builtin_fma(part.sum, part.top == top ? 1. : powers.weight(part.top, top, heat), sum);
        if (part.top == top) best = min(best, part.best);
    }
    sum = dev::wave_sum(sum);
    best = wave_min(best);
    if (top == -kInf) sum = 0.;
    return {sum, top, best};
}

// The weights that a token is drawn from: w of a row (equal logits' sums are
// exact), or max(p - q, 0).
struct Drawn {
    float top;
    double heat, by;   // by: 1 / Z where there is a q, 1 elsewhere
    bool refused;       // less q
    const float* q;    // of the row, or NULL: all at the token
    int token;
    const Powers& powers;

    // A thread's tokens of a chunk, and q of them.
    template <typename T>
    struct Chunk {
        Tokens<T> logits;
        float of_q[kEach];
    };
    template <typename T>
    __device__ __forceinline__ void load(const VerifyArgs& a, int row, int from, bool together, Chunk<T>& c) const {
        c.logits.load(reinterpret_cast<const T*>(a.logits) + row * a.logit_stride, from, a.vocabulary, together, T(-kInf));
        if (!refused || !q) return;
        if (from + kChunk <= a.vocabulary) {
            typedef float float4_a4 __attribute__((ext_vector_type(4), aligned(4)));
#pragma unroll
            for (int i = 0; i < kEach; i += 4) {
                const float4_a4 v = *reinterpret_cast<const float4_a4*>(q + from + Tokens<T>::at(i, together));
#pragma unroll
                for (int e = 0; e < 4; ++e) c.of_q[i + e] = v[e];
            }
        } else {
#pragma unroll
            for (int i = 0; i < kEach; ++i) c.of_q[i] = q[min(from + Tokens<T>::at(i, together), a.vocabulary - 1)];
        }
    }
    // Their weights (places as Tokens<T> has them), four at a time where one of a wave's has any.
    template <typename T>
    __device__ __forceinline__ void weigh(const Chunk<T>& c, int from, bool together, double (&w)[kEach]) const {
        const bool finite = top < kInf && top > -kInf;
        const float least = heat > 0. ? float(top - 64 * 1001 / heat) : -kInf;
#pragma unroll
        for (int i = 0; i < kEach; i += 4) {
            float x[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = c.logits.logit(i + j), w[i + j] = 0.;
            const float high = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
            if (finite && __any(high >= least && high > -kInf)) {
#pragma unroll
                for (int j = 0; j < 4; ++j) w[i + j] = powers.weight<true>(x[j], top, heat) * by;
            } else if (!finite) {
#pragma unroll
                for (int j = 0; j < 4; ++j) w[i + j] = powers.weight(x[j], top, heat) * by;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (refused && q)
                    w[i + j] = fmax(w[i + j] - fmax(double(c.of_q[i + j]), 0.), 0.);
                else if (refused && from + Tokens<T>::at(i + j, together) == token)
                    w[i + j] = 0.;
            }
        }
    }
};
__device__ __forceinline__ Drawn drawn_from(const VerifyArgs& a, const Powers& powers, const Outcome& v, double heat) {
    const bool refused = v.accepted < v.drafted;
    const float* const q = refused && a.draft ? a.draft + v.row * a.draft_stride : nullptr;
    return {uniform(v.top), heat, q ? 1. / v.z : 1., refused, q, v.token, powers};
}

// The sum over the threads before this one, and over all.
__device__ __forceinline__ double sum_before(double x, double* waves, double& all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double upto = x;
#pragma unroll
    for (int off = 1; off < 64; off *= 2) {
        const double other = __shfl_up(upto, off);
        if (lane >= off) upto += other;
    }
    if (lane == 63) waves[wave] = upto;
    double before = __shfl_up(upto, 1);
    if (lane == 0) before = 0.;
    __syncthreads();
    double base = 0.;
    all = 0.;
    for (int w = 0; w < kWaves; ++w) {
        if (w == wave) base = all;
        all += waves[w];
    }
    __syncthreads();
    return base + before;
}

// The lowest of the threads' numbers, and the highest of their others.
__device__ __forceinline__ int lowest(int number, int& other, int* waves) {
    number = wave_min(number);
    other = -wave_min(-other);
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = number, waves[kWaves + (threadIdx.x >> 6)] = other;
    __syncthreads();
    number = min(min(waves[0], waves[1]), min(waves[2], waves[3]));
    other = max(max(waves[4], waves[5]), max(waves[6], waves[7]));
    __syncthreads();
    return number;
}

// What a sequence's rows come to: the first row whose drafted token is not
// accepted, or the last. A wave checks a row, so a workgroup four at a time.
template <typename T>
__device__ __forceinline__ Outcome check_rows(const VerifyArgs& a, const Powers& powers, int s, double heat, bool greedy,
                                              Outcome (&of_wave)[kWaves], int (&fits)[kWaves]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int first;
    const int n = a.rows_of(s, first);
    Outcome v{0., -kInf, -1, -1, -1, 0, max(n - 1, 0)};
    for (int i0 = 0; i0 < n && v.row < 0; i0 += kWaves) {
        const int i = i0 + wave;
        if (i < n) {
            const int row = first + i, token = i + 1 < n ? a.tokens[row + 1] : -1;
            const bool there = token >= 0 && token < a.vocabulary;
            // Loads that only need the token go out before the row's parts are added.
            const float x = there ? logit<T>(a.logits, row * a.logit_stride + token) : -kInf;
            const float of_q = there && a.draft ? a.draft[row * a.draft_stride + token] : 1.f;
            const float number = a.accept[row];
            const Part whole = whole_row(a, powers, row, heat, lane);
            const double w = greedy ? (token == whole.best ? whole.sum : 0.) : powers.weight(x, whole.top, heat);
            const bool fit = there && whole.sum > 0. && double(number) * fmax(double(of_q), 0.) * whole.sum < w;
            if (lane == 0) {
                of_wave[wave] = {whole.sum, whole.top, whole.best, row, token, i, n - 1};
                fits[wave] = fit;
            }
        }
        __syncthreads();
        for (int w = 0; w < kWaves && i0 + w < n; ++w)
            if (!fits[w]) {
                v = of_wave[w];
                break;
            }
        __syncthreads();
    }
    return v;
}

// Sums that other workgroups of the launch read, on other XCDs too.
__device__ __forceinline__ void post(double* p, double x) {
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), __builtin_bit_cast(uint64_t, x), __ATOMIC_RELAXED,
                       __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void posted_stores_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ double posted(const double* p) {
    return __builtin_bit_cast(double, __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED,
                                                        __HIP_MEMORY_SCOPE_AGENT));
}

// Every workgroup of a sequence checks its rows (from sums, which takes no
// longer than to wait for another's word) and adds the weights that the token
// is drawn from up over its own chunks, unless they are a row's own, whose
// sums are there; the last one to do so draws: the chunk (or range) in which
// the sum of the weights passes sample times the whole, then the token in it.
// Sums of one range in two orders may differ in their last place, so that a border can lie between them: the last token with a weight
// stands for what lies behind all. Latency bounds it: 11 us for a sequence of
// two rows, 15 for eight of five, 22 for 64 of up to seven, a chain of loads
// (offsets, tokens, the row's parts, its logits, the posted sums, the chosen
// chunk) with a launch before it.
template <typename T>
__global__ __launch_bounds__(kThreads, 4) void verify_draw_kernel(VerifyArgs a) {
    __shared__ Powers powers;
    __shared__ double waves[kWaves], base_of, chunk_sums[kMostChunks][kWaves];
    __shared__ Outcome of_wave[kWaves];
    __shared__ int fits[kWaves], picks[2 * kWaves], last_one;
    const int groups = (a.chunks + a.draw_chunks - 1) / a.draw_chunks;
    const int s = blockIdx.x / groups, own = blockIdx.x - s * groups, tid = threadIdx.x;
    powers.make();
    __syncthreads();
    const double heat = a.heat(s);
    const bool greedy = a.greedy(s);
    const Outcome v = check_rows<T>(a, powers, s, heat, greedy, of_wave, fits);
    const bool draws = v.row >= 0 && v.z > 0. && !greedy;
    int token = draws || v.row < 0 || !(v.z > 0.) ? -1 : v.best;
    Drawn drawn = drawn_from(a, powers, v, heat);
    double* const rest = a.rest + int64_t(s) * a.chunks;
    // Without a q to subtract, the ranges' sums are those of the first kernel, but for the drafted token's range. (A token
    // for each of 64 sequences 27 us, 41 without this; 64 sequences of up to seven BF16 rows, whose ranges have eight
    // chunks, 48 us with it, 42 without.)
    const bool known = !(drawn.refused && drawn.q) && a.chunks <= a.ranges * max(2, a.draw_chunks);
    if ((!draws || known) && own) return;
    if (draws) {
        // The weights of chunks, the next one's tokens on their way, until f says that it is enough.
        auto walk = [&](int c0, int c1, bool together, auto f) {
            Drawn::Chunk<T> ahead;
            drawn.load<T>(a, v.row, c0 * kChunk, together, ahead);
            for (int c = c0; c < c1; ++c) {
                const Drawn::Chunk<T> here = ahead;
                if (c + 1 < c1) drawn.load<T>(a, v.row, (c + 1) * kChunk, together, ahead);
                double w[kEach];
                drawn.weigh<T>(here, c * kChunk, together, w);
                if (f(c, w)) break;
            }
        };
        auto sum_of = [](const double (&w)[kEach]) {
            double sum = 0.;
#pragma unroll
            for (int i = 0; i < kEach; ++i) sum += w[i];
            return sum;
        };
        // Up to 8 chunks' sums; wave 0 posts them.
        auto add_up = [&](int c0, int c1) {
            walk(c0, c1, false, [&](int c, const double (&w)[kEach]) {
                const double sum = dev::wave_sum(sum_of(w));
                if ((tid & 63) == 0) chunk_sums[c - c0][tid >> 6] = sum;
                return false;
            });
            __syncthreads();
            if (tid < c1 - c0) {
                const double* const of = chunk_sums[tid];
                post(rest + c0 + tid, (of[0] + of[1]) + (of[2] + of[3]));
            }
            if (tid < 64) posted_stores_done();
            __syncthreads();
        };
        // Pieces of the row whose sums are at hand: ranges, or chunks.
        const int pieces = known ? a.ranges : a.chunks;
        auto first_chunk = [&](int piece) { return known ? int(int64_t(a.chunks) * piece / a.ranges) : piece; };
        double all = 0., without = 0.;
        int spared = -1;  // the drafted token's range, whose sum is `without`
        if (known && drawn.refused && v.token >= 0 && v.token < a.vocabulary) {
            spared = int((int64_t(v.token / kChunk + 1) * a.ranges - 1) / a.chunks);
            double sum = 0.;
            walk(first_chunk(spared), first_chunk(spared + 1), false, [&](int, const double (&w)[kEach]) {
                sum += sum_of(w);
                return false;
            });
            (void)sum_before(sum, waves, without);
        } else if (!known) {
            add_up(own * a.draw_chunks, min((own + 1) * a.draw_chunks, a.chunks));
            if (tid == 0)
                last_one = __hip_atomic_fetch_add(a.done + s, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == groups - 1;
            __syncthreads();
            if (!last_one) return;
        }
        auto piece_sum = [&](int i) {
            if (!known) return posted(rest + i);
            const Part part = a.parts[int64_t(v.row) * a.ranges + i];
            return i == spared ? without : part.sum * (part.top == v.top ? 1. : powers.weight(part.top, v.top, heat));
        };
        const int each = (pieces + kThreads - 1) / kThreads, i0 = min(tid * each, pieces), i1 = min(i0 + each, pieces);
        double before = 0., only = 0.;  // only: of up to 256 pieces, the thread's
        for (;;) {
            double sum = 0.;
            for (int i = i0; i < i1; ++i) sum += only = piece_sum(i);
            before = sum_before(sum, waves, all);
            if (!drawn.refused || all > 0.) break;
            drawn.refused = false;  // q is p or more throughout
            drawn.by = 1.;
            spared = -1;
            if (!known)
                for (int c = 0; c < a.chunks; c += kMostChunks) add_up(c, min(c + kMostChunks, a.chunks));
        }
        const double target = double(a.sample[s]) * all;
        int piece = pieces, last = -1;
        double upto = before, base = before, last_base = before;
        for (int i = i0; i < i1; ++i) {
            const double sum = each == 1 ? only : piece_sum(i);
            if (sum > 0.) last = i, last_base = upto;
            if (piece == pieces && upto + sum > target && sum > 0.) piece = i, base = upto;
            upto += sum;
        }
        int last_of_all = last;
        const int first = lowest(piece, last_of_all, picks), found = first < pieces ? first : max(0, last_of_all);
        if (found == piece)
            base_of = base;
        else if (first == pieces && found == last)
            base_of = last_base;
        __syncthreads();
        double from = base_of;  // the sum before a chunk
        walk(first_chunk(found), first_chunk(found + 1), true, [&](int c, const double (&w)[kEach]) {
            double whole;
            double upto = from + sum_before(sum_of(w), waves, whole);
            int pick = a.vocabulary, end = -1;
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const int at = c * kChunk + tid * kEach + i;
                upto += w[i];
                if (w[i] > 0.) {
                    end = at;
                    if (pick == a.vocabulary && upto > target) pick = at;
                }
            }
            pick = lowest(pick, end, picks);
            token = pick < a.vocabulary ? pick : max(token, end);
            from += whole;
            return pick < a.vocabulary;
        });
    }
    if (tid) return;
    a.next[s] = token;
    const int accepted = v.row >= 0 ? v.accepted : 0;
    if (a.accepted) a.accepted[s] = accepted;
    if (a.back) a.back[s] = accepted - v.drafted;
}

struct Plan {
    int64_t chunks, units, ranges, draw_chunks;
    size_t parts, rest, done;
    explicit Plan(const qwen_gpu_draft& d) {
        chunks = (d.vocabulary + kChunk - 1) / kChunk;
        units = chunks * std::max(d.total_rows, d.sequences);
        // About as many workgroups as the GPU holds, of a chunk at least (260 unfiltered FP32 rows 73 us, with 768 78; 40
        // rows 23.5 with either).
        ranges = std::clamp<int64_t>(1536 / std::max(d.total_rows, 1), 1, chunks);
        // 64 sequences of 38 BF16 chunks 42 us, with 320 or 1280 workgroups 44, with a chunk each 53.
        draw_chunks = std::clamp<int64_t>((chunks * d.sequences + 639) / 640, 1, kMostChunks);
        parts = sizeof(Part) * ranges * d.total_rows;
        rest = sizeof(double) * chunks * d.sequences;
        done = sizeof(int) * d.sequences;
    }
    size_t bytes() const { return parts + rest + done; }
};

Plan plan_of(const qwen_gpu_draft& d) {
    require(d.type == QWEN_GPU_F32 || d.type == QWEN_GPU_F16 || d.type == QWEN_GPU_BF16, "Unknown type of logits");
    require(d.vocabulary >= 1 && d.vocabulary <= 1 << 24, "The vocabulary must be in 1..2^24");
    require(d.sequences >= 1 && d.sequences <= 4096, "Draft sequences must be in 1..4096");
    require(d.rows >= 1 && d.rows <= 1024, "Draft rows must be in 1..1024");
    require(d.total_rows >= 0 && d.total_rows <= 1 << 20, "Draft total_rows must be in 0..2^20");
    require(d.offsets || int64_t(d.sequences) * d.rows == d.total_rows,
            "Draft total_rows must be sequences * rows without offsets");
    const Plan plan(d);
    require(plan.units < int64_t(1) << 31, "Too many logits for one call");
    return plan;
}

template <typename T>
void run(const VerifyArgs& a, hipStream_t stream) {
    const unsigned draws = (a.chunks + a.draw_chunks - 1) / a.draw_chunks;
    if (a.total_rows) verify_parts_kernel<T><<<unsigned(a.total_rows * a.ranges), kThreads, 0, stream>>>(a);
    verify_draw_kernel<T><<<a.sequences * draws, kThreads, 0, stream>>>(a);
}

}  // namespace

size_t verify_workspace_bytes(const qwen_gpu_draft& draft) { return plan_of(draft).bytes(); }

void launch_verify_draft(const qwen_gpu_draft& d, int32_t* accepted, int32_t* next, int32_t* back, void* workspace,
                         size_t workspace_bytes, hipStream_t stream) {
    const Plan plan = plan_of(d);
    const int size = d.type == QWEN_GPU_F32 ? 4 : 2;
    const int64_t most = int64_t(1) << 32;
    require(d.total_rows <= 1 || (d.logit_stride >= d.vocabulary && d.logit_stride <= most),
            "Rows of logits overlap or lie too far apart");
    require(!d.draft || d.total_rows <= 1 || (d.draft_stride >= d.vocabulary && d.draft_stride <= most),
            "Rows of draft overlap or lie too far apart");
    const size_t n = size_t(d.sequences) * 4, rows = size_t(d.total_rows) * 4;
    auto span = [&](int64_t stride, int element) {
        return d.total_rows ? (size_t(d.total_rows - 1) * stride + d.vocabulary) * element : size_t(0);
    };
    const OpArray arrays[] = {{"logits", d.logits, span(d.logit_stride, size), true, false, unsigned(size)},
                              {"draft", d.draft, span(d.draft_stride, 4), false, false},
                              {"tokens", d.tokens, rows, true, false},
                              {"offsets", d.offsets, n + 4, false, false},
                              {"temperature", d.temperature, n, false, false},
                              {"accept", d.accept, rows, true, false},
                              {"sample", d.sample, n, true, false},
                              {"accepted", accepted, n, false, true},
                              {"next", next, n, true, true},
                              {"back", back, n, false, true},
                              {"workspace", workspace, plan.bytes(), true, true, 16}};
    check_arrays(arrays, std::size(arrays));
    require(workspace_bytes >= plan.bytes(), "Workspace is too small");
    const OpDevice device(d.logits, "logits", "the logits", stream);
    for (const OpArray& a : arrays)
        if (a.at) device.check(a.at, a.name, a.alignment);
    char* const space = static_cast<char*>(workspace);
    const VerifyArgs a{static_cast<const char*>(d.logits), d.draft, d.tokens, d.offsets, d.temperature, d.accept, d.sample,
                       d.total_rows > 1 ? d.logit_stride : 0, d.total_rows > 1 ? d.draft_stride : 0, d.vocabulary,
                       int(plan.chunks), d.sequences, d.rows, d.total_rows, int(plan.ranges), int(plan.draw_chunks),
                       reinterpret_cast<Part*>(space),
                       reinterpret_cast<double*>(space + plan.parts),
                       reinterpret_cast<int*>(space + plan.parts + plan.rest), accepted, next, back};
    if (d.type == QWEN_GPU_F32)
        run<float>(a, stream);
    else if (d.type == QWEN_GPU_F16)
        run<_Float16>(a, stream);
    else
        run<__bf16>(a, stream);
}

}  // namespace qwen_hip

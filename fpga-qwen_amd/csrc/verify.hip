// Verification of drafted tokens against the target's probabilities.
//
// With w_i = 2^(z_i), z_i = (x_i - m) log2(e) / T and m a row's largest logit,
// p = w / Z, Z = sum w. Which token a number falls on is decided at borders
// between sums over the vocabulary, so weights and sums are FP64: with 32
// bits about one drawn token in a hundred of a peaked row's tail would be
// another one.
#include "verify.hpp"

#include <algorithm>
#include <string>
#include <type_traits>

#include "decode_dev.hpp"
#include "op_device.hpp"
#include "qwen_common.hpp"

namespace qwen_hip {

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64, kEach = 16;
constexpr int kChunk = kThreads * kEach;  // tokens of a workgroup
constexpr float kInf = __builtin_huge_valf();

// Of a row and a chunk: its largest logit, the lowest token that has it, and
// the sum of the weights relative to it.
struct Part {
    double sum;
    float top;
    int best;
};

// What the rows of a sequence come to.
struct Verdict {
    double z;        // of the row that the token is drawn from
    float top;
    int best;        // lowest token of the largest logit
    int row;         // -1: there is none
    int token;       // the drafted one that the row judges, -1: none
    int accepted, drafted;
};

struct VerifyArgs {
    const char* logits;
    const float* draft;
    const int32_t *tokens, *offsets;
    const float *temperature, *accept, *sample;
    int64_t logit_stride, draft_stride;
    int vocabulary, chunks, sequences, rows, total_rows;
    Part* parts;        // [total_rows][chunks]
    double* rest;       // [sequences][chunks]: sums of max(p - q, 0)
    Verdict* verdicts;  // [sequences]
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
    // log2(e) / T; 0: the largest logit alone counts.
    __device__ double heat(int s) const {
        const float t = temperature ? temperature[s] : 1.f;
        return t > 0.f ? 1.44269504088896340736 / t : 0.;
    }
    __device__ bool greedy(int s) const { return temperature && !(temperature[s] > 0.f); }
};

// 2^z for z <= 0, 0 for NaN: the power of the nearest whole number, and the
// exponential series of the rest (at most ln(2) / 2 from 0, where the first
// term left out is 6e-15 of the whole).
__device__ __forceinline__ double power(double z) {
    z = fmax(z, -1100.);
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
// Weight of a logit in a row (or chunk) whose largest is `top`. Minus
// infinity and NaN weigh nothing; with a top of infinity only equal logits do.
__device__ __forceinline__ double weight(float x, float top, double heat) {
    if (top == kInf || top == -kInf) return x == kInf ? 1. : 0.;
    return power((double(x) - double(top)) * heat);
}

template <typename T>
__device__ __forceinline__ float logit(const char* logits, int64_t at) {
    return float(reinterpret_cast<const T*>(logits)[at]);
}

// A thread's 16 tokens of a chunk. `together`: 16 in a row, otherwise the
// pieces of 16 bytes that make a wave's load one range.
template <typename T>
struct Tokens {
    static constexpr int kPiece = 16 / sizeof(T), kPieces = kEach / kPiece;
    typedef T piece_t __attribute__((ext_vector_type(kPiece), aligned(sizeof(T))));
    static __device__ __forceinline__ int at(int piece, bool together) {
        return together ? threadIdx.x * kEach + piece * kPiece : (piece * kThreads + threadIdx.x) * kPiece;
    }
    // x[i] is token at(i / kPiece) + i % kPiece of the chunk; minus infinity behind the vocabulary and for NaN.
    static __device__ __forceinline__ void load(const char* logits, int64_t row, int from, int vocabulary, bool together,
                                                float (&x)[kEach]) {
        const T* const p = reinterpret_cast<const T*>(logits) + row + from;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            const int t = at(i, together);
            if (from + t + kPiece <= vocabulary) {
                const piece_t v = *reinterpret_cast<const piece_t*>(p + t);
#pragma unroll
                for (int j = 0; j < kPiece; ++j) x[i * kPiece + j] = float(v[j]);
            } else {
#pragma unroll
                for (int j = 0; j < kPiece; ++j) x[i * kPiece + j] = from + t + j < vocabulary ? float(p[t + j]) : -kInf;
            }
        }
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (!(x[i] == x[i])) x[i] = -kInf;
    }
};

__device__ __forceinline__ int wave_min(int x) {
    x = min(x, dev::xor_lanes<32>(x));
    x = min(x, dev::xor_lanes<16>(x));
    x = min(x, dev::xor_lanes<8>(x));
    x = min(x, dev::xor_lanes<4>(x));
    x = min(x, dev::xor_lanes<2>(x));
    return min(x, dev::xor_lanes<1>(x));
}

// A chunk of a row: its largest logit and the sum of its weights.
template <typename T>
__global__ __launch_bounds__(kThreads) void verify_parts_kernel(VerifyArgs a) {
    __shared__ double sums[kWaves];
    __shared__ float tops[kWaves];
    __shared__ int bests[kWaves];
    const int row = blockIdx.x / a.chunks, chunk = blockIdx.x - row * a.chunks, from = chunk * kChunk;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float x[kEach];
    Tokens<T>::load(a.logits, row * a.logit_stride, from, a.vocabulary, false, x);
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
    float top = x[0];
#pragma unroll
    for (int i = 1; i < kEach; ++i) top = fmaxf(top, x[i]);
    top = dev::wave_max(top);
    if (lane == 0) tops[wave] = top;
    __syncthreads();
    top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    int best = a.vocabulary;
#pragma unroll
    for (int i = kEach - 1; i >= 0; --i)
        if (x[i] == top) best = from + Tokens<T>::at(i / Tokens<T>::kPiece, false) + i % Tokens<T>::kPiece;
    best = wave_min(best);
    double sum = 0.;
#pragma unroll
    for (int i = 0; i < kEach; ++i) sum += weight(x[i], top, heat);
    sum = dev::wave_sum(sum);
    if (lane == 0) {
        sums[wave] = sum;
        bests[wave] = best;
    }
    __syncthreads();
    if (threadIdx.x == 0)
        a.parts[int64_t(row) * a.chunks + chunk] = {(sums[0] + sums[1]) + (sums[2] + sums[3]), top,
                                                    min(min(bests[0], bests[1]), min(bests[2], bests[3]))};
}

// A row's parts together, by a wave; the same in all lanes.
__device__ __forceinline__ Part whole_row(const VerifyArgs& a, int row, double heat, int lane) {
    const Part* const parts = a.parts + int64_t(row) * a.chunks;
    float top = -kInf;
    for (int c = lane; c < a.chunks; c += 64) top = fmaxf(top, parts[c].top);
    top = dev::wave_max(top);
    double sum = 0.;
    int best = a.vocabulary;
    for (int c = lane; c < a.chunks; c += 64) {
        const Part part = parts[c];
        sum = __builtin_fma(part.sum, part.top == top ? 1. : weight(part.top, top, heat), sum);
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
    bool judged;       // less q
    const float* q;    // of the row, or NULL: all at the token
    int token;

    __device__ __forceinline__ double operator()(float x, float of_q, int at) const {
        const double p = weight(x, top, heat) * by;
        if (!judged) return p;
        if (!q) return at == token ? 0. : p;
        return fmax(p - fmax(double(of_q), 0.), 0.);
    }
    // The weights of a thread's tokens of a chunk (their places as Tokens<T> has them).
    template <typename T>
    __device__ __forceinline__ void load(const VerifyArgs& a, int row, int from, bool together, double (&w)[kEach]) const {
        float x[kEach], of_q[kEach];
        Tokens<T>::load(a.logits, row * a.logit_stride, from, a.vocabulary, together, x);
#pragma unroll
        for (int i = 0; i < Tokens<T>::kPieces; ++i) {
            const int t = Tokens<T>::at(i, together);
#pragma unroll
            for (int j = 0; j < Tokens<T>::kPiece; j += 4) {
                typedef float float4_a4 __attribute__((ext_vector_type(4), aligned(4)));
                float* const to = of_q + i * Tokens<T>::kPiece + j;
                if (judged && q && from + t + j + 4 <= a.vocabulary) {
                    const float4_a4 v = *reinterpret_cast<const float4_a4*>(q + from + t + j);
#pragma unroll
                    for (int e = 0; e < 4; ++e) to[e] = v[e];
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) to[e] = judged && q && from + t + j + e < a.vocabulary ? q[from + t + j + e] : 0.f;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            w[i] = (*this)(x[i], of_q[i], from + Tokens<T>::at(i / Tokens<T>::kPiece, together) + i % Tokens<T>::kPiece);
    }
};
__device__ __forceinline__ Drawn drawn_from(const VerifyArgs& a, const Verdict& v, double heat) {
    const bool judged = v.accepted < v.drafted;
    return {v.top, heat, judged ? 1. / v.z : 1., judged, judged && a.draft ? a.draft + v.row * a.draft_stride : nullptr, v.token};
}

// Every workgroup of a sequence finds, from its rows' parts, the row that the
// token is drawn from, and sums that row's max(p - q, 0) over its own chunk.
template <typename T>
__global__ __launch_bounds__(kThreads) void verify_rest_kernel(VerifyArgs a) {
    __shared__ double sums[kWaves];
    __shared__ Verdict of_wave[kWaves];
    __shared__ int fits[kWaves];
    const int s = blockIdx.x / a.chunks, chunk = blockIdx.x - s * a.chunks;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int first;
    const int n = a.rows_of(s, first);
    const double heat = a.heat(s);
    const bool greedy = a.greedy(s);
    Verdict v{0., -kInf, -1, -1, -1, 0, max(n - 1, 0)};
    for (int i0 = 0; i0 < n && v.row < 0; i0 += kWaves) {
        const int i = i0 + wave;
        if (i < n) {
            const int row = first + i, token = i + 1 < n ? a.tokens[row + 1] : -1;
            const Part whole = whole_row(a, row, heat, lane);
            bool fit = false;
            if (token >= 0 && token < a.vocabulary && whole.sum > 0.) {
                const double q = a.draft ? fmax(double(a.draft[row * a.draft_stride + token]), 0.) : 1.;
                const float x = logit<T>(a.logits, row * a.logit_stride + token);
                const double w = greedy ? (token == whole.best ? whole.sum : 0.) : weight(x, whole.top, heat);
                fit = double(a.accept[row]) * q * whole.sum < w;
            }
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
    if (chunk == 0 && threadIdx.x == 0) a.verdicts[s] = v;
    if (v.row < 0 || greedy || !(v.z > 0.) || v.accepted == v.drafted) return;
    double w[kEach], sum = 0.;
    drawn_from(a, v, heat).load<T>(a, v.row, chunk * kChunk, false, w);
#pragma unroll
    for (int i = 0; i < kEach; ++i) sum += w[i];
    sum = dev::wave_sum(sum);
    if (lane == 0) sums[wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) a.rest[int64_t(s) * a.chunks + chunk] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
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

// The lowest of the threads' numbers, or the highest of `others` where none is below `none`.
__device__ __forceinline__ int lowest_or_last(int number, int none, int other, int* waves) {
    number = wave_min(number);
    other = -wave_min(-other);
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = number, waves[kWaves + (threadIdx.x >> 6)] = other;
    __syncthreads();
    number = min(min(waves[0], waves[1]), min(waves[2], waves[3]));
    other = max(max(waves[4], waves[5]), max(waves[6], waves[7]));
    __syncthreads();
    return number < none ? number : other;
}

// One workgroup a sequence: the chunk in which the sum of the weights passes
// sample times the whole, then the token in it. Sums of one range in two
// orders may differ in their last place, so that a border can lie between them: the last
// token with a weight stands for what lies behind all.
template <typename T>
__global__ __launch_bounds__(kThreads) void verify_draw_kernel(VerifyArgs a) {
    __shared__ double waves[kWaves], base_of;
    __shared__ int picks[2 * kWaves];
    const int s = blockIdx.x, tid = threadIdx.x;
    const Verdict v = a.verdicts[s];
    const double heat = a.heat(s);
    int token = -1;
    if (v.row >= 0 && v.z > 0. && a.greedy(s)) token = v.best;
    if (v.row >= 0 && v.z > 0. && !a.greedy(s)) {
        Drawn drawn = drawn_from(a, v, heat);
        const Part* const parts = a.parts + int64_t(v.row) * a.chunks;
        const double* const rest = a.rest + int64_t(s) * a.chunks;
        const int each = (a.chunks + kThreads - 1) / kThreads, c0 = min(tid * each, a.chunks), c1 = min(c0 + each, a.chunks);
        auto of_chunk = [&](int c) {
            if (drawn.judged) return rest[c];
            const Part part = parts[c];
            return part.sum * (part.top == drawn.top ? 1. : weight(part.top, drawn.top, heat)) * drawn.by;
        };
        double before = 0., all = 0.;
        for (;;) {
            double sum = 0.;
            for (int c = c0; c < c1; ++c) sum += of_chunk(c);
            before = sum_before(sum, waves, all);
            if (!drawn.judged || all > 0.) break;
            drawn.judged = false;  // q is p or more throughout
        }
        const double target = double(a.sample[s]) * all;
        int chunk = a.chunks, last = -1;
        double upto = before, base = before, last_base = before;
        for (int c = c0; c < c1; ++c) {
            const double sum = of_chunk(c);
            if (sum > 0.) last = c, last_base = upto;
            if (chunk == a.chunks && upto + sum > target && sum > 0.) chunk = c, base = upto;
            upto += sum;
        }
        const int found = max(0, lowest_or_last(chunk, a.chunks, last, picks));
        if (found == chunk) base_of = base;
        else if (found == last && found >= c0 && found < c1) base_of = last_base;
        __syncthreads();
        double w[kEach], sum = 0.;
        drawn.load<T>(a, v.row, found * kChunk, true, w);
#pragma unroll
        for (int i = 0; i < kEach; ++i) sum += w[i];
        upto = base_of + sum_before(sum, waves, all);
        int pick = a.vocabulary, end = -1;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int at = found * kChunk + tid * kEach + i;
            upto += w[i];
            if (w[i] > 0.) {
                end = at;
                if (pick == a.vocabulary && upto > target) pick = at;
            }
        }
        token = lowest_or_last(pick, a.vocabulary, end, picks);
    }
    if (tid) return;
    a.next[s] = token;
    const int accepted = v.row >= 0 ? v.accepted : 0;
    if (a.accepted) a.accepted[s] = accepted;
    if (a.back) a.back[s] = accepted - v.drafted;
}

struct Plan {
    int64_t chunks, units;
    size_t parts, rest, verdicts;
    explicit Plan(const qwen_gpu_draft& d) {
        chunks = (d.vocabulary + kChunk - 1) / kChunk;
        units = chunks * std::max(d.total_rows, d.sequences);
        parts = sizeof(Part) * chunks * d.total_rows;
        rest = sizeof(double) * chunks * d.sequences;
        verdicts = sizeof(Verdict) * d.sequences;
    }
    size_t bytes() const { return parts + rest + verdicts; }
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
    if (a.total_rows) verify_parts_kernel<T><<<unsigned(a.total_rows * a.chunks), kThreads, 0, stream>>>(a);
    verify_rest_kernel<T><<<unsigned(a.sequences * a.chunks), kThreads, 0, stream>>>(a);
    verify_draw_kernel<T><<<unsigned(a.sequences), kThreads, 0, stream>>>(a);
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
    struct Array {
        const char* name;
        const void* at;
        size_t bytes;
        bool needed, written;
        unsigned align = 4;
    };
    const Array arrays[] = {{"logits", d.logits, span(d.logit_stride, size), true, false, unsigned(size)},
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
    for (const Array& a : arrays) require(a.at || !a.needed, std::string("Null argument: ") + a.name);
    for (const Array& a : arrays)
        for (const Array& b : arrays)
            if (&a != &b && a.at && b.at && a.written)
                require(apart(a.at, a.bytes, b.at, b.bytes), std::string(a.name) + " overlaps " + b.name);
    require(workspace_bytes >= plan.bytes(), "Workspace is too small");
    const OpDevice device(d.logits, "logits", "the logits", stream);
    for (const Array& a : arrays)
        if (a.at) device.check(a.at, a.name, a.align);
    char* const space = static_cast<char*>(workspace);
    const VerifyArgs a{static_cast<const char*>(d.logits), d.draft, d.tokens, d.offsets, d.temperature, d.accept, d.sample,
                       d.total_rows > 1 ? d.logit_stride : 0, d.total_rows > 1 ? d.draft_stride : 0, d.vocabulary,
                       int(plan.chunks), d.sequences, d.rows, d.total_rows, reinterpret_cast<Part*>(space),
                       reinterpret_cast<double*>(space + plan.parts),
                       reinterpret_cast<Verdict*>(space + plan.parts + plan.rest), accepted, next, back};
    if (d.type == QWEN_GPU_F32)
        run<float>(a, stream);
    else if (d.type == QWEN_GPU_F16)
        run<_Float16>(a, stream);
    else
        run<__bf16>(a, stream);
}

}  // namespace qwen_hip

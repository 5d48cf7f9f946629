// Norm of queries' and keys' heads and their rotation by position.
#include "rotate.hpp"

#include <cmath>
#include <string>
#include <type_traits>
#include <utility>

#include "half_split.hpp"
#include "op_device.hpp"
#include "qwen_common.hpp"

namespace qwen_hip {

// ---- frequencies ----

void rotary_frequencies(int scaling, int dims, double base, double factor, double trained, double slow, double fast,
                        double* frequencies, float* magnitude) {
    require(scaling >= QWEN_GPU_ROTARY_PLAIN && scaling <= QWEN_GPU_ROTARY_RAMP, "Unknown rotary scaling");
    require(dims >= 2 && dims <= 512 && dims % 2 == 0, "Rotary dims must be even, in 2..512");
    require(frequencies, "Null argument: frequencies");
    require(base > 1 && std::isfinite(base), "The rotary base must be above 1");
    require(scaling == QWEN_GPU_ROTARY_PLAIN || (factor >= 1 && std::isfinite(factor)),
            "The rotary factor must be 1 or more");
    require(scaling != QWEN_GPU_ROTARY_BASE || dims > 2, "A rotary base is scaled for more than one pair");
    require(scaling != QWEN_GPU_ROTARY_RAMP || (trained > 0 && std::isfinite(trained) && slow > 0 && fast > slow &&
                                                std::isfinite(fast)),
            "A rotary ramp needs trained positions and 0 < slow < fast");
    if (scaling == QWEN_GPU_ROTARY_BASE) base *= std::pow(factor, double(dims) / (dims - 2));
    require(std::isfinite(base), "The rotary base must be finite, scaled too");  // its last pair would not turn
    constexpr double kTurn = 6.283185307179586476925;
    for (int i = 0; i < dims / 2; ++i) {
        const double f = std::pow(base, -2.0 * i / dims);
        double share = scaling == QWEN_GPU_ROTARY_LINEAR ? 0 : 1;  // of f; the rest is of f / factor
        if (scaling == QWEN_GPU_ROTARY_RAMP)
            share = std::fmin(1, std::fmax(0, (trained * f / kTurn - slow) / (fast - slow)));
        frequencies[i] = share == 1 ? f : f * share + f / factor * (1 - share);
    }
    if (magnitude) *magnitude = scaling == QWEN_GPU_ROTARY_RAMP ? float(0.1 * std::log(factor) + 1) : 1.f;
}

// ---- rotation ----

namespace {

constexpr int kThreads = 256, kMaxDim = 512, kMaxRows = 1 << 24;

struct Side {
    const char* rows;
    char* out;
    const float* norm;
    int64_t row_stride, head_stride, out_row_stride, out_head_stride;  // elements
    int heads;
};

struct RotateArgs {
    Side sides[2];
    const double* frequencies;
    const int32_t* positions;
    int pairs, turned;     // of a head; those that turn are the first
    int lanes;             // of a head, a power of two
    float magnitude, epsilon, over_dim;
};

template <typename T, int V>
struct Vec {
    typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T))));
};
template <typename T>
struct Vec<T, 1> {
    typedef T type;
};

template <typename T, int V>
__device__ __forceinline__ void load(const T* from, float* to) {
    const typename Vec<T, V>::type x = *reinterpret_cast<const typename Vec<T, V>::type*>(from);
    if constexpr (V == 1) {
        to[0] = float(x);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) to[i] = float(x[i]);
    }
}

// Rounded to nearest, from a float that no other operation is fused into.
template <typename T>
__device__ __forceinline__ T rounded(float x) {
    if constexpr (std::is_same_v<T, float>)
        return x;
    else
        return static_cast<T>(fp32_fixed(x));
}

template <typename T, int V>
__device__ __forceinline__ void store(T* to, const float* from) {
    if constexpr (V == 1) {
        *to = rounded<T>(from[0]);
    } else {
        typename Vec<T, V>::type x;
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = rounded<T>(from[i]);
        *reinterpret_cast<typename Vec<T, V>::type*>(to) = x;
    }
}

// A workgroup has a row. Its threads first find the row's angles, one pair
// each: position * frequency in turns and FP64, less the nearest quarter,
// which leaves an eighth of a turn at most, so that rounding it to FP32 costs
// half a step of sine and cosine. Then a head at a time goes through `lanes`
// lanes of a wave, each with V pairs (K times V where there are more): both
// channels of a pair are in one lane, so the rotation moves nothing between
// lanes and the norm is one sum over them. Channels behind the turned ones
// count as pairs that stay.
//
// Memory bounds it: 8191 rows of 40 BF16 heads of 128 (168 MB read and written)
// take 37.8 us, 4.4 TB/s, where a copy of 1 GiB reaches 5.16; 512 rows of 24
// FP32 heads 5.6, 8 rows 4.3, a launch's latency with the angles' FP64 in it.
// Four rows a workgroup, for fewer of them, took 9.7 and 8.6 us for those, two
// 6.4 and 5.4, and no less for many (16384: 70 us with one row, 70 with two, 74
// with four).
template <typename T, int V, int K, bool INTERLEAVED>
__global__ __launch_bounds__(kThreads) void rotate_kernel(RotateArgs a) {
    __shared__ float2 turns[kMaxDim / 2];
    static_assert(kMaxDim / 2 <= kThreads, "a pair each");
    const int64_t row = blockIdx.y * gridDim.x + blockIdx.x;
    const int position = a.positions[row];
    if (position < 0) return;
    if (const int pair = threadIdx.x; pair < a.turned) {
        double turn = position * (a.frequencies[pair] * 0.159154943091895335769);  // 1 / (2 pi)
        const double quarters = rint(4 * turn);
        turn -= quarters / 4;
        float s, c;
        sincospif(2 * float(turn), &s, &c);
        const int quarter = int(quarters - 4 * floor(quarters / 4));
        if (quarter & 1) {
            const float x = c;
            c = -s;
            s = x;
        }
        if (quarter & 2) c = -c, s = -s;
        turns[pair] = float2{c * a.magnitude, s * a.magnitude};
    }
    __syncthreads();
    const int heads = a.sides[0].heads + a.sides[1].heads, slots = kThreads / a.lanes;
    const int lane = threadIdx.x & (a.lanes - 1);
    for (int item = threadIdx.x / a.lanes; item < heads; item += slots) {
        const bool second = item >= a.sides[0].heads;
        const Side& side = a.sides[second];
        const int head = second ? item - a.sides[0].heads : item;
        const T* const from = reinterpret_cast<const T*>(side.rows) + row * side.row_stride + head * side.head_stride;
        T* const to = reinterpret_cast<T*>(side.out) + row * side.out_row_stride + head * side.out_head_stride;
        float x[K][2 * V];
        int at[K], beside[K];
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int pair = (lane + k * a.lanes) * V;
            const bool turned = pair < a.turned;
            if (INTERLEAVED && turned) {
                at[k] = 2 * pair;
                beside[k] = V;
            } else {
                at[k] = turned ? pair : pair + a.turned;
                beside[k] = turned ? a.turned : a.pairs - a.turned;
            }
            if (pair >= a.pairs) continue;
            load<T, V>(from + at[k], x[k]);
            load<T, V>(from + at[k] + beside[k], x[k] + V);
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) sum = __builtin_fmaf(x[k][i], x[k][i], sum);
        }
        if (side.norm) {
            for (int off = 1; off < a.lanes; off *= 2) sum += __shfl_xor(sum, off);
            const float by = 1.f / sqrtf(__builtin_fmaf(sum, a.over_dim, a.epsilon));
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if ((lane + k * a.lanes) * V >= a.pairs) continue;
                float w[2 * V];
                load<float, V>(side.norm + at[k], w);
                load<float, V>(side.norm + at[k] + beside[k], w + V);
#pragma unroll
                for (int i = 0; i < 2 * V; ++i) x[k][i] = x[k][i] * by * w[i];
            }
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int pair = (lane + k * a.lanes) * V;
            if (pair >= a.pairs) continue;
            if (pair < a.turned) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float2 t = turns[pair + i];
                    const int one = INTERLEAVED ? 2 * i : i, two = INTERLEAVED ? 2 * i + 1 : V + i;
                    const float p = x[k][one], q = x[k][two];
                    x[k][one] = __builtin_fmaf(p, t.x, -(q * t.y));
                    x[k][two] = __builtin_fmaf(q, t.x, p * t.y);
                }
            }
            store<T, V>(to + at[k], x[k]);
            store<T, V>(to + at[k] + beside[k], x[k] + V);
        }
    }
}

template <typename T, int V>
void rotate_run(const RotateArgs& args, unsigned rows, bool interleaved, hipStream_t stream) {
    constexpr int K = V >= 4 ? 1 : 4 / V;  // 512 channels are 256 pairs
    RotateArgs a = args;
    a.lanes = 1;
    while (a.lanes < 64 && a.lanes * V < a.pairs) a.lanes *= 2;
    // The threads of a grid's axis are counted in 32 bits: the most rows there are need one more.
    const dim3 grid = rows == kMaxRows ? dim3(kMaxRows / 2, 2) : dim3(rows);
    if (interleaved)
        rotate_kernel<T, V, K, true><<<grid, kThreads, 0, stream>>>(a);
    else
        rotate_kernel<T, V, K, false><<<grid, kThreads, 0, stream>>>(a);
}

// 16 bytes a load, or fewer where the turned and the other pairs do not come in such groups (of the 8191 BF16 rows above:
// 8 bytes 43 us, 4 68, 2 120).
template <typename T>
void rotate_of(const RotateArgs& a, unsigned rows, bool interleaved, hipStream_t stream) {
    auto fits = [&](int v) { return a.turned % v == 0 && a.pairs % v == 0; };
    if constexpr (sizeof(T) == 2)
        if (fits(8)) return rotate_run<T, 8>(a, rows, interleaved, stream);
    if (fits(4)) return rotate_run<T, 4>(a, rows, interleaved, stream);
    if (fits(2)) return rotate_run<T, 2>(a, rows, interleaved, stream);
    rotate_run<T, 1>(a, rows, interleaved, stream);
}

// Where the heads of a side lie, in bytes: [outer][inner] pieces of `piece`.
struct Region {
    const char* at;
    int64_t outer, inner, outers, inners, piece;
    int64_t row() const { return (inners - 1) * inner + piece; }
    int64_t span() const { return (outers - 1) * outer + row(); }
};
Region region(const void* at, int64_t row_stride, int64_t head_stride, int64_t rows, int64_t heads, int64_t dim,
              int64_t size) {
    Region r{static_cast<const char*>(at), row_stride * size, head_stride * size, row_stride ? rows : 1,
             head_stride ? heads : 1, dim * size};
    if (r.outer < r.inner || r.outers == 1) {
        std::swap(r.outer, r.inner);
        std::swap(r.outers, r.inners);
    }
    return r;
}
// Pieces every `stride` bytes keep clear of others, `ahead` bytes further, with that stride.
bool between(int64_t ahead, int64_t stride, int64_t piece, int64_t other) {
    const int64_t off = ((ahead % stride) + stride) % stride;
    return off >= piece && stride - off >= other;
}
bool regions_apart(const Region& a, const Region& b) {
    const int64_t ahead = b.at - a.at;
    if (ahead >= a.span() || -ahead >= b.span()) return true;
    if (a.outers > 1 && a.outer != b.outer && b.outers > 1) return false;
    const int64_t outer = a.outers > 1 ? a.outer : b.outer;
    if ((a.outers > 1 || b.outers > 1) && between(ahead, outer, a.row(), b.row())) return true;
    if (a.inners > 1 && b.inners > 1 && a.inner != b.inner) return false;
    const int64_t inner = a.inners > 1 ? a.inner : b.inner;
    return (a.inners > 1 || b.inners > 1) && (outer % inner == 0 || (a.outers == 1 && b.outers == 1)) &&
           between(ahead, inner, a.piece, b.piece);
}

void check_side(const qwen_gpu_rotary_heads& h, const char* name, int head_dim, int rows) {
    if (!h.rows) throw std::runtime_error(std::string("Null argument: ") + name);
    if (!h.out) throw std::runtime_error(std::string("Null argument: out of ") + name);
    require(h.heads >= 1 && h.heads <= 4096, "Rotary heads must be in 1..4096");
    const int64_t most = int64_t(1) << 32;
    for (int64_t stride : {h.row_stride, h.head_stride, h.out_row_stride, h.out_head_stride})
        require(stride >= 0 && stride <= most, "Rotary strides must be in 0..2^32");
    const bool by_rows = h.heads > 1 && (rows == 1 || h.out_head_stride <= h.out_row_stride);
    const int64_t low = by_rows ? h.out_head_stride : h.out_row_stride, high = by_rows ? h.out_row_stride : h.out_head_stride;
    const int64_t lows = by_rows ? h.heads : rows, highs = by_rows ? rows : h.heads;
    require((lows <= 1 || low >= head_dim) && (highs <= 1 || high >= (lows > 1 ? (lows - 1) * low : 0) + head_dim),
            "Rotary strides let heads of out overlap");
}

}  // namespace

void launch_rotate(const qwen_gpu_rotary& rotary, const qwen_gpu_rotary_heads& queries,
                   const qwen_gpu_rotary_heads* keys, const int32_t* positions, int rows, hipStream_t stream) {
    require(rotary.type == QWEN_GPU_F32 || rotary.type == QWEN_GPU_F16 || rotary.type == QWEN_GPU_BF16,
            "Unknown type of rows");
    require(rotary.head_dim >= 2 && rotary.head_dim <= kMaxDim && rotary.head_dim % 2 == 0,
            "Rotary head_dim must be even, in 2..512");
    require(rotary.dims >= 0 && rotary.dims <= rotary.head_dim && rotary.dims % 2 == 0,
            "Rotary dims must be even, in 0..head_dim");
    require(rotary.layout == QWEN_GPU_ROTARY_HALVES || rotary.layout == QWEN_GPU_ROTARY_INTERLEAVED,
            "Unknown rotary layout");
    require(std::isfinite(rotary.magnitude), "The rotary magnitude must be finite");
    require(rotary.epsilon > 0 && std::isfinite(rotary.epsilon), "The norm's epsilon must be above 0");
    require(rotary.frequencies || !rotary.dims, "Null argument: frequencies");
    require(positions, "Null argument: positions");
    require(rows >= 0 && rows <= kMaxRows, "Rotary rows must be in 0..2^24");
    check_side(queries, "queries", rotary.head_dim, rows);
    if (keys) check_side(*keys, "keys", rotary.head_dim, rows);
    const int size = rotary.type == QWEN_GPU_F32 ? 4 : 2;
    const qwen_gpu_rotary_heads* const sides[2] = {&queries, keys};
    for (const auto* to : sides) {
        if (!to || !rows) continue;
        const Region out = region(to->out, to->out_row_stride, to->out_head_stride, rows, to->heads, rotary.head_dim, size);
        for (const auto* from : sides) {
            if (!from) continue;
            const bool in_place = from == to && to->out == to->rows && to->row_stride == to->out_row_stride &&
                                  to->head_stride == to->out_head_stride;
            require(in_place || regions_apart(out, region(from->rows, from->row_stride, from->head_stride, rows,
                                                          from->heads, rotary.head_dim, size)),
                    "out overlaps heads that are read");
            require(from == to || regions_apart(out, region(from->out, from->out_row_stride, from->out_head_stride, rows,
                                                            from->heads, rotary.head_dim, size)),
                    "The outs of queries and keys overlap");
        }
        auto clear = [&](const void* p, size_t bytes, const char* what) {
            if (p && !apart(out.at, size_t(out.span()), p, bytes))
                throw std::runtime_error(std::string("out overlaps ") + what);
        };
        clear(positions, size_t(rows) * 4, "positions");
        clear(rotary.dims ? rotary.frequencies : nullptr, size_t(rotary.dims) * 4, "frequencies");
        for (const auto* from : sides)
            if (from) clear(from->norm, size_t(rotary.head_dim) * 4, "the norm");
    }
    const OpDevice device(queries.out, "out of queries", "the queries", stream);
    for (const auto* side : sides) {
        if (!side) continue;
        device.check(side->out, side == keys ? "out of keys" : "out of queries", size);
        device.check(side->rows, side == keys ? "keys" : "queries", size);
        if (side->norm) device.check(side->norm, "norm");
    }
    device.check(positions, "positions");
    if (rotary.dims) device.check(rotary.frequencies, "frequencies", 8);
    if (!rows) return;
    RotateArgs a{};
    for (int i = 0; i < 2; ++i)
        if (sides[i])
            a.sides[i] = {static_cast<const char*>(sides[i]->rows),
                          static_cast<char*>(sides[i]->out),
                          sides[i]->norm,
                          sides[i]->row_stride,
                          sides[i]->head_stride,
                          sides[i]->out_row_stride,
                          sides[i]->out_head_stride,
                          sides[i]->heads};
    a.frequencies = rotary.frequencies;
    a.positions = positions;
    a.pairs = rotary.head_dim / 2;
    a.turned = rotary.dims / 2;
    a.magnitude = rotary.magnitude;
    a.epsilon = rotary.epsilon;
    a.over_dim = 1.f / rotary.head_dim;
    const bool interleaved = rotary.layout == QWEN_GPU_ROTARY_INTERLEAVED;
    if (rotary.type == QWEN_GPU_F32)
        rotate_of<float>(a, unsigned(rows), interleaved, stream);
    else if (rotary.type == QWEN_GPU_F16)
        rotate_of<_Float16>(a, unsigned(rows), interleaved, stream);
    else
        rotate_of<__bf16>(a, unsigned(rows), interleaved, stream);
}

}  // namespace qwen_hip

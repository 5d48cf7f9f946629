// Attention of new rows over a paged key-value cache.
#include <algorithm>
#include <string>

#include "paged.hpp"
#include "paged_dev.hpp"
#include "qwen_common.hpp"

namespace qwen_hip {
namespace {

struct AttentionArgs {
    const float* queries;
    int64_t query_stride;
    float* out;
    int64_t out_stride;
    int group;
    float scale;
};

// One element of a row.
template <int TYPE>
__device__ __forceinline__ float element(const char* row, int i, float scale) {
    if constexpr (TYPE == kPagedF16) return float(reinterpret_cast<const _Float16*>(row)[i]);
    if constexpr (TYPE == kPagedBF16) return __builtin_bit_cast(float, unsigned(reinterpret_cast<const uint16_t*>(row)[i]) << 16);
    const bf16x2 pair = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(reinterpret_cast<const uint8_t*>(row)[i], scale, false);
    return float(pair[0]);
}

// One workgroup per sequence and KV head takes its query rows one after the other.
template <int TYPE, int DIM>
__global__ __launch_bounds__(256) void paged_attention_kernel(PagedView v, AttentionArgs a) {
    __shared__ float q[DIM], p[256], acc[256], red[256];
    const int tid = threadIdx.x;
    const int s = blockIdx.x / v.kv_heads, head = blockIdx.x - s * v.kv_heads;
    int first;
    const int n = v.new_rows(s, first), length = v.length(s);
    auto locate = [&](int j, int64_t& at, int64_t& exponents) {
        const PageSlot where = page_slot(j, v.page_size, v.magic);
        const int page = v.page_of(s, where.page);
        if (page < 0) return false;
        at = v.row_at(page, head, where.slot);
        exponents = v.exponents_at(page, head, where.slot);
        return true;
    };
    auto score = [&](int j) {
        int64_t at, e;
        if (!locate(j, at, e)) return -__builtin_huge_valf();
        const float up = TYPE == kPagedE4M3 ? byte_pow2(v.exponents[e]) : 1.f;
        float sum = 0.f;
        for (int d = 0; d < DIM; ++d) sum = fmaf(q[d], element<TYPE>(v.keys + at, d, up), sum);
        return sum * a.scale;
    };
    for (int i = 0; i < n; ++i) {
        const int64_t row = int64_t(first) + i;
        if (row < 0 || row >= v.total_rows) continue;
        const int sees = length - n + i + 1;
        for (int g = 0; g < a.group; ++g) {
            __syncthreads();
            for (int d = tid; d < DIM; d += 256) q[d] = a.queries[row * a.query_stride + (head * a.group + g) * DIM + d];
            float top = -__builtin_huge_valf(), sum = 0.f, mine = 0.f;
            for (int begin = 0; begin < sees; begin += 256) {
                __syncthreads();
                const float x = begin + tid < sees ? score(begin + tid) : -__builtin_huge_valf();
                red[tid] = x;
                __syncthreads();
                float high = top;
                for (int t = 0; t < 256; ++t) high = fmaxf(high, red[t]);
                const float safe = high == -__builtin_huge_valf() ? 0.f : high;
                p[tid] = __expf(x - safe);
                const float keep = __expf(top - safe);
                top = high;
                __syncthreads();
                sum *= keep;
                mine *= keep;
                float part = 0.f;
                for (int t = 0; t < 256; ++t) part += p[t];
                sum += part;
                const int lanes = 256 / DIM;
                for (int t = tid / DIM; t < 256 && begin + t < sees; t += lanes) {
                    int64_t at, e;
                    if (locate(begin + t, at, e))
                        mine = fmaf(p[t], element<TYPE>(v.values + at, tid % DIM, TYPE == kPagedE4M3 ? byte_pow2(v.exponents[e + 1]) : 1.f), mine);
                }
            }
            acc[tid] = mine;
            __syncthreads();
            if (tid < DIM) {
                for (int t = tid + DIM; t < 256; t += DIM) mine += acc[t];
                a.out[row * a.out_stride + (head * a.group + g) * DIM + tid] = sum == 0.f ? 0.f : mine / sum;
            }
            if (v.weights && sum != 0.f)
                for (int j = tid; j < sees; j += 256) v.weights[v.track_at(s, head) + j] += __expf(score(j) - top) / sum;
        }
    }
}

template <int TYPE>
void attention_of(int dim, const PagedView& v, const AttentionArgs& a, hipStream_t stream) {
    const dim3 grid(v.sequences * v.kv_heads);
    if (dim == 64)
        paged_attention_kernel<TYPE, 64><<<grid, 256, 0, stream>>>(v, a);
    else if (dim == 128)
        paged_attention_kernel<TYPE, 128><<<grid, 256, 0, stream>>>(v, a);
    else
        paged_attention_kernel<TYPE, 256><<<grid, 256, 0, stream>>>(v, a);
}

void check_heads(const qwen_gpu_paged_cache& cache, int query_heads) {
    require(query_heads >= cache.kv_heads && query_heads % cache.kv_heads == 0,
            "query_heads must be a multiple of kv_heads");
}

}  // namespace

size_t paged_workspace_bytes(const qwen_gpu_paged_cache& cache, const qwen_gpu_paged_batch& batch, int query_heads) {
    (void)paged_view(cache, batch);
    check_heads(cache, query_heads);
    // Eviction: two lists of the rows that move, at most half of the longest.
    return kPagedCounterBytes + size_t(batch.sequences) * cache.kv_heads * 2 * (size_t(batch.max_length) / 2) * 4 + 16;
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
    const PagedDevice device(cache, batch, stream);
    device.check(queries, "queries");
    device.check(out, "out");
    if (!batch.total_rows) return;
    const AttentionArgs a{queries, query_stride, out, out_stride, query_heads / cache.kv_heads, scale};
    if (cache.type == kPagedF16)
        attention_of<kPagedF16>(cache.head_dim, v, a, stream);
    else if (cache.type == kPagedBF16)
        attention_of<kPagedBF16>(cache.head_dim, v, a, stream);
    else
        attention_of<kPagedE4M3>(cache.head_dim, v, a, stream);
}

}  // namespace qwen_hip

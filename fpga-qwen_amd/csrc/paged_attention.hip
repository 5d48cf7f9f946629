// Attention of new rows over a paged key-value cache: entry point, and the
// weights' part of it.
#include "paged_attention.hpp"

#include <cmath>
#include <cstdlib>
#include <string>

#include "paged.hpp"
#include "qwen_common.hpp"

namespace qwen_hip {

extern template void attention_launch<kPagedF16>(int, const PagedView&, const AttentionArgs&, const AttentionPlan&,
                                                 hipStream_t);
extern template void attention_launch<kPagedBF16>(int, const PagedView&, const AttentionArgs&, const AttentionPlan&,
                                                  hipStream_t);
extern template void attention_launch<kPagedE4M3>(int, const PagedView&, const AttentionArgs&, const AttentionPlan&,
                                                  hipStream_t);

namespace {

// The weights of a sequence and KV head grow by the softmax of the scores that
// the attention left, summed over its query rows in their order: a thread a
// slot, as scores of a row are read in one piece. 8 x 1025 positions of two
// rows take 4 us, a launch behind another.
__global__ __launch_bounds__(256) void paged_track_kernel(PagedView v, AttentionArgs a) {
    constexpr int kStates = 64;
    __shared__ float2 states[kStates];
    __shared__ int sees[kStates];
    const int heads = v.kv_heads, s = blockIdx.x / heads, head = blockIdx.x - s * heads;
    int first;
    const int n = v.new_rows(s, first), length = v.length(s);
    int from_row, to_row;
    v.existing(first, n, from_row, to_row);
    float* const weights = v.weights + v.track_at(s, head);
    const int64_t unit = a.tracked(v, head, first);
    for (int r0 = from_row * a.group; r0 < to_row * a.group; r0 += kStates) {
        const int count = min(kStates, to_row * a.group - r0);
        const float* const scores = a.scores + (unit + r0) * a.score_stride;
        __syncthreads();
        if (int(threadIdx.x) < count) {
            states[threadIdx.x] = a.states[unit + r0 + threadIdx.x];
            sees[threadIdx.x] = length - n + (r0 + int(threadIdx.x)) / a.group + 1;
        }
        __syncthreads();
        for (int j = blockIdx.y * 256 + threadIdx.x; j < length; j += int(gridDim.y) * 256) {
            float w = 0.f;
            for (int q = 0; q < count; ++q)
                if (j < sees[q])
                    w += exp2_fast(scores[q * a.score_stride + j] - states[q].x) * states[q].y;
            weights[j] += w;
        }
    }
}

// The sizes of a call that a launch and 32-bit indices hold. A head's tiles have at most 16 query rows, so the first
// check refuses no more than the second one would, and keeps the plan's products within 64 bits.
AttentionPlan plan_of(const qwen_gpu_paged_cache& cache, const qwen_gpu_paged_batch& batch, int query_heads) {
    const char* const too_many = "Too many new rows or positions for one call";
    require(int64_t(query_heads) * batch.rows <= 65535 * 16, too_many);
    const AttentionPlan plan(cache, batch, query_heads);
    require(plan.grid_rows <= 65535 && plan.blocks < (int64_t(1) << 31) && plan.columns < (int64_t(1) << 23) &&
                plan.score_rows < (int64_t(1) << 31),
            too_many);
    return plan;
}

// Rows of `out` lie on their own queries or apart from all (between them, for one): a workgroup's output would
// otherwise be another's queries.
bool rows_apart(const float* queries, int64_t query_stride, const float* out, int64_t out_stride, int64_t row,
                int64_t total) {
    if (!total || (out == queries && out_stride == query_stride)) return true;
    const int64_t ahead = reinterpret_cast<intptr_t>(out) - reinterpret_cast<intptr_t>(queries), bytes = row * 4;
    if (ahead >= ((total - 1) * query_stride + row) * 4 || -ahead >= ((total - 1) * out_stride + row) * 4) return true;
    const int64_t stride = query_stride * 4, off = std::abs(ahead) % stride;
    return query_stride == out_stride && off >= bytes && stride - off >= bytes;
}

}  // namespace

size_t paged_workspace_bytes(const qwen_gpu_paged_cache& cache, const qwen_gpu_paged_batch& batch, int query_heads) {
    (void)paged_view(cache, batch);
    // Eviction: at most half of the longest sequence moves.
    const size_t lists = kPagedCounterBytes + paged_moves_bytes(cache, batch, batch.max_length / 2) + 16;
    if (!query_heads) return lists;
    paged_check_heads(cache, query_heads);
    paged_check_rows(batch);
    return std::max(plan_of(cache, batch, query_heads).bytes() + 16, lists);
}

void launch_paged_attention(const qwen_gpu_paged_cache& cache, const qwen_gpu_paged_batch& batch, const float* queries,
                            int64_t query_stride, int query_heads, float scale, float* out, int64_t out_stride,
                            void* workspace, size_t workspace_bytes, hipStream_t stream) {
    const PagedView v = paged_view(cache, batch);
    paged_check_rows(batch);
    require(queries, "Null argument: queries");
    require(out, "Null argument: out");
    paged_check_heads(cache, query_heads);
    const float scale_of_2 = scale * 1.44269504088896340736f;  // the kernels' exponentials are powers of 2
    require(std::isfinite(scale_of_2), "The scale must be finite, times log2(e) too");
    const int64_t row = int64_t(query_heads) * cache.head_dim;
    require(query_stride >= row && out_stride >= row, "Paged rows overlap: stride below query_heads * head_dim");
    require(query_stride <= (int64_t(1) << 32) && out_stride <= (int64_t(1) << 32), "Paged row stride is too large");
    require(rows_apart(queries, query_stride, out, out_stride, row, batch.total_rows), "out overlaps other rows' queries");
    const AttentionPlan plan = plan_of(cache, batch, query_heads);
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
                          0xffffffffu / unsigned(query_heads / cache.kv_heads),
                          int(shares_of(cache.head_dim) / plan.grid_rows) + 1,
                          int(plan.pitch),
                          int(plan.tiles),
                          scale_of_2,
                          reinterpret_cast<float*>(space),
                          static_cast<int*>(workspace),
                          plan.adds,
                          reinterpret_cast<float2*>(space + plan.partial_bytes),
                          reinterpret_cast<float*>(space + plan.partial_bytes + plan.state_bytes),
                          plan.score_stride};
    if (cache.type == kPagedF16)
        attention_launch<kPagedF16>(cache.head_dim, v, a, plan, stream);
    else if (cache.type == kPagedBF16)
        attention_launch<kPagedBF16>(cache.head_dim, v, a, plan, stream);
    else
        attention_launch<kPagedE4M3>(cache.head_dim, v, a, plan, stream);
    if (!v.weights || plan.adds) return;
    // Enough workgroups for the positions of few units.
    const unsigned units = unsigned(v.sequences) * v.kv_heads;
    const unsigned share = unsigned(std::max(1, std::min((v.max_length + 255) / 256, int(1024 / units) + 1)));
    paged_track_kernel<<<dim3(units, share), 256, 0, stream>>>(v, a);
}

}  // namespace qwen_hip

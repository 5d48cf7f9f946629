// Attention behind shared prefixes: entry point, and the join of the parts.
#include "paged_shared.hpp"

#include <cmath>
#include <string>

#include "paged.hpp"
#include "qwen_common.hpp"

namespace qwen_hip {

extern template void shared_launch<kPagedF16>(int, const PagedView&, const SharedArgs&, const SharedPlan&, hipStream_t);
extern template void shared_launch<kPagedBF16>(int, const PagedView&, const SharedArgs&, const SharedPlan&, hipStream_t);
extern template void shared_launch<kPagedE4M3>(int, const PagedView&, const SharedArgs&, const SharedPlan&, hipStream_t);

namespace {

SharedPlan plan_of(const qwen_gpu_paged_cache& cache, const qwen_gpu_paged_batch& batch, const qwen_gpu_paged_prefix& prefix,
                   int query_heads) {
    (void)paged_view(cache, batch);
    paged_check_rows(batch);
    paged_check_heads(cache, query_heads);
    require(!batch.weights && !batch.positions, "Attention behind shared prefixes tracks no weights");
    require(prefix.lengths, "Null argument: lengths of the prefixes");
    require(prefix.groups >= 1 && prefix.groups <= batch.sequences && (prefix.offsets || prefix.groups == 1),
            "Groups must be in 1..sequences, 1 without offsets");
    require(prefix.max_length >= 0 && prefix.max_length <= batch.max_length,
            "The prefixes' max_length must be in 0..max_length");
    require(prefix.max_rest >= 1 && prefix.max_rest <= batch.max_length, "max_rest must be in 1..max_length");
    const char* const too_many = "Too many new rows or positions for one call";
    // Query rows fit 31 bits, which keeps the plan's products within 64. A launch counts its threads in 32 bits, so
    // each has fewer than 2^24 workgroups of 256: those of the attention, and one for each new row to join its parts.
    require(int64_t(query_heads) * std::max(batch.rows, batch.total_rows) < int64_t(1) << 31, too_many);
    const SharedPlan plan(cache, batch, prefix, query_heads);
    constexpr int64_t kMostGroups = int64_t(1) << 24;
    require(plan.groups() < kMostGroups && batch.total_rows < kMostGroups, too_many);
    return plan;
}

}  // namespace

size_t paged_shared_workspace_bytes(const qwen_gpu_paged_cache& cache, const qwen_gpu_paged_batch& batch,
                                    const qwen_gpu_paged_prefix& prefix, int query_heads) {
    return plan_of(cache, batch, prefix, query_heads).bytes();
}

void launch_paged_attention_shared(const qwen_gpu_paged_cache& cache, const qwen_gpu_paged_batch& batch,
                                   const qwen_gpu_paged_prefix& prefix, const float* queries, int64_t query_stride,
                                   int query_heads, float scale, float* out, int64_t out_stride, void* workspace,
                                   size_t workspace_bytes, hipStream_t stream) {
    const SharedPlan plan = plan_of(cache, batch, prefix, query_heads);
    const PagedView v = paged_view(cache, batch);
    require(queries, "Null argument: queries");
    require(out, "Null argument: out");
    const float scale_of_2 = scale * 1.44269504088896340736f;  // the kernels' exponentials are powers of 2
    require(std::isfinite(scale_of_2), "The scale must be finite, times log2(e) too");
    const int64_t row = int64_t(query_heads) * cache.head_dim;
    require(query_stride >= row && out_stride >= row, "Paged rows overlap: stride below query_heads * head_dim");
    require(query_stride <= (int64_t(1) << 32) && out_stride <= (int64_t(1) << 32), "Paged row stride is too large");
    const PagedDevice device(cache, batch, stream);
    device.check(prefix.lengths, "lengths of the prefixes");
    if (prefix.offsets) device.check(prefix.offsets, "offsets of the prefixes");
    device.check(queries, "queries");
    device.check(out, "out");
    if (!batch.total_rows) return;
    device.check(workspace, "workspace", 16);
    require(workspace_bytes >= plan.bytes(), "Workspace is too small");
    const int64_t rows = batch.total_rows - 1;
    require(apart(workspace, plan.bytes(), queries, size_t(rows * query_stride + row) * 4) &&
                apart(workspace, plan.bytes(), out, size_t(rows * out_stride + row) * 4),
            "The workspace overlaps queries or out");
    const int group = query_heads / cache.kv_heads;
    const SharedArgs a{queries,
                       query_stride,
                       out,
                       out_stride,
                       group,
                       query_heads,
                       0xffffffffu / unsigned(group),
                       scale_of_2,
                       prefix.lengths,
                       prefix.offsets,
                       prefix.groups,
                       int(plan.rest_tiles),
                       int(plan.parts),
                       int(plan.rest_parts),
                       int(plan.part),
                       int(plan.rest_part),
                       int(plan.jobs),
                       int(plan.rest_jobs),
                       plan.compact,
                       reinterpret_cast<float*>(static_cast<char*>(workspace) + plan.state_bytes),
                       static_cast<float2*>(workspace)};
    if (cache.type == kPagedF16)
        shared_launch<kPagedF16>(cache.head_dim, v, a, plan, stream);
    else if (cache.type == kPagedBF16)
        shared_launch<kPagedBF16>(cache.head_dim, v, a, plan, stream);
    else
        shared_launch<kPagedE4M3>(cache.head_dim, v, a, plan, stream);
    // (Without the parts there is nothing to join.)
    if (const hipError_t e = hipGetLastError(); e != hipSuccess)
        throw std::runtime_error(std::string("HIP error: ") + hipGetErrorString(e));
    // A workgroup for each piece of few rows; of many, it finds its row's parts once for several pieces.
    const int64_t pieces = (row / 4 + kJoinItems - 1) / kJoinItems;
    const dim3 grid(unsigned(batch.total_rows), unsigned(std::clamp<int64_t>(2048 / batch.total_rows, 1, pieces)));
    if (cache.head_dim == 64)
        shared_join_kernel<64><<<grid, 256, 0, stream>>>(v, a);
    else if (cache.head_dim == 128)
        shared_join_kernel<128><<<grid, 256, 0, stream>>>(v, a);
    else
        shared_join_kernel<256><<<grid, 256, 0, stream>>>(v, a);
}

}  // namespace qwen_hip

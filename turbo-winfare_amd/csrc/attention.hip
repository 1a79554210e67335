// Attention of a batch over the quantised cache: how a call is split, and what joins the partial results.
#include <stdexcept>

#include "dt_attend.h"

namespace tdt {
namespace {

constexpr uint32_t kJoinStats = 1024;

// Joins the partial results of a row. kThreads / (head_dim / 4) groups of threads; a group takes four values
// to a thread of every per_row-th part of a row, and the groups of a row add up through LDS: with few
// rows the parts' loads run side by side.
template <bool F32>
__global__ __launch_bounds__(kThreads) void k_join(const AttnArgs a, uint32_t head_dim, uint32_t rows, uint32_t per_row) {
    __shared__ float4 sum[kThreads];
    __shared__ float part_total[kThreads];
    __shared__ float2 stats[kJoinStats];
    const uint32_t width = head_dim / 4u, group = threadIdx.x / width, col = (threadIdx.x % width) * 4u;
    const uint32_t per_block = kThreads / width / per_row, r0 = blockIdx.x * per_block;
    const uint32_t r = r0 + group / per_row, first = group % per_row;
    const bool exists = r < rows;
    // the rows' statistics through LDS where they fit: one load each, side by side
    const bool held = per_block * a.parts <= kJoinStats;
    const float2* st = a.stats + (uint64_t)(exists ? r : r0) * a.parts;
    if (held) {
        const uint32_t n = min(per_block, rows - r0) * a.parts;
        for (uint32_t i = threadIdx.x; i < n; i += kThreads) stats[i] = a.stats[(uint64_t)r0 * a.parts + i];
        __syncthreads();
    }
    const float2* mine = stats + (exists ? r - r0 : 0u) * a.parts;
    auto stat = [&](uint32_t i) { return held ? mine[i] : st[i]; };
    float top = kNegInf;
#pragma unroll 8
    for (uint32_t i = 0; i < a.parts; ++i) top = fmaxf(top, stat(i).x);
    float total = 0.0f;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const float* from = a.sums + (uint64_t)(exists ? r : r0) * a.parts * head_dim + col;
    auto take = [&](uint32_t i, float4 x) {
        const float2 s = stat(i);
        if (s.y == 0.0f) return;  // its sums were not written
        const float w = __builtin_amdgcn_exp2f(s.x - top);
        total += w * s.y;
        v.x = fmaf(w, x.x, v.x), v.y = fmaf(w, x.y, v.y), v.z = fmaf(w, x.z, v.z), v.w = fmaf(w, x.w, v.w);
    };
    auto load = [&](uint32_t i) { return *reinterpret_cast<const float4*>(from + (uint64_t)i * head_dim); };
    uint32_t i = first;
    for (; i + 7u * per_row < a.parts; i += 8u * per_row) {
        float4 x[8];
#pragma unroll
        for (uint32_t j = 0; j < 8u; ++j) x[j] = load(i + j * per_row);
#pragma unroll
        for (uint32_t j = 0; j < 8u; ++j) take(i + j * per_row, x[j]);
    }
    for (; i < a.parts; i += per_row) take(i, load(i));
    if (per_row > 1u) {
        sum[threadIdx.x] = v;
        part_total[threadIdx.x] = total;
        __syncthreads();
        if (first != 0u) return;
        for (uint32_t i = 1; i < per_row; ++i) {
            const float4 x = sum[threadIdx.x + i * width];
            total += part_total[threadIdx.x + i * width];
            v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
        }
    }
    if (!exists) return;
    const float r1 = total != 0.0f ? 1.0f / total : 0.0f;
    const uint32_t token = r / a.q_heads, head = r % a.q_heads;
    store_out<F32>(a.out, token * a.out_stride + (uint64_t)head * head_dim + col, make_float4(v.x * r1, v.y * r1, v.z * r1, v.w * r1));
}

Divider divider(uint32_t d) {  // ceil(2^(31 + L) / d) with 2^(L - 1) < d <= 2^L: exact for dividends below 2^31
    uint32_t bits = 0u;
    while (bits < 31u && (1u << bits) < d) ++bits;
    if (bits == 0u) return Divider{0u, 0u};
    return Divider{(uint32_t)(((1ull << (31u + bits)) + d - 1u) / d), bits - 1u};
}

}  // namespace

void launch_attention(AttnArgs& a, const AttnPlan& plan, uint32_t head_dim, int dtype, hipStream_t st) {
    a.prefix_tiles = plan.prefix_tiles, a.prefix_splits = plan.prefix_splits;
    a.own_tiles = plan.own_tiles, a.own_splits = plan.own_splits;
    a.prefix_items = (uint32_t)plan.prefix_items, a.items = (uint32_t)plan.items;
    a.wide_tiles = plan.wide_tiles, a.wide_splits = plan.wide_splits, a.wide_items = (uint32_t)plan.wide_items;
    a.parts = plan.parts;
    a.by_rows = divider(a.q_len * a.group), a.by_group = divider(a.group);
    if (a.masks) launch_tree_attend(a, plan, head_dim, dtype, st);
    else if (dtype == TURBO_HIDDEN_F32) launch_dtype<true, false>(a, plan, head_dim, st);
    else launch_dtype<false, false>(a, plan, head_dim, st);
    check_hip(hipGetLastError(), "attention");
    if (plan.parts > 1u) {
        const uint32_t groups = kThreads / (head_dim / 4u), rows = (uint32_t)plan.rows;
        uint32_t per_row = 1u;  // more groups to a row while there are parts for them and the card has room
        while (per_row < groups && per_row * 2u <= plan.parts && (uint64_t)rows * per_row < 4096u) per_row *= 2u;
        const uint32_t per_block = groups / per_row;
        const dim3 grid((rows + per_block - 1u) / per_block), block(kThreads);
        if (dtype == TURBO_HIDDEN_F32) hipLaunchKernelGGL((k_join<true>), grid, block, 0, st, a, head_dim, rows, per_row);
        else hipLaunchKernelGGL((k_join<false>), grid, block, 0, st, a, head_dim, rows, per_row);
        check_hip(hipGetLastError(), "attention");
    }
}

}  // namespace tdt

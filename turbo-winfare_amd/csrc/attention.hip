// Attention of a batch over the quantised cache: how a call is split, and what joins the partial results.
#include <algorithm>
#include <cmath>
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

uint32_t tiles_for(uint64_t rows, uint32_t most) {
    uint32_t mt = 1u;
    while (mt < most && rows > 16u * mt) mt *= 2u;
    return mt;
}
Divider divider(uint32_t d) {  // ceil(2^(31 + L) / d) with 2^(L - 1) < d <= 2^L: exact for dividends below 2^31
    uint32_t bits = 0u;
    while (bits < 31u && (1u << bits) < d) ++bits;
    if (bits == 0u) return Divider{0u, 0u};
    return Divider{(uint32_t)(((1ull << (31u + bits)) + d - 1u) / d), bits - 1u};
}

}  // namespace

// Keys are split until every compute unit has two workgroups (one at a head_dim of 512, whose registers hold no
// more). Three or four, which the registers of smaller heads hold, bring more partial results to join: 29.5 -> 31.7
// and 33.7 us (32 sequences of 2,000 with heads of 128), 38 -> 40 and 41 us (64 behind 4,000); only 300 prompt
// tokens with heads of 128 gain, 40 -> 37 us. No split is below 4 records, one to a wave: with 8 at least one
// sequence of 2,000 measured 12.7 -> 13.6 us, 8 sequences behind 2,000 14.3 -> 15.1.
// The prefix is taken apart from the sequences' own keys where that leaves two thirds of the tiles or fewer: 16
// sequences of 8 rows behind 6,000 (heads of 512) measured 44 us together, 34 apart. With as many rows in a
// sequence as in a tile, a tile goes on from the prefix to its own keys, without partial results to join.
// Two tiles of rows to a workgroup share the widening of codes, one makes more workgroups: one is taken
// where two left fewer than 16 records to each. With a border of 8 records 16 sequences of 2,000 measured
// 17 -> 19 us and 7 x 8 drafts 18 -> 19, though 3 x 10 drafts behind 4,000 31 -> 27; with one of 32, 32 sequences
// behind 8,000 30 -> 36 us, though 300 prompt tokens 40 -> 34.
// Trees, whose sequences have many rows each, weigh tiles of 32 and 16 rows and numbers of splits against each other. Figures
// in microseconds: 8 to begin and end, 3.2 (32 rows) or 2 (16) for a record to each of four waves, 4 for the join and its
// bytes at 4 TB/s. With few records to a wave the chain of a record's loads and products counts, and so do whole rounds of
// workgroups; with many the vector unit is full, and a round that is not takes less. A window's records are counted once,
// not for the prefix and the own tokens each. 7 trees of 17 nodes with a window of 1,024: 32.3 -> 22.3.
// Trees of many rows in BF16 without a window may take workgroups of 128 rows that widen a record once for all of them
// (tree_attention.hip). Figures: a record of each of n workgroups on a compute unit, measured in rounds of as many as it holds;
// 16 to begin and end, the tree's own records among it; the partial results, written and read at 4 TB/s. With heads of 256
// the other kind's figures, which are those of short chains, are a quarter below what many records take. Of 40 mixed shapes
// four take 11 to 33 % less time than in the other kind, one 7 % more.
AttnPlan plan_attention(uint32_t batch, uint32_t q_len, uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim, int dtype,
                        uint32_t prefix_len, uint32_t own_most, uint32_t window, uint32_t cus, bool tree) {
    const uint64_t group = q_heads / kv_heads, own_rows = q_len * group, all_rows = batch * own_rows;
    auto records = [&](uint64_t keys, uint64_t spread) {
        if (window) keys = std::min<uint64_t>(keys, (uint64_t)window + spread);
        return (keys + kKvBlock - 1u) / kKvBlock;
    };
    const uint64_t pr = prefix_len ? records(prefix_len, prefix_len / 4u) : 0u, orr = own_most ? records(own_most, q_len) : 0u;
    AttnPlan p{};
    p.rows = (uint64_t)batch * q_len * q_heads;
    double best = 0.0;
    AttnPlan chosen{};
    for (uint32_t most = most_tiles(head_dim, dtype == TURBO_HIDDEN_F32);; most /= 2u) {
        p.own_tile_rows = 16u * tiles_for(own_rows, most);
        const uint64_t ot = (own_rows + p.own_tile_rows - 1u) / p.own_tile_rows;
        p.prefix_tile_rows = 16u * tiles_for(all_rows, most);
        uint64_t pt = (all_rows + p.prefix_tile_rows - 1u) / p.prefix_tile_rows;
        const bool shared = pr && 2u * batch * ot > 3u * pt;
        if (!shared) p.prefix_tile_rows = p.own_tile_rows, pt = 0u;
        uint64_t alone = shared ? orr : pr + orr;  // records of a workgroup's sequence
        if (tree && !shared && window) alone = std::min(alone, records((uint64_t)prefix_len + own_most, q_len) + 1u);
        const uint64_t work = kv_heads * (pt * pr + batch * ot * alone);
        const uint64_t groups = head_dim <= 256u ? 2u * cus : cus, per = std::max<uint64_t>(4u, (work + groups - 1u) / groups);
        p.prefix_tiles = (uint32_t)pt;
        p.prefix_splits = shared ? (uint32_t)((pr + per - 1u) / per) : 0u;
        p.own_tiles = (uint32_t)ot;
        p.own_splits = (uint32_t)((alone + per - 1u) / per);
        // without any keys a call still writes zeros, or NaN past the tables
        if (!shared && !alone) p.own_splits = 1u;
        p.prefix_items = kv_heads * pt * p.prefix_splits;
        p.items = p.prefix_items + (uint64_t)batch * kv_heads * ot * p.own_splits;
        if (tree && !shared) {
            const uint64_t tiles = (uint64_t)batch * kv_heads * ot, most_splits = std::min<uint64_t>(64u, (alone + 3u) / 4u);
            for (uint64_t s = 1u; s <= std::max<uint64_t>(1u, most_splits); ++s) {
                const double each = (double)(((alone + s - 1u) / s + 3u) / 4u), full = (double)(tiles * s) / (double)groups;
                const double rounds = each < 16.0 ? std::ceil(full) : std::max(1.0, full);
                const double join = s > 1u ? 4.0 + (double)p.rows * s * head_dim * 8.0 / 4e6 : 0.0;
                const double cost = rounds * (8.0 + each * (p.own_tile_rows == 32u ? 3.2 : 2.0)) + join;
                if (best == 0.0 || cost < best) {
                    best = cost;
                    chosen = p;
                    chosen.own_splits = (uint32_t)s;
                    chosen.items = tiles * s;
                }
            }
            if (most > 1u) continue;
            p = chosen;
            break;
        }
        if (most == 1u || per >= 16u) break;
    }
    if (tree && best > 0.0 && !window && dtype == TURBO_HIDDEN_BF16 && head_dim <= 256u) {
        const uint64_t tiles = (own_rows + 127u) / 128u, at_once = wide_groups(head_dim), all = pr + orr;
        auto record = [&](uint64_t n) {  // of each of n workgroups
            if (n == 0u) return 0.0;
            return head_dim == 64u ? 1.1 + 0.32 * (double)n : head_dim == 128u ? 0.95 + 0.67 * (double)n : 1.65 + 0.65 * (double)n;
        };
        double least = head_dim == 256u ? 1.3 * best : best;
        for (uint64_t s = 1u; s <= std::min<uint64_t>(64u, all / 8u); ++s) {
            const uint64_t on_one = (batch * kv_heads * tiles * s + cus - 1u) / cus;
            const double records = (double)((all + s - 1u) / s), rounds = (double)(on_one / at_once);
            if (p.rows * (s + 1u) * head_dim > (1u << 27)) break;  // partial results of 512 MB at most
            const double parts = (double)p.rows * (s + 1u) * head_dim * 8.0 / 4e6;
            const double cost = 16.0 + records * (rounds * record(at_once) + record(on_one % at_once)) + parts;
            if (cost >= least) continue;
            least = cost;
            p.wide_tiles = (uint32_t)tiles, p.wide_splits = (uint32_t)s;
        }
        if (p.wide_splits) {
            p.own_tile_rows = p.prefix_tile_rows = 32u;
            p.own_tiles = (uint32_t)((own_rows + 31u) / 32u), p.own_splits = 1u;
            p.wide_items = (uint64_t)batch * kv_heads * p.wide_tiles * p.wide_splits;
            p.items = p.wide_items + (uint64_t)batch * kv_heads * p.own_tiles;
        }
    }
    p.parts = p.prefix_splits + p.wide_splits + p.own_splits;
    if (p.parts > 1u) {
        p.stats_bytes = (p.rows * p.parts * sizeof(float2) + 15u) / 16u * 16u;
        p.bytes = p.stats_bytes + p.rows * p.parts * head_dim * sizeof(float);
    }
    return p;
}

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

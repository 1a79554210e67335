// How an attention call over the quantised cache is split: tiles of rows, splits of the keys and the partial results that
// they leave. Host code alone, so that it can be run for any sizes without a GPU.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>

namespace tdt {

constexpr uint32_t kKvBlock = 32;  // tokens per record of the cache

struct AttnPlan {
    uint32_t prefix_tile_rows, own_tile_rows;  // rows to a workgroup: 16 or 32
    uint32_t prefix_tiles, prefix_splits, own_tiles, own_splits;
    uint32_t wide_tiles, wide_splits;
    uint64_t wide_items, prefix_items, items, rows;
    uint32_t parts;
    uint64_t stats_bytes, bytes;
};
// Workgroups of 128 rows of a tree that a compute unit holds at once, by their registers.
constexpr uint32_t wide_groups(uint32_t head_dim) { return head_dim == 64u ? 4u : head_dim == 128u ? 3u : 2u; }
// 16-row tiles of a workgroup at most: what the registers of two waves per SIMD hold without spills (heads of 256:
// all 256). One in place of two: 94 -> 117 us (2 x 512 prompt tokens behind 2,000), 100 -> 121 us (128 sequences
// behind 16,000, heads of 128), but 40 -> 34 us (300 prompt tokens with heads of 128, whose workgroups then fill the
// card).
constexpr int most_tiles(uint32_t head_dim, bool f32) { return head_dim <= (f32 ? 128u : 256u) ? 2 : 1; }

inline uint32_t tiles_for(uint64_t rows, uint32_t most) {
    uint32_t mt = 1u;
    while (mt < most && rows > 16u * mt) mt *= 2u;
    return mt;
}

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
// four take 11 to 33 % less time than in the other kind, one 7 % more. Where tiles of 16 rows take the prefix apart, that is
// what runs, whatever tiles of 32 rows would have cost: 18 trees of 10 nodes, 64 / 32 heads of 64 behind 1,536, 40 us in place
// of 80; 57 of 21 behind 1,000, 44 in place of 72.
// A tree's plan leaves at most most_bytes of partial results; one part, which leaves none, always does.
inline AttnPlan plan_attention(uint32_t batch, uint32_t q_len, uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim, bool f32,
                               uint32_t prefix_len, uint32_t own_most, uint32_t window, uint32_t cus, bool tree,
                               uint64_t most_bytes = ~0ull) {
    const uint64_t group = q_heads / kv_heads, own_rows = q_len * group, all_rows = batch * own_rows;
    auto records = [&](uint64_t keys, uint64_t spread) {
        if (window) keys = std::min<uint64_t>(keys, (uint64_t)window + spread);
        return (keys + kKvBlock - 1u) / kKvBlock;
    };
    const uint64_t pr = prefix_len ? records(prefix_len, prefix_len / 4u) : 0u, orr = own_most ? records(own_most, q_len) : 0u;
    AttnPlan p{};
    p.rows = (uint64_t)batch * q_len * q_heads;
    auto stats_bytes = [&](uint64_t parts) { return parts > 1u ? (p.rows * parts * 2u * sizeof(float) + 15u) / 16u * 16u : 0u; };
    auto bytes = [&](uint64_t parts) { return parts > 1u ? stats_bytes(parts) + p.rows * parts * head_dim * sizeof(float) : 0u; };
    double best = 0.0;
    AttnPlan chosen{};
    for (uint32_t most = most_tiles(head_dim, f32);; most /= 2u) {
        p.own_tile_rows = 16u * tiles_for(own_rows, most);
        const uint64_t ot = (own_rows + p.own_tile_rows - 1u) / p.own_tile_rows;
        p.prefix_tile_rows = 16u * tiles_for(all_rows, most);
        uint64_t pt = (all_rows + p.prefix_tile_rows - 1u) / p.prefix_tile_rows;
        const uint64_t groups = head_dim <= 256u ? 2u * cus : cus;
        auto share_of = [&](uint64_t work) { return std::max<uint64_t>(4u, (work + groups - 1u) / groups); };  // records
        bool shared = pr && 2u * batch * ot > 3u * pt;
        if (tree && shared) {
            const uint64_t per = share_of(kv_heads * (pt * pr + batch * ot * orr));
            shared = bytes((pr + per - 1u) / per + (orr + per - 1u) / per) <= most_bytes;
        }
        if (!shared) p.prefix_tile_rows = p.own_tile_rows, pt = 0u;
        uint64_t alone = shared ? orr : pr + orr;  // records of a workgroup's sequence
        if (tree && !shared && window) alone = std::min(alone, records((uint64_t)prefix_len + own_most, q_len) + 1u);
        const uint64_t per = share_of(kv_heads * (pt * pr + batch * ot * alone));
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
            for (uint64_t s = 1u; s <= std::max<uint64_t>(1u, most_splits) && bytes(s) <= most_bytes; ++s) {
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
    if (tree && !p.prefix_splits && !window && !f32 && head_dim <= 256u) {
        const uint64_t tiles = (own_rows + 127u) / 128u, at_once = wide_groups(head_dim), all = pr + orr;
        auto record = [&](uint64_t n) {  // of each of n workgroups
            if (n == 0u) return 0.0;
            return head_dim == 64u ? 1.1 + 0.32 * (double)n : head_dim == 128u ? 0.95 + 0.67 * (double)n : 1.65 + 0.65 * (double)n;
        };
        double least = head_dim == 256u ? 1.3 * best : best;
        for (uint64_t s = 1u; s <= std::min<uint64_t>(64u, all / 8u); ++s) {
            const uint64_t on_one = (batch * kv_heads * tiles * s + cus - 1u) / cus;
            const double records = (double)((all + s - 1u) / s), rounds = (double)(on_one / at_once);
            if (p.rows * (s + 1u) * head_dim > (1u << 27) || bytes(s + 1u) > most_bytes) break;  // partial results of 512 MB at most
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
    p.stats_bytes = stats_bytes(p.parts), p.bytes = bytes(p.parts);
    return p;
}

}  // namespace tdt

// The key/value cache in memory, and the arguments of the kernels that write, read and attend over it.
//
// A page holds, for each of its heads, one record per 32 tokens. With NG = head_dim / 64 groups a
// record is [key codes][value codes][scales and biases], each part in the order in which the
// attention's matrix instructions (16 x 16 outputs, 32 deep) take it, so a wave streams a record with
// 16-byte loads, 64 lanes side by side, and needs no exchange between lanes:
//   key codes: per group 64 lanes x 16 bytes per 16-token half (8 bits) or per 32 tokens (4 bits: bytes
//     0-7 the first half's, 8-15 the second's). Lane 16 g + i holds token i's values 16 g .. 16 g + 15
//     of the group, in order, two to a byte (even one low) at 4 bits.
//   value codes: per 32 values (8 bits) or 64 values (4 bits) 64 lanes x 16 bytes. Lane 16 g + i, byte
//     8 x + j holds token 16 (j / 4) + 4 g + j % 4 at value 32 c + 16 x + i (8 bits, chunk c), or at
//     values 64 c + 32 x + i (low half) and + 16 (high half) (4 bits). Those are the tokens whose
//     scores the same lane holds after the first product, so weights need no transposing either.
//   scales: [keys, values][group][32 tokens] words of scale BF16 << 16 | bias BF16.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>
#include <stdexcept>

namespace tdt {

constexpr uint32_t kKvBlock = 32;  // tokens per record

struct KvView {
    uint8_t* base;
    uint64_t slots;         // pages * page_tokens
    uint32_t pages;
    uint32_t page_shift;    // log2(page_tokens)
    uint32_t heads;
    uint32_t bits;
    uint32_t groups;        // head_dim / 64
    uint32_t record;        // bytes of a record
};

__host__ __device__ inline uint32_t kv_part_bytes(uint32_t groups, uint32_t bits) { return groups * 64u * kKvBlock * bits / 8u; }
__host__ __device__ inline uint32_t kv_record_bytes(uint32_t groups, uint32_t bits) {
    return 2u * kv_part_bytes(groups, bits) + 2u * groups * kKvBlock * 4u;
}
// Workgroups of 256 threads in one dimension of a grid, which holds fewer than 2^32 threads.
inline uint32_t grid_blocks(uint64_t blocks) {
    if (blocks >> 24) throw std::runtime_error("tokens * heads is too large for one call");
    return (uint32_t)blocks;
}
// Byte offset of the record of 32 tokens number `block` of (page, head); 64 bits: caches pass 4 GiB.
__host__ __device__ inline uint64_t kv_record_at(const KvView& kv, uint32_t page, uint32_t head, uint32_t block) {
    const uint32_t per_page = (1u << kv.page_shift) / kKvBlock;
    return ((uint64_t)page * kv.heads + head) * ((uint64_t)per_page * kv.record) + (uint64_t)block * kv.record;
}
// Offset in the key codes of the byte that holds value d of token t (t < 32); at 4 bits value d is the
// low half of it when d is even.
__host__ __device__ inline uint32_t kv_key_byte(uint32_t bits, uint32_t t, uint32_t d) {
    const uint32_t group = d >> 6, lane = (t & 15u) + 16u * ((d >> 4) & 3u), e = d & 15u;
    return bits == 8u ? ((group * 2u + (t >> 4)) * 64u + lane) * 16u + e
                      : (group * 64u + lane) * 16u + (t >> 4) * 8u + (e >> 1);
}
// Offset in the value codes; at 4 bits value d is the low half of the byte when d & 16 is 0.
__host__ __device__ inline uint32_t kv_value_byte(uint32_t bits, uint32_t t, uint32_t d) {
    const uint32_t lane = (d & 15u) + 16u * ((t & 15u) >> 2), j = (t >> 4) * 4u + (t & 3u);
    return bits == 8u ? ((d >> 5) * 64u + lane) * 16u + ((d >> 4) & 1u) * 8u + j
                      : ((d >> 6) * 64u + lane) * 16u + ((d >> 5) & 1u) * 8u + j;
}
// Offset in the scales of the word of token t and a group, of the keys (which 0) or the values (1).
__host__ __device__ inline uint32_t kv_scale_byte(uint32_t groups, uint32_t which, uint32_t t, uint32_t group) {
    return ((which * groups + group) * kKvBlock + t) * 4u;
}

constexpr uint32_t kXcds = 8;
// Workgroups are dealt out to the eight dies in turn. Those that read or write the same lines are neighbours
// in the returned number; this takes neighbours to one die, whose L2 then holds the lines for all of them.
__host__ __device__ inline uint32_t same_die(uint32_t id, uint32_t n) {
    const uint32_t per = n / kXcds, rest = n % kXcds, die = id % kXcds;
    return die * per + (die < rest ? die : rest) + id / kXcds;
}

// kv_cache.hip: norms, rotation and the cache's write in one pass. Any part may be absent: q, k and v
// null, turns null (no rotation), cache.base null.
struct QkvArgs {
    const void *q, *k, *v;
    void *q_out, *k_out;
    uint64_t q_stride, k_stride, v_stride, q_out_stride, k_out_stride;
    const uint32_t* positions;
    const uint32_t* slots;
    const uint16_t *q_norm, *k_norm;   // [head_dim] bf16 or null
    const uint64_t* turns;             // [rotary_dim / 2] turns per position, 64-bit fixed point
    uint32_t tokens, q_heads, kv_heads, rotary_dim;
    int pairs;                         // 0: halves
    int still;                         // some frequency is 0
    uint32_t norms;                    // TURBO_NORM_*
    float eps;
    KvView kv;
};
void launch_qkv(const QkvArgs& a, uint32_t head_dim, int dtype, hipStream_t st);

struct KvReadArgs {
    KvView kv;
    const uint32_t* slots;
    void *k, *v;
    uint64_t k_stride, v_stride;
    uint32_t tokens;
};
void launch_kv_read(const KvReadArgs& a, uint32_t head_dim, int dtype, hipStream_t st);

// attention.hip
struct Divider {
    uint32_t factor, shift;  // factor 0: by one
};
struct AttnArgs {
    KvView kv;
    const void* q;
    void* out;
    uint64_t q_stride, out_stride;
    const uint32_t* kv_len;
    const uint32_t* prefix_pages;
    const uint32_t* pages;
    uint32_t prefix_len, page_stride;
    uint32_t batch, q_len, q_heads, group;   // group: query heads per key/value head
    uint32_t window;
    float scale_log2e;                       // times 2^scale_power: scale * log2(e), which may leave FP32
    int scale_power;
    // the plan
    uint32_t prefix_tiles, prefix_splits;    // row tiles and key splits of the prefix, per key/value head (0: the
                                             // sequences take it with their own keys)
    uint32_t own_tiles, own_splits;          // of one sequence's own keys
    uint32_t prefix_items, items;            // workgroups
    Divider by_rows, by_group;               // by q_len * group, by group
    uint32_t parts;                          // partial results per row (1: written to out directly)
    float2* stats;                           // [rows][parts] (running maximum, sum)
    float* sums;                             // [rows][parts][head_dim]
};
struct AttnPlan {
    uint32_t prefix_tile_rows, own_tile_rows;  // rows to a workgroup: 16 or 32
    uint32_t prefix_tiles, prefix_splits, own_tiles, own_splits;
    uint64_t prefix_items, items, rows;
    uint32_t parts;
    uint64_t stats_bytes, bytes;
};
AttnPlan plan_attention(uint32_t batch, uint32_t q_len, uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim, int dtype,
                        uint32_t prefix_len, uint32_t own_most, uint32_t window, uint32_t cus);
void launch_attention(AttnArgs& a, const AttnPlan& plan, uint32_t head_dim, int dtype, hipStream_t st);

}  // namespace tdt

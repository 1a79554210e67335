// Tokens of the quantised cache moved from slot to slot, codes, scales and biases as they are.
//
// A workgroup takes one row of moves, one key/value head and the key or the value codes. It reads everything that
// the row moves into LDS before it writes anything, so a row may move tokens onto slots that it reads. A token's
// codes share no byte with another token's, so rows need no order among themselves. The bytes are few; what bounds a
// call is the chain of slots, codes, LDS and stores.
#include "dt_internal.h"
#include "dt_step.h"

namespace tdt {
namespace {

constexpr uint32_t kThreads = 256;

// LDS of a token's key or value codes and their scales, in whole 16 bytes.
__host__ __device__ inline uint32_t held_bytes(uint32_t groups, uint32_t bits) { return (groups * (8u * bits + 4u) + 15u) & ~15u; }

__global__ __launch_bounds__(kThreads) void k_kv_move(const KvMoveArgs a) {
    extern __shared__ uint4 held[];
    __shared__ uint64_t source[kTreeNodes], target[kTreeNodes];  // byte offsets of the tokens' records
    __shared__ uint32_t source_at[kTreeNodes], target_at[kTreeNodes];
    __shared__ uint32_t count;
    const uint32_t head = blockIdx.y;
    const bool values = blockIdx.z != 0u;
    if (threadIdx.x < 64u) {
        const uint32_t i = threadIdx.x;
        const bool in = i < a.width;
        const uint32_t f = in ? a.source[(uint64_t)blockIdx.x * a.width + i] : 0xFFFFFFFFu;
        const uint32_t t = in ? a.target[(uint64_t)blockIdx.x * a.width + i] : 0xFFFFFFFFu;
        const bool moves = f < a.kv.slots && t < a.kv.slots && f != t;
        const unsigned long long all = __ballot(moves);
        if (moves) {
            const uint32_t at = (uint32_t)__popcll(all & ((1ull << i) - 1ull)), mask = (1u << a.kv.page_shift) - 1u;
            source[at] = kv_record_at(a.kv, f >> a.kv.page_shift, head, (f & mask) / kKvBlock);
            target[at] = kv_record_at(a.kv, t >> a.kv.page_shift, head, (t & mask) / kKvBlock);
            source_at[at] = f % kKvBlock, target_at[at] = t % kKvBlock;
        }
        if (i == 0u) count = (uint32_t)__popcll(all);
    }
    __syncthreads();
    const uint32_t n = count;
    if (n == 0u) return;
    const uint32_t bits = a.kv.bits, groups = a.kv.groups, part = kv_part_bytes(groups, bits);
    const uint32_t bytes = groups * 8u * bits, words = held_bytes(groups, bits);  // a token's codes, and its place in LDS
    uint8_t* lds = reinterpret_cast<uint8_t*>(held);
    // piece p of a token's codes: 16 key codes in order (8 or 16 bytes), or one byte of value codes
    const uint32_t pieces = values ? bytes : groups * 4u, size = values ? 1u : 2u * bits;
    auto piece_at = [&](uint32_t t, uint32_t p) {
        if (!values) return kv_key_byte(bits, t, p * 16u);
        return part + kv_value_byte(bits, t, bits == 8u ? p : (p >> 4) * 32u + (p & 15u));
    };
    auto scale_at = [&](uint32_t t, uint32_t g) { return 2u * part + kv_scale_byte(groups, values ? 1u : 0u, t, g); };
    auto all_pieces = [&](auto&& code, auto&& scale) {
        const uint32_t per = pieces + groups;
        for (uint32_t i = threadIdx.x; i < n * per; i += kThreads) {
            const uint32_t m = i / per, p = i - m * per;
            if (p < pieces) code(m, p, lds + m * words + p * size);
            else scale(m, p - pieces, reinterpret_cast<uint32_t*>(lds + m * words + bytes) + p - pieces);
        }
    };
    auto copy = [&](uint8_t* to, const uint8_t* from) {
        if (size == 1u) *to = *from;
        else if (size == 8u) *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(from);
        else
            *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(from),
            *reinterpret_cast<uint2*>(to + 8) = *reinterpret_cast<const uint2*>(from + 8);
    };
    all_pieces([&](uint32_t m, uint32_t p, uint8_t* at) { copy(at, a.kv.base + source[m] + piece_at(source_at[m], p)); },
               [&](uint32_t m, uint32_t g, uint32_t* at) {
                   *at = *reinterpret_cast<const uint32_t*>(a.kv.base + source[m] + scale_at(source_at[m], g));
               });
    __syncthreads();
    all_pieces([&](uint32_t m, uint32_t p, uint8_t* at) { copy(a.kv.base + target[m] + piece_at(target_at[m], p), at); },
               [&](uint32_t m, uint32_t g, uint32_t* at) {
                   *reinterpret_cast<uint32_t*>(a.kv.base + target[m] + scale_at(target_at[m], g)) = *at;
               });
}

}  // namespace

void launch_kv_move(const KvMoveArgs& a, hipStream_t st) {
    hipLaunchKernelGGL(k_kv_move, dim3(a.rows, a.kv.heads, 2), dim3(kThreads), a.width * held_bytes(a.kv.groups, a.kv.bits), st, a);
    check_hip(hipGetLastError(), "cache move");
}

}  // namespace tdt

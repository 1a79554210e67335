// Tokens of the quantised cache moved from slot to slot, codes, scales and biases as they are.
//
// A workgroup takes one row of moves, one key/value head and the key or the value codes. Everything that the row moves
// is read, into LDS, before anything is written, so a row may move tokens onto slots that it reads. A token's codes
// share no byte with another token's, so rows need no order among themselves. The bytes are few; what bounds a call
// is the chain of slots, codes and stores.
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
    // A thread takes the same pieces of every token, kAhead tokens' loads side by side. Those of other threads never meet
    // its own, so it waits for nobody.
    constexpr uint32_t kAhead = 8u;
    for (uint32_t p = threadIdx.x; p < pieces + groups; p += kThreads) {
        uint8_t* const at = lds + (p < pieces ? p * size : bytes + (p - pieces) * 4u);
        auto move_piece = [&](auto unit) {
            typedef decltype(unit) Unit;
            auto place = [&](uint64_t record, uint32_t t) {
                return reinterpret_cast<Unit*>(a.kv.base + record + (p < pieces ? piece_at(t, p) : scale_at(t, p - pieces)));
            };
            for (uint32_t m = 0; m < n; m += kAhead) {
                Unit x[kAhead];
#pragma unroll
                for (uint32_t i = 0; i < kAhead; ++i)
                    if (m + i < n) x[i] = *place(source[m + i], source_at[m + i]);
#pragma unroll
                for (uint32_t i = 0; i < kAhead; ++i)
                    if (m + i < n) *reinterpret_cast<Unit*>(at + (m + i) * words) = x[i];
            }
            for (uint32_t m = 0; m < n; ++m) *place(target[m], target_at[m]) = *reinterpret_cast<const Unit*>(at + m * words);
        };
        if (p >= pieces) move_piece(uint32_t{});
        else if (values) move_piece(uint8_t{});
        else if (bits == 4u) move_piece(uint2{});
        else move_piece(uint4{});
    }
}

}  // namespace

void launch_kv_move(const KvMoveArgs& a, hipStream_t st) {
    hipLaunchKernelGGL(k_kv_move, dim3(a.rows, a.kv.heads, 2), dim3(kThreads), a.width * held_bytes(a.kv.groups, a.kv.bits), st, a);
    check_hip(hipGetLastError(), "cache move");
}

}  // namespace tdt

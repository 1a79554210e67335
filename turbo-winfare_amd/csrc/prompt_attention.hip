// Causal attention over whole prompts, packed one after another, keys and values as the projections leave them.
//
// With s_j = scale q . k_j over the keys j that a query at position i sees (j <= i, and i - j < window):
//   out = sum_j 2^(c s_j - m) v_j / sum_j 2^(c s_j - m),  c = scale log2(e), m a running maximum of the c s_j,
// one pass over the keys, sums and statistics in FP32. A workgroup takes 32 query rows of one head; its four waves
// take the blocks of 32 keys in turn, each with its own maximum and sums, and join at the end.
//   S^T = K Q^T, keys as the first operand: a lane holds 16 scores of one row.
//   O^T += V^T P^T: those 16 keys are the lane's part of the second operand as they are, if the first operand takes
//     the keys in the same order.
#include <type_traits>

#include "dt_internal.h"
#include "dt_step.h"

namespace tdt {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short short4v __attribute__((ext_vector_type(4)));

constexpr uint32_t kThreads = 256, kWaves = 4;
constexpr uint32_t kRows = 32, kKeys = 32;
constexpr float kNegInf = -__builtin_inff();
constexpr float kSlack = 8.0f;  // a weight is at most 2^kSlack before the maximum moves

union Frag {
    uint4 u;
    uint32_t w[4];
    bf16x8 b;
    short4v h[2];
};

__device__ inline f32x16 zeros() {
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.0f;
    return z;
}
// Two numbers rounded to BF16 (nearest even, NaN stays NaN), one instruction on gfx950.
__device__ inline uint32_t pack_bf16(float lo, float hi) {
    typedef float float2v __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((float2v{lo, hi}), bf16x2));
}
// v of the lanes that hold the same row (lane, lane ^ 32)
template <class Op>
__device__ inline float halves_reduce(float v, Op op) {
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return op(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ inline float halves_max(float v) { return halves_reduce(v, [](float a, float b) { return fmaxf(a, b); }); }
__device__ inline float halves_sum(float v) { return halves_reduce(v, [](float a, float b) { return a + b; }); }
// A key of a block that element r of a lane's scores belongs to, and a column of O
__device__ inline uint32_t element(uint32_t r, uint32_t half) { return 8u * (r >> 2) + 4u * half + (r & 3u); }

struct Item {
    uint32_t first, len, tile;  // the sequence's first row of q, k, v and out, its tokens, and its tile of rows
    bool exists;
};

// Tile number `id` of all sequences' tiles of `rows` rows: the last tiles, which have most keys, come first, and
// among equal ones the sequences in order. Every wave finds it for itself: the number of tiles at a level or above
// falls with the level, so the level is found by halving.
__device__ inline Item locate(const PromptArgs& a, uint32_t id, uint32_t rows) {
    const uint32_t lane = threadIdx.x & 63u;
    auto bounds = [&](uint32_t b, uint32_t& first, uint32_t& len) {
        first = min(a.starts[b], a.tokens);
        len = max(min(a.starts[b + 1u], a.tokens), first) - first;
    };
    uint32_t first0 = 0, len0 = 0;
    if (lane < a.batch) bounds(lane, first0, len0);
    auto tiles_of = [&](uint32_t b) {
        uint32_t first = first0, len = len0;
        if (b >= 64u) bounds(b, first, len);
        return (len + rows - 1u) / rows;
    };
    auto at_least = [&](uint32_t level) {  // tiles of all sequences from this level on
        uint32_t n = 0;
        for (uint32_t b = lane; b < a.batch; b += 64u) {
            const uint32_t t = tiles_of(b);
            n += t > level ? t - level : 0u;
        }
        return (uint32_t)__builtin_amdgcn_readfirstlane((int)wave_reduce(n, [](uint32_t x, uint32_t y) { return x + y; }));
    };
    Item it{};
    uint32_t lo = 0u, hi = (a.tokens + rows - 1u) / rows;  // at_least(lo) > id >= at_least(hi)
    if (at_least(0u) <= id) return it;
    while (hi - lo > 1u) {
        const uint32_t mid = (lo + hi) / 2u;
        if (at_least(mid) > id) lo = mid;
        else hi = mid;
    }
    uint32_t rank = id - at_least(lo + 1u);
    for (uint32_t b0 = 0; b0 < a.batch; b0 += 64u) {
        const uint32_t b = b0 + lane;
        const unsigned long long have = __ballot(b < a.batch && tiles_of(b) > lo);
        const uint32_t n = (uint32_t)__popcll(have);
        if (rank >= n) {
            rank -= n;
            continue;
        }
        const unsigned long long mine = __ballot(((have >> lane) & 1ull) && (uint32_t)__popcll(have & ((1ull << lane) - 1ull)) == rank);
        const uint32_t found = b0 + (uint32_t)__ffsll(mine) - 1u;
        bounds(found, it.first, it.len);
        it.first = (uint32_t)__builtin_amdgcn_readfirstlane((int)it.first);
        it.len = (uint32_t)__builtin_amdgcn_readfirstlane((int)it.len);
        it.tile = lo;
        it.exists = true;
        break;
    }
    return it;
}

// A row's running maximum (times scale) and sum, and the weights of a block's 16 scores of a lane.
struct Softmax {
    float m = kNegInf, l = 0.0f;
    // Scores to weights; true where the sums have to be multiplied by alpha first.
    __device__ inline bool weights(f32x16& s, float c, float& alpha) {
        float top = kNegInf;
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, s[r]);
        top = halves_max(top) * c;
        const bool moves = __any(top > m + kSlack || (m == kNegInf && top > kNegInf));
        alpha = 1.0f;
        if (moves) {
            const float now = fmaxf(m, top);
            alpha = now == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(m - now);
            m = now;
            l *= alpha;
        }
        const float zero = m == kNegInf ? 0.0f : m;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, -zero));
            l += s[r];
        }
        return moves;
    }
};

__device__ inline bool not_finite(float v) { return !(fabsf(v) < __builtin_inff()); }
// Whether one of two BF16 numbers is infinite or NaN, and the pair with 0 in its place
__device__ inline bool odd_pair(uint32_t w) { return (w & 0x7F80u) == 0x7F80u || (w & 0x7F800000u) == 0x7F800000u; }
__device__ inline uint32_t clean_pair(uint32_t w) {
    if ((w & 0x7F80u) == 0x7F80u) w &= 0xFFFF0000u;
    if ((w & 0x7F800000u) == 0x7F800000u) w &= 0x0000FFFFu;
    return w;
}

template <int D, bool F32>
struct Shared {
    union {
        float4 q[F32 ? D / 8 : 1][64];                 // FP32 queries as second operands
        uint4 v[F32 ? 1 : kWaves][kKeys * D / 8];      // a wave's block of BF16 values, [key][D]
        float sums[kWaves][kRows][68];
    };
    float m[kWaves][kRows], l[kWaves][kRows];
};

template <int D, bool F32>
__global__ __launch_bounds__(kThreads, D <= 256 ? 2 : 1) void k_prompt(const PromptArgs a) {
    __shared__ Shared<D, F32> sh;
    const uint32_t lane = threadIdx.x & 63u, col = lane & 31u, half = lane >> 5;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // heads change fastest, the key/value heads before the heads that share one
    const uint32_t turn = blockIdx.x % a.q_heads, kv_head = turn % a.kv_heads, head = kv_head * a.group + turn / a.kv_heads;
    const Item it = locate(a, blockIdx.x / a.q_heads, kRows);
    if (!it.exists) return;
    const uint32_t row0 = it.tile * kRows, pos = row0 + col, last = it.len - 1u;
    const uint32_t end = min(it.len, row0 + kRows);
    const uint32_t begin = a.window && row0 + 1u > a.window ? row0 + 1u - a.window : 0u;
    const uint32_t lo = a.window && pos + 1u > a.window ? pos + 1u - a.window : 0u;  // what this lane's row sees: lo .. pos
    // rows from full0 .. full1 on see every key of a block that lies between them
    const uint32_t all_lo = a.window && end > a.window ? end - a.window : 0u;

    typedef typename std::conditional<F32, float, uint16_t>::type E;
    const E* q = static_cast<const E*>(a.q) + (uint64_t)(it.first + min(pos, last)) * a.q_stride + (uint64_t)head * D;
    const E* k = static_cast<const E*>(a.k) + (uint64_t)it.first * a.k_stride + (uint64_t)kv_head * D;
    const E* v = static_cast<const E*>(a.v) + (uint64_t)it.first * a.v_stride + (uint64_t)kv_head * D;

    Frag qf[F32 ? 1 : D / 16];
    if constexpr (F32) {
        for (int i = wave; i < D / 8; i += kWaves) {
            uint4 x = *reinterpret_cast<const uint4*>(q + i * 8 + half * 4u);
            x.x ^= a.flip, x.y ^= a.flip, x.z ^= a.flip, x.w ^= a.flip;
            sh.q[i][lane] = __builtin_bit_cast(float4, x);
        }
        __syncthreads();
    } else {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            qf[i].u = *reinterpret_cast<const uint4*>(q + i * 16 + half * 8u);
#pragma unroll
            for (int j = 0; j < 4; ++j) qf[i].w[j] ^= a.flip;
        }
    }

    f32x16 o[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) o[i] = zeros();
    Softmax sm;

    for (uint32_t base = begin / kKeys * kKeys + wave * kKeys; base < end; base += kWaves * kKeys) {
        const bool masked = base < all_lo || base + kKeys > row0 + 1u;
        // ---- scores
        const E* krow = k + (uint64_t)min(base + col, last) * a.k_stride;
        f32x16 s = zeros();
        if constexpr (F32) {
#pragma unroll 8
            for (int i = 0; i < D / 8; ++i) {
                const float4 x = *reinterpret_cast<const float4*>(krow + i * 8 + half * 4u), y = sh.q[i][lane];
                s = __builtin_amdgcn_mfma_f32_32x32x2f32(x.x, y.x, s, 0, 0, 0);
                s = __builtin_amdgcn_mfma_f32_32x32x2f32(x.y, y.y, s, 0, 0, 0);
                s = __builtin_amdgcn_mfma_f32_32x32x2f32(x.z, y.z, s, 0, 0, 0);
                s = __builtin_amdgcn_mfma_f32_32x32x2f32(x.w, y.w, s, 0, 0, 0);
            }
        } else {
            // the values' block on its way to LDS meanwhile, whole rows of D
            constexpr int kLoads = kKeys * D / 512;
            uint4 held[kLoads];
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const uint32_t at = i * 512u + lane * 8u, row = at / D;
                held[i] = *reinterpret_cast<const uint4*>(v + (uint64_t)min(base + row, last) * a.v_stride + at % D);
            }
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
                Frag x;
                x.u = *reinterpret_cast<const uint4*>(krow + i * 16 + half * 8u);
                s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x.b, qf[i].b, s, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < kLoads; ++i) sh.v[wave][i * 64u + lane] = held[i];
        }
        if (masked) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const uint32_t key = base + element(r, half);
                if (key < lo || key > pos) s[r] = kNegInf;
            }
        }
        // ---- weights
        float alpha;
        if (sm.weights(s, a.scale_log2e, alpha)) {
#pragma unroll
            for (int i = 0; i < D / 32; ++i) o[i] *= alpha;
        }
        // ---- weighted values. A value that is infinite or NaN has no part in a row that does not see it, where
        // its weight is 0: such values are taken out of the product and added to the rows that see them.
        bool odd = false;
        if constexpr (F32) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const E* vrow = v + (uint64_t)min(base + element(r, half), last) * a.v_stride + col;
#pragma unroll
                for (int i = 0; i < D / 32; ++i) {
                    float x = vrow[i * 32];
                    if (masked && not_finite(x)) odd = true, x = 0.0f;
                    o[i] = __builtin_amdgcn_mfma_f32_32x32x2f32(x, s[r], o[i], 0, 0, 0);
                }
            }
        } else {
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            Frag p[2];
#pragma unroll
            for (int j = 0; j < 8; ++j) p[j >> 2].w[j & 3] = pack_bf16(s[2 * j], s[2 * j + 1]);
            if (masked) {
                bool any = false;
#pragma unroll 4
                for (int i = 0; i < (int)kKeys * D / 512; ++i) {
                    const uint4 x = sh.v[wave][i * 64u + lane];
                    any = any || odd_pair(x.x) || odd_pair(x.y) || odd_pair(x.z) || odd_pair(x.w);
                }
                odd = __any(any);
            }
            // keys 4 half .. and 8 + 4 half .. of 16, columns col of 32: 16 lanes read four keys of 16 columns and
            // get a column each
            const uint16_t* vs = reinterpret_cast<const uint16_t*>(sh.v[wave]) + (4u * half + ((lane & 15u) >> 2)) * D + (lane & 16u) + (lane & 3u) * 4u;
#pragma unroll
            for (int i = 0; i < D / 32; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    Frag x;
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        x.h[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (__attribute__((address_space(3))) short4v*)(vs + (16 * j + 8 * e) * D + i * 32));
                    if (odd) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) x.w[e] = clean_pair(x.w[e]);
                    }
                    o[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x.b, p[j].b, o[i], 0, 0, 0);
                }
        }
        if (masked && __any(odd)) {
#pragma unroll
            for (int i = 0; i < D / 32; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    float add = 0.0f;
#pragma unroll 1
                    for (uint32_t j = 0; j < kKeys; ++j) {
                        const uint32_t key = base + j;
                        if (key < lo || key > pos || key > last) continue;
                        const E x = v[(uint64_t)key * a.v_stride + i * 32 + element(r, half)];
                        float y;
                        if constexpr (F32) y = x;
                        else y = __uint_as_float((uint32_t)x << 16);
                        if (not_finite(y)) add += y;
                    }
                    o[i][r] += add;
                }
        }
    }

    // ---- the four waves join
    sm.l = halves_sum(sm.l);
    if (half == 0u) sh.m[wave][col] = sm.m, sh.l[wave][col] = sm.l;
    __syncthreads();
    float top = fmaxf(fmaxf(sh.m[0][col], sh.m[1][col]), fmaxf(sh.m[2][col], sh.m[3][col]));  // of the lane's row
    const float mine = sm.m == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(sm.m - top);
    const bool counts = sm.m != kNegInf || sm.l != 0.0f;
    // thread tid writes 8 values of row tid / 8
    const uint32_t row = threadIdx.x >> 3, c8 = (threadIdx.x & 7u) * 8u;
    float total = 0.0f;
    top = fmaxf(fmaxf(sh.m[0][row], sh.m[1][row]), fmaxf(sh.m[2][row], sh.m[3][row]));
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w)
        if (sh.l[w][row] != 0.0f) total += sh.l[w][row] * __builtin_amdgcn_exp2f(sh.m[w][row] - top);
    const float by = 1.0f / total;
#pragma unroll
    for (int n = 0; n < D / 64; ++n) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 16; r += 4) {
                const f32x16& x = o[n * 2 + i];
                const float4 y = counts ? make_float4(x[r] * mine, x[r + 1] * mine, x[r + 2] * mine, x[r + 3] * mine) : make_float4(0, 0, 0, 0);
                *reinterpret_cast<float4*>(&sh.sums[wave][col][i * 32 + element(r, half)]) = y;
            }
        __syncthreads();
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            x[i] = 0.0f;
#pragma unroll
            for (uint32_t w = 0; w < kWaves; ++w) x[i] += sh.sums[w][row][c8 + i];
            x[i] *= by;
        }
        if (row0 + row < it.len) {
            E* to = static_cast<E*>(a.out) + (uint64_t)(it.first + row0 + row) * a.out_stride + (uint64_t)head * D + n * 64u + c8;
            if constexpr (F32) {
                *reinterpret_cast<float4*>(to) = make_float4(x[0], x[1], x[2], x[3]);
                *reinterpret_cast<float4*>(to + 4) = make_float4(x[4], x[5], x[6], x[7]);
            } else {
                *reinterpret_cast<uint4*>(to) = make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
            }
        }
    }
}

template <int D>
void launch_dim(const PromptArgs& a, int dtype, uint32_t items, hipStream_t st) {
    if (dtype == TURBO_HIDDEN_F32) hipLaunchKernelGGL((k_prompt<D, true>), dim3(items), dim3(kThreads), 0, st, a);
    else hipLaunchKernelGGL((k_prompt<D, false>), dim3(items), dim3(kThreads), 0, st, a);
}

}  // namespace

void launch_prompt(const PromptArgs& a, uint32_t head_dim, int dtype, uint32_t cus, hipStream_t st) {
    (void)cus;
    // as many tiles as the sequences can have: all but one row of each sequence's last tile may be missing
    const uint64_t tiles = ((uint64_t)a.tokens + (uint64_t)a.batch * (kRows - 1u)) / kRows;
    const uint32_t items = grid_blocks(tiles * a.q_heads);
    switch (head_dim) {
        case 64u: launch_dim<64>(a, dtype, items, st); break;
        case 128u: launch_dim<128>(a, dtype, items, st); break;
        case 256u: launch_dim<256>(a, dtype, items, st); break;
        default: launch_dim<512>(a, dtype, items, st); break;
    }
    check_hip(hipGetLastError(), "prompt attention");
}

}  // namespace tdt

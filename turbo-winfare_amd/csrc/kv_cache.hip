// Norms and rotation of query and key heads, and the quantised cache's write and read.
//
// k_qkv: a workgroup takes one role (queries, keys or values), a run of tokens and a run of heads. A
//   head sits in head_dim / E neighbouring lanes, E values (16 bytes) to a lane where that leaves at
//   most a wave, so a wave holds one to eight heads at once; the mean square is a reduction over those
//   lanes, and the other value of a pair in halves comes from the lane rotary_dim / 2 / E away. The
//   sine and cosine of a token's angles are computed once and used for all the heads a wave takes.
//   Angle: position * turns[i] modulo 2^64 is the fraction of a turn in fixed point, exact whatever the
//   position; its quadrant is removed as an integer and the remainder, at most pi / 4, goes through the
//   Taylor series to degree 9 and 10 (first term left out below 2^-28).
//   Keys and values for the cache: the group's range over 64 / E lanes, then the codes. Keys are stored
//   straight from the registers, E values to a lane. A value's 32 tokens are neighbours in the cache, so
//   values pass through LDS and four tokens in a row become one 4-byte store; a decode step's lone
//   tokens are single bytes.
// k_kv_read is its inverse.
#include <stdexcept>

#include "dt_internal.h"
#include "dt_kv.h"

namespace tdt {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kMaxChunk = 32;      // tokens of a workgroup
constexpr uint32_t kMaxHeads = 8;       // heads of a workgroup at most (LDS of the values' codes)
constexpr uint32_t kStageBytes = 32768; // LDS for the codes of a workgroup's tokens and heads

template <class T> struct Vec;
template <> struct Vec<float> {
    template <int E> static __device__ void load(const float* p, float (&x)[E]) {
#pragma unroll
        for (int i = 0; i < E; i += 4) {
            const float4 v = *reinterpret_cast<const float4*>(p + i);
            x[i] = v.x, x[i + 1] = v.y, x[i + 2] = v.z, x[i + 3] = v.w;
        }
    }
    template <int E> static __device__ void store(float* p, const float (&x)[E]) {
#pragma unroll
        for (int i = 0; i < E; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
    }
};
// BF16 as its bits; rounding to nearest even, NaN stays NaN
__device__ inline uint32_t bf16_bits(float f) {
    const uint32_t u = __float_as_uint(f);
    if ((u & 0x7FFFFFFFu) > 0x7F800000u) return (u >> 16) | 0x40u;
    return (u + 0x7FFFu + ((u >> 16) & 1u)) >> 16;
}
template <> struct Vec<uint16_t> {
    template <int E> static __device__ void load(const uint16_t* p, float (&x)[E]) {
        static_assert(E == 8);
        const uint4 v = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
    template <int E> static __device__ void store(uint16_t* p, const float (&x)[E]) {
        static_assert(E == 8);
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = bf16_bits(x[2 * i]) | bf16_bits(x[2 * i + 1]) << 16;
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
};

// op over N neighbouring lanes (N a power of two), the result in each of them.
template <int N, class Op>
__device__ inline float lanes_reduce(float v, Op op) {
    if (N >= 2) v = op(v, dpp_mov<dpp::kXor1>(v));
    if (N >= 4) v = op(v, dpp_mov<dpp::kXor2>(v));
    if (N >= 8) v = op(v, dpp_mov<dpp::kHalfMirror>(v));
    if (N >= 16) v = op(v, dpp_mov<dpp::kRor8>(v));
    if (N >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
    if (N >= 64) {
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
    return v;
}

// cos and sin of `turn` / 2^32 turns
__device__ inline void turn_cos_sin(uint32_t turn, float& c, float& s) {
    const uint32_t quadrant = (turn + 0x20000000u) >> 30;
    const float x = (float)(int32_t)(turn - (quadrant << 30)) * 1.46291807926715968e-9f;  // 2 pi / 2^32
    const float z = x * x;
    const float sn = x + x * z * (-1.0f / 6 + z * (1.0f / 120 + z * (-1.0f / 5040 + z * (1.0f / 362880))));
    const float cs = 1.0f + z * (-0.5f + z * (1.0f / 24 + z * (-1.0f / 720 + z * (1.0f / 40320 + z * (-1.0f / 3628800)))));
    const float a = (quadrant & 1u) ? sn : cs, b = (quadrant & 1u) ? cs : sn;
    c = ((quadrant + 1u) & 2u) ? -a : a;
    s = (quadrant & 2u) ? -b : b;
}

// x rounded to BF16 upwards or downwards: the low half is cut off, which rounds towards zero, and one
// unit is added where that went the wrong way (|x| is far below the largest number).
__device__ inline float bf16_outward(float x, bool up) {
    const uint32_t u = __float_as_uint(x), cut = u & 0xFFFF0000u;
    const bool right = cut == u || (up ? (u >> 31) != 0u : (u >> 31) == 0u);
    return __uint_as_float(right ? cut : cut + 0x10000u);
}

// The codes of a lane's E values and the group's word of scale and bias. N lanes share a group. A group
// with a value of 2^103 or more, infinite or NaN is NaN: below that a score's sum over 512 products with
// queries of 2^15 stays in FP32.
template <int E, int N>
__device__ inline uint32_t quantise(const float (&x)[E], uint32_t top, uint32_t (&code)[E]) {
    float lo = x[0], hi = x[0];
    uint32_t mag = 0u;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        lo = fminf(lo, x[i]);
        hi = fmaxf(hi, x[i]);
        mag = max(mag, __float_as_uint(x[i]) & 0x7FFFFFFFu);
    }
    const uint32_t lane = threadIdx.x & 63u;
    const unsigned long long odd = __ballot(mag >= 0x73000000u) >> (lane & ~(uint32_t)(N - 1));
    const bool finite = (odd & ((1ull << N) - 1ull)) == 0ull;
    lo = lanes_reduce<N>(lo, [](float a, float b) { return fminf(a, b); });
    hi = lanes_reduce<N>(hi, [](float a, float b) { return fmaxf(a, b); });
    const float bias = bf16_outward(lo, false);
    const float scale = fmaxf(bf16_outward((hi - bias) / (float)top, true), 0x1p-126f);
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const float t = rintf((x[i] - bias) / scale);
        code[i] = finite ? (uint32_t)fminf(fmaxf(t, 0.0f), (float)top) : 0u;
    }
    return finite ? __float_as_uint(scale) | __float_as_uint(bias) >> 16 : 0x7FC07FC0u;
}

// What a workgroup knows of its tokens' places (slot 0xFFFFFFFF: none), and which of them begin four
// consecutive slots of one aligned quad (2), lie inside such a quad (1) or stand alone (0).
struct Places {
    uint32_t slot[kMaxChunk];
    uint32_t quad[kMaxChunk];
};

__device__ inline void find_places(Places& p, const uint32_t* slots, uint32_t t0, uint32_t n, uint64_t limit) {
    const uint32_t tid = threadIdx.x;
    if (tid < kMaxChunk) {
        const uint32_t s = tid < n ? slots[t0 + tid] : 0xFFFFFFFFu;
        p.slot[tid] = s < limit ? s : 0xFFFFFFFFu;
    }
    __syncthreads();
    if (tid < kMaxChunk) {
        auto leads = [&](uint32_t i) {
            const uint32_t s = p.slot[i];
            return i + 3u < n && s != 0xFFFFFFFFu && (s & 3u) == 0u && p.slot[i + 1] == s + 1u && p.slot[i + 2] == s + 2u &&
                   p.slot[i + 3] == s + 3u;
        };
        uint32_t kind = leads(tid) ? 2u : 0u;
        for (uint32_t back = 1; back <= 3u && kind == 0u; ++back)
            if (tid >= back && leads(tid - back)) kind = 1u;
        p.quad[tid] = kind;
    }
    __syncthreads();
}

__device__ inline uint8_t* record_of(const KvView& kv, uint32_t slot, uint32_t head) {
    const uint32_t page = slot >> kv.page_shift, at = slot & ((1u << kv.page_shift) - 1u);
    return kv.base + kv_record_at(kv, page, head, at / kKvBlock);
}

// Values from LDS codes [head][chunk][head_dim] to the cache.
template <int NG, uint32_t BITS>
__device__ inline void store_values(const KvView& kv, const Places& p, const uint8_t* stage, uint32_t n, uint32_t head0,
                                    uint32_t heads) {
    constexpr uint32_t D = NG * 64u;
    constexpr uint32_t W = BITS == 8u ? D : D / 2u;  // bytes of a token
    for (uint32_t i = threadIdx.x; i < heads * n * W; i += kThreads) {
        const uint32_t w = i % W, t = (i / W) % n, h = i / (W * n);
        const uint32_t kind = p.quad[t], slot = p.slot[t];
        if (slot == 0xFFFFFFFFu || kind == 1u) continue;
        const uint32_t d = BITS == 8u ? w : (w & 15u) | (w & ~15u) << 1;  // 4 bits: values d and d + 16
        const uint8_t* src = stage + (h * n + t) * D + d;
        uint8_t* dst = record_of(kv, slot, head0 + h) + kv_part_bytes(NG, BITS) + kv_value_byte(BITS, slot & 31u, d);
        uint32_t word = 0u;
        const uint32_t many = kind == 2u ? 4u : 1u;
        for (uint32_t j = 0; j < many; ++j) {
            const uint32_t c = BITS == 8u ? src[j * D] : src[j * D] | (uint32_t)src[j * D + 16u] << 4;
            word |= c << (8u * j);
        }
        if (kind == 2u) *reinterpret_cast<uint32_t*>(dst) = word;
        else *dst = (uint8_t)word;
    }
}

template <int NG, class T, int E, uint32_t BITS>
__global__ __launch_bounds__(kThreads) void k_qkv(const QkvArgs a, uint32_t chunk, uint32_t heads_per, uint32_t q_parts,
                                                  uint32_t kv_parts) {
    constexpr uint32_t D = NG * 64u, LPH = D / E, HP = 64u / LPH;  // lanes per head, heads per wave
    extern __shared__ uint8_t stage[];
    __shared__ Places places;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t t0 = blockIdx.x * chunk, n = min(chunk, a.tokens - t0);
    uint32_t part = blockIdx.y;
    const uint32_t role = part < q_parts ? 0u : part < q_parts + kv_parts ? 1u : 2u;
    part -= role == 0u ? 0u : role == 1u ? q_parts : q_parts + kv_parts;
    const uint32_t all = role == 0u ? a.q_heads : a.kv_heads;
    const uint32_t h0 = part * heads_per, heads = min(heads_per, all - h0);
    const bool stored = BITS != 0u && role != 0u;
    if (stored) find_places(places, a.slots, t0, n, a.kv.slots);

    const T* src = static_cast<const T*>(role == 0u ? a.q : role == 1u ? a.k : a.v);
    T* dst = static_cast<T*>(role == 0u ? a.q_out : role == 1u ? a.k_out : nullptr);
    const uint64_t stride = role == 0u ? a.q_stride : role == 1u ? a.k_stride : a.v_stride;
    const uint64_t out_stride = role == 0u ? a.q_out_stride : a.k_out_stride;
    const uint16_t* weight = role == 0u ? a.q_norm : role == 1u ? a.k_norm : nullptr;
    const bool normed = (a.norms >> role) & 1u;
    const uint32_t rot = role == 2u || !a.turns ? 0u : a.rotary_dim;
    const uint32_t d0 = (lane % LPH) * E, sub = lane / LPH;

    float w[E];
#pragma unroll
    for (int i = 0; i < E; ++i) w[i] = weight && normed ? bf16_to_f32(weight[d0 + i]) : 1.0f;
    // the lane with the other values of this lane's pairs (halves), and the sign of their sines
    const uint32_t half = rot / 2u;
    const bool turning = d0 < rot, first = d0 < half;
    const uint32_t other = !turning || a.pairs ? lane : first ? lane + half / E : lane - half / E;

    // four tokens at a time, or the heads of a token divided among the waves
    const uint32_t tstep = chunk >= 4u ? 4u : 1u, tfirst = chunk >= 4u ? wave : 0u;
    const uint32_t pstep = (chunk >= 4u ? 1u : 4u) * HP, pfirst = chunk >= 4u ? 0u : wave * HP;
    for (uint32_t t = tfirst; t < n; t += tstep) {
        float cs[E], sn[E];
        if (rot) {
            const uint64_t pos = a.positions[t0 + t];
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const uint32_t d = d0 + i;
                cs[i] = 1.0f, sn[i] = 0.0f;
                if (d < rot && !(a.pairs && (i & 1))) {
                    const uint64_t turn = pos * a.turns[a.pairs ? d / 2u : d < half ? d : d - half];
                    turn_cos_sin((uint32_t)((turn + 0x80000000ull) >> 32), cs[i], sn[i]);
                }
            }
        }
        for (uint32_t h = pfirst; h < heads; h += pstep) {
            const bool here = h + sub < heads;  // lanes past the last head take it again and store nothing
            const uint32_t head = h0 + (here ? h + sub : heads - 1u);
            float x[E];
            Vec<T>::template load<E>(src + (uint64_t)(t0 + t) * stride + (uint64_t)head * D + d0, x);
            if (normed) {
                float sq = 0.0f;
#pragma unroll
                for (int i = 0; i < E; ++i) sq = fmaf(x[i], x[i], sq);
                sq = lanes_reduce<LPH>(sq, [](float p, float q) { return p + q; });
                const float r = 1.0f / sqrtf(sq * (1.0f / D) + a.eps);
#pragma unroll
                for (int i = 0; i < E; ++i) x[i] = x[i] * r * w[i];
            }
            if (rot) {
                if (a.pairs) {
#pragma unroll
                    for (int i = 0; i < E; i += 2) {
                        const float u = x[i], v = x[i + 1];
                        x[i] = u * cs[i] - v * sn[i];
                        x[i + 1] = v * cs[i] + u * sn[i];
                    }
                } else {
                    float y[E];
#pragma unroll
                    for (int i = 0; i < E; ++i) y[i] = __shfl(x[i], (int)other);
#pragma unroll
                    for (int i = 0; i < E; ++i) {
                        if (turning) x[i] = first ? x[i] * cs[i] - y[i] * sn[i] : x[i] * cs[i] + y[i] * sn[i];
                    }
                }
            }
            if (dst && here) Vec<T>::template store<E>(dst + (uint64_t)(t0 + t) * out_stride + (uint64_t)head * D + d0, x);
            if (stored) {
                uint32_t code[E];
                constexpr int N = 64 / E;
                const uint32_t word = quantise<E, N>(x, (1u << BITS) - 1u, code);
                const uint32_t slot = places.slot[t];
                if (here && slot != 0xFFFFFFFFu) {
                    uint8_t* rec = record_of(a.kv, slot, head);
                    if (lane % N == 0u)
                        *reinterpret_cast<uint32_t*>(rec + 2u * kv_part_bytes(NG, BITS) +
                                                     kv_scale_byte(NG, role - 1u, slot & 31u, d0 / 64u)) = word;
                    if (role == 1u) {
                        uint8_t* at = rec + kv_key_byte(BITS, slot & 31u, d0);
                        if (BITS == 8u) {
#pragma unroll
                            for (int i = 0; i < E; i += 4)
                                *reinterpret_cast<uint32_t*>(at + i) = code[i] | code[i + 1] << 8 | code[i + 2] << 16 | code[i + 3] << 24;
                        } else {
#pragma unroll
                            for (int i = 0; i < E; i += 4)
                                *reinterpret_cast<uint16_t*>(at + i / 2) =
                                    (uint16_t)(code[i] | code[i + 1] << 4 | code[i + 2] << 8 | code[i + 3] << 12);
                        }
                    }
                }
                if (role == 2u && here) {
                    uint8_t* at = stage + ((h + sub) * n + t) * D + d0;
#pragma unroll
                    for (int i = 0; i < E; i += 4)
                        *reinterpret_cast<uint32_t*>(at + i) = code[i] | code[i + 1] << 8 | code[i + 2] << 16 | code[i + 3] << 24;
                }
            }
        }
    }
    if constexpr (BITS != 0u) {
        if (role == 2u) {
            __syncthreads();
            store_values<NG, BITS>(a.kv, places, stage, n, h0, heads);
        }
    }
}

template <int NG, class T, int E, uint32_t BITS>
__global__ __launch_bounds__(kThreads) void k_kv_read(const KvReadArgs a, uint32_t chunk, uint32_t heads_per, uint32_t parts) {
    constexpr uint32_t D = NG * 64u, LPH = D / E, HP = 64u / LPH;
    constexpr uint32_t W = BITS == 8u ? D : D / 2u;
    extern __shared__ uint8_t stage[];
    __shared__ Places places;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t t0 = blockIdx.x * chunk, n = min(chunk, a.tokens - t0);
    const bool values = !a.k || blockIdx.y >= parts;
    const uint32_t h0 = (blockIdx.y % parts) * heads_per, heads = min(heads_per, a.kv.heads - h0);
    T* dst = static_cast<T*>(values ? a.v : a.k);
    const uint64_t stride = values ? a.v_stride : a.k_stride;
    find_places(places, a.slots, t0, n, a.kv.slots);
    if (values) {
        for (uint32_t i = threadIdx.x; i < heads * n * W; i += kThreads) {
            const uint32_t w = i % W, t = (i / W) % n, h = i / (W * n);
            const uint32_t kind = places.quad[t], slot = places.slot[t];
            if (slot == 0xFFFFFFFFu || kind == 1u) continue;
            const uint32_t d = BITS == 8u ? w : (w & 15u) | (w & ~15u) << 1;
            const uint8_t* src = record_of(a.kv, slot, h0 + h) + kv_part_bytes(NG, BITS) + kv_value_byte(BITS, slot & 31u, d);
            const uint32_t word = kind == 2u ? *reinterpret_cast<const uint32_t*>(src) : *src;
            const uint32_t many = kind == 2u ? 4u : 1u;
            for (uint32_t j = 0; j < many; ++j) {
                const uint32_t c = (word >> (8u * j)) & 255u;
                uint8_t* at = stage + (h * n + t + j) * D + d;
                if (BITS == 8u) at[0] = (uint8_t)c;
                else at[0] = (uint8_t)(c & 15u), at[16] = (uint8_t)(c >> 4);
            }
        }
        __syncthreads();
    }
    const uint32_t d0 = (lane % LPH) * E, sub = lane / LPH;
    const uint32_t tstep = chunk >= 4u ? 4u : 1u, tfirst = chunk >= 4u ? wave : 0u;
    const uint32_t pstep = (chunk >= 4u ? 1u : 4u) * HP, pfirst = chunk >= 4u ? 0u : wave * HP;
    for (uint32_t t = tfirst; t < n; t += tstep) {
        for (uint32_t h = pfirst + sub; h < heads; h += pstep) {
            const uint32_t slot = places.slot[t];
            float x[E];
            if (slot == 0xFFFFFFFFu) {
#pragma unroll
                for (int i = 0; i < E; ++i) x[i] = __builtin_nanf("");
            } else {
                const uint8_t* rec = record_of(a.kv, slot, h0 + h);
                const uint32_t word = *reinterpret_cast<const uint32_t*>(
                    rec + 2u * kv_part_bytes(NG, BITS) + kv_scale_byte(NG, values ? 1u : 0u, slot & 31u, d0 / 64u));
                const float scale = __uint_as_float(word & 0xFFFF0000u), bias = __uint_as_float(word << 16);
                uint32_t code[E];
                if (values || BITS == 8u) {
                    const uint8_t* at = values ? stage + (h * n + t) * D + d0 : rec + kv_key_byte(BITS, slot & 31u, d0);
#pragma unroll
                    for (int i = 0; i < E; i += 4) {
                        const uint32_t four = *reinterpret_cast<const uint32_t*>(at + i);
#pragma unroll
                        for (int j = 0; j < 4; ++j) code[i + j] = (four >> (8 * j)) & 255u;
                    }
                } else {
                    const uint8_t* at = rec + kv_key_byte(BITS, slot & 31u, d0);
#pragma unroll
                    for (int i = 0; i < E; i += 4) {
                        const uint32_t four = *reinterpret_cast<const uint16_t*>(at + i / 2);
#pragma unroll
                        for (int j = 0; j < 4; ++j) code[i + j] = (four >> (4 * j)) & 15u;
                    }
                }
#pragma unroll
                for (int i = 0; i < E; ++i) x[i] = fmaf((float)code[i], scale, bias);
            }
            Vec<T>::template store<E>(dst + (uint64_t)(t0 + t) * stride + (uint64_t)(h0 + h) * D + d0, x);
        }
    }
}

// Tokens and heads of a workgroup. A longer run of tokens turns the values' bytes into 4-byte stores and
// a longer run of heads shares a token's sines, but the card needs a thousand workgroups to be busy:
// the run of tokens is halved from 32, then the heads from as many as LDS holds, until there are.
struct Shape {
    uint32_t chunk, heads;
};
Shape shape_for(uint32_t tokens, uint32_t heads, uint32_t all_heads, uint32_t head_dim, uint32_t wave_heads) {
    Shape s{kMaxChunk, heads < kMaxHeads ? heads : kMaxHeads};
    while (s.heads > 1u && s.chunk * s.heads * head_dim > kStageBytes) s.heads = (s.heads + 1u) / 2u;
    auto groups = [&] { return (uint64_t)((tokens + s.chunk - 1u) / s.chunk) * ((all_heads + s.heads - 1u) / s.heads); };
    while (s.chunk > 1u && groups() < 1024u) s.chunk /= 2u;
    while (s.heads > wave_heads && groups() < 1024u) s.heads = (s.heads + 1u) / 2u;
    return s;
}

template <int NG, class T, int E>
void launch_qkv_typed(const QkvArgs& a, hipStream_t st) {
    constexpr uint32_t D = NG * 64u;
    const bool keys = a.k != nullptr, values = a.v != nullptr && a.kv.base != nullptr;
    const uint32_t all = (a.q ? a.q_heads : 0u) + (keys ? a.kv_heads : 0u) + (values ? a.kv_heads : 0u);
    const Shape s = shape_for(a.tokens, a.q ? max(a.q_heads, a.kv_heads) : a.kv_heads, all, D, 64u / (D / E));
    const uint32_t qp = a.q ? (a.q_heads + s.heads - 1u) / s.heads : 0u;
    const uint32_t kp = (a.kv_heads + s.heads - 1u) / s.heads;
    const dim3 grid((a.tokens + s.chunk - 1u) / s.chunk, qp + (keys ? kp : 0u) + (values ? kp : 0u));
    const uint32_t key_parts = keys ? kp : 0u;
    const size_t lds = values ? (size_t)s.chunk * s.heads * D : 0u;
    if (!a.kv.base) hipLaunchKernelGGL((k_qkv<NG, T, E, 0u>), grid, dim3(kThreads), 0, st, a, s.chunk, s.heads, qp, key_parts);
    else if (a.kv.bits == 8u) hipLaunchKernelGGL((k_qkv<NG, T, E, 8u>), grid, dim3(kThreads), lds, st, a, s.chunk, s.heads, qp, key_parts);
    else hipLaunchKernelGGL((k_qkv<NG, T, E, 4u>), grid, dim3(kThreads), lds, st, a, s.chunk, s.heads, qp, key_parts);
}

template <int NG, class T, int E>
void launch_read_typed(const KvReadArgs& a, hipStream_t st) {
    constexpr uint32_t D = NG * 64u;
    const uint32_t both = (a.k ? 1u : 0u) + (a.v ? 1u : 0u);
    const Shape s = shape_for(a.tokens, a.kv.heads, a.kv.heads * both, D, 64u / (D / E));
    const uint32_t parts = (a.kv.heads + s.heads - 1u) / s.heads;
    const dim3 grid((a.tokens + s.chunk - 1u) / s.chunk, parts * both);
    const size_t lds = a.v ? (size_t)s.chunk * s.heads * D : 0u;
    if (a.kv.bits == 8u) hipLaunchKernelGGL((k_kv_read<NG, T, E, 8u>), grid, dim3(kThreads), lds, st, a, s.chunk, s.heads, parts);
    else hipLaunchKernelGGL((k_kv_read<NG, T, E, 4u>), grid, dim3(kThreads), lds, st, a, s.chunk, s.heads, parts);
}

}  // namespace

void launch_qkv(const QkvArgs& a, uint32_t head_dim, int dtype, hipStream_t st) {
    if (dtype == TURBO_HIDDEN_BF16) {
        if (head_dim == 64u) launch_qkv_typed<1, uint16_t, 8>(a, st);
        else if (head_dim == 128u) launch_qkv_typed<2, uint16_t, 8>(a, st);
        else if (head_dim == 256u) launch_qkv_typed<4, uint16_t, 8>(a, st);
        else launch_qkv_typed<8, uint16_t, 8>(a, st);
    } else {
        if (head_dim == 64u) launch_qkv_typed<1, float, 4>(a, st);
        else if (head_dim == 128u) launch_qkv_typed<2, float, 4>(a, st);
        else if (head_dim == 256u) launch_qkv_typed<4, float, 4>(a, st);
        else launch_qkv_typed<8, float, 8>(a, st);
    }
    check_hip(hipGetLastError(), "norms, rotation and cache write");
}

void launch_kv_read(const KvReadArgs& a, uint32_t head_dim, int dtype, hipStream_t st) {
    if (dtype == TURBO_HIDDEN_BF16) {
        if (head_dim == 64u) launch_read_typed<1, uint16_t, 8>(a, st);
        else if (head_dim == 128u) launch_read_typed<2, uint16_t, 8>(a, st);
        else if (head_dim == 256u) launch_read_typed<4, uint16_t, 8>(a, st);
        else launch_read_typed<8, uint16_t, 8>(a, st);
    } else {
        if (head_dim == 64u) launch_read_typed<1, float, 4>(a, st);
        else if (head_dim == 128u) launch_read_typed<2, float, 4>(a, st);
        else if (head_dim == 256u) launch_read_typed<4, float, 4>(a, st);
        else launch_read_typed<8, float, 8>(a, st);
    }
    check_hip(hipGetLastError(), "cache read");
}

}  // namespace tdt

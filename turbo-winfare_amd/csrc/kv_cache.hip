// Norms and rotation of query and key heads, and the quantised cache's write and read.
//
// k_qkv has two kinds of workgroups. Both take a run of tokens and a run of heads; a head sits in head_dim / E
// neighbouring lanes, E values (16 bytes) to a lane where that leaves at most a wave, so a wave holds one
// to eight heads at once, and the mean square and a group's range are reductions over neighbouring lanes.
// The next heads' values are on their way while these are worked on.
//   Queries and keys: the sines of the run's tokens are computed once, into LDS, and serve all its heads.
//     Angle: position * turns[i] modulo 2^64 is the fraction of a turn in fixed point, exact for turns[i]
//     (rounded to 2^-64) whatever the position; its quadrant is removed as an integer and the remainder, at
//     most pi / 4, goes through the Taylor series to degree 9 and 10 (first term left out below 2^-28). The other value of a pair in
//     halves comes from the lane rotary_dim / 2 / E away. A key's codes go to the cache straight from the
//     registers.
//   Values: 32 tokens are neighbours in the cache, so the codes pass through LDS, and four tokens in a row
//     are transposed in registers to one 4-byte store per value; a decode step's lone tokens are bytes.
// The cache's write takes about 200 instructions per 512 values: at 4,001 tokens the vector units are busy 65 % of its
// time, and waves wait 43 % of theirs, so divisions are products with a group's reciprocal and one correction step.
// k_kv_read: a thread takes four values of four tokens, 4-byte loads where the tokens are neighbours.
#include <stdexcept>

#include "dt_internal.h"
#include "dt_kv.h"

namespace tdt {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kMaxChunk = 32;      // tokens of a workgroup
constexpr uint32_t kMaxHeads = 8;       // heads of a workgroup
constexpr uint32_t kGroups = 1000u;     // workgroups that a call is divided into, at least (shape_for)
constexpr uint32_t kLdsBytes = 32768;   // for a workgroup's sines, or its values' codes

typedef float float2v __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
// Two numbers rounded to BF16 (nearest even, NaN stays NaN), one instruction on gfx950.
__device__ inline uint32_t pack_bf16(float lo, float hi) {
    union {
        bf16x2 b;
        uint32_t u;
    } x;
    x.b = __builtin_convertvector((float2v{lo, hi}), bf16x2);
    return x.u;
}

// E values of a lane as they lie in memory, and as FP32.
template <class T, int E>
struct Vec {
    static constexpr int kWords = E * (int)sizeof(T) / 16;
    uint4 raw[kWords];
    __device__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) raw[i] = reinterpret_cast<const uint4*>(p)[i];
    }
    __device__ void get(float (&x)[E]) const {
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (sizeof(T) == 4) x[4 * i + j] = __uint_as_float(w[j]);
                else x[8 * i + 2 * j] = __uint_as_float(w[j] << 16), x[8 * i + 2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
            }
        }
    }
    static __device__ void store(T* p, const float (&x)[E]) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (sizeof(T) == 4) w[j] = __float_as_uint(x[4 * i + j]);
                else w[j] = pack_bf16(x[8 * i + 2 * j], x[8 * i + 2 * j + 1]);
            }
            reinterpret_cast<uint4*>(p)[i] = make_uint4(w[0], w[1], w[2], w[3]);
        }
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

// 1 / sqrt(mean(x^2) + eps) of a head that lies in D / E lanes. Where the squares leave FP32 (or eps is 0 and they
// vanish), x is brought near 1 by a power of two first; the lanes of other heads get the bits that they get alone.
template <uint32_t D, int E>
__device__ inline float norm_factor(float (&x)[E], float eps) {
    auto mean = [&](float e) {
        float sq = 0.0f;
#pragma unroll
        for (int i = 0; i < E; ++i) sq = fmaf(x[i], x[i], sq);
        return lanes_reduce<D / E>(sq, [](float p, float q) { return p + q; }) * (1.0f / D) + e;
    };
    float m = mean(eps);
    const bool out = !(m > 0x1p-100f && m < 0x1p127f);
    if (__any(out)) {
        asm volatile("");
        float top = sqrtf(eps);
#pragma unroll
        for (int i = 0; i < E; ++i) top = fmaxf(top, fabsf(x[i]));
        top = lanes_reduce<D / E>(top, [](float p, float q) { return fmaxf(p, q); });
        const int by = out ? 127 - (int)(__float_as_uint(top) >> 23) : 0;
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = ldexpf(x[i], by);
        m = mean(ldexpf(eps, 2 * by));
    }
    return 1.0f / sqrtf(m);
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

// The codes of a lane's E values, four to a word, and the group's word of scale and bias. N lanes share a
// group. A group with a value of 2^103 or more, infinite or NaN is NaN: below that a score's sum over 512
// products with queries of 2^15 stays in FP32.
template <int E, int N, uint32_t BITS>
__device__ inline uint32_t quantise(const float (&x)[E], uint32_t (&code)[E / 4]) {
    constexpr float top = (float)((1u << BITS) - 1u);
    float lo = x[0], hi = x[0], size = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        lo = fminf(lo, x[i]);
        hi = fmaxf(hi, x[i]);
        size = fmaf(x[i], 0.0f, size);  // NaN where a value is NaN or infinite
    }
    const bool in = size == 0.0f && fmaxf(-lo, hi) < 0x1p103f;
    const uint32_t lane = threadIdx.x & 63u;
    const bool finite = ((__ballot(!in) >> (lane & ~(uint32_t)(N - 1))) & ((1ull << N) - 1ull)) == 0ull;
    lo = lanes_reduce<N>(lo, [](float a, float b) { return fminf(a, b); });
    hi = lanes_reduce<N>(hi, [](float a, float b) { return fmaxf(a, b); });
    const float bias = bf16_outward(lo, false);
    // quotients as IEEE division gives them: one correction step of a product with the correctly rounded
    // reciprocal (Markstein's theorem); scale has 8 significant bits, so one Newton step rounds its
    // reciprocal correctly
    const float range = hi - bias, share = range * (1.0f / top);
    const float scale = fmaxf(bf16_outward(fmaf(fmaf(-share, top, range), 1.0f / top, share), true), 0x1p-126f);
    const float near = __builtin_amdgcn_rcpf(scale);
    const float inv = finite ? fmaf(fmaf(-scale, near, 1.0f), near, near) : __builtin_nanf("");  // a code of NaN is 0
    // scale is rounded up and bias down, so the codes are within 0 .. top as they are
    float q[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const float y = x[i] - bias, t = y * inv;
        q[i] = rintf(fmaf(fmaf(-t, scale, y), inv, t));
    }
#pragma unroll
    for (int i = 0; i < E; i += 4) {
        uint32_t w = __builtin_amdgcn_cvt_pk_u8_f32(q[i], 0u, 0u);
        w = __builtin_amdgcn_cvt_pk_u8_f32(q[i + 1], 1u, w);
        w = __builtin_amdgcn_cvt_pk_u8_f32(q[i + 2], 2u, w);
        code[i / 4] = __builtin_amdgcn_cvt_pk_u8_f32(q[i + 3], 3u, w);
    }
    return finite ? __float_as_uint(scale) | __float_as_uint(bias) >> 16 : 0x7FC07FC0u;
}

// The places of a workgroup's tokens (0xFFFFFFFF: none). Tokens 0 .. lead - 1 come before the first slot
// that is a multiple of four; from there on four at a time may be neighbours.
struct Places {
    uint32_t slot[kMaxChunk];
};
__device__ inline void find_places(Places& p, const uint32_t* slots, uint32_t t0, uint32_t n, uint64_t limit) {
    if (threadIdx.x < kMaxChunk) {
        const uint32_t s = threadIdx.x < n ? slots[t0 + threadIdx.x] : 0xFFFFFFFFu;
        p.slot[threadIdx.x] = s < limit ? s : 0xFFFFFFFFu;
    }
    __syncthreads();
}
// Token groups of a workgroup: number i is tokens first .. first + count - 1, neighbours when quad.
struct Group {
    uint32_t first, count;
    bool quad;
};
__device__ inline uint32_t lead_of(const Places& p, uint32_t n) { return min(n, (4u - (p.slot[0] & 3u)) & 3u); }
__device__ inline uint32_t groups_of(uint32_t lead, uint32_t n) { return (lead ? 1u : 0u) + (n - lead + 3u) / 4u; }
__device__ inline Group group_of(const Places& p, uint32_t lead, uint32_t n, uint32_t i) {
    Group g;
    const uint32_t at = lead ? i - 1u : i;
    g.first = lead && i == 0u ? 0u : lead + 4u * at;
    g.count = lead && i == 0u ? lead : min(4u, n - g.first);
    const uint32_t s = p.slot[g.first];
    g.quad = g.count == 4u && s != 0xFFFFFFFFu && (s & 3u) == 0u && p.slot[g.first + 1u] == s + 1u && p.slot[g.first + 2u] == s + 2u &&
             p.slot[g.first + 3u] == s + 3u;
    return g;
}

__device__ inline uint8_t* record_of(const KvView& kv, uint32_t slot, uint32_t head) {
    const uint32_t page = slot >> kv.page_shift, at = slot & ((1u << kv.page_shift) - 1u);
    return kv.base + kv_record_at(kv, page, head, at / kKvBlock);
}

// Four words of four bytes, transposed: word i of the result has byte i of each.
__device__ inline void transpose4(uint32_t (&w)[4]) {
    const uint32_t a = __builtin_amdgcn_perm(w[1], w[0], 0x05010400u), b = __builtin_amdgcn_perm(w[1], w[0], 0x07030602u);
    const uint32_t c = __builtin_amdgcn_perm(w[3], w[2], 0x05010400u), d = __builtin_amdgcn_perm(w[3], w[2], 0x07030602u);
    w[0] = __builtin_amdgcn_perm(c, a, 0x05040100u), w[1] = __builtin_amdgcn_perm(c, a, 0x07060302u);
    w[2] = __builtin_amdgcn_perm(d, b, 0x05040100u), w[3] = __builtin_amdgcn_perm(d, b, 0x07060302u);
}

// Values from LDS codes [head][token][head_dim] to the cache: four values to a lane (4 bits: and the four 16
// further), the tokens of a group.
template <int NG, uint32_t BITS>
__device__ inline void store_values(const KvView& kv, const Places& p, const uint8_t* stage, uint32_t n, uint32_t head0, uint32_t heads) {
    constexpr uint32_t D = NG * 64u, W = BITS == 8u ? D / 4u : D / 8u;  // lanes of a token
    const uint32_t lead = lead_of(p, n), groups = groups_of(lead, n);
    const uint32_t w = threadIdx.x % W * 4u, d = BITS == 8u ? w : (w & 15u) | (w & ~15u) << 1;
    for (uint32_t u = threadIdx.x / W; u < groups * heads; u += kThreads / W) {
        const uint32_t h = u % heads;
        const Group g = group_of(p, lead, n, u / heads);
        const uint8_t* src = stage + (h * n + g.first) * D + d;
        uint32_t c[4];
#pragma unroll
        for (uint32_t j = 0; j < 4u; ++j) {
            c[j] = 0u;
            if (j < g.count) {
                c[j] = *reinterpret_cast<const uint32_t*>(src + j * D);
                if constexpr (BITS == 4u) c[j] |= *reinterpret_cast<const uint32_t*>(src + j * D + 16u) << 4;
            }
        }
        if (g.quad) {
            transpose4(c);
            const uint32_t slot = p.slot[g.first];
            uint8_t* dst = record_of(kv, slot, head0 + h) + kv_part_bytes(NG, BITS) + kv_value_byte(BITS, slot & 31u, d);
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i) *reinterpret_cast<uint32_t*>(dst + i * 16u) = c[i];
        } else {
            for (uint32_t j = 0; j < g.count; ++j) {
                const uint32_t slot = p.slot[g.first + j];
                if (slot == 0xFFFFFFFFu) continue;
                uint8_t* dst = record_of(kv, slot, head0 + h) + kv_part_bytes(NG, BITS) + kv_value_byte(BITS, slot & 31u, d);
                const uint32_t x = j == 0u ? c[0] : j == 1u ? c[1] : j == 2u ? c[2] : c[3];
#pragma unroll
                for (uint32_t i = 0; i < 4u; ++i) dst[i * 16u] = (uint8_t)(x >> (8u * i));
            }
        }
    }
}

// How a call is divided: workgroups of turn_chunk tokens and turn_heads heads of the queries or keys, then
// those of value_chunk tokens and value_heads heads of the values.
struct Division {
    uint32_t turn_chunk, turn_heads, q_parts, turn_parts, turn_items;
    uint32_t value_chunk, value_heads, value_parts;
};

// A wave's walk over a workgroup's tokens and heads: whole tokens in turn where there are four or more, else
// the heads of a token divided among the waves.
struct Walk {
    uint32_t t, h, tokens, heads, tstep, hfirst, hstep;
    __device__ Walk(uint32_t n, uint32_t heads_, uint32_t wave, uint32_t wave_heads) : tokens(n), heads(heads_) {
        const bool whole = n >= 4u;
        t = whole ? wave : 0u, tstep = whole ? 4u : 1u;
        hfirst = whole ? 0u : wave * wave_heads, hstep = (whole ? 1u : 4u) * wave_heads;
        h = hfirst;
        if (h >= heads) t = tokens;
    }
    __device__ bool more() const { return t < tokens; }
    __device__ void next() {
        h += hstep;
        if (h >= heads) h = hfirst, t += tstep;
    }
};

template <int NG, class T, int E, uint32_t BITS>
__device__ inline void turn_heads(const QkvArgs& a, const Division& v, uint32_t id, uint8_t* lds) {
    constexpr uint32_t D = NG * 64u, LPH = D / E, HP = 64u / LPH;  // lanes per head, heads per wave
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint32_t part = id % v.turn_parts;
    const uint32_t t0 = id / v.turn_parts * v.turn_chunk, n = min(v.turn_chunk, a.tokens - t0);
    const bool keys = part >= v.q_parts;
    if (keys) part -= v.q_parts;
    const uint32_t h0 = part * v.turn_heads, heads = min(v.turn_heads, (keys ? a.kv_heads : a.q_heads) - h0);
    const T* src = static_cast<const T*>(keys ? a.k : a.q);
    T* dst = static_cast<T*>(keys ? a.k_out : a.q_out);
    const uint64_t stride = keys ? a.k_stride : a.q_stride, out_stride = keys ? a.k_out_stride : a.q_out_stride;
    const uint16_t* weight = keys ? a.k_norm : a.q_norm;
    const bool normed = (a.norms >> (keys ? 1 : 0)) & 1u;
    const bool stored = BITS != 0u && keys;
    const uint32_t rot = a.turns ? a.rotary_dim : 0u, half = rot / 2u;
    const uint32_t d0 = (lane % LPH) * E, sub = lane / LPH;

    Walk at(n, heads, wave, HP);
    // lanes past the last head take it again and store nothing
    auto from = [&](const Walk& w) {
        return src + (uint64_t)(t0 + w.t) * stride + ((h0 + min(w.h + sub, heads - 1u)) * D + d0);
    };
    Vec<T, E> next;
    if (at.more()) next.load(from(at));
    float w[E];
#pragma unroll
    for (int i = 0; i < E; ++i) w[i] = weight && normed ? bf16_to_f32(weight[d0 + i]) : 1.0f;
    float *cosines = reinterpret_cast<float*>(lds), *sines = cosines + n * half;
    if (rot) {
        const uint32_t first = n >= 4u ? lane : threadIdx.x, step = n >= 4u ? 64u : kThreads;
        for (uint32_t t = n >= 4u ? wave : 0u; t < n; t += n >= 4u ? 4u : 1u) {
            const uint64_t pos = a.positions[t0 + t];
            for (uint32_t i = first; i < half; i += step)
                turn_cos_sin((uint32_t)((pos * a.turns[i] + 0x80000000ull) >> 32), cosines[t * half + i], sines[t * half + i]);
        }
        __syncthreads();
    }
    // the lane with the other values of this lane's pairs (halves), and the sign of their sines
    const bool turning = d0 < rot, first = d0 < half;
    const bool still = a.still || rot % E != 0u;  // pairs that do not turn lie in turning lanes
    const uint32_t other = !turning || a.pairs ? lane : first ? lane + half / E : lane - half / E;

    float cs[E], sn[E];
#pragma unroll
    for (int i = 0; i < E; ++i) cs[i] = 1.0f, sn[i] = 0.0f;
    uint32_t angles = 0xFFFFFFFFu;  // the token whose sines are held
    while (at.more()) {
        const Walk now = at;
        float x[E];
        next.get(x);
        at.next();
        if (at.more()) next.load(from(at));
        if (rot && now.t != angles) {
            angles = now.t;
            if (turning) {
                const uint32_t p = now.t * half + (a.pairs ? d0 / 2u : first ? d0 : d0 - half);
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    if (a.pairs) {
                        if (!(i & 1) && d0 + i < rot) cs[i] = cosines[p + i / 2], sn[i] = sines[p + i / 2];
                    } else {
                        cs[i] = cosines[p + i], sn[i] = sines[p + i];
                    }
                }
            }
        }
        const bool here = now.h + sub < heads;
        const uint32_t t = now.t, head = h0 + min(now.h + sub, heads - 1u);
        if (normed) {
            const float r = norm_factor<D, E>(x, a.eps);
#pragma unroll
            for (int i = 0; i < E; ++i) x[i] = x[i] * r * w[i];
        }
        if (rot) {
            // what does not turn stays as it is: a product with a sine of 0 would make NaN of infinities
            float y[E], z[E];
            if (a.pairs) {
#pragma unroll
                for (int i = 0; i < E; i += 2) {
                    y[i] = x[i] * cs[i] - x[i + 1] * sn[i];
                    y[i + 1] = x[i + 1] * cs[i] + x[i] * sn[i];
                }
            } else {
#pragma unroll
                for (int i = 0; i < E; ++i) z[i] = __shfl(x[i], (int)other);
#pragma unroll
                for (int i = 0; i < E; ++i) y[i] = first ? x[i] * cs[i] - z[i] * sn[i] : x[i] * cs[i] + z[i] * sn[i];
            }
            if (still) {
                asm volatile("");
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    const int at = a.pairs ? i & ~1 : i;
                    if (sn[at] == 0.0f && cs[at] == 1.0f) y[i] = x[i];
                }
            }
#pragma unroll
            for (int i = 0; i < E; ++i) x[i] = turning ? y[i] : x[i];
        }
        if (dst && here) Vec<T, E>::store(dst + (uint64_t)(t0 + t) * out_stride + (head * D + d0), x);
        if constexpr (BITS != 0u) {
            if (stored) {
                uint32_t code[E / 4];
                constexpr int N = 64 / E;
                const uint32_t word = quantise<E, N, BITS>(x, code);
                const uint32_t slot = __builtin_amdgcn_readfirstlane(a.slots[t0 + t]);
                if (here && slot < a.kv.slots) {
                    uint8_t* rec = record_of(a.kv, slot, head);
                    if (lane % N == 0u)
                        *reinterpret_cast<uint32_t*>(rec + 2u * kv_part_bytes(NG, BITS) + kv_scale_byte(NG, 0u, slot & 31u, d0 / 64u)) = word;
                    uint8_t* to = rec + kv_key_byte(BITS, slot & 31u, d0);
#pragma unroll
                    for (int i = 0; i < E / 4; ++i) {
                        if constexpr (BITS == 8u) {
                            reinterpret_cast<uint32_t*>(to)[i] = code[i];
                        } else {
                            const uint32_t two = code[i] | code[i] >> 4;  // bytes 0 and 2 hold two codes each
                            reinterpret_cast<uint16_t*>(to)[i] = (uint16_t)__builtin_amdgcn_perm(0u, two, 0x0C0C0200u);
                        }
                    }
                }
            }
        }
    }
}

template <int NG, class T, int E, uint32_t BITS>
__device__ inline void store_value_heads(const QkvArgs& a, const Division& v, uint32_t id, uint8_t* stage, Places& places) {
    constexpr uint32_t D = NG * 64u, LPH = D / E, HP = 64u / LPH;
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t h0 = id % v.value_parts * v.value_heads, heads = min(v.value_heads, a.kv_heads - h0);
    const uint32_t t0 = id / v.value_parts * v.value_chunk, n = min(v.value_chunk, a.tokens - t0);
    const uint32_t d0 = (lane % LPH) * E, sub = lane / LPH;
    Walk at(n, heads, wave, HP);
    auto from = [&](const Walk& w) {
        return static_cast<const T*>(a.v) + (uint64_t)(t0 + w.t) * a.v_stride + ((h0 + min(w.h + sub, heads - 1u)) * D + d0);
    };
    Vec<T, E> next;
    if (at.more()) next.load(from(at));
    find_places(places, a.slots, t0, n, a.kv.slots);
    const bool normed = (a.norms >> 2) & 1u;
    while (at.more()) {
        const Walk now = at;
        float x[E];
        next.get(x);
        at.next();
        if (at.more()) next.load(from(at));
        if (normed) {
            const float r = norm_factor<D, E>(x, a.eps);
#pragma unroll
            for (int i = 0; i < E; ++i) x[i] *= r;
        }
        uint32_t code[E / 4];
        constexpr int N = 64 / E;
        const uint32_t word = quantise<E, N, BITS>(x, code);
        if (now.h + sub < heads) {
            const uint32_t slot = __builtin_amdgcn_readfirstlane(places.slot[now.t]);
            if (lane % N == 0u && slot != 0xFFFFFFFFu)
                *reinterpret_cast<uint32_t*>(record_of(a.kv, slot, h0 + now.h + sub) + 2u * kv_part_bytes(NG, BITS) +
                                             kv_scale_byte(NG, 1u, slot & 31u, d0 / 64u)) = word;
            uint32_t* to = reinterpret_cast<uint32_t*>(stage + ((now.h + sub) * n + now.t) * D + d0);
#pragma unroll
            for (int i = 0; i < E / 4; ++i) to[i] = code[i];
        }
    }
    __syncthreads();
    store_values<NG, BITS>(a.kv, places, stage, n, h0, heads);
}

template <int NG, class T, int E, uint32_t BITS>
__global__ __launch_bounds__(kThreads) void k_qkv(const QkvArgs a, const Division v) {
    extern __shared__ __align__(16) uint8_t lds[];
    // workgroups of neighbouring tokens on one die: they write the same lines of the cache
    if (blockIdx.x < v.turn_items) {
        turn_heads<NG, T, E, BITS>(a, v, BITS != 0u ? same_die(blockIdx.x, v.turn_items) : blockIdx.x, lds);
    } else if constexpr (BITS != 0u) {
        __shared__ Places places;
        store_value_heads<NG, T, E, BITS>(a, v, same_die(blockIdx.x - v.turn_items, gridDim.x - v.turn_items), lds, places);
    }
}

// A thread takes four values of the up to four tokens of a group, of the keys or of the values.
template <int NG, class T, uint32_t BITS>
__global__ __launch_bounds__(kThreads) void k_kv_read(const KvReadArgs a, uint32_t chunk, uint32_t heads_per, uint32_t parts) {
    constexpr uint32_t D = NG * 64u, W = D / 4u;
    __shared__ Places places;
    const uint32_t t0 = blockIdx.x * chunk, n = min(chunk, a.tokens - t0);
    const bool values = !a.k || blockIdx.y >= parts;
    const uint32_t h0 = (blockIdx.y % parts) * heads_per, heads = min(heads_per, a.kv.heads - h0);
    T* dst = static_cast<T*>(values ? a.v : a.k);
    const uint64_t stride = values ? a.v_stride : a.k_stride;
    find_places(places, a.slots, t0, n, a.kv.slots);
    const uint32_t lead = lead_of(places, n), groups = groups_of(lead, n);
    const uint32_t d = threadIdx.x % W * 4u;
    for (uint32_t u = threadIdx.x / W; u < groups * heads; u += kThreads / W) {
        const uint32_t h = u % heads;
        const Group g = group_of(places, lead, n, u / heads);
        uint32_t c[4], word[4];  // by token: four codes, and the scale and bias of its group
        if (values && g.quad) {
            const uint32_t slot = places.slot[g.first];
            const uint8_t* rec = record_of(a.kv, slot, h0 + h);
            const uint8_t* from = rec + kv_part_bytes(NG, BITS) + kv_value_byte(BITS, slot & 31u, d);
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i) c[i] = *reinterpret_cast<const uint32_t*>(from + i * 16u);
            const uint4 s = *reinterpret_cast<const uint4*>(rec + 2u * kv_part_bytes(NG, BITS) + kv_scale_byte(NG, 1u, slot & 31u, d / 64u));
            word[0] = s.x, word[1] = s.y, word[2] = s.z, word[3] = s.w;
            if constexpr (BITS == 4u)
#pragma unroll
                for (uint32_t i = 0; i < 4u; ++i) c[i] = (c[i] >> ((d & 16u) ? 4 : 0)) & 0x0F0F0F0Fu;
            transpose4(c);
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 4u; ++j) {
                const uint32_t slot = j < g.count ? places.slot[g.first + j] : 0xFFFFFFFFu;
                c[j] = 0u, word[j] = 0x7FC07FC0u;
                if (slot == 0xFFFFFFFFu) continue;
                const uint8_t* rec = record_of(a.kv, slot, h0 + h);
                word[j] = *reinterpret_cast<const uint32_t*>(rec + 2u * kv_part_bytes(NG, BITS) +
                                                            kv_scale_byte(NG, values ? 1u : 0u, slot & 31u, d / 64u));
                if (values) {
                    const uint8_t* from = rec + kv_part_bytes(NG, BITS) + kv_value_byte(BITS, slot & 31u, d);
#pragma unroll
                    for (uint32_t i = 0; i < 4u; ++i) c[j] |= (uint32_t)from[i * 16u] << (8u * i);
                    if constexpr (BITS == 4u) c[j] = (c[j] >> ((d & 16u) ? 4 : 0)) & 0x0F0F0F0Fu;
                } else if constexpr (BITS == 8u) {
                    c[j] = *reinterpret_cast<const uint32_t*>(rec + kv_key_byte(BITS, slot & 31u, d));
                } else {
                    const uint32_t two = *reinterpret_cast<const uint16_t*>(rec + kv_key_byte(BITS, slot & 31u, d));
                    c[j] = (two & 15u) | (two & 0xF0u) << 4 | (two & 0xF00u) << 8 | (two & 0xF000u) << 12;
                }
            }
        }
#pragma unroll
        for (uint32_t j = 0; j < 4u; ++j) {
            if (j >= g.count) break;
            const float scale = __uint_as_float(word[j] & 0xFFFF0000u), bias = __uint_as_float(word[j] << 16);
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = fmaf((float)((c[j] >> (8 * i)) & 255u), scale, bias);
            T* to = dst + (uint64_t)(t0 + g.first + j) * stride + (uint64_t)(h0 + h) * D + d;
            if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(to) = make_float4(x[0], x[1], x[2], x[3]);
            else *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]));
        }
    }
}

// Tokens and heads of a workgroup, from the most that are useful, halved until there are a thousand workgroups:
// the tokens first, which share a token's sines among more heads, or the heads first, which fill whole lines
// of the cache (eight neighbouring tokens' keys, 32 tokens' values): a cache write of 4,001 tokens and its
// read back measured 38.8 us with the tokens halved first, 32.5 so. With 500 workgroups in place of a thousand that
// is 33 -> 36 us, 1,500 tokens rotated into the cache and read 27 -> 31, but 256 of them 18 -> 15; with 2,000 workgroups
// 35 and 31 us, and a rotation of 2,048 tokens 15 -> 19. Heads stay as many as least_heads, what
// the waves hold at once, while tokens are left to halve.
struct Shape {
    uint32_t chunk, heads;
};
Shape shape_for(uint32_t tokens, uint32_t all_heads, uint32_t chunk, uint32_t heads, uint32_t least_heads, bool heads_first) {
    Shape s{chunk, heads};
    auto few = [&] { return (uint64_t)((tokens + s.chunk - 1u) / s.chunk) * ((all_heads + s.heads - 1u) / s.heads) < kGroups; };
    auto fewer_heads = [&] {
        while (s.heads > least_heads && few()) s.heads = (s.heads + 1u) / 2u;
    };
    if (heads_first) fewer_heads();
    while (s.chunk > 1u && few()) s.chunk /= 2u;
    fewer_heads();
    return s;
}
uint32_t parts_of(uint32_t n, uint32_t per) { return (n + per - 1u) / per; }

template <int NG, class T, int E>
void launch_qkv_typed(const QkvArgs& a, hipStream_t st) {
    constexpr uint32_t D = NG * 64u, HP = 64u / (D / E);
    const bool keys = a.k != nullptr, values = a.v != nullptr && a.kv.base != nullptr;
    Division v{};
    uint64_t turn_items = 0u, value_items = 0u;  // more than 32 bits at the most tokens of 1,024 heads of 512
    size_t lds = 0u;
    const uint32_t turned = (a.q ? a.q_heads : 0u) + (keys ? a.kv_heads : 0u);
    if (turned) {
        const bool lines = keys && a.kv.base != nullptr;
        uint32_t chunk = lines ? kMaxChunk : kMaxChunk / 2u;
        while (a.turns && chunk > 1u && chunk * a.rotary_dim * 4u > kLdsBytes) chunk /= 2u;
        const uint32_t heads = min(max(a.q ? a.q_heads : 0u, keys ? a.kv_heads : 0u), kMaxHeads);
        const Shape s = shape_for(a.tokens, turned, chunk, heads, min(lines ? HP : 4u * HP, heads), lines);
        v.turn_chunk = s.chunk, v.turn_heads = s.heads;
        v.q_parts = a.q ? parts_of(a.q_heads, s.heads) : 0u;
        v.turn_parts = v.q_parts + (keys ? parts_of(a.kv_heads, s.heads) : 0u);
        turn_items = (uint64_t)v.turn_parts * parts_of(a.tokens, s.chunk);
        if (a.turns) lds = (size_t)s.chunk * a.rotary_dim * 4u;
    }
    if (values) {
        uint32_t heads = min(a.kv_heads, kMaxHeads);
        while (heads > 1u && kMaxChunk * heads * D > kLdsBytes) heads = (heads + 1u) / 2u;
        const Shape s = shape_for(a.tokens, a.kv_heads, kMaxChunk, heads, min(HP, heads), true);
        v.value_chunk = s.chunk, v.value_heads = s.heads, v.value_parts = parts_of(a.kv_heads, s.heads);
        value_items = (uint64_t)v.value_parts * parts_of(a.tokens, s.chunk);
        lds = max(lds, (size_t)s.chunk * s.heads * D);
    }
    const dim3 grid(grid_blocks(turn_items + value_items)), block(kThreads);
    v.turn_items = (uint32_t)turn_items;
    if (!a.kv.base) hipLaunchKernelGGL((k_qkv<NG, T, E, 0u>), grid, block, lds, st, a, v);
    else if (a.kv.bits == 8u) hipLaunchKernelGGL((k_qkv<NG, T, E, 8u>), grid, block, lds, st, a, v);
    else hipLaunchKernelGGL((k_qkv<NG, T, E, 4u>), grid, block, lds, st, a, v);
}

template <int NG, class T>
void launch_read_typed(const KvReadArgs& a, hipStream_t st) {
    const uint32_t both = (a.k ? 1u : 0u) + (a.v ? 1u : 0u);
    const Shape s = shape_for(a.tokens, a.kv.heads * both, kMaxChunk, min(a.kv.heads, kMaxHeads), 1u, true);
    const uint32_t parts = parts_of(a.kv.heads, s.heads);
    const dim3 grid(parts_of(a.tokens, s.chunk), parts * both), block(kThreads);
    if (a.kv.bits == 8u) hipLaunchKernelGGL((k_kv_read<NG, T, 8u>), grid, block, 0, st, a, s.chunk, s.heads, parts);
    else hipLaunchKernelGGL((k_kv_read<NG, T, 4u>), grid, block, 0, st, a, s.chunk, s.heads, parts);
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
        if (head_dim == 64u) launch_read_typed<1, uint16_t>(a, st);
        else if (head_dim == 128u) launch_read_typed<2, uint16_t>(a, st);
        else if (head_dim == 256u) launch_read_typed<4, uint16_t>(a, st);
        else launch_read_typed<8, uint16_t>(a, st);
    } else {
        if (head_dim == 64u) launch_read_typed<1, float>(a, st);
        else if (head_dim == 128u) launch_read_typed<2, float>(a, st);
        else if (head_dim == 256u) launch_read_typed<4, float>(a, st);
        else launch_read_typed<8, float>(a, st);
    }
    check_hip(hipGetLastError(), "cache read");
}

}  // namespace tdt

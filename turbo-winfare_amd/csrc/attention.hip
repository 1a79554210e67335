// Attention of a batch over the quantised cache, its shared prefix read once for all sequences.
//
// A workgroup takes one key/value head, a tile of 16 or 32 query rows and a range of keys: of the prefix
// (rows of every sequence of the batch) or of one sequence's own keys (its rows). Its four waves take the
// range's 32-token records in turn, each with its own running maximum and sum, and join at the end; a
// second kernel joins the workgroups' partial results. Everything stays in registers:
//   S^T = K Q^T with the codes as the first operand. A code widened to 16 bits is the fp16 denormal
//     code * 2^-24, exact, so widening costs one byte permute per two codes; with q the row's values in
//     fp16 (scaled by a power of two of the row), scale and bias of a key enter afterwards, in fp32:
//     sum_g s_g (codes_g . q_g) + b_g sum(q_g) over the groups of 64.
//   O^T += V^T P^T: a lane holds the scores of 8 keys of one row, and those 8 keys' value codes are its
//     bytes of the record, so the weights p * s_v go into the second product as they are; the biases add
//     sum_j p_j b_j per group. The weights are scaled by a power of two that keeps the record's largest
//     value scale just inside fp16, so scales of any size are held.
// BF16 queries: q is exact in one fp16 operand, the weights are rounded to 11 bits (2^-12 of each, against
// the output's 2^-9). FP32 queries: q and the weights are split into two fp16 parts each (22 bits), and
// the codes are centred (code - 128 or - 8, one packed addition more per two codes): products of
// denormals add up with 4 (8 bits) to 7 (4 bits) bits less than FP32 has, and a sum of codes that are all
// positive cancels against the biases. Measured against 64 bits at 777 keys, 4 bits: plain codes 5e-5.
#include <algorithm>
#include <cmath>
#include <stdexcept>

#include "dt_internal.h"
#include "dt_kv.h"

namespace tdt {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float float4v __attribute__((ext_vector_type(4)));

constexpr uint32_t kThreads = 256;
constexpr uint32_t kWaves = 4;
constexpr uint32_t kXcds = 8;
constexpr float kNegInf = -__builtin_inff();

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
union Frag {
    half8 h;
    bf16x8 b;
    uint32_t u[4];
};

__device__ inline uint32_t out_bits(float f) {
    const uint32_t u = __float_as_uint(f);
    if ((u & 0x7FFFFFFFu) > 0x7F800000u) return (u >> 16) | 0x40u;
    return (u + 0x7FFFu + ((u >> 16) & 1u)) >> 16;
}
// v over the lanes that hold the same row (lane, lane ^ 16, lane ^ 32, lane ^ 48)
template <class Op>
__device__ inline float rows_reduce(float v, Op op) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return op(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ inline float rows_max(float v) { return rows_reduce(v, [](float a, float b) { return fmaxf(a, b); }); }
__device__ inline float rows_sum(float v) { return rows_reduce(v, [](float a, float b) { return a + b; }); }

// A pair of 16-bit codes as fp16: plain, the denormals code * 2^-24, or centred, the numbers
// code - 128 (8 bits) or code - 8 (4 bits), by way of 1024 + code.
template <uint32_t BITS, bool CENTRED>
__device__ inline uint32_t as_fp16(uint32_t pair) {
    if constexpr (!CENTRED) return pair;
    typedef _Float16 half2v __attribute__((ext_vector_type(2)));
    union {
        uint32_t u;
        half2v h;
    } x;
    x.u = pair | 0x64006400u;
    const _Float16 middle = (_Float16)(BITS == 8u ? -1152.0f : -1032.0f);
    x.h += half2v{middle, middle};
    return x.u;
}
// eight bytes, in order
template <bool CENTRED>
__device__ inline Frag widen_bytes(uint32_t a, uint32_t b) {
    constexpr uint32_t top = CENTRED ? 0x64646464u : 0u;  // the upper bytes, taken by the same permute
    Frag f;
    f.u[0] = as_fp16<8u, CENTRED>(__builtin_amdgcn_perm(top, a, CENTRED ? 0x04010400u : 0x0C010C00u));
    f.u[1] = as_fp16<8u, CENTRED>(__builtin_amdgcn_perm(top, a, CENTRED ? 0x04030402u : 0x0C030C02u));
    f.u[2] = as_fp16<8u, CENTRED>(__builtin_amdgcn_perm(top, b, CENTRED ? 0x04010400u : 0x0C010C00u));
    f.u[3] = as_fp16<8u, CENTRED>(__builtin_amdgcn_perm(top, b, CENTRED ? 0x04030402u : 0x0C030C02u));
    return f;
}
// eight nibbles of one word: operand elements 2 p, 2 p + 1 are nibbles p, p + 4 (the queries are laid out alike)
template <bool CENTRED>
__device__ inline Frag widen_nibbles(uint32_t w) {
    Frag f;
#pragma unroll
    for (int p = 0; p < 4; ++p) f.u[p] = as_fp16<4u, CENTRED>((w >> (4 * p)) & 0x000F000Fu);
    return f;
}
// the low (shift 0) or high (shift 4) halves of eight bytes: elements are bytes 0, 2, 1, 3 of each word
// (the weights are laid out alike)
template <bool CENTRED>
__device__ inline Frag widen_halves(uint32_t a, uint32_t b, uint32_t shift) {
    Frag f;
    f.u[0] = as_fp16<4u, CENTRED>((a >> shift) & 0x000F000Fu);
    f.u[1] = as_fp16<4u, CENTRED>((a >> (8u + shift)) & 0x000F000Fu);
    f.u[2] = as_fp16<4u, CENTRED>((b >> shift) & 0x000F000Fu);
    f.u[3] = as_fp16<4u, CENTRED>((b >> (8u + shift)) & 0x000F000Fu);
    return f;
}
// A key's scale, and its bias as the products need it: that of code 0, or of the middle code
template <uint32_t BITS, bool CENTRED>
__device__ inline float scale_of(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
template <uint32_t BITS, bool CENTRED>
__device__ inline float bias_of(uint32_t w) {
    const float b = __uint_as_float(w << 16);
    return CENTRED ? fmaf(BITS == 8u ? 128.0f : 8.0f, __uint_as_float(w & 0xFFFF0000u), b) : b;
}

// Two numbers rounded to fp16, and back. The packed word is opaque to the compiler: it would otherwise
// round a product anew for each use, once from FP32 and once, fused with the product, from the exact
// value, and what is left of a number after its first part would miss a step near a tie.
__device__ inline uint32_t pack_fp16(float lo, float hi) {
    typedef _Float16 half2v __attribute__((ext_vector_type(2)));
    union {
        half2v h;
        uint32_t u;
    } x;
    x.h = half2v{(_Float16)lo, (_Float16)hi};
    asm("" : "+v"(x.u));
    return x.u;
}
struct Pair {
    float lo, hi;
};
__device__ inline Pair unpack_fp16(uint32_t w) {
    typedef _Float16 half2v __attribute__((ext_vector_type(2)));
    union {
        uint32_t u;
        half2v h;
    } x;
    x.u = w;
    return Pair{(float)x.h[0], (float)x.h[1]};
}

struct Item {
    bool prefix;
    uint32_t head, row0, rows;     // key/value head, first row of the tile, rows of the segment
    uint32_t seq;                  // own keys: the sequence
    uint32_t split, splits, part;
    const uint32_t* pages;
    uint32_t table;                // entries of pages
};

struct Row {
    uint32_t token, head;          // of q and out
    int lo, hi;                    // visible keys of the segment
    bool exists, over;             // over: passes its page table
};

__device__ inline Row row_of(const AttnArgs& a, const Item& it, uint32_t r) {
    Row w;
    w.exists = r < it.rows;
    if (!w.exists) r = it.rows - 1u;
    const uint32_t per = a.q_len * a.group;
    const uint32_t b = it.prefix ? r / per : it.seq, in = it.prefix ? r % per : r;
    const uint32_t t = in / a.group;
    w.token = b * a.q_len + t;
    w.head = it.head * a.group + in % a.group;
    const long long pos = (long long)a.kv_len[b] - (long long)a.q_len + t;
    const long long room = (long long)a.prefix_len + ((long long)a.page_stride << a.kv.page_shift);
    w.over = pos >= room;
    long long lo = a.window ? pos - (long long)a.window + 1 : 0, hi = pos + 1;
    if (it.prefix) hi = hi < (long long)a.prefix_len ? hi : (long long)a.prefix_len;
    else lo -= a.prefix_len, hi -= a.prefix_len;
    w.lo = (int)(lo > 0 ? (lo < 0x7FFFFFFF ? lo : 0x7FFFFFFF) : 0);
    w.hi = w.over ? 0 : (int)(hi > 0 ? hi : 0);
    return w;
}

template <bool F32>
__device__ inline void load_q8(const void* q, uint64_t at, float (&x)[8]) {
    if constexpr (F32) {
        const float4 u = *reinterpret_cast<const float4*>(static_cast<const float*>(q) + at);
        const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(q) + at + 4);
        x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w, x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
    } else {
        const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(q) + at);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
}

template <bool F32>
__device__ inline void store_out(void* out, uint64_t at, float4 v) {
    if constexpr (F32) *reinterpret_cast<float4*>(static_cast<float*>(out) + at) = v;
    else *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + at) = make_uint2(out_bits(v.x) | out_bits(v.y) << 16, out_bits(v.z) | out_bits(v.w) << 16);
}

template <int NG, bool F32, int MT>
struct Shared {
    static constexpr uint32_t kRow = 68;  // floats of a row of 64, padded
    union {
        struct {
            uint4 q[MT][NG][F32 ? 4 : 2][64];  // the queries as second operands: [.., chunk of 32 (and low parts)][lane]
            uint32_t scales[kWaves][2 * NG * kKvBlock];
        };
        float sums[kWaves][16 * MT][kRow];
    };
    float m[kWaves][16 * MT], l[kWaves][16 * MT];
};

template <int NG, uint32_t BITS, bool F32, int MT>
__device__ inline void attend(const AttnArgs& a, const Item& it, Shared<NG, F32, MT>& sh) {
    constexpr int KU = BITS == 8u ? 2 : 1;       // 16-byte loads per group of keys or values
    constexpr int kUnit = F32 ? 0 : 24;          // codes are in units of 2^-kUnit
    constexpr uint32_t D = NG * 64u, PART = NG * 64u * kKvBlock * BITS / 8u, RECORD = 2u * PART + 2u * NG * kKvBlock * 4u;
    const uint32_t lane = threadIdx.x & 63u, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    // ---- the rows and what they see
    Row row[MT];
    bool live[MT];
    int lo_min = 0x7FFFFFFF, lo_max = 0, hi_min = 0x7FFFFFFF, hi_max = 0;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        row[mt] = row_of(a, it, it.row0 + mt * 16u + (lane & 15u));
        live[mt] = row[mt].exists && row[mt].lo < row[mt].hi;
        if (live[mt]) {
            lo_min = min(lo_min, row[mt].lo), lo_max = max(lo_max, row[mt].lo);
            hi_min = min(hi_min, row[mt].hi), hi_max = max(hi_max, row[mt].hi);
        } else {
            row[mt].lo = 0, row[mt].hi = 0x7FFFFFFF;  // hides nothing and is left out at the end
        }
    }
    auto least = [](int x, int y) { return min(x, y); };
    auto most = [](int x, int y) { return max(x, y); };
    lo_min = wave_reduce(lo_min, least), lo_max = wave_reduce(lo_max, most);
    hi_min = wave_reduce(hi_min, least), hi_max = wave_reduce(hi_max, most);
    int s0 = 0, s1 = 0;  // this split's records
    if (hi_max > 0) {
        const int b0 = lo_min / (int)kKvBlock, b1 = (hi_max + (int)kKvBlock - 1) / (int)kKvBlock;
        const int per = (b1 - b0 + (int)it.splits - 1) / (int)it.splits;
        s0 = min(b1, b0 + (int)it.split * per), s1 = min(b1, s0 + per);
    }

    // ---- the queries, fp16 after a power of two that takes the row's largest to 2^14 .. 2^15, in LDS for
    // all four waves; a negative scale is theirs, so that larger scores are larger weights
    float factor[MT], qsum[F32 ? MT : 1][F32 ? NG : 1];
    Frag qbias[MT];  // the groups' sums of q in three BF16 parts, part major, as the second operand against biases
    const float sign = a.scale_log2e < 0.0f ? -1.0f : a.scale_log2e == 0.0f ? 0.0f : 1.0f;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const uint64_t at = row[mt].token * a.q_stride + (uint64_t)row[mt].head * D + g * 16u;
        float top = 0.0f;
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float x[8];
                load_q8<F32>(a.q, at + n * 64u + c * 8u, x);
#pragma unroll
                for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[i]));
            }
        top = rows_max(top);
        const int shift = top > 0.0f ? 14 - ((int)(__float_as_uint(top) >> 23) - 127) : 0;
        factor[mt] = sign == 0.0f ? 1.0f : ldexpf(fabsf(a.scale_log2e), kUnit - shift);
        qbias[mt].u[0] = qbias[mt].u[1] = qbias[mt].u[2] = qbias[mt].u[3] = 0u;
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            float sum = 0.0f;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float v[8];
                load_q8<F32>(a.q, at + n * 64u + c * 8u, v);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = ldexpf(v[i], shift) * sign, sum += v[i];
                Frag h, low;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int j = BITS == 8u ? 2 * i : i, k = j + (BITS == 8u ? 1 : 4);
                    h.u[i] = pack_fp16(v[j], v[k]);
                    if constexpr (F32) {
                        const Pair u = unpack_fp16(h.u[i]);
                        low.u[i] = pack_fp16(v[j] - u.lo, v[k] - u.hi);
                    }
                }
                if ((n & 3) == (int)wave) {
                    sh.q[mt][n][c][lane] = make_uint4(h.u[0], h.u[1], h.u[2], h.u[3]);
                    if constexpr (F32) sh.q[mt][n][2 + c][lane] = make_uint4(low.u[0], low.u[1], low.u[2], low.u[3]);
                }
            }
            sum = rows_sum(sum);
            if constexpr (F32) {
                qsum[mt][n] = sum;
            } else {
                float rest = sum * 0x1p-24f;
#pragma unroll
                for (int part = 0; part < 3; ++part) {
                    const uint32_t w = out_bits(rest);  // BF16
                    rest -= __uint_as_float(w << 16);
                    const int slot = part * NG + n;
                    if (g == (uint32_t)slot / 8u) qbias[mt].u[(slot % 8) / 2] |= w << (16 * (slot % 2));
                }
            }
        }
    }
    // no wave reads the queries before all have written their part
    __syncthreads();

    float4v o[MT][NG * 4];
    float obias[MT][NG], m[MT], l[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        m[mt] = kNegInf, l[mt] = 0.0f;
#pragma unroll
        for (int n = 0; n < NG; ++n) obias[mt][n] = 0.0f;
#pragma unroll
        for (int i = 0; i < NG * 4; ++i) o[mt][i] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
    }
    int vexp = -1000;  // the sums are in units of 2^(kUnit + vexp)

    const uint32_t page_mask = (1u << a.kv.page_shift) / kKvBlock - 1u, block_shift = a.kv.page_shift - 5u;
    auto page_at = [&](int blk) {  // the page of a record; past the table or the cache: none
        const uint32_t i = (uint32_t)blk >> block_shift;
        const uint32_t p = i < it.table ? it.pages[i] : 0xFFFFFFFFu;
        return p;
    };
    auto record_at = [&](int blk, uint32_t page) {
        return a.kv.base + kv_record_at(a.kv, page < a.kv.pages ? page : 0u, it.head, (uint32_t)blk & page_mask);
    };
    auto query = [&](int mt, int n, int c) {
        Frag f;
        const uint4 v = sh.q[mt][n][c][lane];
        f.u[0] = v.x, f.u[1] = v.y, f.u[2] = v.z, f.u[3] = v.w;
        return f;
    };
    uint4 kc[NG * KU];
    uint32_t sw[NG];
    auto load_keys = [&](const uint8_t* rec) {
#pragma unroll
        for (int i = 0; i < NG * KU; ++i) kc[i] = *reinterpret_cast<const uint4*>(rec + i * 1024u + lane * 16u);
        const uint32_t* s = reinterpret_cast<const uint32_t*>(rec + 2u * PART) + lane * NG;
        if constexpr (NG == 1) sw[0] = s[0];
        if constexpr (NG == 2) {
            const uint2 v = *reinterpret_cast<const uint2*>(s);
            sw[0] = v.x, sw[1] = v.y;
        }
        if constexpr (NG >= 4)
#pragma unroll
            for (int i = 0; i < NG; i += 4) {
                const uint4 v = *reinterpret_cast<const uint4*>(s + i);
                sw[i] = v.x, sw[i + 1] = v.y, sw[i + 2] = v.z, sw[i + 3] = v.w;
            }
    };
    uint32_t* scales = sh.scales[wave];

    int blk = s0 + (int)wave;
    uint32_t page = 0xFFFFFFFFu;
    const uint8_t* rec = a.kv.base;
    if (blk < s1) {
        page = page_at(blk);
        rec = record_at(blk, page);
        load_keys(rec);
    }
    while (blk < s1) {
        const int next = blk + (int)kWaves, base = blk * (int)kKvBlock;
        const bool bad = page >= a.kv.pages;
        uint4 vc[NG * KU];
#pragma unroll
        for (int i = 0; i < NG * KU; ++i) vc[i] = *reinterpret_cast<const uint4*>(rec + PART + i * 1024u + lane * 16u);
        const uint32_t next_page = next < s1 ? page_at(next) : 0xFFFFFFFFu;

        // scales and biases through LDS, where a lane finds those of its four keys side by side; the
        // largest value scale of the keys that any row sees sets the weights' power of two
        uint32_t vmax = 0u;
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            scales[lane * NG + i] = sw[i];
            const int key = base + (int)((lane * NG + i) & 31u);
            if (lane >= 32u && key >= lo_min && key < hi_max && sw[i] < 0x7F800000u) vmax = max(vmax, sw[i]);  // not NaN's
        }
        vmax = wave_max_u(vmax);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        const int want = min(max((int)(vmax >> 23) - 141, -120), 113);
        if (want > vexp) {
            if (vexp > -1000) {
                const int d = vexp - want;
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int i = 0; i < NG * 4; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[mt][i][e] = ldexpf(o[mt][i][e], d);
            }
            vexp = want;
        }

        // ---- scores of the rows against 32 keys
        float s[MT][8];
#pragma unroll
        for (int tile = 0; tile < 2; ++tile) {
            if constexpr (F32) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[mt][tile * 4 + i] = 0.0f;
            } else {
                // sum_n b_n sum(q_n): the biases are BF16 as they are; depth 8 g + i holds group i % NG
                uint32_t w[NG];
#pragma unroll
                for (int n = 0; n < NG; ++n) w[n] = scales[n * kKvBlock + tile * 16u + (lane & 15u)];
                Frag b;
#pragma unroll
                for (int i = 0; i < 4; ++i) b.u[i] = __builtin_amdgcn_perm(w[(2 * i + 1) % NG], w[(2 * i) % NG], 0x05040100u);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    const float4v acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b.b, qbias[mt].b, float4v{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[mt][tile * 4 + i] = acc[i];
                }
            }
#pragma unroll
            for (int n = 0; n < NG; ++n) {
                const uint4 w4 = *reinterpret_cast<const uint4*>(scales + n * kKvBlock + tile * 16u + g * 4u);
                const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
                Frag k0, k1;
                if constexpr (BITS == 8u) {
                    const uint4 c = kc[n * 2 + tile];
                    k0 = widen_bytes<F32>(c.x, c.y), k1 = widen_bytes<F32>(c.z, c.w);
                } else {
                    const uint4 c = kc[n];
                    k0 = widen_nibbles<F32>(tile ? c.z : c.x), k1 = widen_nibbles<F32>(tile ? c.w : c.y);
                }
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    float4v acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int part = 0; part < (F32 ? 4 : 2); part += 2) {
                        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0.h, query(mt, n, part).h, acc, 0, 0, 0);
                        acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1.h, query(mt, n, part + 1).h, acc, 0, 0, 0);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float& to = s[mt][tile * 4 + i];
                        to = fmaf(scale_of<BITS, F32>(w[i]), acc[i], to);
                        if constexpr (F32) to = fmaf(bias_of<BITS, F32>(w[i]), qsum[mt][n], to);
                    }
                }
            }
        }
        const uint8_t* next_rec = rec;
        if (next < s1) {
            next_rec = record_at(next, next_page);
            load_keys(next_rec);
        }

        // ---- weights
        const bool masked = base < lo_max || base + (int)kKvBlock > hi_min;
        float p[MT][8];
        uint32_t seen[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            float top = kNegInf;
            seen[mt] = 0xFFu;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (bad) s[mt][j] = __builtin_nanf("");
            if (masked) {
                asm volatile("");  // a branch, not selects: few records are masked
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int key = base + (j >> 2) * 16 + (int)g * 4 + (j & 3);
                    if (key < row[mt].lo || key >= row[mt].hi) s[mt][j] = kNegInf, seen[mt] &= ~(1u << j);
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) top = fmaxf(top, s[mt][j]);
            top = fmaxf(m[mt], rows_max(top) * factor[mt]);
            const float zero = top == kNegInf ? 0.0f : top;
            if (__any(top > m[mt])) {
                const float alpha = __builtin_amdgcn_exp2f(m[mt] - zero);
                l[mt] *= alpha;
#pragma unroll
                for (int n = 0; n < NG; ++n) obias[mt][n] *= alpha;
#pragma unroll
                for (int i = 0; i < NG * 4; ++i) o[mt][i] *= alpha;
                m[mt] = top;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                p[mt][j] = __builtin_amdgcn_exp2f(fmaf(s[mt][j], factor[mt], -zero));
                l[mt] += p[mt][j];
            }
        }

        // ---- weighted values
        const float unit = __uint_as_float((uint32_t)(127 - vexp) << 23);
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            const uint4 wa = *reinterpret_cast<const uint4*>(scales + (NG + n) * kKvBlock + g * 4u);
            const uint4 wb = *reinterpret_cast<const uint4*>(scales + (NG + n) * kKvBlock + 16u + g * 4u);
            Frag ph[MT], pl[MT];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                uint32_t w[8] = {wa.x, wa.y, wa.z, wa.w, wb.x, wb.y, wb.z, wb.w};
                if (masked) {
                    asm volatile("");
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (!((seen[mt] >> j) & 1u)) w[j] = 0u;  // what the slot holds may be anything, NaN too
                }
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float scale = scale_of<BITS, F32>(w[j]), bias = bias_of<BITS, F32>(w[j]);
                    v[j] = p[mt][j] * unit * scale;
                    obias[mt][n] = fmaf(p[mt][j], bias, obias[mt][n]);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int x = BITS == 8u ? 2 * i : (i & 2) * 2 + (i & 1), y = x + (BITS == 8u ? 1 : 2);
                    ph[mt].u[i] = pack_fp16(v[x], v[y]);
                    if constexpr (F32) {
                        const Pair h = unpack_fp16(ph[mt].u[i]);
                        pl[mt].u[i] = pack_fp16(v[x] - h.lo, v[y] - h.hi);
                    }
                }
            }
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                Frag f;
                if constexpr (BITS == 8u) {
                    const uint4 c = vc[n * 2 + (d >> 1)];
                    f = (d & 1) ? widen_bytes<F32>(c.z, c.w) : widen_bytes<F32>(c.x, c.y);
                } else {
                    const uint4 c = vc[n];
                    f = (d & 2) ? widen_halves<F32>(c.z, c.w, (d & 1) * 4u) : widen_halves<F32>(c.x, c.y, (d & 1) * 4u);
                }
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    o[mt][n * 4 + d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f.h, ph[mt].h, o[mt][n * 4 + d], 0, 0, 0);
                    if constexpr (F32) o[mt][n * 4 + d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(f.h, pl[mt].h, o[mt][n * 4 + d], 0, 0, 0);
                }
            }
        }
        blk = next;
        page = next_page;
        rec = next_rec;
    }

    // ---- the four waves join: every wave scales its sums to the workgroup's maximum
    __syncthreads();
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        l[mt] = rows_sum(l[mt]);
#pragma unroll
        for (int n = 0; n < NG; ++n) obias[mt][n] = rows_sum(obias[mt][n]);
        if (!live[mt]) m[mt] = kNegInf, l[mt] = 0.0f;
        if (row[mt].over) m[mt] = 0.0f, l[mt] = __builtin_nanf("");
        if (g == 0u) sh.m[wave][mt * 16 + lane] = m[mt], sh.l[wave][mt * 16 + lane] = l[mt];
    }
    __syncthreads();
    float own[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const uint32_t r = mt * 16u + (lane & 15u);
        const float top = fmaxf(fmaxf(sh.m[0][r], sh.m[1][r]), fmaxf(sh.m[2][r], sh.m[3][r]));
        own[mt] = live[mt] && top != kNegInf ? __builtin_amdgcn_exp2f(m[mt] - top) : 0.0f;
    }
    // thread tid writes 4 values of row tid / 16 (and 16 + that); these are that row's
    const uint32_t out_row = threadIdx.x >> 4, col = (threadIdx.x & 15u) * 4u;
    float top[MT], total[MT];
    Row to[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const uint32_t r = mt * 16u + out_row;
        to[mt] = row_of(a, it, it.row0 + r);
        top[mt] = fmaxf(fmaxf(sh.m[0][r], sh.m[1][r]), fmaxf(sh.m[2][r], sh.m[3][r]));
        total[mt] = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < kWaves; ++w)
            if (sh.l[w][r] != 0.0f) total[mt] += sh.l[w][r] * __builtin_amdgcn_exp2f(sh.m[w][r] - top[mt]);
        if (a.parts > 1u && col == 0u && to[mt].exists)
            a.stats[((uint64_t)to[mt].token * a.q_heads + to[mt].head) * a.parts + it.part] = make_float2(top[mt], total[mt]);
    }
#pragma unroll
    for (int n = 0; n < NG; ++n) {
        if (n) __syncthreads();
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    v[e] = own[mt] != 0.0f ? own[mt] * (ldexpf(o[mt][n * 4 + d][e], kUnit + vexp) + obias[mt][n]) : 0.0f;
                *reinterpret_cast<float4*>(&sh.sums[wave][mt * 16 + (lane & 15u)][d * 16 + g * 4]) = make_float4(v[0], v[1], v[2], v[3]);
            }
        __syncthreads();
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            const uint32_t r = mt * 16u + out_row;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (uint32_t w = 0; w < kWaves; ++w) {
                const float4 x = *reinterpret_cast<const float4*>(&sh.sums[w][r][col]);
                v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
            }
            if (!to[mt].exists) continue;
            if (a.parts > 1u) {
                if (total[mt] != 0.0f)
                    *reinterpret_cast<float4*>(a.sums + (((uint64_t)to[mt].token * a.q_heads + to[mt].head) * a.parts + it.part) * D +
                                               n * 64u + col) = v;
            } else {
                const float r1 = total[mt] != 0.0f ? 1.0f / total[mt] : 0.0f;
                store_out<F32>(a.out, to[mt].token * a.out_stride + (uint64_t)to[mt].head * D + n * 64u + col,
                               make_float4(v.x * r1, v.y * r1, v.z * r1, v.w * r1));
            }
        }
    }
}

// ---- many rows ------------------------------------------------------------------------------------
// A tile of 64 MT rows of BF16 queries, 16 MT to a wave. The workgroup widens each record once, to fp16
// values in LDS (key and value = (code - middle) * s' + b', one packed fused multiply-add per two codes, s'
// and b' brought to the record's size by a power of two, so a value is rounded to 11 bits or to 2^-25 of
// the record's largest), and every wave takes them from there as operands: the per-key scales, 144
// instructions per 16 rows and record above, are paid once per workgroup. While a record is multiplied,
// the next one is widened into the other half of LDS and the one after it is on its way to registers.
template <int NG>
struct Wide {
    uint4 k[2][NG][2][2][64];   // [half][group][tile of 16 keys][chunk of 32 values][lane]
    uint4 v[2][NG][4][64];      // [half][group][tile of 16 values][lane]
    int range[kWaves][2];
};

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
union Half2 {
    uint32_t u;
    half2v h;
};
__device__ inline uint32_t fma_fp16(uint32_t x, uint32_t s, uint32_t b) {
    Half2 p, q, r;
    p.u = x, q.u = s, r.u = b;
    p.h = p.h * q.h + r.h;
    return p.u;
}

template <int NG, uint32_t BITS, int MT>
__device__ inline void attend_many(const AttnArgs& a, const Item& it, Wide<NG>& sh) {
    constexpr int KU = BITS == 8u ? 2 : 1, UNITS = NG * KU, PER = (UNITS + 3) / 4;  // 16-byte loads of a wave, of keys and of values
    constexpr uint32_t D = NG * 64u, PART = NG * 64u * kKvBlock * BITS / 8u;
    constexpr float kMiddle = BITS == 8u ? 128.0f : 8.0f;
    const uint32_t lane = threadIdx.x & 63u, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    Row row[MT];
    bool live[MT];
    int lo_min = 0x7FFFFFFF, lo_max = 0, hi_min = 0x7FFFFFFF, hi_max = 0;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        row[mt] = row_of(a, it, it.row0 + (wave * MT + mt) * 16u + (lane & 15u));
        live[mt] = row[mt].exists && row[mt].lo < row[mt].hi;
        if (live[mt]) {
            lo_min = min(lo_min, row[mt].lo), lo_max = max(lo_max, row[mt].lo);
            hi_min = min(hi_min, row[mt].hi), hi_max = max(hi_max, row[mt].hi);
        } else {
            row[mt].lo = 0, row[mt].hi = 0x7FFFFFFF;
        }
    }
    auto least = [](int x, int y) { return min(x, y); };
    auto most = [](int x, int y) { return max(x, y); };
    lo_min = wave_reduce(lo_min, least), lo_max = wave_reduce(lo_max, most);
    hi_min = wave_reduce(hi_min, least), hi_max = wave_reduce(hi_max, most);
    if (lane == 0u) sh.range[wave][0] = lo_min, sh.range[wave][1] = hi_max;
    __syncthreads();
    int all_lo = 0x7FFFFFFF, all_hi = 0;  // keys that some row of the tile sees
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) all_lo = min(all_lo, sh.range[w][0]), all_hi = max(all_hi, sh.range[w][1]);
    int s0 = 0, s1 = 0;
    if (all_hi > 0) {
        const int b0 = all_lo / (int)kKvBlock, b1 = (all_hi + (int)kKvBlock - 1) / (int)kKvBlock;
        const int per = (b1 - b0 + (int)it.splits - 1) / (int)it.splits;
        s0 = min(b1, b0 + (int)it.split * per), s1 = min(b1, s0 + per);
    }

    float factor[MT];
    Frag q[MT][NG][2];
    const float sign = a.scale_log2e < 0.0f ? -1.0f : a.scale_log2e == 0.0f ? 0.0f : 1.0f;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const uint64_t at = row[mt].token * a.q_stride + (uint64_t)row[mt].head * D + g * 16u;
        float top = 0.0f;
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float x[8];
                load_q8<false>(a.q, at + n * 64u + c * 8u, x);
#pragma unroll
                for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[i]));
            }
        top = rows_max(top);
        const int shift = top > 0.0f ? 14 - ((int)(__float_as_uint(top) >> 23) - 127) : 0;
        factor[mt] = sign == 0.0f ? 1.0f : ldexpf(fabsf(a.scale_log2e), -shift);
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float v[8];
                load_q8<false>(a.q, at + n * 64u + c * 8u, v);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = ldexpf(v[i], shift) * sign;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int j = BITS == 8u ? 2 * i : i, k = j + (BITS == 8u ? 1 : 4);
                    q[mt][n][c].u[i] = pack_fp16(v[j], v[k]);
                }
            }
    }
    float4v o[MT][NG * 4];
    float m[MT], l[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        m[mt] = kNegInf, l[mt] = 0.0f;
#pragma unroll
        for (int i = 0; i < NG * 4; ++i) o[mt][i] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
    }

    // ---- a record on its way: registers, then LDS
    const uint32_t page_mask = (1u << a.kv.page_shift) / kKvBlock - 1u, block_shift = a.kv.page_shift - 5u;
    auto page_at = [&](int blk) {
        const uint32_t i = (uint32_t)blk >> block_shift;
        return i < it.table ? it.pages[i] : 0xFFFFFFFFu;
    };
    auto record_at = [&](int blk, uint32_t page) {
        return a.kv.base + kv_record_at(a.kv, page < a.kv.pages ? page : 0u, it.head, (uint32_t)blk & page_mask);
    };
    uint4 kr[PER], vr[PER];
    uint32_t kw[PER * (BITS == 8u ? 1 : 2)], all[NG];
    constexpr int VG = BITS == 8u ? (PER + 1) / 2 : PER;  // groups that a wave's value units belong to
    uint4 vw[VG][2];
    const uint32_t first = wave * PER;
    auto load = [&](const uint8_t* rec) {
        const uint32_t* words = reinterpret_cast<const uint32_t*>(rec + 2u * PART);
#pragma unroll
        for (int i = 0; i < NG; ++i) all[i] = words[lane * NG + i];
        if (first < UNITS) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const uint32_t u = first + i;
                kr[i] = *reinterpret_cast<const uint4*>(rec + u * 1024u + lane * 16u);
                vr[i] = *reinterpret_cast<const uint4*>(rec + PART + u * 1024u + lane * 16u);
                if constexpr (BITS == 8u) {
                    kw[i] = words[(u >> 1) * kKvBlock + (u & 1u) * 16u + (lane & 15u)];
                } else {
                    kw[2 * i] = words[u * kKvBlock + (lane & 15u)];
                    kw[2 * i + 1] = words[u * kKvBlock + 16u + (lane & 15u)];
                }
            }
#pragma unroll
            for (int i = 0; i < VG; ++i) {
                const uint32_t n = BITS == 8u ? (first + 2 * i) >> 1 : first + i;
                vw[i][0] = *reinterpret_cast<const uint4*>(words + (NG + n) * kKvBlock + g * 4u);
                vw[i][1] = *reinterpret_cast<const uint4*>(words + (NG + n) * kKvBlock + 16u + g * 4u);
            }
        }
    };
    // The powers of two of a record's keys and values: below 2^(e + 15) with a scale's largest code and its
    // bias. Words of keys that no row sees are left out, and NaN. The values' is the largest so far.
    int kexp = 0, vexp = -1000;
    bool vnan = false;
    auto sizes = [&](int base) {
        uint32_t top = 0u;
        bool nan = false;
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const int key = base + (int)((lane * NG + i) & 31u);
            const bool in = key >= all_lo && key < all_hi;
            const uint32_t s = all[i] >> 23, b = (all[i] >> 7) & 0xFFu;
            if (in && s < 255u) top = max(top, max(s + BITS, b));
            nan |= in && s >= 255u;
        }
        const uint32_t kt = wave_max_u(lane < 32u ? top : 0u), vt = wave_max_u(lane < 32u ? 0u : top);
        kexp = min(max((int)kt - 140, -120), 113);
        vexp = max(vexp, min(max((int)vt - 140, -120), 113));
        vnan = __ballot(nan && lane >= 32u) != 0ull;
    };
    // s' and b' of a word; outside the visible keys, and (values) where it is NaN, both 0
    auto scaled = [&](uint32_t w, int key, float unit, bool values) {
        const bool in = key >= all_lo && key < all_hi && !(values && w >= 0x7F800000u);
        const float s = __uint_as_float(w & 0xFFFF0000u) * unit, b = __uint_as_float(w << 16) * unit;
        return Pair{in ? s : 0.0f, in ? fmaf(kMiddle, s, b) : 0.0f};
    };
    auto widen = [&](int half, int base) {
        if (first >= UNITS) return;
        const float kunit = __uint_as_float((uint32_t)(127 - kexp) << 23), vunit = __uint_as_float((uint32_t)(127 - vexp) << 23);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const uint32_t u = first + i;
#pragma unroll
            for (int t = 0; t < (BITS == 8u ? 1 : 2); ++t) {
                const uint32_t n = BITS == 8u ? u >> 1 : u, tile = BITS == 8u ? u & 1u : (uint32_t)t;
                const Pair p = scaled(kw[BITS == 8u ? i : 2 * i + t], base + (int)(tile * 16u + (lane & 15u)), kunit, false);
                const uint32_t s = pack_fp16(p.lo, p.lo), b = pack_fp16(p.hi, p.hi);
                Frag f[2];
                if constexpr (BITS == 8u) f[0] = widen_bytes<true>(kr[i].x, kr[i].y), f[1] = widen_bytes<true>(kr[i].z, kr[i].w);
                else f[0] = widen_nibbles<true>(t ? kr[i].z : kr[i].x), f[1] = widen_nibbles<true>(t ? kr[i].w : kr[i].y);
#pragma unroll
                for (int c = 0; c < 2; ++c) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) f[c].u[e] = fma_fp16(f[c].u[e], s, b);
                    sh.k[half][n][tile][c][lane] = make_uint4(f[c].u[0], f[c].u[1], f[c].u[2], f[c].u[3]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < VG; ++i) {
            const uint32_t w[8] = {vw[i][0].x, vw[i][0].y, vw[i][0].z, vw[i][0].w, vw[i][1].x, vw[i][1].y, vw[i][1].z, vw[i][1].w};
            uint32_t s[4], b[4];  // in the order of the codes
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int x = BITS == 8u ? 2 * e : (e & 2) * 2 + (e & 1), y = x + (BITS == 8u ? 1 : 2);
                const Pair p = scaled(w[x], base + (x >> 2) * 16 + (int)g * 4 + (x & 3), vunit, true);
                const Pair r = scaled(w[y], base + (y >> 2) * 16 + (int)g * 4 + (y & 3), vunit, true);
                s[e] = pack_fp16(p.lo, r.lo), b[e] = pack_fp16(p.hi, r.hi);
            }
#pragma unroll
            for (int j = 0; j < (BITS == 8u ? 2 : 1); ++j) {
                const int iu = BITS == 8u ? 2 * i + j : i;
                if (iu >= PER) break;
                const uint32_t u = first + iu;
                const uint4 c = vr[iu];
#pragma unroll
                for (int d = 0; d < (BITS == 8u ? 2 : 4); ++d) {
                    Frag f;
                    if constexpr (BITS == 8u) f = d ? widen_bytes<true>(c.z, c.w) : widen_bytes<true>(c.x, c.y);
                    else f = (d & 2) ? widen_halves<true>(c.z, c.w, (d & 1) * 4u) : widen_halves<true>(c.x, c.y, (d & 1) * 4u);
#pragma unroll
                    for (int e = 0; e < 4; ++e) f.u[e] = fma_fp16(f.u[e], s[e], b[e]);
                    const uint32_t n = BITS == 8u ? u >> 1 : u, tile = BITS == 8u ? (u & 1u) * 2u + d : (uint32_t)d;
                    sh.v[half][n][tile][lane] = make_uint4(f.u[0], f.u[1], f.u[2], f.u[3]);
                }
            }
        }
    };
    auto operand = [&](const uint4& v) {
        Frag f;
        f.u[0] = v.x, f.u[1] = v.y, f.u[2] = v.z, f.u[3] = v.w;
        return f;
    };

    uint32_t page = 0xFFFFFFFFu, next_page = 0xFFFFFFFFu;
    int ov = -1000;  // the power of two that the sums are in
    if (s0 < s1) {
        page = page_at(s0);
        load(record_at(s0, page));
        sizes(s0 * (int)kKvBlock);
        widen(0, s0 * (int)kKvBlock);
        if (s0 + 1 < s1) {
            next_page = page_at(s0 + 1);
            load(record_at(s0 + 1, next_page));
        }
    }
    for (int blk = s0; blk < s1; ++blk) {
        __syncthreads();  // this record is in LDS, and nobody reads the other half any more
        const int half = (blk - s0) & 1, base = blk * (int)kKvBlock, kx = kexp, vx = vexp;
        const bool bad = page >= a.kv.pages, values_nan = vnan;
        page = next_page;
        if (blk + 1 < s1) {
            sizes(base + (int)kKvBlock);
            widen(half ^ 1, base + (int)kKvBlock);
            if (blk + 2 < s1) {
                next_page = page_at(blk + 2);
                load(record_at(blk + 2, next_page));
            }
        }
        if (base >= hi_max || base + (int)kKvBlock <= lo_min) continue;  // none of this wave's rows sees it
        if (vx > ov) {
            if (ov > -1000) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                    for (int i = 0; i < NG * 4; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[mt][i][e] = ldexpf(o[mt][i][e], ov - vx);
            }
            ov = vx;
        }
        float4v s[MT][2];
#pragma unroll
        for (int tile = 0; tile < 2; ++tile) {
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) s[mt][tile] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int n = 0; n < NG; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const Frag k = operand(sh.k[half][n][tile][c][lane]);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) s[mt][tile] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k.h, q[mt][n][c].h, s[mt][tile], 0, 0, 0);
                }
        }
        const bool masked = base < lo_max || base + (int)kKvBlock > hi_min;
        Frag p[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            const float f = ldexpf(factor[mt], kx);
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = s[mt][j >> 2][j & 3];
            if (bad || masked) {
                asm volatile("");
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int key = base + (j >> 2) * 16 + (int)g * 4 + (j & 3);
                    x[j] = key < row[mt].lo || key >= row[mt].hi ? kNegInf : bad ? __builtin_nanf("") : x[j];
                }
            }
            float top = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
            // weights are up to 2^14: small ones stay normal numbers in fp16
            top = fmaxf(m[mt], fmaf(rows_max(top), f, -14.0f));
            const float zero = top == kNegInf ? 0.0f : top;
            if (__any(top > m[mt])) {
                const float alpha = __builtin_amdgcn_exp2f(m[mt] - zero);
                l[mt] *= alpha;
#pragma unroll
                for (int i = 0; i < NG * 4; ++i) o[mt][i] *= alpha;
                m[mt] = top;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[j] = __builtin_amdgcn_exp2f(fmaf(x[j], f, -zero));
                l[mt] += x[j];
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = BITS == 8u ? 2 * e : (e & 2) * 2 + (e & 1), j = i + (BITS == 8u ? 1 : 2);
                p[mt].u[e] = pack_fp16(x[i], x[j]);
            }
        }
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                const Frag v = operand(sh.v[half][n][d][lane]);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) o[mt][n * 4 + d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v.h, p[mt].h, o[mt][n * 4 + d], 0, 0, 0);
            }
        if (values_nan) {  // rows that see a group of NaN: they were taken as 0
            const uint32_t pg = page_at(blk);
            const uint32_t* words = reinterpret_cast<const uint32_t*>(record_at(blk, pg) + 2u * PART);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int n = 0; n < NG; ++n) {
                    float hit = 0.0f;
                    for (int j = 0; j < 8; ++j) {
                        const int t = (j >> 2) * 16 + (int)g * 4 + (j & 3), key = base + t;
                        if (key >= row[mt].lo && key < row[mt].hi && words[(NG + n) * kKvBlock + t] >= 0x7F800000u) hit = 1.0f;
                    }
                    if (rows_max(hit) != 0.0f)
#pragma unroll
                        for (int i = n * 4; i < n * 4 + 4; ++i)
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[mt][i][e] = __builtin_nanf("");
                }
        }
    }

#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        float total = rows_sum(l[mt]);
        if (!live[mt]) m[mt] = kNegInf, total = 0.0f;
        if (row[mt].over) m[mt] = 0.0f, total = __builtin_nanf("");
        if (!row[mt].exists) continue;
        const uint64_t r = (uint64_t)row[mt].token * a.q_heads + row[mt].head;
        const float by = a.parts > 1u ? 1.0f : total != 0.0f ? 1.0f / total : 0.0f;
        if (a.parts > 1u && g == 0u) a.stats[r * a.parts + it.part] = make_float2(m[mt], total);
#pragma unroll
        for (int i = 0; i < NG * 4; ++i) {
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = total != 0.0f && live[mt] ? ldexpf(o[mt][i][e], ov) * by : total;
            const float4 x = make_float4(v[0], v[1], v[2], v[3]);
            if (a.parts > 1u) *reinterpret_cast<float4*>(a.sums + (r * a.parts + it.part) * D + i * 16u + g * 4u) = x;
            else store_out<false>(a.out, row[mt].token * a.out_stride + (uint64_t)row[mt].head * D + i * 16u + g * 4u, x);
        }
    }
}

// Workgroups are dealt out to the eight dies in turn. Tiles that read the same keys are neighbours in
// `index`; this takes neighbours to one die, whose L2 then holds the keys for all of them.
__device__ inline uint32_t same_die(uint32_t id, uint32_t n) {
    const uint32_t per = n / kXcds, rest = n % kXcds, die = id % kXcds;
    return die * per + min(die, rest) + id / kXcds;
}

// MTP and MTO: rows of a prefix's and an own tile, as the multiple of 16 that a wave holds; kMany and
// more is attend_many, with MT = that - kMany.
constexpr int kMany = 8;
constexpr uint32_t tile_rows(int mt) { return mt > kMany ? 64u * (mt - kMany) : 16u * mt; }
template <int NG, uint32_t BITS, bool F32, int MT>
struct Body {
    typedef Shared<NG, F32, MT> Lds;
    static __device__ void run(const AttnArgs& a, const Item& it, Lds& sh) { attend<NG, BITS, F32, MT>(a, it, sh); }
};
template <int NG, uint32_t BITS, int MT>
    requires(MT > kMany)
struct Body<NG, BITS, false, MT> {
    typedef Wide<NG> Lds;
    static __device__ void run(const AttnArgs& a, const Item& it, Lds& sh) { attend_many<NG, BITS, MT - kMany>(a, it, sh); }
};

template <int NG, uint32_t BITS, bool F32, int MTP, int MTO>
__global__ __launch_bounds__(kThreads, NG <= 4 ? 2 : 1) void k_attend(const AttnArgs a) {
    typedef Body<NG, BITS, F32, MTP> Prefix;
    typedef Body<NG, BITS, F32, MTO> Own;
    __shared__ union {
        typename Prefix::Lds p;
        typename Own::Lds o;
    } sh;
    Item it;
    uint32_t id = blockIdx.x;
    it.prefix = id < a.prefix_items;
    if (it.prefix) {
        id = same_die(id, a.prefix_items);
        const uint32_t tile = id % a.prefix_tiles, rest = id / a.prefix_tiles;
        it.split = rest % a.prefix_splits, it.splits = a.prefix_splits, it.part = it.split;
        it.head = rest / a.prefix_splits;
        it.seq = 0u, it.row0 = tile * tile_rows(MTP), it.rows = a.batch * a.q_len * a.group;
        it.pages = a.prefix_pages, it.table = (a.prefix_len + (1u << a.kv.page_shift) - 1u) >> a.kv.page_shift;
    } else {
        id -= a.prefix_items;
        if (a.own_tiles > 1u) id = same_die(id, a.items - a.prefix_items);
        const uint32_t tile = id % a.own_tiles;
        uint32_t rest = id / a.own_tiles;
        it.split = rest % a.own_splits, it.splits = a.own_splits, it.part = a.prefix_splits + it.split;
        rest /= a.own_splits;
        it.head = rest % a.kv.heads, it.seq = rest / a.kv.heads;
        it.row0 = tile * tile_rows(MTO), it.rows = a.q_len * a.group;
        it.pages = a.pages + (uint64_t)it.seq * a.page_stride, it.table = a.page_stride;
    }
    if constexpr (MTP == MTO) {
        Prefix::run(a, it, sh.p);
    } else {
        if (it.prefix) Prefix::run(a, it, sh.p);
        else Own::run(a, it, sh.o);
    }
}

// Joins the partial results of a row: its largest maximum, then the weighted sums. head_dim / 4 threads
// to a row.
template <bool F32>
__global__ __launch_bounds__(kThreads) void k_join(const AttnArgs a, uint32_t head_dim, uint32_t rows) {
    const uint32_t per = head_dim / 4u, r = blockIdx.x * (kThreads / per) + threadIdx.x / per, col = (threadIdx.x % per) * 4u;
    if (r >= rows) return;
    const float2* st = a.stats + (uint64_t)r * a.parts;
    float top = kNegInf;
    for (uint32_t i = 0; i < a.parts; ++i) top = fmaxf(top, st[i].x);
    float total = 0.0f;
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (uint32_t i = 0; i < a.parts; ++i) {
        if (st[i].y == 0.0f) continue;  // its sums were not written
        const float w = __builtin_amdgcn_exp2f(st[i].x - top);
        total += w * st[i].y;
        const float4 x = *reinterpret_cast<const float4*>(a.sums + ((uint64_t)r * a.parts + i) * head_dim + col);
        v.x = fmaf(w, x.x, v.x), v.y = fmaf(w, x.y, v.y), v.z = fmaf(w, x.z, v.z), v.w = fmaf(w, x.w, v.w);
    }
    const float r1 = total != 0.0f ? 1.0f / total : 0.0f;
    const uint32_t token = r / a.q_heads, head = r % a.q_heads;
    store_out<F32>(a.out, token * a.out_stride + (uint64_t)head * head_dim + col, make_float4(v.x * r1, v.y * r1, v.z * r1, v.w * r1));
}

// Rows of a tile: one row of 16 to a wave up to 16 rows, two (where registers hold them: head_dim up to 128)
// up to kFewRows, the many-row body beyond.
template <int NG, bool F32>
struct Tiles {
    static constexpr int kFew = NG <= 2 ? 2 : 1, kLarge = F32 ? kFew : kMany + (NG <= 2 ? 2 : 1);
};
constexpr uint32_t kFewRows = 32;

template <int NG, uint32_t BITS, bool F32, int MTP, int MTO>
void launch_tiles(const AttnArgs& a, hipStream_t st) {
    hipLaunchKernelGGL((k_attend<NG, BITS, F32, MTP, MTO>), dim3(a.items), dim3(kThreads), 0, st, a);
}

template <int NG, uint32_t BITS, bool F32>
void launch_typed(const AttnArgs& a, const AttnPlan& plan, hipStream_t st) {
    typedef Tiles<NG, F32> X;
    const uint32_t p = plan.prefix_tile_rows, o = plan.own_tile_rows;
    if constexpr (!F32) {
        if (o == tile_rows(X::kLarge)) return launch_tiles<NG, BITS, F32, X::kLarge, X::kLarge>(a, st);
        if (p == tile_rows(X::kLarge)) {
            if (X::kFew > 1 && o == tile_rows(X::kFew)) return launch_tiles<NG, BITS, F32, X::kLarge, X::kFew>(a, st);
            return launch_tiles<NG, BITS, F32, X::kLarge, 1>(a, st);
        }
    }
    if constexpr (X::kFew > 1) {
        if (o == tile_rows(X::kFew)) return launch_tiles<NG, BITS, F32, X::kFew, X::kFew>(a, st);
        if (p == tile_rows(X::kFew)) return launch_tiles<NG, BITS, F32, X::kFew, 1>(a, st);
    }
    launch_tiles<NG, BITS, F32, 1, 1>(a, st);
}

uint32_t tile_for(uint64_t rows, uint32_t head_dim, int dtype) {
    if (rows <= 16u) return 16u;
    const uint32_t few = head_dim <= 128u ? 32u : 16u;
    if (rows <= kFewRows || dtype == TURBO_HIDDEN_F32) return few;
    return head_dim <= 128u ? 128u : 64u;
}

template <bool F32>
void launch_dtype(const AttnArgs& a, const AttnPlan& plan, uint32_t head_dim, hipStream_t st) {
    const bool wide = a.kv.bits == 8u;
    switch (head_dim) {
        case 64u: wide ? launch_typed<1, 8u, F32>(a, plan, st) : launch_typed<1, 4u, F32>(a, plan, st); break;
        case 128u: wide ? launch_typed<2, 8u, F32>(a, plan, st) : launch_typed<2, 4u, F32>(a, plan, st); break;
        case 256u: wide ? launch_typed<4, 8u, F32>(a, plan, st) : launch_typed<4, 4u, F32>(a, plan, st); break;
        default: wide ? launch_typed<8, 8u, F32>(a, plan, st) : launch_typed<8, 4u, F32>(a, plan, st); break;
    }
}

}  // namespace

// Rows of 32 to a workgroup halve the widening of codes per row where registers hold them (head_dim up to
// 256, FP32 up to 128). Keys are split until about two workgroups per compute unit have work, but not
// below 8 records (two to a wave): then a workgroup's start and end weigh more than its keys.
AttnPlan plan_attention(uint32_t batch, uint32_t q_len, uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim, int dtype,
                        uint32_t prefix_len, uint32_t own_most, uint32_t window, uint32_t cus) {
    AttnPlan p{};
    const uint64_t group = q_heads / kv_heads, own_rows = q_len * group, all_rows = batch * own_rows;
    p.own_tile_rows = tile_for(own_rows, head_dim, dtype);
    p.prefix_tile_rows = prefix_len ? std::max(tile_for(all_rows, head_dim, dtype), p.own_tile_rows) : p.own_tile_rows;
    auto records = [&](uint64_t keys, uint64_t spread) {
        if (window) keys = std::min<uint64_t>(keys, (uint64_t)window + spread);
        return (keys + kKvBlock - 1u) / kKvBlock;
    };
    const uint64_t pr = prefix_len ? records(prefix_len, prefix_len / 4u) : 0u, orr = own_most ? records(own_most, q_len) : 0u;
    const uint64_t pt = prefix_len ? (all_rows + p.prefix_tile_rows - 1u) / p.prefix_tile_rows : 0u;
    const uint64_t ot = (own_rows + p.own_tile_rows - 1u) / p.own_tile_rows;
    const uint64_t work = kv_heads * (pt * pr + batch * ot * orr);
    const uint64_t per = std::max<uint64_t>(8u, (work + 2u * cus - 1u) / (2u * cus));
    p.prefix_tiles = (uint32_t)pt;
    p.prefix_splits = prefix_len ? (uint32_t)((pr + per - 1u) / per) : 0u;
    p.own_tiles = (uint32_t)ot;
    p.own_splits = own_most ? (uint32_t)((orr + per - 1u) / per) : 0u;
    if (!prefix_len && !own_most) p.own_splits = 1u;  // still writes zeros, or NaN past the tables
    p.prefix_items = kv_heads * pt * p.prefix_splits;
    p.items = p.prefix_items + (uint64_t)batch * kv_heads * ot * p.own_splits;
    p.parts = p.prefix_splits + p.own_splits;
    p.rows = (uint64_t)batch * q_len * q_heads;
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
    a.parts = plan.parts;
    if (dtype == TURBO_HIDDEN_F32) launch_dtype<true>(a, plan, head_dim, st);
    else launch_dtype<false>(a, plan, head_dim, st);
    check_hip(hipGetLastError(), "attention");
    if (plan.parts > 1u) {
        const uint32_t per_group = kThreads / (head_dim / 4u), rows = (uint32_t)plan.rows;
        const dim3 grid((rows + per_group - 1u) / per_group), block(kThreads);
        if (dtype == TURBO_HIDDEN_F32) hipLaunchKernelGGL((k_join<true>), grid, block, 0, st, a, head_dim, rows);
        else hipLaunchKernelGGL((k_join<false>), grid, block, 0, st, a, head_dim, rows);
        check_hip(hipGetLastError(), "attention");
    }
}

}  // namespace tdt

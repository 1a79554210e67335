// Attention of a batch over the quantised cache; the rows of all sequences share a workgroup over the prefix.
//
// A workgroup takes one key/value head, a tile of 16 MT query rows and a range of keys: of the prefix
// (rows of every sequence of the batch) or of one sequence's own keys (its rows). Its four waves take the
// range's 32-token records in turn, each with its own running maximum and sum, and join at the end; a
// second kernel joins the workgroups' partial results. A record goes from memory to registers in the
// order of the matrix instructions' operands, and the waves never wait for each other on the way:
//   S^T = K Q^T, keys as the first operand; the rows' queries lie in LDS as the second, in fp16 after a
//     power of two of the row.
//   O^T += V^T P^T: a lane holds the scores of 8 keys of one row, and those 8 keys' value codes are its
//     bytes of the record, so the weights are the second operand as they are.
// A code enters as a whole number in fp16, exact: code - 128 (8 bits) or code - 8 (4 bits), two by one byte
// permute and one packed addition. (As denormals, code * 2^-24, they need no addition, but products of
// denormals add up with 4 to 7 bits less than FP32 has; uncentred, sums of codes that are all positive cancel
// against the biases: 5e-5 of the result in place of 2e-7, 777 keys of 4 bits.)
//   A key's scale and centre (the value of the middle code) enter its score in FP32: sum over the groups of 64 of
//   scale (codes . q) + centre sum(q), the second part by one FP32 matrix instruction per 16 keys and four groups.
//   A value's scale enters its weight, sum of (weight * scale) codes, and the centres are added with the weights
//   themselves, in FP32 matrix instructions.
//   BF16 queries: q is exact in fp16 (to 2^-40 of the row's largest), weights times scale are rounded to 11
//   bits, 2^-12 of each, against the output's 2^-9. FP32 queries: q and the weights times scale in two fp16
//   parts each (22 bits).
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
constexpr uint32_t kJoinStats = 1024;
constexpr float kNegInf = -__builtin_inff();

union Frag {
    half8 h;
    uint32_t u[4];
};

// Two numbers rounded to BF16 (nearest even, NaN stays NaN), one instruction on gfx950.
__device__ inline uint32_t pack_bf16(float lo, float hi) {
    typedef float float2v __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    union {
        bf16x2 b;
        uint32_t u;
    } x;
    x.b = __builtin_convertvector((float2v{lo, hi}), bf16x2);
    return x.u;
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

// A pair of 16-bit codes as fp16 numbers, code - 128 (8 bits) or code - 8 (4 bits), by way of 1024 + code,
// whose upper bytes (0x64) are in the pair already.
template <uint32_t BITS>
__device__ inline uint32_t centred(uint32_t pair) {
    typedef _Float16 half2v __attribute__((ext_vector_type(2)));
    union {
        uint32_t u;
        half2v h;
    } x;
    x.u = pair;
    const _Float16 middle = (_Float16)(BITS == 8u ? -1152.0f : -1032.0f);
    x.h += half2v{middle, middle};
    return x.u;
}
// eight bytes, in order; the permute takes the upper bytes from a constant
__device__ inline Frag widen_bytes(uint32_t a, uint32_t b) {
    constexpr uint32_t top = 0x64646464u;
    Frag f;
    f.u[0] = centred<8u>(__builtin_amdgcn_perm(top, a, 0x04010400u));
    f.u[1] = centred<8u>(__builtin_amdgcn_perm(top, a, 0x04030402u));
    f.u[2] = centred<8u>(__builtin_amdgcn_perm(top, b, 0x04010400u));
    f.u[3] = centred<8u>(__builtin_amdgcn_perm(top, b, 0x04030402u));
    return f;
}
// eight nibbles of one word: operand elements 2 p, 2 p + 1 are nibbles p, p + 4 (the queries are laid out alike)
__device__ inline Frag widen_nibbles(uint32_t w) {
    Frag f;
#pragma unroll
    for (int p = 0; p < 4; ++p) f.u[p] = centred<4u>(((w >> (4 * p)) & 0x000F000Fu) | 0x64006400u);
    return f;
}
// the low (shift 0) or high (shift 4) halves of eight bytes: elements are bytes 0, 2, 1, 3 of each word
// (the weights are laid out alike)
__device__ inline Frag widen_halves(uint32_t a, uint32_t b, uint32_t shift) {
    Frag f;
    f.u[0] = centred<4u>(((a >> shift) & 0x000F000Fu) | 0x64006400u);
    f.u[1] = centred<4u>(((a >> (8u + shift)) & 0x000F000Fu) | 0x64006400u);
    f.u[2] = centred<4u>(((b >> shift) & 0x000F000Fu) | 0x64006400u);
    f.u[3] = centred<4u>(((b >> (8u + shift)) & 0x000F000Fu) | 0x64006400u);
    return f;
}
// A word's scale, and its centre: the value of the middle code
__device__ inline float scale_of(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
template <uint32_t BITS>
__device__ inline float centre_of(uint32_t w) {
    return fmaf(BITS == 8u ? 128.0f : 8.0f, scale_of(w), __uint_as_float(w << 16));
}

// floor(log2(x)) of a number that is not negative (-127 below 2^-126)
__device__ inline float power_of(float x) { return (float)((int)(__float_as_uint(x) >> 23) - 127); }

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
// Word i of a table that no kernel of the call writes, by a scalar load: a vector load would wait for the
// record's loads before it (they return in order), a microsecond per record.
__device__ inline uint32_t table_word(const uint32_t* table, uint32_t i) {
    typedef const uint32_t __attribute__((address_space(4))) * Constant;
    return ((Constant) reinterpret_cast<uintptr_t>(table))[i];
}
// A value that is the same in all lanes, in a scalar register.
__device__ inline int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
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

// n / d for n below 2^31, by the multiplier that divider() made of d
__device__ inline uint32_t quotient(uint32_t n, Divider d) { return d.factor ? __umulhi(n, d.factor) >> d.shift : n; }

// What a workgroup takes. Records are numbered in order: the prefix's, whose last one may hold fewer than 32 of
// its tokens, then the sequence's own.
struct Item {
    bool shared;                   // rows of every sequence, over the prefix alone
    uint32_t head, row0, rows;     // key/value head, first row of the tile, rows there are
    uint32_t seq;                  // otherwise: the sequence
    uint32_t split, splits, part;
    int begin, end;                // positions of the keys
    const uint32_t* pages;         // of the sequence's own tokens
};

struct Row {
    uint32_t token, head;          // of q and out
    int lo, hi;                    // positions it sees, of the item's
    bool exists, over;             // over: passes its page table
};

__device__ inline Row row_of(const AttnArgs& a, const Item& it, uint32_t r) {
    Row w;
    w.exists = r < it.rows;
    if (!w.exists) r = it.rows - 1u;
    const uint32_t b = it.shared ? quotient(r, a.by_rows) : it.seq, in = it.shared ? r - b * (a.q_len * a.group) : r;
    const uint32_t t = quotient(in, a.by_group);
    w.token = b * a.q_len + t;
    w.head = it.head * a.group + in - t * a.group;
    const long long pos = (long long)a.kv_len[b] - (long long)a.q_len + t;
    w.over = pos >= (long long)a.prefix_len + ((long long)a.page_stride << a.kv.page_shift);
    const long long lo = a.window ? pos - (long long)a.window + 1 : 0;
    w.lo = max(it.begin, (int)(lo > 0 ? (lo < 0x7FFFFFFF ? lo : 0x7FFFFFFF) : 0));
    w.hi = w.over ? 0 : min(it.end, (int)(pos >= 0 ? pos + 1 : 0));
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
    else *reinterpret_cast<uint2*>(static_cast<uint16_t*>(out) + at) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
}

__device__ inline Frag operand(uint4 v) {
    Frag f;
    f.u[0] = v.x, f.u[1] = v.y, f.u[2] = v.z, f.u[3] = v.w;
    return f;
}

template <int NG, bool F32, int MT>
struct Shared {
    static constexpr uint32_t kRow = 68;  // floats of a row of 64, padded
    union {
        struct {
            uint4 q[MT][NG][F32 ? 4 : 2][64];            // the queries as second operands: [.., chunk of 32 (and low parts)][lane]
            // a wave's record: scales and centres, [keys, values][group][32 tokens]
            float scale[kWaves][2 * NG * kKvBlock], centre[kWaves][2 * NG * kKvBlock];
        };
        float sums[kWaves][16 * MT][kRow];
    };
    float m[kWaves][16 * MT], l[kWaves][16 * MT], factor[16 * MT];
    int lo[16 * MT], hi[16 * MT];           // what the rows see, read where a record is not seen whole
    float qsum[16 * MT][NG + 1];  // of a row's groups
};

template <int NG, uint32_t BITS, bool F32, int MT>
__device__ inline void attend(const AttnArgs& a, const Item& it, Shared<NG, F32, MT>& sh) {
    constexpr int KU = BITS == 8u ? 2 : 1;       // 16-byte loads per group of keys or values
    // Registers hold a record's keys and values at once; otherwise the next keys are loaded when all but the last
    // group's values are used. Earlier, two tiles of heads of 256 spill (64 sequences behind 32,768: 139 -> 186 us).
    constexpr bool kEarly = NG * MT <= 4;
    // A row's weights p are relative to m, a running maximum that is left alone while they stay below 2^kSlack:
    // of 16 rows one has a new maximum in most records, and the sums would be rescaled there.
    // The sums of weighted values are in units of 2^(m + u - kUnit). u is a whole number for each row: 2^u is at most
    // the largest p * size that the row has met, a value's size being the larger of 128 scale and |centre| over its
    // head, and u rises where a p * size could pass 2^(u + kRoom + 1). A weight times a scale is then below 2^15,
    // and one that fp16 holds with fewer than 11 bits is off by 2^-32 of the row's largest weighted size. Tokens
    // that a row does not see, or gives no weight, do not enter.
    constexpr float kSlack = 7.0f, kRoom = 7.0f;
    constexpr int kUnit = 14, kScaleUnit = 20;  // scales of values lie in LDS times 2^20, so that no power leaves FP32
    constexpr uint32_t D = NG * 64u, PART = NG * 64u * kKvBlock * BITS / 8u;
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
    lo_min = uniform(wave_reduce(lo_min, least)), lo_max = uniform(wave_reduce(lo_max, most));
    hi_min = uniform(wave_reduce(hi_min, least)), hi_max = uniform(wave_reduce(hi_max, most));
    // records: of the prefix up to prefix_records, then of the sequence's own tokens
    const int prefix_len = (int)a.prefix_len, prefix_records = (prefix_len + (int)kKvBlock - 1) / (int)kKvBlock;
    auto record_of = [&](int pos) {
        return pos < prefix_len ? pos / (int)kKvBlock : prefix_records + (pos - prefix_len) / (int)kKvBlock;
    };
    int s0 = 0, s1 = 0;  // this split's records
    if (hi_max > 0) {
        const int b0 = record_of(lo_min), b1 = record_of(hi_max - 1) + 1;
        const int per = (b1 - b0 + (int)it.splits - 1) / (int)it.splits;
        s0 = min(b1, b0 + (int)it.split * per), s1 = min(b1, s0 + per);
    }

    // ---- the queries, fp16 after a power of two that takes the row's largest to 2^14 .. 2^15, in LDS for
    // all four waves, which divide the tiles among them and then a tile's groups; a negative scale is
    // theirs, so that larger scores are larger weights
    const float sign = a.scale_log2e < 0.0f ? -1.0f : a.scale_log2e == 0.0f ? 0.0f : 1.0f;
    constexpr int kSharers = (int)kWaves / MT;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        if (mt != (int)wave % MT) continue;
        const uint64_t at = row[mt].token * a.q_stride + (uint64_t)row[mt].head * D + g * 16u;
        float x[NG][2][8], top = 0.0f, bad = 0.0f;
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                load_q8<F32>(a.q, at + n * 64u + c * 8u, x[n][c]);
#pragma unroll
                for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[n][c][i])), bad = fmaf(x[n][c][i], 0.0f, bad);
            }
        top = rows_max(top);
        bad = rows_sum(bad);  // NaN where a value is infinite or NaN: so is the row then, whatever its scores' signs
        const int shift = top > 0.0f ? 14 - ((int)(__float_as_uint(top) >> 23) - 127) : 0;
        const float factor = sign == 0.0f ? 1.0f : fminf(ldexpf(fabsf(a.scale_log2e), a.scale_power - shift), 0x1.fffffep127f);
        if (g == 0u && (int)wave < MT) sh.factor[mt * 16 + lane] = factor + bad;
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            if (n % kSharers != (int)wave / MT) continue;
            float sum = 0.0f;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = ldexpf(x[n][c][i], shift) * sign, sum += v[i];
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
                sh.q[mt][n][c][lane] = make_uint4(h.u[0], h.u[1], h.u[2], h.u[3]);
                if constexpr (F32) sh.q[mt][n][2 + c][lane] = make_uint4(low.u[0], low.u[1], low.u[2], low.u[3]);
            }
            sum = rows_sum(sum);
            if (g == 0u) sh.qsum[mt * 16 + lane][n] = sum;
        }
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
        if (threadIdx.x < 16u) sh.lo[mt * 16 + lane] = row[mt].lo, sh.hi[mt * 16 + lane] = row[mt].hi;
    __syncthreads();
    // the groups' sums as the FP32 products' second operand: that of group 4 h + lane / 16
    constexpr int kFours = NG > 4 ? NG / 4 : 1;
    float qsum[MT][kFours];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int h = 0; h < kFours; ++h) qsum[mt][h] = g < (uint32_t)NG ? sh.qsum[mt * 16 + (lane & 15u)][min(4u * h + g, NG - 1u)] : 0.0f;

    float4v o[MT][NG * 4];
    float4v oc[MT];  // the centres' sums, rows of the product: element e of lane / 16 is group (4 (lane / 16) + e) mod NG
    float m[MT], l[MT], u[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        m[mt] = kNegInf, l[mt] = 0.0f, u[mt] = -119.0f, oc[mt] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < NG * 4; ++i) o[mt][i] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
    }

    const uint32_t page_mask = (1u << a.kv.page_shift) / kKvBlock - 1u, block_shift = a.kv.page_shift - 5u;
    const uint32_t prefix_table = (a.prefix_len + (1u << a.kv.page_shift) - 1u) >> a.kv.page_shift;
    auto page_at = [&](int rec) {  // the page of a record; past the table or the cache: none
        const int r = uniform(rec);
        const bool own = r >= prefix_records;
        const uint32_t i = (uint32_t)(own ? r - prefix_records : r) >> block_shift;
        return i < (own ? a.page_stride : prefix_table) ? table_word(own ? it.pages : a.prefix_pages, i) : 0xFFFFFFFFu;
    };
    auto record_at = [&](int rec, uint32_t page) {
        const uint32_t r = (uint32_t)(rec >= prefix_records ? rec - prefix_records : rec);
        return a.kv.base + kv_record_at(a.kv, page < a.kv.pages ? page : 0u, it.head, r & page_mask);
    };
    const uint32_t at16 = lane * 16u, at_words = lane * (NG * 4u);
    uint4 kc[NG * KU], vc[NG * KU];
    uint32_t sw[NG];  // the record's scales and biases, NG words to a lane: the keys' in the first 32 lanes
    auto load_keys = [&](const uint8_t* rec) {
#pragma unroll
        for (int i = 0; i < NG * KU; ++i) kc[i] = *reinterpret_cast<const uint4*>(rec + i * 1024u + at16);
        const uint8_t* w = rec + 2u * PART;
        if constexpr (NG == 1) sw[0] = *reinterpret_cast<const uint32_t*>(w + at_words);
        if constexpr (NG == 2) {
            const uint2 v = *reinterpret_cast<const uint2*>(w + at_words);
            sw[0] = v.x, sw[1] = v.y;
        }
        if constexpr (NG >= 4)
#pragma unroll
            for (int i = 0; i < NG; i += 4) {
                const uint4 v = *reinterpret_cast<const uint4*>(w + i * 4 + at_words);
                sw[i] = v.x, sw[i + 1] = v.y, sw[i + 2] = v.z, sw[i + 3] = v.w;
            }
    };
    auto load_values = [&](const uint8_t* rec) {
#pragma unroll
        for (int i = 0; i < NG * KU; ++i) vc[i] = *reinterpret_cast<const uint4*>(rec + PART + i * 1024u + at16);
    };
    float *scales = sh.scale[wave], *centres = sh.centre[wave];

    // A record's scales and centres, and the power of two of its largest value's size. Words of keys that no row
    // sees become 0, as do a value's of NaN.
    float largest = 0.0f;
    bool vnan = false;
    auto prepare = [&](int base, int end) {
        end = min(end, hi_max);
        if (base < lo_min || base + (int)kKvBlock > end) {
            asm volatile("");  // a branch, not selects: few records are not seen whole
#pragma unroll
            for (int i = 0; i < NG; ++i) {
                const int key = base + (int)((lane * NG + i) & 31u);
                if (key < lo_min || key >= end) sw[i] = 0u;
            }
        }
        uint32_t top = 0u;
#pragma unroll
        for (int i = 0; i < NG; ++i) top = max(top, sw[i]);
        vnan = false;
        if (__any(lane >= 32u && top >= 0x7F800000u)) {
            asm volatile("");
#pragma unroll
            for (int i = 0; i < NG; ++i)
                if (lane >= 32u && sw[i] >= 0x7F800000u) sw[i] = 0u, vnan = true;
            vnan = __any(vnan);
        }
        float sc[NG], ce[NG], size = 0.0f;
        const float by = lane < 32u ? 1.0f : (float)(1 << kScaleUnit);
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            sc[i] = scale_of(sw[i]), ce[i] = centre_of<BITS>(sw[i]);
            size = fmaxf(size, fmaxf(128.0f * sc[i], fabsf(ce[i])));
            sc[i] *= by;
        }
        size = fmaxf(size, dpp_mov<dpp::kXor1>(size));
        size = fmaxf(size, dpp_mov<dpp::kXor2>(size));
        size = fmaxf(size, dpp_mov<dpp::kRor4>(size));
        size = fmaxf(size, dpp_mov<dpp::kRor8>(size));
        largest = power_of(fmaxf(lane_read(size, 32), lane_read(size, 48)));
        auto put = [&](float* to, const float (&x)[NG]) {
            if constexpr (NG == 1) to[lane] = x[0];
            if constexpr (NG == 2) *reinterpret_cast<float2*>(to + lane * 2u) = make_float2(x[0], x[1]);
            if constexpr (NG >= 4)
#pragma unroll
                for (int i = 0; i < NG; i += 4) *reinterpret_cast<float4*>(to + lane * NG + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
        };
        put(scales, sc);
        put(centres, ce);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    };

    int blk = s0 + (int)wave;
    uint32_t page = 0xFFFFFFFFu;
    const uint8_t* rec = a.kv.base;
    if (blk < s1) {
        page = page_at(blk);
        rec = record_at(blk, page);
        load_keys(rec);
    }
    while (blk < s1) {
        // position of the record's first token, and of the end of the tokens of its kind
        const bool own_keys = blk >= prefix_records;
        const int next = blk + (int)kWaves;
        const int base = own_keys ? prefix_len + (blk - prefix_records) * (int)kKvBlock : blk * (int)kKvBlock;
        const int end = own_keys ? 0x7FFFFFFF : prefix_len;
        const bool bad = page >= a.kv.pages;
        if constexpr (kEarly) load_values(rec);
        const uint32_t next_page = next < s1 ? page_at(next) : 0xFFFFFFFFu;
        prepare(base, end);

        // ---- scores of the rows against 32 keys
        float4v s[MT][2];
#pragma unroll
        for (int tile = 0; tile < 2; ++tile)
#pragma unroll
            for (int h = 0; h < kFours; ++h) {
                const float c = centres[(NG < 4 ? g % NG : 4u * h + g) * kKvBlock + tile * 16u + (lane & 15u)];
#pragma unroll
                for (int mt = 0; mt < MT; ++mt)
                    s[mt][tile] = __builtin_amdgcn_mfma_f32_16x16x4f32(c, qsum[mt][h], h ? s[mt][tile] : float4v{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0);
            }
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            Frag q[MT][F32 ? 4 : 2];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int c = 0; c < (F32 ? 4 : 2); ++c) q[mt][c] = operand(sh.q[mt][n][c][lane]);
#pragma unroll
            for (int tile = 0; tile < 2; ++tile) {
                Frag k[2];
                if constexpr (BITS == 8u) {
                    const uint4 c = kc[n * 2 + tile];
                    k[0] = widen_bytes(c.x, c.y), k[1] = widen_bytes(c.z, c.w);
                } else {
                    const uint4 c = kc[n];
                    k[0] = widen_nibbles(tile ? c.z : c.x), k[1] = widen_nibbles(tile ? c.w : c.y);
                }
                const float4 sc = *reinterpret_cast<const float4*>(scales + n * kKvBlock + tile * 16u + g * 4u);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    float4v acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int c = 0; c < (F32 ? 4 : 2); ++c) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[c & 1].h, q[mt][c].h, acc, 0, 0, 0);
                    s[mt][tile][0] = fmaf(sc.x, acc[0], s[mt][tile][0]);
                    s[mt][tile][1] = fmaf(sc.y, acc[1], s[mt][tile][1]);
                    s[mt][tile][2] = fmaf(sc.z, acc[2], s[mt][tile][2]);
                    s[mt][tile][3] = fmaf(sc.w, acc[3], s[mt][tile][3]);
                }
            }
        }
        // The sums end here: left to itself the compiler moves them past the next loads, to where the scores are
        // used, with all products and scales alive (100 registers).
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) asm volatile("" : "+v"(s[mt][0]), "+v"(s[mt][1]));
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (!kEarly) load_values(rec);
        const uint8_t* next_rec = rec;
        if (next < s1) next_rec = record_at(next, next_page);
        if constexpr (kEarly) {
            if (next < s1) load_keys(next_rec);
        }

        // ---- weights
        const bool masked = base < lo_max || base + (int)kKvBlock > min(hi_min, end);
        float p[MT][8];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            // The factor may leave FP32 (small queries, a large scale): a score of 0 stays 0, and a hidden key's
            // -infinity is set after the product, which would make it NaN.
#pragma unroll
            for (int j = 0; j < 8; ++j) p[mt][j] = s[mt][j >> 2][j & 3] * sh.factor[mt * 16 + (lane & 15u)];
            if (bad || masked) {
                asm volatile("");
                const int lo = sh.lo[mt * 16 + (lane & 15u)], hi = min(sh.hi[mt * 16 + (lane & 15u)], end);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int key = base + (j >> 2) * 16 + (int)g * 4 + (j & 3);
                    if (key < lo || key >= hi) p[mt][j] = kNegInf;
                    else if (bad) p[mt][j] = __builtin_nanf("");
                }
            }
            float top = kNegInf;
#pragma unroll
            for (int j = 0; j < 8; ++j) top = fmaxf(top, p[mt][j]);
            top = rows_max(top);
            // the differences that the exponential takes: a sum of m and a bound would round at large scores
            const float rise = top - m[mt];
            if (__any(rise > kSlack || rise + largest > u[mt] + kRoom)) {  // a bound; the row's own is found here
                asm volatile("");
                if (rise > kSlack) m[mt] = top;
                const float by = rise > kSlack ? rise : 0.0f;
                float need = kNegInf;
#pragma unroll
                for (int tile = 0; tile < 2; ++tile) {
                    float4 size = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma nounroll
                    for (int n = NG; n < 2 * NG; ++n) {
                        constexpr float by = 128.0f / (1 << kScaleUnit);
                        const uint32_t at = n * kKvBlock + tile * 16u + g * 4u;
                        const float4 sc = *reinterpret_cast<const float4*>(scales + at), ce = *reinterpret_cast<const float4*>(centres + at);
                        size.x = fmaxf(size.x, fmaxf(by * sc.x, fabsf(ce.x))), size.y = fmaxf(size.y, fmaxf(by * sc.y, fabsf(ce.y)));
                        size.z = fmaxf(size.z, fmaxf(by * sc.z, fabsf(ce.z))), size.w = fmaxf(size.w, fmaxf(by * sc.w, fabsf(ce.w)));
                    }
                    const float s4[4] = {size.x, size.y, size.z, size.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) need = fmaxf(need, p[mt][tile * 4 + j] - m[mt] + power_of(s4[j]));
                }
                need = fmaxf(fmaxf(floorf(rows_max(need)), floorf(u[mt] - by)), -119.0f);
                const float alpha = __builtin_amdgcn_exp2f(u[mt] - need - by);
                l[mt] *= __builtin_amdgcn_exp2f(-by);
                oc[mt] *= alpha;
#pragma unroll
                for (int i = 0; i < NG * 4; ++i) o[mt][i] *= alpha;
                u[mt] = need;
            }
            const float zero = m[mt] == kNegInf ? 0.0f : m[mt], unit = ldexpf(1.0f, kUnit - kScaleUnit - (int)u[mt]);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                p[mt][j] = __builtin_amdgcn_exp2f(p[mt][j] - zero);
                l[mt] += p[mt][j];
                p[mt][j] *= unit;
            }
        }

        // ---- weighted values
        {
            const float* c = centres + (NG + lane % NG) * kKvBlock + g * 4u;
            const float4 ca = *reinterpret_cast<const float4*>(c), cb = *reinterpret_cast<const float4*>(c + 16u);
            const float c8[8] = {ca.x, ca.y, ca.z, ca.w, cb.x, cb.y, cb.z, cb.w};
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int j = 0; j < 8; ++j) oc[mt] = __builtin_amdgcn_mfma_f32_16x16x4f32(c8[j], p[mt][j], oc[mt], 0, 0, 0);
        }
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            const float* sn = scales + (NG + n) * kKvBlock + g * 4u;
            const float4 sa = *reinterpret_cast<const float4*>(sn), sb = *reinterpret_cast<const float4*>(sn + 16u);
            const float s8[8] = {sa.x, sa.y, sa.z, sa.w, sb.x, sb.y, sb.z, sb.w};
            if constexpr (!kEarly)
                if (n == NG - 1) {
                    if (next < s1) {
                        load_keys(next_rec);
                    } else {  // the old ones end here: kept alive for a loop that is over, they cost their registers
#pragma unroll
                        for (int i = 0; i < NG * KU; ++i) kc[i] = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
                        for (int i = 0; i < NG; ++i) sw[i] = 0u;
                    }
                }
            Frag ph[MT], pl[F32 ? MT : 1];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {  // in the order of the codes
                    const int x = BITS == 8u ? 2 * e : (e & 2) * 2 + (e & 1), y = x + (BITS == 8u ? 1 : 2);
                    const float u = p[mt][x] * s8[x], v = p[mt][y] * s8[y];
                    ph[mt].u[e] = pack_fp16(u, v);
                    if constexpr (F32) {
                        const Pair h = unpack_fp16(ph[mt].u[e]);
                        pl[mt].u[e] = pack_fp16(u - h.lo, v - h.hi);
                    }
                }
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                Frag f;
                if constexpr (BITS == 8u) {
                    const uint4 c = vc[n * 2 + (d >> 1)];
                    f = (d & 1) ? widen_bytes(c.z, c.w) : widen_bytes(c.x, c.y);
                } else {
                    const uint4 c = vc[n];
                    f = (d & 2) ? widen_halves(c.z, c.w, (d & 1) * 4u) : widen_halves(c.x, c.y, (d & 1) * 4u);
                }
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    float4v& to = o[mt][n * 4 + d];
                    to = __builtin_amdgcn_mfma_f32_16x16x32_f16(f.h, ph[mt].h, to, 0, 0, 0);
                    if constexpr (F32) to = __builtin_amdgcn_mfma_f32_16x16x32_f16(f.h, pl[mt].h, to, 0, 0, 0);
                }
            }
        }
        if (vnan) {  // rows that see a group of NaN, which was taken as 0
            const uint32_t* raw = reinterpret_cast<const uint32_t*>(rec + 2u * PART);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int n = 0; n < NG; ++n) {
                    float hit = 0.0f;
                    const int lo = sh.lo[mt * 16 + (lane & 15u)], hi = min(sh.hi[mt * 16 + (lane & 15u)], end);
#pragma nounroll
                    for (int j = 0; j < 8; ++j) {
                        const int in = (j >> 2) * 16 + (int)g * 4 + (j & 3);
                        if (base + in >= lo && base + in < hi && raw[(NG + n) * kKvBlock + in] >= 0x7F800000u) hit = __builtin_nanf("");
                    }
                    hit = rows_sum(hit);
#pragma unroll
                    for (int i = n * 4; i < n * 4 + 4; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[mt][i][e] += hit;
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
        if (!live[mt]) m[mt] = kNegInf, l[mt] = 0.0f;
        if (row[mt].over) m[mt] = 0.0f, l[mt] = __builtin_nanf("");
        if (g == 0u) sh.m[wave][mt * 16 + lane] = m[mt], sh.l[wave][mt * 16 + lane] = l[mt];
    }
    __syncthreads();
    float own[MT];
    bool counts[MT];  // also with a factor of 0, against which NaN stays NaN
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        const uint32_t r = mt * 16u + (lane & 15u);
        const float top = fmaxf(fmaxf(sh.m[0][r], sh.m[1][r]), fmaxf(sh.m[2][r], sh.m[3][r]));
        counts[mt] = live[mt] && top != kNegInf;
        own[mt] = counts[mt] ? __builtin_amdgcn_exp2f(m[mt] - top) : 0.0f;
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
        float centre[MT];  // of group n
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            centre[mt] = oc[mt][NG < 4 ? n : n & 3];
            if constexpr (NG == 8) {
                const float across = __shfl_xor(centre[mt], 16);
                if ((g & 1u) != (uint32_t)n / 4u) centre[mt] = across;
            }
            centre[mt] = ldexpf(centre[mt], (int)u[mt] + kScaleUnit - kUnit);
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = counts[mt] ? own[mt] * (ldexpf(o[mt][n * 4 + d][e], (int)u[mt] - kUnit) + centre[mt]) : 0.0f;
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

template <int NG, uint32_t BITS, bool F32, int MTP, int MTO>
__global__ __launch_bounds__(kThreads, NG <= 4 ? 2 : 1) void k_attend(const AttnArgs a) {
    __shared__ union {
        Shared<NG, F32, MTP> p;
        Shared<NG, F32, MTO> o;
    } sh;
    Item it;
    uint32_t id = blockIdx.x;
    it.shared = id < a.prefix_items;
    if (it.shared) {
        id = same_die(id, a.prefix_items);
        const uint32_t tile = id % a.prefix_tiles, rest = id / a.prefix_tiles;
        it.split = rest % a.prefix_splits, it.splits = a.prefix_splits, it.part = it.split;
        it.head = rest / a.prefix_splits;
        it.seq = 0u, it.row0 = tile * 16u * MTP, it.rows = a.batch * a.q_len * a.group;
        it.begin = 0, it.end = (int)a.prefix_len;
        it.pages = nullptr;
    } else {
        id -= a.prefix_items;
        if (a.own_tiles > 1u) id = same_die(id, a.items - a.prefix_items);
        const uint32_t tile = id % a.own_tiles;
        uint32_t rest = id / a.own_tiles;
        it.split = rest % a.own_splits, it.splits = a.own_splits, it.part = a.prefix_splits + it.split;
        rest /= a.own_splits;
        it.head = rest % a.kv.heads, it.seq = rest / a.kv.heads;
        it.row0 = tile * 16u * MTO, it.rows = a.q_len * a.group;
        it.begin = a.prefix_splits ? (int)a.prefix_len : 0, it.end = 0x7FFFFFFF;
        it.pages = a.pages + (uint64_t)it.seq * a.page_stride;
    }
    if constexpr (MTP == MTO) {
        attend<NG, BITS, F32, MTP>(a, it, sh.p);
    } else {
        if (it.shared) attend<NG, BITS, F32, MTP>(a, it, sh.p);
        else attend<NG, BITS, F32, MTO>(a, it, sh.o);
    }
}

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

// 16-row tiles of a workgroup at most: what the registers of two waves per SIMD hold without spills (heads of 256:
// all 256). One in place of two: 94 -> 117 us (2 x 512 prompt tokens behind 2,000), 100 -> 121 us (128 sequences
// behind 16,000, heads of 128), but 40 -> 34 us (300 prompt tokens with heads of 128, whose workgroups then fill the
// card).
constexpr int most_tiles(uint32_t head_dim, bool f32) { return head_dim <= (f32 ? 128u : 256u) ? 2 : 1; }
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

template <int NG, uint32_t BITS, bool F32, int MTP, int MTO>
void launch_tiles(const AttnArgs& a, hipStream_t st) {
    hipLaunchKernelGGL((k_attend<NG, BITS, F32, MTP, MTO>), dim3(a.items), dim3(kThreads), 0, st, a);
}

template <int NG, uint32_t BITS, bool F32, int MTP>
void launch_own(const AttnArgs& a, uint32_t mto, hipStream_t st) {
    if (mto == MTP) return launch_tiles<NG, BITS, F32, MTP, MTP>(a, st);
    if constexpr (MTP > 1) launch_tiles<NG, BITS, F32, MTP, 1>(a, st);
}

template <int NG, uint32_t BITS, bool F32>
void launch_typed(const AttnArgs& a, const AttnPlan& plan, hipStream_t st) {
    constexpr int most = most_tiles(NG * 64u, F32);
    const uint32_t p = plan.prefix_tile_rows / 16u, o = plan.own_tile_rows / 16u;
    if constexpr (most >= 2)
        if (p == 2u) return launch_own<NG, BITS, F32, 2>(a, o, st);
    launch_own<NG, BITS, F32, 1>(a, o, st);
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
AttnPlan plan_attention(uint32_t batch, uint32_t q_len, uint32_t q_heads, uint32_t kv_heads, uint32_t head_dim, int dtype,
                        uint32_t prefix_len, uint32_t own_most, uint32_t window, uint32_t cus) {
    const uint64_t group = q_heads / kv_heads, own_rows = q_len * group, all_rows = batch * own_rows;
    auto records = [&](uint64_t keys, uint64_t spread) {
        if (window) keys = std::min<uint64_t>(keys, (uint64_t)window + spread);
        return (keys + kKvBlock - 1u) / kKvBlock;
    };
    const uint64_t pr = prefix_len ? records(prefix_len, prefix_len / 4u) : 0u, orr = own_most ? records(own_most, q_len) : 0u;
    AttnPlan p{};
    p.rows = (uint64_t)batch * q_len * q_heads;
    for (uint32_t most = most_tiles(head_dim, dtype == TURBO_HIDDEN_F32);; most /= 2u) {
        p.own_tile_rows = 16u * tiles_for(own_rows, most);
        const uint64_t ot = (own_rows + p.own_tile_rows - 1u) / p.own_tile_rows;
        p.prefix_tile_rows = 16u * tiles_for(all_rows, most);
        uint64_t pt = (all_rows + p.prefix_tile_rows - 1u) / p.prefix_tile_rows;
        const bool shared = pr && 2u * batch * ot > 3u * pt;
        if (!shared) p.prefix_tile_rows = p.own_tile_rows, pt = 0u;
        const uint64_t alone = shared ? orr : pr + orr;  // records of a workgroup's sequence
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
        if (most == 1u || per >= 16u) break;
    }
    p.parts = p.prefix_splits + p.own_splits;
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
    a.by_rows = divider(a.q_len * a.group), a.by_group = divider(a.group);
    if (dtype == TURBO_HIDDEN_F32) launch_dtype<true>(a, plan, head_dim, st);
    else launch_dtype<false>(a, plan, head_dim, st);
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

// Attention of drafted trees over the quantised cache: the rows of a tree see the tokens before it and, of its own
// nodes, those whose bits their masks have. Small calls take the workgroups' kernel of dt_attend.h with the masks.
//
// Its time for trees of many rows is the vector unit's: 32 rows widen every code for themselves. Here a workgroup of 128
// rows of one sequence widens a record once, each wave a quarter of it, into the matrix instructions' operands in LDS, and
// its four waves, 32 rows each, read them from there; the next record is widened meanwhile. It takes the records that all
// its rows see whole, those before the tree; the rest, the tree's own among them, goes to workgroups of the other kind in
// the same launch, and the join adds the parts up.
//   A key or value enters as scale * code + bias in fp16 after a power of two of the token that takes its head's largest
//   near the middle of the exponents: one rounding, 2^-11 of it at most, and 2^-22 (4 bits: 2^-18) of its head's largest
//   where it is small against that. The power of a key multiplies its score in FP32, that of a value its weight before the
//   weight is rounded to 11 bits. Statistics and sums are FP32.
// 24 trees of 64 nodes behind 8,192 shared tokens (heads of 256) 476 -> 391 us, 16 of 64 behind 8,000 with heads of 128
// 397 -> 285, of 64 267 -> 185. What bounds it: the vector unit issues in 53 % of the cycles, the matrix unit is busy in 27 %,
// and the waves wait 27 % of their time, for LDS and at the two barriers of a record. Records come by way of LDS, two
// ahead: in registers they spill with heads of 256 (612 us).
#include "dt_attend.h"
#include "dt_tile.h"

namespace tdt {
namespace {

constexpr uint32_t kWideRows = 128;

// Records of a sequence that end before its tree (a tree that begins inside the prefix leaves the prefix's before it).
__device__ inline int whole_records(const AttnArgs& a, uint32_t seq) {
    const long long before = (long long)a.kv_len[seq] - (long long)a.q_len, prefix = a.prefix_len;
    if (before <= 0) return 0;
    if (before < prefix) return (int)(before / kKvBlock);
    return (int)((prefix + kKvBlock - 1) / kKvBlock + (before - prefix) / kKvBlock);
}

// LDS of a workgroup: a record's operands, and two more records as they come from memory.
template <int NG, uint32_t BITS>
struct Wide {
    // units of 16 codes to a lane that a wave widens, of keys and of values, and loads of 1 KB for them
    static constexpr int kUnits = NG >= 2 ? NG / 2 : 1, kLoads = BITS == 8u ? kUnits : kUnits > 1 ? kUnits / 2 : 1;
    uint4 k[NG * 4][64], v[NG * 4][64];         // keys [group][16 tokens][chunk of 32], values [16 values]
    int k_power[2][kKvBlock], v_power[2][kKvBlock];
    uint32_t words[kWaves][2 * NG * kKvBlock];  // a wave's: scale and bias of [keys, values][group][token] in fp16
    struct {
        uint4 k[kLoads][64], v[kLoads][64];
        uint32_t words[256];                    // [keys, values][group][token]
    } raw[2][kWaves];                           // what a wave widens
};

// scale * code + bias of two codes, each a fp16 denormal (code * 2^-24) and the scale times 2^24
__device__ inline uint32_t widened(uint32_t codes, uint32_t scale, uint32_t bias) {
    typedef _Float16 half2v __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(half2v, codes), __builtin_bit_cast(half2v, scale),
                                                                  __builtin_bit_cast(half2v, bias)));
}
__device__ inline uint32_t lows(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }
__device__ inline uint32_t highs(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }
__device__ inline uint32_t bytes01(uint32_t a) { return __builtin_amdgcn_perm(a, a, 0x0C010C00u); }
__device__ inline uint32_t bytes23(uint32_t a) { return __builtin_amdgcn_perm(a, a, 0x0C030C02u); }

template <int NG, uint32_t BITS>
__device__ inline void wide(const AttnArgs& a, const Item& it, int records, Wide<NG, BITS>& sh) {
    constexpr uint32_t D = NG * 64u, PART = NG * 64u * kKvBlock * BITS / 8u;
    constexpr float kSlack = 8.0f;
    constexpr int kUnit = 7;                          // weights are at most 2^kSlack and lie times 2^kUnit in fp16
    constexpr int kMiddle = BITS == 8u ? -3 : -7;     // power of two of a widened token's largest: its scale times 2^24 is below 2^16
    constexpr float kMost = BITS == 8u ? 255.0f : 15.0f;
    constexpr int KU = Wide<NG, BITS>::kUnits, kLoads = Wide<NG, BITS>::kLoads;
    const uint32_t lane = threadIdx.x & 63u, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    Row row[2];
    bool some = false;
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
        row[mt] = row_of<true>(a, it, it.row0 + wave * 32u + mt * 16u + (lane & 15u));
        some = some || (row[mt].exists && row[mt].hi > 0);
    }
    const bool some_rows = it.row0 + wave * 32u < it.rows;  // of this wave's
    const int per = (records + (int)it.splits - 1) / (int)it.splits;
    const int s0 = min(records, (int)it.split * per);
    const int s1 = __syncthreads_or(some) ? min(records, s0 + per) : s0;

    // ---- the queries as second operands, fp16 after a power of two that takes the row's largest to 2^14 .. 2^15
    const float sign = a.scale_log2e < 0.0f ? -1.0f : a.scale_log2e == 0.0f ? 0.0f : 1.0f;
    Frag q[2][NG][2];
    float factor[2];
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
        const uint64_t at = row[mt].token * a.q_stride + (uint64_t)row[mt].head * D + g * 16u;
        float top = 0.0f, bad = 0.0f;
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) + at + n * 64u + c * 8u);
                q[mt][n][c] = operand(v);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float x = __uint_as_float(q[mt][n][c].u[i] << 16), y = __uint_as_float(q[mt][n][c].u[i] & 0xFFFF0000u);
                    top = fmaxf(top, fmaxf(fabsf(x), fabsf(y))), bad = fmaf(x, 0.0f, fmaf(y, 0.0f, bad));
                }
            }
        top = rows_max(top);
        bad = rows_sum(bad);  // NaN where a value is infinite or NaN: so is the row then, whatever its scores' signs
        const int shift = top > 0.0f ? 14 - ((int)(__float_as_uint(top) >> 23) - 127) : 0;
        factor[mt] = bad + (sign == 0.0f ? 1.0f : fminf(ldexpf(fabsf(a.scale_log2e), a.scale_power - shift), 0x1.fffffep127f));
#pragma unroll
        for (int n = 0; n < NG; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float v[8];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t w = q[mt][n][c].u[i];
                    v[2 * i] = ldexpf(__uint_as_float(w << 16), shift) * sign;
                    v[2 * i + 1] = ldexpf(__uint_as_float(w & 0xFFFF0000u), shift) * sign;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {  // in the order of the codes
                    const int j = BITS == 8u ? 2 * i : i, k = j + (BITS == 8u ? 1 : 4);
                    q[mt][n][c].u[i] = pack_fp16(v[j], v[k]);
                }
            }
    }

    float4v o[2][NG * 4];
    float m[2], l[2];
    constexpr int kNoUnit = -1000;  // below all that a record needs
    int unit[2] = {kNoUnit, kNoUnit};  // a row's sums are in units of 2^(unit - kUnit)
#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
        m[mt] = kNegInf, l[mt] = 0.0f;
#pragma unroll
        for (int i = 0; i < NG * 4; ++i) o[mt][i] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
    }

    // A lane's number, made anew where the loop has no registers for what follows from it.
    auto this_lane = [&] {
        uint32_t l = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
        asm volatile("" : "+v"(l));
        return l;
    };
    // ---- records from memory to registers, one ahead of their widening
    const int prefix_len = (int)a.prefix_len, prefix_records = (prefix_len + (int)kKvBlock - 1) / (int)kKvBlock;
    const uint32_t page_mask = (1u << a.kv.page_shift) / kKvBlock - 1u, block_shift = a.kv.page_shift - 5u;
    const uint32_t prefix_table = (a.prefix_len + (1u << a.kv.page_shift) - 1u) >> a.kv.page_shift;
    auto page_at = [&](int rec) {  // the page of a record; past the table or the cache: none
        const int r = uniform(rec);
        const bool own = r >= prefix_records;
        const uint32_t i = (uint32_t)(own ? r - prefix_records : r) >> block_shift;
        return i < (own ? a.page_stride : prefix_table) ? table_word(own ? it.pages : a.prefix_pages, i) : 0xFFFFFFFFu;
    };
    const bool keys_wave = NG > 1 || wave < 2u, values_wave = NG > 1 || wave >= 2u;
    const uint32_t unit0 = NG > 1 ? wave * KU : wave & 1u, load0 = BITS == 8u ? unit0 : unit0 / 2u;
    uint32_t bad_pages = 0u;  // bit r % 4
    auto fetch = [&](int r, uint32_t page) {
        const bool bad = page >= a.kv.pages;
        bad_pages = (bad_pages & ~(1u << (r & 3))) | (uint32_t)bad << (r & 3);
        const uint32_t in = (uint32_t)(r >= prefix_records ? r - prefix_records : r) & page_mask;
        const TileSource from(a.kv.base + kv_record_at(a.kv, bad ? 0u : page, it.head, in), a.kv.record);
        const uint32_t lane = this_lane();
        auto& to = sh.raw[(r - s0) & 1][wave];
        from.load(to.words, 2u * PART + min(lane, NG * 16u - 1u) * 16u);
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            from.load(to.k[j], (load0 + j) * 1024u + lane * 16u);
            from.load(to.v[j], PART + (load0 + j) * 1024u + lane * 16u);
        }
    };
    auto landed = [&](int r) {  // record r is there, of which this wave reads only what it fetched itself
        if (r + 1 < s1) __builtin_amdgcn_s_waitcnt(vm_wait(2 * kLoads + 1));
        else __builtin_amdgcn_s_waitcnt(vm_wait(0));
        asm volatile("" ::: "memory");
    };

    // ---- a record into the operands
    uint32_t* const mine = sh.words[wave];
    auto unit_words = [&](const uint4 (&from)[kLoads][64], int j, uint32_t lane, uint32_t (&to)[BITS / 2u]) {
        if constexpr (BITS == 8u) {
            const uint4 x = from[j][lane];
            to[0] = x.x, to[1] = x.y, to[2] = x.z, to[3] = x.w;
        } else {
            const uint2 x = reinterpret_cast<const uint2*>(&from[KU > 1 ? j >> 1 : 0][lane])[(unit0 + j) & 1u];
            to[0] = x.x, to[1] = x.y;
        }
    };
    // scales, biases and powers, and the keys; returns the largest power of the values
    auto widen_keys = [&](int r) {
        const auto& raw = sh.raw[(r - s0) & 1][wave];
        const uint32_t lane = this_lane(), token = lane & 31u, half = lane >> 5;
        uint32_t words[NG];
#pragma unroll
        for (int n = 0; n < NG; ++n) words[n] = raw.words[(half * NG + n) * kKvBlock + token];
        if (r < prefix_records && (r + 1) * (int)kKvBlock > prefix_len)  // behind the prefix: no row sees it
#pragma unroll
            for (int n = 0; n < NG; ++n) words[n] = r * (int)kKvBlock + (int)token < prefix_len ? words[n] : 0u;
        float size = 0.0f;
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            const float s = scale_of(words[n]), b = __uint_as_float(words[n] << 16);
            size = fmaxf(size, words[n] < 0x7F800000u ? fmaxf(fabsf(b), fabsf(fmaf(kMost, s, b))) : 0.0f);
        }
        const int power = (int)(__float_as_uint(size) >> 23) - 127 - kMiddle;
        const bool bad = (bad_pages >> (r & 3)) & 1u;
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            const uint32_t w = pack_fp16(ldexpf(scale_of(words[n]), 24 - power), ldexpf(__uint_as_float(words[n] << 16), -power));
            mine[(half * NG + n) * kKvBlock + token] = words[n] >= 0x7F800000u || (bad && half == 0u) ? 0x7E007E00u : w;
        }
        if (wave == 0u) (half ? sh.v_power : sh.k_power)[r & 1][token] = power;
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int j = 0; j < KU; ++j) {
            if (!keys_wave) break;
            const uint32_t u = unit0 + j, w = mine[(u >> 1) * kKvBlock + (u & 1u) * 16u + (lane & 15u)], s = lows(w, w), b = highs(w, w);
            uint32_t from[BITS / 2u];
            unit_words(raw.k, j, lane, from);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                Frag f;
                if constexpr (BITS == 8u) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        f.u[2 * i] = widened(bytes01(from[c * 2 + i]), s, b);
                        f.u[2 * i + 1] = widened(bytes23(from[c * 2 + i]), s, b);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) f.u[i] = widened((from[c] >> (4 * i)) & 0x000F000Fu, s, b);
                }
                sh.k[u * 2u + c][lane] = make_uint4(f.u[0], f.u[1], f.u[2], f.u[3]);
            }
        }
        int most = power;
        most = max(most, dpp_mov<dpp::kXor1>(most));
        most = max(most, dpp_mov<dpp::kXor2>(most));
        most = max(most, dpp_mov<dpp::kRor4>(most));
        most = max(most, dpp_mov<dpp::kRor8>(most));
        return max(lane_read(most, 32), lane_read(most, 48));
    };
    auto widen_values = [&](int r) {
        const auto& raw = sh.raw[(r - s0) & 1][wave];
        if (!values_wave) return;
        const uint32_t lane = this_lane(), g = lane >> 4;
#pragma unroll
        for (int j = 0; j < KU; ++j) {
            const uint32_t u = unit0 + j;
            const uint32_t* at = mine + (NG + (u >> 1)) * kKvBlock + g * 4u;
            const uint4 x4 = *reinterpret_cast<const uint4*>(at), y4 = *reinterpret_cast<const uint4*>(at + 16u);
            const uint32_t w[8] = {x4.x, x4.y, x4.z, x4.w, y4.x, y4.y, y4.z, y4.w};
            uint32_t s[4], b[4], from[BITS / 2u];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int x = BITS == 8u ? 2 * e : (e & 2) * 2 + (e & 1), y = x + (BITS == 8u ? 1 : 2);
                s[e] = lows(w[x], w[y]), b[e] = highs(w[x], w[y]);
            }
            unit_words(raw.v, j, lane, from);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                Frag f;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t codes;
                    if constexpr (BITS == 8u) codes = (e & 1) ? bytes23(from[c * 2 + (e >> 1)]) : bytes01(from[c * 2 + (e >> 1)]);
                    else codes = (from[e >> 1] >> ((e & 1) * 8 + c * 4)) & 0x000F000Fu;
                    f.u[e] = widened(codes, s[e], b[e]);
                }
                sh.v[u * 2u + c][lane] = make_uint4(f.u[0], f.u[1], f.u[2], f.u[3]);
            }
        }
    };

    constexpr int kReads = NG * 4;
    constexpr int kAhead = 4;  // operands that are on their way while one is multiplied
    Frag x[kAhead];
    int next_power = 0;  // the largest of the next record's values
    if (s0 < s1) {
        fetch(s0, page_at(s0));
        if (s0 + 1 < s1) fetch(s0 + 1, page_at(s0 + 1));
        landed(s0);
        next_power = widen_keys(s0);
        widen_values(s0);
        if (s0 + 2 < s1) fetch(s0 + 2, page_at(s0 + 2));
    }
    __syncthreads();
    for (int r = s0; r < s1; ++r) {
        const int this_power = next_power;
        const uint32_t page = r + 3 < s1 ? page_at(r + 3) : 0xFFFFFFFFu;
        float4v s[2][2];
        if (some_rows) {
            // ---- scores
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) s[mt][0] = s[mt][1] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int n = 0; n < kAhead; ++n) x[n] = operand(sh.k[n][lane]);
#pragma unroll
            for (int n = 0; n < kReads; ++n) {
                const int tile = (n >> 1) & 1;
#pragma unroll
                for (int mt = 0; mt < 2; ++mt)
                    s[mt][tile] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[n % kAhead].h, q[mt][n >> 2][n & 1].h, s[mt][tile], 0, 0, 0);
                if (n + kAhead < kReads) x[n % kAhead] = operand(sh.k[n + kAhead][lane]);
                __builtin_amdgcn_sched_barrier(0);
            }
            __builtin_amdgcn_s_setprio(0);
        }
        __syncthreads();  // all have read the keys, and written the values
        if (r + 1 < s1) {
            landed(r + 1);
            next_power = widen_keys(r + 1);
        }

        if (some_rows) {
            // ---- weights
#pragma unroll
            for (int tile = 0; tile < 2; ++tile) {
                const int4 power = *reinterpret_cast<const int4*>(&sh.k_power[r & 1][tile * 16 + (this_lane() >> 4) * 4u]);
                const int by[4] = {power.x, power.y, power.z, power.w};
#pragma unroll
                for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[mt][tile][e] = ldexpf(s[mt][tile][e], by[e]) * factor[mt];
            }
            __builtin_amdgcn_sched_barrier(0);
            if (r < prefix_records && (r + 1) * (int)kKvBlock > prefix_len) {
#pragma unroll
                for (int mt = 0; mt < 2; ++mt) asm volatile("" : "+v"(s[mt][0]), "+v"(s[mt][1]));  // a branch, not selects
                const int behind = prefix_len - r * (int)kKvBlock - (int)(this_lane() >> 4) * 4;
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if ((j >> 2) * 16 + (j & 3) >= behind) s[0][j >> 2][j & 3] = s[1][j >> 2][j & 3] = kNegInf;
            }
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
                float top = kNegInf;
#pragma unroll
                for (int j = 0; j < 8; ++j) top = fmaxf(top, s[mt][j >> 2][j & 3]);
                top = rows_max(top);
                const float rise = top - m[mt];
                if (__any(rise > kSlack)) {
                    asm volatile("");
                    const float by = rise > kSlack ? rise : 0.0f;
                    if (rise > kSlack) m[mt] = top;
                    l[mt] *= __builtin_amdgcn_exp2f(-by);
                    // The unit falls with the sums, which then lose less than a bit: what large values under keys that led
                    // leave behind does not take the later ones' bits.
                    const int to = max(unit[mt] - (int)fminf(by, 4000.0f), kNoUnit);
                    const float alpha = __builtin_amdgcn_exp2f((float)(unit[mt] - to) - by);
#pragma unroll
                    for (int i = 0; i < NG * 4; ++i) o[mt][i] *= alpha;
                    unit[mt] = to;
                }
                const float zero = m[mt] == kNegInf ? 0.0f : m[mt];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float p = __builtin_amdgcn_exp2f(s[mt][j >> 2][j & 3] - zero);
                    s[mt][j >> 2][j & 3] = p;
                    l[mt] += p;
                }
                if (__any(this_power > unit[mt])) {
                    // The row's unit becomes that power, or, where all such values have next to no weight, what they need:
                    // large values that a row gives no weight do not cost it the bits of others.
                    int need = -2000;
#pragma nounroll
                    for (int tile = 0; tile < 2; ++tile) {
                        const int4 power = *reinterpret_cast<const int4*>(&sh.v_power[r & 1][tile * 16 + (this_lane() >> 4) * 4u]);
                        const int of[4] = {power.x, power.y, power.z, power.w};
                        const float4v t = tile ? s[mt][1] : s[mt][0];
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (t[e] != 0.0f) need = max(need, (int)power_of(t[e]) + of[e]);
                    }
                    need = (int)rows_max((float)need);
                    const int to = max(unit[mt], need >= this_power - 12 ? this_power : need - 7);
                    const float by = ldexpf(1.0f, unit[mt] - to);
#pragma unroll
                    for (int i = 0; i < NG * 4; ++i) o[mt][i] *= by;
                    unit[mt] = to;
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            Frag w[2];
            {
                int by[8];
#pragma unroll
                for (int tile = 0; tile < 2; ++tile) {
                    const int4 power = *reinterpret_cast<const int4*>(&sh.v_power[r & 1][tile * 16 + (this_lane() >> 4) * 4u]);
                    by[tile * 4] = power.x, by[tile * 4 + 1] = power.y, by[tile * 4 + 2] = power.z, by[tile * 4 + 3] = power.w;
                }
#pragma unroll
                for (int mt = 0; mt < 2; ++mt) {
                    int from = kUnit - unit[mt];
                    asm("" : "+v"(from));
#pragma unroll
                    for (int e = 0; e < 4; ++e) {  // in the order of the codes
                        const int x = BITS == 8u ? 2 * e : (e & 2) * 2 + (e & 1), y = x + (BITS == 8u ? 1 : 2);
                        w[mt].u[e] = pack_fp16(ldexpf(s[mt][x >> 2][x & 3], by[x] + from), ldexpf(s[mt][y >> 2][y & 3], by[y] + from));
                    }
                }
            }

            // ---- weighted values
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int n = 0; n < kAhead; ++n) x[n] = operand(sh.v[n][lane]);
#pragma unroll
            for (int n = 0; n < kReads; ++n) {
#pragma unroll
                for (int mt = 0; mt < 2; ++mt) o[mt][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[n % kAhead].h, w[mt].h, o[mt][n], 0, 0, 0);
                if (n + kAhead < kReads) x[n % kAhead] = operand(sh.v[n + kAhead][lane]);
                __builtin_amdgcn_sched_barrier(0);
            }
            __builtin_amdgcn_s_setprio(0);
        }
        __syncthreads();  // all have read the values, and written the next keys
        if (r + 1 < s1) {
            widen_values(r + 1);
            if (r + 3 < s1) fetch(r + 3, page);
        }
    }

#pragma unroll
    for (int mt = 0; mt < 2; ++mt) {
        l[mt] = rows_sum(l[mt]);
        const Row to_row = row_of<true>(a, it, it.row0 + wave * 32u + mt * 16u + (lane & 15u));
        if (!to_row.exists) continue;
        if (to_row.hi <= 0) m[mt] = kNegInf, l[mt] = 0.0f;
        const uint64_t at = ((uint64_t)to_row.token * a.q_heads + to_row.head) * a.parts + it.part;
        if (g == 0u) a.stats[at] = make_float2(m[mt], l[mt]);
        if (l[mt] == 0.0f) continue;
        float* to = a.sums + at * D + g * 4u;
#pragma unroll
        for (int i = 0; i < NG * 4; ++i) {
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = ldexpf(o[mt][i][e], unit[mt] - kUnit);
            *reinterpret_cast<float4*>(to + i * 16) = make_float4(v[0], v[1], v[2], v[3]);
        }
    }
}

template <int NG, uint32_t BITS>
__global__ __launch_bounds__(kThreads, wide_groups(NG * 64u)) void k_tree_wide(const AttnArgs a) {
    __shared__ union {
        Wide<NG, BITS> wide;
        Shared<NG, false, 2, true> rest;
    } sh;
    Item it;
    uint32_t id = blockIdx.x;
    const bool is_wide = id < a.wide_items;
    it.shared = false;
    it.rows = a.q_len * a.group;
    it.begin = 0, it.end = 0x7FFFFFFF;
    // neighbours read the same keys: a sequence's tiles, then, over the prefix, the sequences
    id = is_wide ? same_die(id, a.wide_items) : same_die(id - a.wide_items, a.items - a.wide_items);
    const uint32_t tiles = is_wide ? a.wide_tiles : a.own_tiles, tile = id % tiles;
    id /= tiles;
    it.seq = id % a.batch, id /= a.batch;
    it.splits = is_wide ? a.wide_splits : 1u;
    it.split = id % it.splits, it.head = id / it.splits;
    it.part = is_wide ? it.split : a.wide_splits;
    it.row0 = tile * (is_wide ? kWideRows : 32u);
    it.pages = a.pages + (uint64_t)it.seq * a.page_stride;
    it.first = whole_records(a, it.seq);
    if (is_wide) wide<NG, BITS>(a, it, it.first, sh.wide);
    else attend<NG, BITS, false, 2, true>(a, it, sh.rest);
}

template <int NG>
void launch_wide(const AttnArgs& a, hipStream_t st) {
    if (a.kv.bits == 8u) hipLaunchKernelGGL((k_tree_wide<NG, 8u>), dim3(a.items), dim3(kThreads), 0, st, a);
    else hipLaunchKernelGGL((k_tree_wide<NG, 4u>), dim3(a.items), dim3(kThreads), 0, st, a);
}

}  // namespace

void launch_tree_attend(const AttnArgs& a, const AttnPlan& plan, uint32_t head_dim, int dtype, hipStream_t st) {
    if (plan.wide_splits) {
        if (head_dim == 64u) launch_wide<1>(a, st);
        else if (head_dim == 128u) launch_wide<2>(a, st);
        else launch_wide<4>(a, st);
    } else if (dtype == TURBO_HIDDEN_F32) launch_dtype<true, true>(a, plan, head_dim, st);
    else launch_dtype<false, true>(a, plan, head_dim, st);
    check_hip(hipGetLastError(), "tree attention");
}

}  // namespace tdt

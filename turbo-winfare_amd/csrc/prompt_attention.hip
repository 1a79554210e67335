// Causal attention over whole prompts, packed one after another, keys and values as the projections leave them.
//
// With s_j = scale q . k_j over the keys j that a query at position i sees (j <= i, and i - j < window):
//   out = sum_j 2^(c s_j - m) v_j / sum_j 2^(c s_j - m),  c = scale log2(e), m a running maximum of the c s_j,
// one pass over the keys, statistics and sums in FP32. Rows are (token, head) pairs: the heads that share keys lie side by
// side, so a tile of rows reads its keys once for all of them. A wave has 32 rows and takes 32 or 64 keys at a time:
//   S^T = K Q^T, keys as the first operand: a lane holds 16 scores of one row for every 32 keys.
//   O^T += V^T P^T: those 16 keys are the lane's part of the second operand as they are, if the first operand takes the
//     keys in the same order; values are transposed on their way out of LDS.
// The maximum, and with it the sums, is left alone while weights stay below 2^8. Weights are rounded to BF16 for BF16 inputs
// (2^-8 of each at most, as the result itself), the sum of weights is that of the unrounded ones.
#include "dt_internal.h"
#include "dt_mfma.h"
#include "dt_step.h"
#include "dt_tile.h"

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
    u32x4 x;
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

// Tile number `id` of all sequences' tiles of `rows` rows (a token has one for each of its heads that share keys). Every
// wave finds it for itself.
// Up to 64 sequences: the last tiles, which have most keys, come first, and among equal ones the sequences in order. The
// number of tiles at a level or above falls with the level, so the level is found by halving.
// More sequences, whose tiles fill the card in any order: sequence b's tiles begin at number (its first row) / rows + b, which
// leaves room for them all, and a number belongs to the last sequence that begins at or before it.
__device__ inline Item locate(const PromptArgs& a, uint32_t id, uint32_t rows) {
    const uint32_t lane = threadIdx.x & 63u;
    auto start_of = [&](uint32_t b) { return min(a.starts[b], a.tokens); };
    auto uniform = [](uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); };
    Item it{};
    uint32_t found;
    if (a.batch <= 64u) {
        const uint32_t first = lane < a.batch ? start_of(lane) : 0u, len = lane < a.batch ? max(start_of(lane + 1u), first) - first : 0u;
        const uint32_t tiles = (len * a.group + rows - 1u) / rows;
        auto at_least = [&](uint32_t level) {  // tiles of all sequences from this level on
            return uniform(wave_reduce(tiles > level ? tiles - level : 0u, [](uint32_t x, uint32_t y) { return x + y; }));
        };
        uint32_t lo = 0u, hi = (a.tokens * a.group + rows - 1u) / rows;  // at_least(lo) > id >= at_least(hi)
        if (at_least(0u) <= id) return it;
        while (hi - lo > 1u) {
            const uint32_t mid = (lo + hi) / 2u;
            if (at_least(mid) > id) lo = mid;
            else hi = mid;
        }
        const uint32_t rank = id - at_least(lo + 1u);  // by all lanes: a reduction
        const unsigned long long have = __ballot(tiles > lo);
        const unsigned long long mine = __ballot(tiles > lo && (uint32_t)__popcll(have & ((1ull << lane) - 1ull)) == rank);
        if (mine == 0ull) return it;
        found = (uint32_t)__ffsll(mine) - 1u;
        it.tile = lo;
    } else {
        uint32_t lo = 0u, n = a.batch, begins = 0u;  // the sequence is one of n from lo on
        while (true) {
            const uint32_t step = (n + 63u) / 64u, b = lo + lane * step;
            const uint32_t at = lane * step < n ? start_of(b) * a.group / rows + b : 0xFFFFFFFFu;
            const uint32_t before = (uint32_t)__popcll(__ballot(at <= id));
            if (before == 0u) return it;
            lo += (before - 1u) * step;
            n = min(step, n - (before - 1u) * step);
            begins = uniform(__shfl(at, (int)before - 1));
            if (n == 1u) break;
        }
        found = lo;
        it.tile = id - begins;
    }
    it.first = uniform(start_of(found));
    it.len = max(uniform(start_of(found + 1u)), it.first) - it.first;
    it.exists = it.tile < (it.len * a.group + rows - 1u) / rows;
    return it;
}

// A row's running maximum (times scale) and sum, and the weights of a lane's scores.
struct Softmax {
    float m = kNegInf, l = 0.0f;
    // Scores to weights; true where the sums have to be multiplied by alpha first.
    template <int N>
    __device__ inline bool weights(f32x16 (&s)[N], float c, float& alpha) {
        float top = kNegInf;
#pragma unroll
        for (int b = 0; b < N; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, s[b][r]);
        top = halves_max(top) * c;
        const bool moves = __any(top > m + kSlack);
        alpha = 1.0f;
        if (moves) {
            const float now = fmaxf(m, top);
            alpha = now == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(m - now);
            m = now;
            l *= alpha;
        }
        const float zero = m == kNegInf ? 0.0f : m;
#pragma unroll
        for (int b = 0; b < N; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[b][r] = __builtin_amdgcn_exp2f(fmaf(s[b][r], c, -zero));
                l += s[b][r];
            }
        return moves;
    }
};

__device__ inline bool not_finite(float v) { return !(fabsf(v) < __builtin_inff()); }
__device__ inline float number(float x) { return x; }
__device__ inline float number(uint16_t x) { return __uint_as_float((uint32_t)x << 16); }

// The 32 rows of a wave, or of a workgroup: row r of a sequence is head r % group of token r / group, so the heads that
// share keys lie side by side and their rows end at the same key.
struct Rows {
    uint32_t pos, lo;      // of the lane's row: its token, and the first key that it sees
    uint32_t first, last;  // tokens of the 32 rows
    uint32_t head;
    bool exists;
    __device__ inline Rows(const PromptArgs& a, const Item& it, uint32_t kv_head, uint32_t row0) {
        const uint32_t col = threadIdx.x & 31u, all = it.len * a.group;
        const uint32_t r = min(row0 + col, all - 1u);
        exists = row0 + col < all;
        pos = r / a.group;
        head = kv_head * a.group + r - pos * a.group;
        lo = from(a, pos);
        first = min(row0, all - 1u) / a.group;
        last = min(row0 + kRows - 1u, all - 1u) / a.group;
    }
    static __device__ inline uint32_t from(const PromptArgs& a, uint32_t token) {
        return a.window && token + 1u > a.window ? token + 1u - a.window : 0u;
    }
    // Whether some row sees some of n keys from base on, and whether all rows see all of them
    __device__ inline bool some(const PromptArgs& a, uint32_t base, uint32_t n) const { return base <= last && base + n > from(a, first); }
    __device__ inline bool all(const PromptArgs& a, uint32_t base, uint32_t n) const { return base + n <= first + 1u && base >= from(a, last); }
};

// A value that is infinite or NaN turns every row of its tile to NaN, also those that do not see it, as its weight is 0 there, and a
// key that is infinite does where FP32 enters in parts. What has to be computed again for that is found at the end, among the rows
// (bits of `left`, from row0 on) whose result is not finite. Where a row's sum of weights is NaN or 0 its scores make it so, and
// it stays. The others stay where each column that is not finite in one of them has such a value at a key that all of them see;
// the keys are gone through from the first on. NaN in the first token of 6,000, which every later row sees: 0.11 ms as without it,
// 22 if all rows are computed again (heads of 128, 8 / 2 of them).
template <int D, int DW, class E>
__device__ inline bool stays(const PromptArgs& a, const Item& it, uint32_t kv_head, uint32_t row0, uint32_t left, uint32_t column) {
    constexpr uint32_t kAtOnce = 8u;
    constexpr int kCols = DW > 64 ? DW / 64 : 1;  // of a lane
    const uint32_t lane = min(threadIdx.x & 63u, DW - 1u);
    const uint32_t from = Rows::from(a, (row0 + 31u - (uint32_t)__clz((int)left)) / a.group), to = (row0 + (uint32_t)__ffs(left) - 1u) / a.group;
    bool open[kCols];  // columns that are not finite, until a value is found
#pragma unroll
    for (int i = 0; i < kCols; ++i) open[i] = false;
#pragma nounroll
    for (uint32_t rest = left; rest; rest &= rest - 1u) {
        const uint32_t row = row0 + (uint32_t)__ffs(rest) - 1u, token = row / a.group;
        const E* out = static_cast<const E*>(a.out) + (uint64_t)(it.first + token) * a.out_stride + (uint64_t)(kv_head * a.group + row - token * a.group) * D + column + lane;
#pragma unroll
        for (int i = 0; i < kCols; ++i) open[i] = open[i] || not_finite(number(out[i * 64]));
    }
    const E* v = static_cast<const E*>(a.v) + (uint64_t)it.first * a.v_stride + (uint64_t)kv_head * D + column + lane;
    auto some_open = [&] {
        bool some = false;
#pragma unroll
        for (int i = 0; i < kCols; ++i) some = some || open[i];
        return __any(some);
    };
    bool some = some_open();
#pragma nounroll
    for (uint32_t base = from; some && base <= to; base += kAtOnce) {
        E x[kAtOnce][kCols];
#pragma unroll
        for (uint32_t j = 0; j < kAtOnce; ++j)
#pragma unroll
            for (int i = 0; i < kCols; ++i) x[j][i] = v[(uint64_t)min(base + j, to) * a.v_stride + i * 64];
#pragma unroll
        for (uint32_t j = 0; j < kAtOnce; ++j)
#pragma unroll
            for (int i = 0; i < kCols; ++i) open[i] = open[i] && !not_finite(number(x[j][i]));
        some = some_open();
    }
    return !some;
}

// DW columns of up to kRedo rows again (bits of `rows`, from row0 on), by one wave: number by number, from what a row sees alone;
// infinite and NaN values are added as they are. A lane takes a key for the scores and a column of 64 for the values. The rows go
// over the keys together, one after the other NaN amid 6,000 tokens of FP32 takes 20 ms in place of 7. A score of NaN or +infinity decides a row at once.
constexpr uint32_t kRedo = 4;
template <int D, int DW, class E>
__device__ inline void redo_rows(const PromptArgs& a, const Item& it, uint32_t kv_head, uint32_t row0, uint32_t rows, uint32_t column) {
    constexpr int kPiece = 16 / sizeof(E);  // numbers of 16 bytes
    constexpr uint32_t kAtOnce = 8u;
    constexpr int kCols = DW > 64 ? DW / 64 : 1;  // of a lane
    const uint32_t lane = threadIdx.x & 63u, n = (uint32_t)__popc(rows);
    uint32_t token[kRedo], head[kRedo], lo[kRedo];  // of the rows, the last one again where there are fewer
    float m[kRedo], l[kRedo], sum[kRedo][kCols];
#pragma unroll
    for (uint32_t r = 0; r < kRedo; ++r) {
        const uint32_t row = row0 + (uint32_t)__ffs(rows) - 1u;
        if (r + 1u < n) rows &= rows - 1u;
        token[r] = row / a.group, head[r] = kv_head * a.group + row - token[r] * a.group;
        lo[r] = Rows::from(a, token[r]);
        m[r] = kNegInf, l[r] = 0.0f;
#pragma unroll
        for (int i = 0; i < kCols; ++i) sum[r][i] = 0.0f;
    }
    const E* k = static_cast<const E*>(a.k) + (uint64_t)it.first * a.k_stride + (uint64_t)kv_head * D;
    const E* v = static_cast<const E*>(a.v) + (uint64_t)it.first * a.v_stride + (uint64_t)kv_head * D + column + min(lane, DW - 1u);
    auto query = [&](uint32_t r) { return static_cast<const E*>(a.q) + (uint64_t)(it.first + token[r]) * a.q_stride + (uint64_t)head[r] * D; };
    union Piece {
        uint4 u;
        E e[kPiece];
    };
    const uint32_t last = token[kRedo - 1u];
#pragma nounroll
    for (uint32_t base = lo[0]; base <= last; base += 64u) {
        const E* key = k + (uint64_t)min(base + lane, last) * a.k_stride;
        float s[kRedo];
#pragma unroll
        for (uint32_t r = 0; r < kRedo; ++r) s[r] = 0.0f;
#pragma nounroll
        for (int i0 = 0; i0 < D; i0 += 4 * kPiece) {
            Piece y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) y[i].u = *reinterpret_cast<const uint4*>(key + i0 + i * kPiece);
#pragma unroll
            for (uint32_t r = 0; r < kRedo; ++r)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    Piece x;
                    x.u = *reinterpret_cast<const uint4*>(query(r) + i0 + i * kPiece);
#pragma unroll
                    for (int j = 0; j < kPiece; ++j) s[r] = fmaf(number(x.e[j]), number(y[i].e[j]), s[r]);
                }
        }
        bool some = false;  // of the rows goes on
#pragma unroll
        for (uint32_t r = 0; r < kRedo; ++r) {
            const bool sees = base + lane >= lo[r] && base + lane <= token[r];
            const float t = sees ? (a.flip ? -s[r] : s[r]) * a.scale_log2e : kNegInf;
            if (__any(!(t < __builtin_inff()))) l[r] = __builtin_nanf("");
            some = some || l[r] == l[r];
            const float now = fmaxf(m[r], wave_max(t)), zero = now == kNegInf ? 0.0f : now;
            const float alpha = __builtin_amdgcn_exp2f(m[r] - zero);
            s[r] = __builtin_amdgcn_exp2f(t - zero);
            m[r] = now;
            l[r] = l[r] * alpha + wave_sum(s[r]);
#pragma unroll
            for (int i = 0; i < kCols; ++i) sum[r][i] *= alpha;
        }
        if (!some) break;
        const uint32_t keys = min(64u, last + 1u - base);
#pragma nounroll
        for (uint32_t j0 = 0; j0 < keys; j0 += kAtOnce) {
            E x[kAtOnce][kCols];
#pragma unroll
            for (uint32_t j = 0; j < kAtOnce; ++j)
#pragma unroll
                for (int i = 0; i < kCols; ++i) x[j][i] = v[(uint64_t)min(base + j0 + j, last) * a.v_stride + i * 64];
#pragma unroll
            for (uint32_t j = 0; j < kAtOnce; ++j)
#pragma unroll
                for (uint32_t r = 0; r < kRedo; ++r) {
                    const uint32_t at = base + j0 + j;
                    if (at < lo[r] || at > token[r]) continue;
                    const float w = lane_read(s[r], (int)(j0 + j));
#pragma unroll
                    for (int i = 0; i < kCols; ++i) {
                        const float y = number(x[j][i]);
                        sum[r][i] = not_finite(y) ? sum[r][i] + y : fmaf(w, y, sum[r][i]);
                    }
                }
        }
    }
#pragma unroll
    for (uint32_t r = 0; r < kRedo; ++r) {
        if (r >= n || lane >= (uint32_t)DW) break;
        E* to = static_cast<E*>(a.out) + (uint64_t)(it.first + token[r]) * a.out_stride + (uint64_t)head[r] * D + column + lane;
        if (l[r] == 0.0f) l[r] = __builtin_nanf("");  // no weight is left, for an infinite value either
#pragma unroll
        for (int i = 0; i < kCols; ++i) {
            if constexpr (sizeof(E) == 4) to[i * 64] = sum[r][i] / l[r];
            else to[i * 64] = (uint16_t)pack_bf16(sum[r][i] / l[r], 0.0f);
        }
    }
}
// All the rows of `left`, or the shares of `sharers` waves that have the same rows.
template <int D, int DW, class E>
__device__ inline void redo(const PromptArgs& a, const Item& it, uint32_t kv_head, uint32_t row0, uint32_t left, uint32_t column, uint32_t sharers = 1u,
                            uint32_t share = 0u) {
#pragma nounroll
    for (uint32_t n = 0; left; ++n) {
        uint32_t rows = 0u;
        for (uint32_t r = 0; r < kRedo && left; ++r) rows |= left & -left, left &= left - 1u;
        if (n % sharers == share) redo_rows<D, DW, E>(a, it, kv_head, row0, rows, column);
    }
}

// Few rows of FP32: a workgroup takes 32 of them. Its four waves take the blocks of 32 keys in turn, each with its own
// maximum and sums, and join at the end. The matrix unit takes FP32 numbers as they are, at a sixteenth of its rate of
// 16-bit ones.
template <int D>
struct Few {
    union {
        float4 q[D / 8][64];  // the queries as second operands
        float sums[kWaves][kRows][68];
    };
    float m[kWaves][kRows], l[kWaves][kRows];
    uint32_t odd;  // rows whose result is not finite
};

template <int D>
__global__ __launch_bounds__(kThreads, 2) void k_few32(const PromptArgs a) {
    __shared__ Few<D> sh;
    const uint32_t lane = threadIdx.x & 63u, col = lane & 31u, half = lane >> 5;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t kv_head = blockIdx.x % a.kv_heads;
    const Item it = locate(a, blockIdx.x / a.kv_heads, kRows);
    if (!it.exists) return;
    const uint32_t last = it.len - 1u;
    const Rows rows(a, it, kv_head, it.tile * kRows);
    const uint32_t begin = Rows::from(a, rows.first), end = rows.last + 1u;
    const float* q = static_cast<const float*>(a.q) + (uint64_t)(it.first + rows.pos) * a.q_stride + (uint64_t)rows.head * D;
    const float* k = static_cast<const float*>(a.k) + (uint64_t)it.first * a.k_stride + (uint64_t)kv_head * D;
    const float* v = static_cast<const float*>(a.v) + (uint64_t)it.first * a.v_stride + (uint64_t)kv_head * D;
    for (int i = wave; i < D / 8; i += kWaves) {
        uint4 x = *reinterpret_cast<const uint4*>(q + i * 8 + half * 4u);
        x.x ^= a.flip, x.y ^= a.flip, x.z ^= a.flip, x.w ^= a.flip;
        sh.q[i][lane] = __builtin_bit_cast(float4, x);
    }
    __syncthreads();
    f32x16 o[D / 32];
    Softmax sm;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) o[i] = zeros();
    for (uint32_t base = begin / kKeys * kKeys + wave * kKeys; base < end; base += kWaves * kKeys) {
        // ---- scores
        const float* krow = k + (uint64_t)min(base + col, last) * a.k_stride;
        f32x16 s[1] = {zeros()};
#pragma unroll 8
        for (int i = 0; i < D / 8; ++i) {
            const float4 x = *reinterpret_cast<const float4*>(krow + i * 8 + half * 4u), y = sh.q[i][lane];
            s[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(x.x, y.x, s[0], 0, 0, 0);
            s[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(x.y, y.y, s[0], 0, 0, 0);
            s[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(x.z, y.z, s[0], 0, 0, 0);
            s[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(x.w, y.w, s[0], 0, 0, 0);
        }
        if (!rows.all(a, base, kKeys)) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const uint32_t key = base + element(r, half);
                if (key < rows.lo || key > rows.pos) s[0][r] = kNegInf;
            }
        }
        // ---- weights
        float alpha;
        if (sm.weights(s, a.scale_log2e, alpha)) {
#pragma unroll
            for (int i = 0; i < D / 32; ++i) o[i] *= alpha;
        }
        // ---- weighted values
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float* vrow = v + (uint64_t)min(base + element(r, half), last) * a.v_stride + col;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) o[i] = __builtin_amdgcn_mfma_f32_32x32x2f32(vrow[i * 32], s[0][r], o[i], 0, 0, 0);
        }
    }

    // ---- the four waves join
    sm.l = halves_sum(sm.l);
    if (half == 0u) sh.m[wave][col] = sm.m, sh.l[wave][col] = sm.l;
    if (threadIdx.x == 0u) sh.odd = 0u;
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
    bool odd = false;
    const uint32_t out_row = it.tile * kRows + row, token = out_row / a.group;
    float* to = static_cast<float*>(a.out) + (uint64_t)(it.first + token) * a.out_stride +
            (uint64_t)(kv_head * a.group + out_row - token * a.group) * D + c8;
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
            odd = odd || not_finite(x[i]);
        }
        if (token < it.len) {
            *reinterpret_cast<float4*>(to + n * 64) = make_float4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<float4*>(to + n * 64 + 4) = make_float4(x[4], x[5], x[6], x[7]);
        }
    }
    if (odd && token < it.len && total > 0.0f) atomicOr(&sh.odd, 1u << row);
    __syncthreads();  // what was written is written over, in order
    uint32_t left = sh.odd;
    if (left == 0u || stays<D, D, float>(a, it, kv_head, it.tile * kRows, left, 0u)) return;
    __syncthreads();  // all have read what is written over
    redo<D, D, float>(a, it, kv_head, it.tile * kRows, left, 0u, kWaves, wave);
}

// Many rows: every wave has 32 rows of its own, and tiles of KT keys and values go from memory to LDS, without passing
// registers, for all of them, one tile ahead. A row of a tile is D values, whose 16-byte chunks are exchanged (chunk c lies
// at c ^ f(row)) so that neither the key reads, 16 bytes of 32 rows, nor the transposing value reads, 64 bytes of 8 rows,
// meet in a bank.
template <int D, int KT, int W, int PARTS, int TEAMS>
struct Many {
    static constexpr int kBuffers = W > 1 ? 2 : 1;
    union {
        struct {
            uint16_t k[kBuffers][KT * D], v[kBuffers][KT * D];
        } tile[TEAMS];
        // the sums that a team makes for another one, which joins and writes those columns
        float4 sums[TEAMS > 1 ? W : 1][TEAMS > 1 ? TEAMS * (TEAMS - 1) : 1][TEAMS > 1 ? D / 8 / TEAMS : 1][64];
    };
    union {
        float2 stats[TEAMS][TEAMS > 1 ? W : 1][64];  // (m, l) of every row
        float4 scores[PARTS > 1 ? W : 1][PARTS > 1 ? 4 : 1][64];
    };
};
template <int D>
__device__ inline uint32_t key_turn(uint32_t row) { return D >= 128 ? row & 15u : (row >> 1) & 7u; }
template <int D>
__device__ inline uint32_t value_turn(uint32_t row) {
    const uint32_t r = row & 3u;
    return (D >= 128 ? r | (r & 1u) << 2 : r) << 1;
}
template <class T>
__device__ inline uint32_t lds_at(T* p) { return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) T*)p; }

// W waves in pairs (PARTS 2) or alone, of which each has DW columns of the queries, keys, values and sums of 32 rows:
// the registers of two waves per SIMD hold 256. WAVES waves per SIMD; C operands are read from LDS while the C products
// before them run. TEAMS of W waves take a workgroup's tiles of keys in turn for the same rows, with maxima and sums of
// their own, and join at the end. A team of one wave has one tile's place and waits for no other until then.
template <int D, int W, int KT, int PARTS, int C, int WAVES, int TEAMS>
__global__ __launch_bounds__(64 * W * TEAMS, WAVES) void k_many(const PromptArgs a) {
    constexpr int DW = D / PARTS, kBlocks = KT / 32, kLoads = KT * D / 512 / W;  // kLoads: a wave's loads of 1 KB
    constexpr uint32_t kChunks = D / 8, kLoadRows = 64 / kChunks, kStep = W * kLoadRows, R = 32 * W / PARTS;
    __shared__ __attribute__((aligned(1024))) Many<D, KT, W, PARTS, TEAMS> sh;
    const uint32_t lane = threadIdx.x & 63u, col = lane & 31u, half = lane >> 5;
    const uint32_t team = TEAMS > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / (64u * W)) : 0u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) - team * W;
    auto& mem = sh.tile[team];
    const uint32_t kv_head = blockIdx.x % a.kv_heads;
    const Item it = locate(a, blockIdx.x / a.kv_heads, R);
    if (!it.exists) return;
    const uint32_t all = it.len * a.group, row0 = it.tile * R, mine = row0 + wave / PARTS * 32u, column = wave % PARTS * DW;
    const uint32_t begin = Rows::from(a, row0 / a.group) / KT * KT, end = min(row0 + R - 1u, all - 1u) / a.group + 1u;
    const uint16_t* k = static_cast<const uint16_t*>(a.k) + (uint64_t)it.first * a.k_stride + (uint64_t)kv_head * D;
    const uint16_t* v = static_cast<const uint16_t*>(a.v) + (uint64_t)it.first * a.v_stride + (uint64_t)kv_head * D;

    // Load n of a wave fills rows (wave + W n) kLoadRows .. of a tile, lane l chunk l % kChunks of row l / kChunks of
    // these. Rows past the sequence are its last row again.
    const uint32_t load_row = wave * kLoadRows + lane / kChunks, chunk = lane % kChunks;
    const uint32_t k_bytes = (uint32_t)a.k_stride * 2u, v_bytes = (uint32_t)a.v_stride * 2u;
    auto fetch_keys = [&](uint32_t base, uint16_t* to) {
        const uint32_t there = min((uint32_t)KT, it.len - base);
        const TileSource from(k + (uint64_t)base * a.k_stride, (there - 1u) * k_bytes + D * 2u);
#pragma unroll
        for (int n = 0; n < kLoads; ++n) {
            const uint32_t row = load_row + n * kStep;
            from.load(to + (wave + W * n) * 512u, min(row, there - 1u) * k_bytes + ((chunk ^ key_turn<D>(row)) * 16u));
        }
    };
    auto fetch_values = [&](uint32_t base, uint16_t* to) {
        const uint32_t there = min((uint32_t)KT, it.len - base);
        const TileSource from(v + (uint64_t)base * a.v_stride, (there - 1u) * v_bytes + D * 2u);
#pragma unroll
        for (int n = 0; n < kLoads; ++n) {
            const uint32_t row = load_row + n * kStep;
            from.load(to + (wave + W * n) * 512u, min(row, there - 1u) * v_bytes + ((chunk ^ value_turn<D>(row)) * 16u));
        }
    };
    const uint32_t my_begin = begin + team * KT;  // a team's tiles
    if (my_begin < end) fetch_keys(my_begin, mem.k[0]), fetch_values(my_begin, mem.v[0]);

    const Rows rows(a, it, kv_head, mine);
    Frag qf[DW / 16];
    const uint16_t* q = static_cast<const uint16_t*>(a.q) + (uint64_t)(it.first + rows.pos) * a.q_stride + (uint64_t)rows.head * D + column;
#pragma unroll
    for (int i = 0; i < DW / 16; ++i) {
        qf[i].u = *reinterpret_cast<const uint4*>(q + i * 16 + half * 8u);
#pragma unroll
        for (int j = 0; j < 4; ++j) qf[i].w[j] ^= a.flip;
    }

    // Where a lane's operands lie in buffer 0. A chunk's number is exchanged in its low four bits (three for heads of 64),
    // so the addresses repeat after kKeyTurns key reads and kValueTurns values' blocks of 32.
    constexpr int kKeyTurns = D >= 128 ? 8 : 4, kValueTurns = D >= 128 ? 4 : 2;
    uint32_t key_at[kKeyTurns], value_at[kValueTurns];
#pragma unroll
    for (int i = 0; i < kKeyTurns; ++i) key_at[i] = lds_at(mem.k[0]) + (col * D + column) * 2u + (((2u * i) ^ half ^ key_turn<D>(col)) * 16u);
#pragma unroll
    for (int i = 0; i < kValueTurns; ++i)
        value_at[i] = lds_at(mem.v[0]) + ((4u * half + ((lane >> 2) & 3u)) * D + column + (lane & 1u) * 4u) * 2u +
                      ((4u * i ^ ((lane >> 4) & 1u) * 2u ^ ((lane & 3u) >> 1) ^ value_turn<D>(lane >> 2)) * 16u);
    uint32_t buf_at = 0u;  // of the tile in hand
    auto key_read = [&](int n) {
        const int i = n / kBlocks;
        Frag x;
        x.x = *(const __attribute__((address_space(3))) u32x4*)(key_at[i % kKeyTurns] + buf_at +
                                                                 (uint32_t)(n % kBlocks * 32 * D * 2 + i / kKeyTurns * kKeyTurns * 32));
        return x;
    };
    auto value_read = [&](int n) {
        const int i = n / (2 * kBlocks);
        Frag x;
#pragma unroll
        for (int e = 0; e < 2; ++e)
            x.h[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)(
                value_at[i % kValueTurns] + buf_at + (uint32_t)((16 * (n % (2 * kBlocks)) + 8 * e) * D * 2 + i / kValueTurns * kValueTurns * 64)));
        return x;
    };

    f32x16 o[DW / 32], s[kBlocks];
    Softmax sm;
    Frag x[2][C], p[2 * kBlocks];
    constexpr int kKeyReads = DW / 16 * kBlocks, kValueReads = DW / 32 * 2 * kBlocks;
    static_assert(kKeyReads / C % 2 == 0 && kValueReads % C == 0);
    // The sched_barriers keep the compiler from asking for all operands of a step at once, which spills.
    auto scores = [&] {
#pragma unroll
        for (int n = 0; n < C; ++n) x[0][n] = key_read(n);
#pragma unroll
        for (int b = 0; b < kBlocks; ++b) s[b] = zeros();
#pragma unroll
        for (int c = 0; c < kKeyReads / C; ++c) {
            if (c + 1 < kKeyReads / C) {
#pragma unroll
                for (int n = 0; n < C; ++n) x[(c + 1) & 1][n] = key_read((c + 1) * C + n);
            }
#pragma unroll
            for (int n = 0; n < C; ++n) {
                f32x16& to = s[(c * C + n) % kBlocks];
                to = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[c & 1][n].b, qf[(c * C + n) / kBlocks].b, to, 0, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto weigh = [&](uint32_t base, f32x16 (&t)[kBlocks]) {
        if (!rows.all(a, base, KT)) {
            asm volatile("");  // a branch, not selects: few blocks are not seen whole
            const uint32_t from = rows.lo - base - 4u * half, to = rows.pos - base - 4u * half;  // of the lane's first key
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int key = 32 * b + (int)element(r, 0u);
                    if (key < (int)from || key > (int)to) t[b][r] = kNegInf;
                }
        }
        float alpha;
        if (sm.weights(t, a.scale_log2e, alpha)) {
#pragma unroll
            for (int i = 0; i < DW / 32; ++i) o[i] *= alpha;
        }
#pragma unroll
        for (int b = 0; b < kBlocks; ++b)
#pragma unroll
            for (int j = 0; j < 8; ++j) p[2 * b + (j >> 2)].w[j & 3] = pack_bf16(t[b][2 * j], t[b][2 * j + 1]);
        __builtin_amdgcn_sched_barrier(0);
    };
    auto first_values = [&] {
#pragma unroll
        for (int n = 0; n < C; ++n) x[0][n] = value_read(n);
    };
    auto sums = [&] {
#pragma unroll
        for (int c = 0; c < kValueReads / C; ++c) {
            if (c + 1 < kValueReads / C) {
#pragma unroll
                for (int n = 0; n < C; ++n) x[(c + 1) & 1][n] = value_read((c + 1) * C + n);
            }
#pragma unroll
            for (int n = 0; n < C; ++n) {
                f32x16& to = o[(c * C + n) / (2 * kBlocks)];
                to = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x[c & 1][n].b, p[(c * C + n) % (2 * kBlocks)].b, to, 0, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto landed = [&] {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's part of the tile is there
        if constexpr (W > 1) __syncthreads();             // the others' too, and nobody reads what is fetched next any more
    };
#pragma unroll
    for (int i = 0; i < DW / 32; ++i) o[i] = zeros();

    for (uint32_t at = begin, buf = 0; at < end; at += KT * TEAMS, buf ^= 1u) {
        const uint32_t base = at + team * KT, next = base + KT * TEAMS;
        landed();
        if constexpr (W > 1) {
            if (next < end) fetch_keys(next, mem.k[buf ^ 1u]), fetch_values(next, mem.v[buf ^ 1u]);
            buf_at = buf * (KT * D * 2u);
        }
        if (PARTS == 1 && (mine >= all || (TEAMS > 1 && base >= end) || !rows.some(a, base, KT))) {
            if (W == 1 && next < end) fetch_keys(next, mem.k[0]), fetch_values(next, mem.v[0]);
            continue;
        }
        // The waves of a SIMD are at different places of their steps; the one that multiplies goes first. Pairs keep step by
        // their barrier, and there it costs 3 %.
        if constexpr (PARTS == 1) __builtin_amdgcn_s_setprio(1);
        scores();
        if constexpr (PARTS == 1) __builtin_amdgcn_s_setprio(0);
        if constexpr (PARTS > 1) {  // the pair's products are each over half of the columns and meet in LDS
            static_assert(PARTS == 2 && kBlocks == 1);
#pragma unroll
            for (int e = 0; e < 4; ++e) sh.scores[wave][e][lane] = make_float4(s[0][4 * e], s[0][4 * e + 1], s[0][4 * e + 2], s[0][4 * e + 3]);
            __syncthreads();
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float4 y = sh.scores[wave ^ 1u][e][lane];
                s[0][4 * e] += y.x, s[0][4 * e + 1] += y.y, s[0][4 * e + 2] += y.z, s[0][4 * e + 3] += y.w;
            }
        }
        first_values();
        weigh(base, s);
        if constexpr (PARTS == 1) __builtin_amdgcn_s_setprio(1);
        sums();
        if constexpr (PARTS == 1) __builtin_amdgcn_s_setprio(0);
        if constexpr (W == 1)
            if (next < end) fetch_keys(next, mem.k[0]), fetch_values(next, mem.v[0]);  // the tile has been read
    }

    // Unit n of a lane's sums, o[n / 4][n % 4 * 4 ..], are columns 8 n + 4 half .. of its row.
    constexpr int kUnits = DW / 8 / TEAMS;  // of a team
    float l = halves_sum(sm.l);
    if constexpr (TEAMS > 1) {
        static_assert(PARTS == 1);
        __syncthreads();  // the tiles' places are free
        sh.stats[team][wave][lane] = make_float2(sm.m, l);
        auto place = [](int from, int to) { return from * (TEAMS - 1) + (to < from ? to : to - 1); };
#pragma unroll
        for (int n = 0; n < DW / 8; ++n)
            if (n / kUnits != (int)team)
                sh.sums[wave][place((int)team, n / kUnits)][n % kUnits][lane] =
                    make_float4(o[n / 4][n % 4 * 4], o[n / 4][n % 4 * 4 + 1], o[n / 4][n % 4 * 4 + 2], o[n / 4][n % 4 * 4 + 3]);
        __syncthreads();
        float top = kNegInf, factor[TEAMS];
#pragma unroll
        for (int n = 0; n < TEAMS; ++n) top = fmaxf(top, sh.stats[n][wave][lane].x);
        l = 0.0f;
#pragma unroll
        for (int n = 0; n < TEAMS; ++n) {
            const float2 x = sh.stats[n][wave][lane];
            factor[n] = __builtin_amdgcn_exp2f(x.x - (top == kNegInf ? 0.0f : top));
            l = fmaf(x.y, factor[n], l);
        }
#pragma unroll
        for (int u = 0; u < TEAMS; ++u) {
            if (u != (int)team) continue;
#pragma unroll
            for (int n = u * kUnits; n < (u + 1) * kUnits; ++n) {
                float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int from = 0; from < TEAMS; ++from) {
                    float4 y;
                    if (from == u) y = make_float4(o[n / 4][n % 4 * 4], o[n / 4][n % 4 * 4 + 1], o[n / 4][n % 4 * 4 + 2], o[n / 4][n % 4 * 4 + 3]);
                    else y = sh.sums[wave][place(from, u)][n % kUnits][lane];
                    x.x = fmaf(y.x, factor[from], x.x), x.y = fmaf(y.y, factor[from], x.y);
                    x.z = fmaf(y.z, factor[from], x.z), x.w = fmaf(y.w, factor[from], x.w);
                }
                const int m = n - u * kUnits;  // to the front, where every team's are written from
                o[m / 4][m % 4 * 4] = x.x, o[m / 4][m % 4 * 4 + 1] = x.y, o[m / 4][m % 4 * 4 + 2] = x.z, o[m / 4][m % 4 * 4 + 3] = x.w;
            }
        }
    }
    const float by = 1.0f / l;
    uint16_t* to = static_cast<uint16_t*>(a.out) + (uint64_t)(it.first + rows.pos) * a.out_stride + (uint64_t)rows.head * D + column + team * (kUnits * 8u) + half * 4u;
    bool odd = false;
#pragma unroll
    for (int n = 0; n < kUnits; ++n) {
        const f32x16 y = o[n / 4];
        float z[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) z[e] = y[n % 4 * 4 + e] * by, odd = odd || not_finite(z[e]);
        if (rows.exists) *reinterpret_cast<uint2*>(to + n * 8) = make_uint2(pack_bf16(z[0], z[1]), pack_bf16(z[2], z[3]));
    }
    const unsigned long long both = __ballot(odd && rows.exists && l > 0.0f);
    const uint32_t left = (uint32_t)both | (uint32_t)(both >> 32);
    // a wave has its columns of a row to itself, a team's after the join too
    constexpr int kOwn = DW / TEAMS;
    if (__builtin_expect(left != 0u, 0) && !stays<D, kOwn, uint16_t>(a, it, kv_head, mine, left, column + team * kOwn))
        redo<D, kOwn, uint16_t>(a, it, kv_head, mine, left, column + team * kOwn);
}

// Many rows of FP32. The matrix unit multiplies 16-bit numbers at 16 times its rate of FP32 ones, so every number enters as
// a sum of such: queries and keys as two of fp16 after a power of two of the row or key (22 bits, and 2^-40 of the largest;
// the product of the two small parts, 2^-22, is left out), weights and values, which need no power there, as three of BF16
// (24 bits; of the nine products those of 2^-24 are left out). A tile's numbers are split once, on their way to LDS, by
// the whole workgroup.
// Heads above 128 are divided among PARTS waves, 128 columns each, whose score products meet in LDS; where the tile's keys
// and values do not fit there together (heads of 512), the values take the keys' place.
template <int D, int W, int PARTS>
struct Many32 {
    static constexpr bool kOnePlace = D > 256;
    static constexpr int kKeyWords = 2 * kKeys * D, kValueWords = 3 * kKeys * D;
    // fp16 keys: the number rounded, and what is left of it; BF16 values in three parts
    uint16_t k[kOnePlace ? kValueWords : kKeyWords], v[kOnePlace ? 8 : kValueWords];
    float4 scores[PARTS > 1 ? W : 1][PARTS > 1 ? 4 : 1][64];
    int power[kKeys];  // of the keys
    int infinite;      // some key holds an infinity, of which the parts are not numbers
};

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
// Two numbers rounded to fp16 in the first word, what is left of them in the second.
__device__ inline void split_fp16(float a, float b, uint32_t& high, uint32_t& low) {
    const half2v h = {(_Float16)a, (_Float16)b};
    const half2v l = {(_Float16)(a - (float)h[0]), (_Float16)(b - (float)h[1])};
    high = __builtin_bit_cast(uint32_t, h), low = __builtin_bit_cast(uint32_t, l);
}
__device__ inline void split_bf16(float a, float b, uint32_t (&w)[3]) {
#pragma unroll
    for (int n = 0; n < 3; ++n) {
        w[n] = pack_bf16(a, b);
        a -= __uint_as_float(w[n] << 16), b -= __uint_as_float(w[n] & 0xFFFF0000u);
    }
}
// The power of two that takes a number's largest magnitude to 2^14 .. 2^15
__device__ inline int power_to_fp16(float top) { return top > 0.0f ? 14 - ((int)(__float_as_uint(top) >> 23) - 127) : 0; }

template <int D, int W, int PARTS>
__global__ __launch_bounds__(64 * W, 2) void k_many32(const PromptArgs a) {
    constexpr uint32_t R = 32 * W / PARTS, kPerKey = 64 * W / kKeys;  // rows, threads that share a key
    constexpr int DW = D / PARTS, kPieces = D / 4 / kPerKey;          // columns of a wave, four numbers each of a thread
    typedef Many32<D, W, PARTS> Tile;
    __shared__ __attribute__((aligned(1024))) Tile sh;
    uint16_t* const values = Tile::kOnePlace ? sh.k : sh.v;
    const uint32_t lane = threadIdx.x & 63u, col = lane & 31u, half = lane >> 5;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t kv_head = blockIdx.x % a.kv_heads;
    const Item it = locate(a, blockIdx.x / a.kv_heads, R);
    if (!it.exists) return;
    const uint32_t all = it.len * a.group, row0 = it.tile * R, mine = row0 + wave / PARTS * 32u, column = wave % PARTS * DW, last = it.len - 1u;
    const uint32_t begin = Rows::from(a, row0 / a.group) / kKeys * kKeys, end = min(row0 + R - 1u, all - 1u) / a.group + 1u;
    const uint32_t my_key = threadIdx.x / kPerKey, my_col = threadIdx.x % kPerKey * 4u;
    const float* k = static_cast<const float*>(a.k) + (uint64_t)it.first * a.k_stride + (uint64_t)kv_head * D + my_col;
    const float* v = static_cast<const float*>(a.v) + (uint64_t)it.first * a.v_stride + (uint64_t)kv_head * D + my_col;
    float4 kn[kPieces], vn[kPieces];  // of the next tile
    auto fetch_keys = [&](uint32_t base) {
        const uint64_t row = min(base + my_key, last);
#pragma unroll
        for (int i = 0; i < kPieces; ++i) kn[i] = *reinterpret_cast<const float4*>(k + row * a.k_stride + i * (int)kPerKey * 4);
    };
    auto fetch_values = [&](uint32_t base) {
        const uint64_t row = min(base + my_key, last);
#pragma unroll
        for (int i = 0; i < kPieces; ++i) vn[i] = *reinterpret_cast<const float4*>(v + row * a.v_stride + i * (int)kPerKey * 4);
    };
    fetch_keys(begin);
    if constexpr (!Tile::kOnePlace) fetch_values(begin);

    const Rows rows(a, it, kv_head, mine);
    Frag qh[DW / 16], ql[DW / 16];
    int q_power;
    {
        const float* q = static_cast<const float*>(a.q) + (uint64_t)(it.first + rows.pos) * a.q_stride + (uint64_t)rows.head * D + half * 8u;
        float top = 0.0f;
#pragma unroll 8
        for (int i = 0; i < D / 16; ++i) {
            const float4 x = *reinterpret_cast<const float4*>(q + i * 16), y = *reinterpret_cast<const float4*>(q + i * 16 + 4);
            top = fmaxf(top, fmaxf(fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))),
                                   fmaxf(fmaxf(fabsf(y.x), fabsf(y.y)), fmaxf(fabsf(y.z), fabsf(y.w)))));
        }
        q_power = power_to_fp16(halves_max(top));
        const float sign = a.flip ? -1.0f : 1.0f;
#pragma unroll
        for (int i = 0; i < DW / 16; ++i) {
            const float4 x = *reinterpret_cast<const float4*>(q + column + i * 16), y = *reinterpret_cast<const float4*>(q + column + i * 16 + 4);
            const float z[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) split_fp16(sign * ldexpf(z[2 * j], q_power), sign * ldexpf(z[2 * j + 1], q_power), qh[i].w[j], ql[i].w[j]);
        }
    }

    // places in LDS, as in k_many
    constexpr int kKeyTurns = D >= 128 ? 8 : 4, kValueTurns = D >= 128 ? 4 : 2;
    uint32_t key_at[kKeyTurns], value_at[kValueTurns];
#pragma unroll
    for (int i = 0; i < kKeyTurns; ++i) key_at[i] = lds_at(sh.k) + (col * D + column) * 2u + (((2u * i) ^ half ^ key_turn<D>(col)) * 16u);
#pragma unroll
    for (int i = 0; i < kValueTurns; ++i)
        value_at[i] = lds_at(values) + ((4u * half + ((lane >> 2) & 3u)) * D + column + (lane & 1u) * 4u) * 2u +
                      ((4u * i ^ ((lane >> 4) & 1u) * 2u ^ ((lane & 3u) >> 1) ^ value_turn<D>(lane >> 2)) * 16u);
    auto key_read = [&](int part, int i) {
        Frag x;
        x.x = *(const __attribute__((address_space(3))) u32x4*)(key_at[i % kKeyTurns] + (uint32_t)(part * kKeys * D * 2 + i / kKeyTurns * kKeyTurns * 32));
        return x;
    };
    auto value_read = [&](int part, int i, int j) {
        Frag x;
#pragma unroll
        for (int e = 0; e < 2; ++e)
            x.h[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4v*)(
                value_at[i % kValueTurns] + (uint32_t)((part * kKeys + 16 * j + 8 * e) * D * 2 + i / kValueTurns * kValueTurns * 64)));
        return x;
    };
    // where a thread's pieces go: an eighth or sixteenth of the row apart, so the exchanged chunks repeat after kTurns
    constexpr int kApart = (int)kPerKey / 2, kTurns = (D >= 128 ? 16 : 8) / kApart;
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    typedef __attribute__((address_space(3))) u32x2* Place;
    uint32_t key_to[kTurns], value_to[kTurns];
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
        const uint32_t chunk = i * kApart + (my_col >> 3), in = (my_key * D + (my_col & 4u)) * 2u;
        key_to[i] = lds_at(sh.k) + in + (chunk ^ key_turn<D>(my_key)) * 16u;
        value_to[i] = lds_at(values) + in + (chunk ^ value_turn<D>(my_key)) * 16u;
    }
    auto split_keys = [&] {
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) top = fmaxf(top, fmaxf(fmaxf(fabsf(kn[i].x), fabsf(kn[i].y)), fmaxf(fabsf(kn[i].z), fabsf(kn[i].w))));
#pragma unroll
        for (uint32_t d = 1; d < kPerKey; d *= 2u) top = fmaxf(top, __shfl_xor(top, (int)d));
        const int power = power_to_fp16(top);
        if (my_col == 0u) sh.power[my_key] = -power;
        if (not_finite(top)) sh.infinite = 1;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            uint2 h, l;
            split_fp16(ldexpf(kn[i].x, power), ldexpf(kn[i].y, power), h.x, l.x);
            split_fp16(ldexpf(kn[i].z, power), ldexpf(kn[i].w, power), h.y, l.y);
            const uint32_t to = key_to[i % kTurns] + (uint32_t)(i / kTurns * kTurns * kApart * 16);
            *(Place)(to) = u32x2{h.x, h.y};
            *(Place)(to + (uint32_t)(kKeys * D * 2)) = u32x2{l.x, l.y};
        }
    };
    auto split_values = [&] {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            uint32_t x[3], y[3];
            split_bf16(vn[i].x, vn[i].y, x);
            split_bf16(vn[i].z, vn[i].w, y);
            const uint32_t to = value_to[i % kTurns] + (uint32_t)(i / kTurns * kTurns * kApart * 16);
#pragma unroll
            for (int n = 0; n < 3; ++n) *(Place)(to + (uint32_t)(n * kKeys * D * 2)) = u32x2{x[n], y[n]};
        }
    };

    f32x16 o[DW / 32];
    Softmax sm;
#pragma unroll
    for (int i = 0; i < DW / 32; ++i) o[i] = zeros();
    if (threadIdx.x == 0u) sh.infinite = 0;
    for (uint32_t base = begin; base < end; base += kKeys) {
        if constexpr (D == 512) {
            // from one place each, made anew here: kept over the loop they spill
            asm volatile("" : "+v"(key_at[0]), "+v"(value_at[0]));
#pragma unroll
            for (int i = 1; i < kKeyTurns; ++i) key_at[i] = key_at[0] ^ (i * 32u);
#pragma unroll
            for (int i = 1; i < kValueTurns; ++i) value_at[i] = value_at[0] ^ (i * 64u);
        }
        __syncthreads();  // nobody reads the tile before any more
        split_keys();
        if constexpr (!Tile::kOnePlace) split_values();
        __syncthreads();
        if (!Tile::kOnePlace && base + kKeys < end) {
            fetch_keys(base + kKeys);
            fetch_values(base + kKeys);
        }
        if (PARTS == 1 && (mine >= all || !rows.some(a, base, kKeys))) continue;
        f32x16 s[1] = {zeros()};
#pragma unroll
        for (int i = 0; i < DW / 16; ++i) {
            const Frag h = key_read(0, i), l = key_read(1, i);
            const half8v kh = __builtin_bit_cast(half8v, h.x), kl = __builtin_bit_cast(half8v, l.x);
            const half8v xh = __builtin_bit_cast(half8v, qh[i].x), xl = __builtin_bit_cast(half8v, ql[i].x);
            s[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kl, xh, s[0], 0, 0, 0);
            s[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, xl, s[0], 0, 0, 0);
            s[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, xh, s[0], 0, 0, 0);
            if (i % 2) __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (PARTS > 1) {
            // in one place the values follow the keys, asked for here: the registers hold no more beside the queries
            if constexpr (Tile::kOnePlace) fetch_values(base);
#pragma unroll
            for (int e = 0; e < 4; ++e) sh.scores[wave][e][lane] = make_float4(s[0][4 * e], s[0][4 * e + 1], s[0][4 * e + 2], s[0][4 * e + 3]);
            __syncthreads();
            s[0] = zeros();
#pragma unroll
            for (uint32_t n = 0; n < PARTS; ++n) {  // in the same order for every wave of the row: so are their weights
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float4 y = sh.scores[wave / PARTS * PARTS + n][e][lane];
                    s[0][4 * e] += y.x, s[0][4 * e + 1] += y.y, s[0][4 * e + 2] += y.z, s[0][4 * e + 3] += y.w;
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if constexpr (Tile::kOnePlace) {
                split_values();
                __syncthreads();
                if (base + kKeys < end) fetch_keys(base + kKeys);
            }
        }
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int4 e = *reinterpret_cast<const int4*>(&sh.power[element(r, half)]);
            s[0][r] = ldexpf(s[0][r], e.x - q_power), s[0][r + 1] = ldexpf(s[0][r + 1], e.y - q_power);
            s[0][r + 2] = ldexpf(s[0][r + 2], e.z - q_power), s[0][r + 3] = ldexpf(s[0][r + 3], e.w - q_power);
        }
        if (!rows.all(a, base, kKeys)) {
            asm volatile("");
            const int from = (int)(rows.lo - base - 4u * half), to = (int)(rows.pos - base - 4u * half);
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if ((int)element(r, 0u) < from || (int)element(r, 0u) > to) s[0][r] = kNegInf;
        }
        float alpha;
        if (sm.weights(s, a.scale_log2e, alpha)) {
#pragma unroll
            for (int i = 0; i < DW / 32; ++i) o[i] *= alpha;
        }
        Frag p[3][2];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            uint32_t w[3];
            split_bf16(s[0][2 * j], s[0][2 * j + 1], w);
#pragma unroll
            for (int n = 0; n < 3; ++n) p[n][j >> 2].w[j & 3] = w[n];
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < DW / 32; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const Frag h = value_read(0, i, j), m = value_read(1, i, j), l = value_read(2, i, j);
                f32x16& to = o[i];
                to = __builtin_amdgcn_mfma_f32_32x32x16_bf16(l.b, p[0][j].b, to, 0, 0, 0);
                to = __builtin_amdgcn_mfma_f32_32x32x16_bf16(h.b, p[2][j].b, to, 0, 0, 0);
                to = __builtin_amdgcn_mfma_f32_32x32x16_bf16(m.b, p[1][j].b, to, 0, 0, 0);
                to = __builtin_amdgcn_mfma_f32_32x32x16_bf16(m.b, p[0][j].b, to, 0, 0, 0);
                to = __builtin_amdgcn_mfma_f32_32x32x16_bf16(h.b, p[1][j].b, to, 0, 0, 0);
                to = __builtin_amdgcn_mfma_f32_32x32x16_bf16(h.b, p[0][j].b, to, 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
    }

    const float l = halves_sum(sm.l), by = 1.0f / l;
    float* to = static_cast<float*>(a.out) + (uint64_t)(it.first + rows.pos) * a.out_stride + (uint64_t)rows.head * D + column + half * 4u;
    bool odd = false;
#pragma unroll
    for (int i = 0; i < DW / 32; ++i)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const f32x16 y = o[i];
            float z[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) z[e] = y[r + e] * by, odd = odd || not_finite(z[e]);
            if (rows.exists) *reinterpret_cast<float4*>(to + i * 32 + 2 * r) = make_float4(z[0], z[1], z[2], z[3]);
        }
    const unsigned long long both = __ballot(odd && rows.exists && (l > 0.0f || sh.infinite));
    uint32_t left = (uint32_t)both | (uint32_t)(both >> 32);
    if (left && !sh.infinite && stays<D, DW, float>(a, it, kv_head, mine, left, column)) return;
    redo<D, DW, float>(a, it, kv_head, mine, left, column);
}

// As many workgroups of up to 512 threads as locate() may give numbers to, over all key/value heads.
uint32_t items_of(const PromptArgs& a, uint32_t rows) {
    const uint64_t all = (uint64_t)a.tokens * a.group;
    const uint64_t tiles = a.batch <= 64u ? (all + (uint64_t)a.batch * (rows - 1u)) / rows : all / rows + a.batch;
    return grid_blocks(tiles * a.kv_heads * 2u) / 2u;  // its limit is that of 256 threads
}

template <int D>
void launch_few(const PromptArgs& a, hipStream_t st) {
    hipLaunchKernelGGL((k_few32<D>), dim3(items_of(a, kRows)), dim3(kThreads), 0, st, a);
}

template <int D, int W, int PARTS>
void launch_many32(const PromptArgs& a, hipStream_t st) {
    hipLaunchKernelGGL((k_many32<D, W, PARTS>), dim3(items_of(a, 32u * W / PARTS)), dim3(64 * W), 0, st, a);
}

template <int D, int W, int KT, int PARTS, int C, int WAVES, int TEAMS>
void launch_many(const PromptArgs& a, hipStream_t st) {
    hipLaunchKernelGGL((k_many<D, W, KT, PARTS, C, WAVES, TEAMS>), dim3(items_of(a, 32u * W / PARTS)), dim3(64 * W * TEAMS), 0, st, a);
}

// Which form, by the tiles of 128 rows that the sequences may have (measured in us, heads of 256 unless said):
// - Few tiles leave compute units without work: 32 rows to a workgroup while those fit the card at once (one of them to a
//   compute unit with heads of 256, two with 128, four with 64): 1 x 512 tokens 27.7 -> 17.7, 1 x 256 with heads of 128
//   11.5 -> 7.8; past that 4 x 256 would take 22.6 in place of 19.0.
// - At most two tiles to a compute unit whose sequences are long: two teams, 1 x 2,048 88 -> 67, 1 x 2,048 with heads of 64
//   39.5 -> 36; 4 x 512 with heads of 64 would take 18.4 in place of 14.0, more tiles more (4 x 1,000: 58 in place of 54).
// - Heads of 512 take pairs at every size.
// - FP32: 32 rows to a workgroup and FP32 products below a tile to each compute unit, 1 x 500 84 -> 45, 4 x 256 53 -> 42;
//   from there on 16-bit parts, 4 x 512 119 -> 88. Heads of 512 take the parts at every size (1 x 64: 57 -> 42), four waves
//   of 32 rows below a tile to each compute unit, 1 x 512 137 -> 107, and eight of 64 from there on (1 x 1,024: the same).
template <int D>
void launch_dim(const PromptArgs& a, int dtype, uint32_t cus, hipStream_t st) {
    if (dtype == TURBO_HIDDEN_F32) {
        constexpr int kParts = D <= 128 ? 1 : D / 128, kManyWaves = kParts == 1 ? 4 : 8;
        const uint32_t items = items_of(a, 32u * kManyWaves / kParts);
        if (items < cus) {
            if constexpr (D <= 256) launch_few<D>(a, st);
            else launch_many32<D, 4, kParts>(a, st);
            return;
        }
        return launch_many32<D, kManyWaves, kParts>(a, st);
    }
    if constexpr (D == 512) {
        launch_many<D, 8, 32, 2, 2, 2, 1>(a, st);
    } else {
        const uint32_t tiles = items_of(a, 128u);
        if ((uint64_t)tiles * D <= cus * 64u) return launch_many<D, 1, 32, 1, 2, (D <= 128 ? 2 : 1), 4>(a, st);
        constexpr int kTile = D <= 128 ? 64 : 32, kAhead = D <= 128 ? 4 : 2;
        if (tiles <= 2u * cus && (uint64_t)a.tokens >= 1000ull * a.batch) return launch_many<D, 4, kTile, 1, kAhead, 2, 2>(a, st);
        launch_many<D, 4, kTile, 1, kAhead, (D == 64 ? 3 : 2), 1>(a, st);
    }
}

}  // namespace

void launch_prompt(const PromptArgs& a, uint32_t head_dim, int dtype, uint32_t cus, hipStream_t st) {
    switch (head_dim) {
        case 64u: launch_dim<64>(a, dtype, cus, st); break;
        case 128u: launch_dim<128>(a, dtype, cus, st); break;
        case 256u: launch_dim<256>(a, dtype, cus, st); break;
        default: launch_dim<512>(a, dtype, cus, st); break;
    }
    check_hip(hipGetLastError(), "prompt attention");
}

}  // namespace tdt

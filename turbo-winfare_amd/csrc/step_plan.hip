// What a serving step needs before and after its layers: page tables, slots and positions from the lengths of
// the sequences, the masks of drafted trees, the pages' way back, and the path of a tree that the model confirms.
//
// All of it is integer work on a few bytes per token, so a call costs its launch and a chain of dependent
// loads. Every workgroup of a plan adds up the whole batch's lengths for itself (two words per sequence in
// LDS), which takes less time than a launch in front that would do it once.
#include "dt_internal.h"
#include "dt_step.h"

namespace tdt {
namespace {

constexpr uint32_t kThreads = 256, kWaves = kThreads / 64u;
constexpr uint32_t kPerThread = 4u, kTokensPerBlock = kPerThread * kThreads;
constexpr uint32_t kNone = 0xFFFFFFFFu;
constexpr uint32_t kCopied = 2048u;

__device__ inline uint32_t saturate(uint64_t v) { return v < kNone ? (uint32_t)v : kNone; }

// Pages of a sequence's own tokens when it holds `len` tokens.
__device__ inline uint64_t pages_for(uint64_t len, uint32_t prefix, uint32_t shift) {
    return len > prefix ? (len - prefix + (1u << shift) - 1u) >> shift : 0u;
}

// Exclusive sums of v over the workgroup's threads, in v's place, and the sums of all.
template <int N>
__device__ inline void block_scan(uint64_t (&v)[N], uint64_t (&total)[N], uint64_t (&sums)[N][kWaves]) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    uint64_t upto[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        upto[n] = wave_incl_scan((unsigned long long)v[n], lane);
        if (lane == 63u) sums[n][wave] = upto[n];
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) {
        uint64_t before = 0;
        total[n] = 0;
#pragma unroll
        for (uint32_t w = 0; w < kWaves; ++w) {
            if (w < wave) before += sums[n][w];
            total[n] += sums[n][w];
        }
        v[n] = before + upto[n] - v[n];
    }
}

// The last i with at[i] <= x (at[0] is 0; among equal ones the last, so empty sequences are passed over).
__device__ inline uint32_t find(const uint32_t* at, uint32_t n, uint32_t x) {
    uint32_t lo = 0, hi = n;
    while (hi - lo > 1u) {
        const uint32_t mid = (lo + hi) / 2u;
        if (at[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

struct Need {
    uint32_t past, add, held, take;  // tokens added, pages held, pages taken (a table's end limits both)
    uint64_t wanted;           // pages that it lacks
};
__device__ inline Need need_of(const PlanArgs& a, uint32_t b) {
    Need n;
    const uint32_t add = a.add[b];
    n.past = a.past[b];
    n.add = a.row_tokens ? min(add, a.row_tokens) : add;
    n.held = min(a.held[b], a.page_stride);
    const uint64_t all = pages_for((uint64_t)n.past + n.add, a.prefix_len, a.page_shift);
    n.wanted = all > n.held ? all - n.held : 0u;
    const uint32_t room = (uint32_t)(all < a.page_stride ? all : a.page_stride);
    n.take = room > n.held ? room - n.held : 0u;
    return n;
}

// kPerThread tokens of a thread go through every load together: one by one they would wait for three loads in turn
// each (24 prompts, 32,762 tokens: 11 us, and 3.3 for the launch behind it).
__global__ __launch_bounds__(kThreads) void k_plan(const PlanArgs a) {
    extern __shared__ uint32_t lds[];
    __shared__ uint64_t sums[4][kWaves];
    uint32_t *first = lds, *taken = lds + a.batch + 1u;  // tokens and taken pages before each sequence
    // the tokens that it holds and its pages, for batches of a usual size
    const bool copies = a.batch <= kCopied;
    uint32_t *past_of = taken + a.batch + 1u, *held_of = past_of + a.batch;
    const uint32_t block = blockIdx.x;
    const uint32_t per = (a.batch + kThreads - 1u) / kThreads, b0 = threadIdx.x * per, b1 = min(a.batch, b0 + per);
    const uint32_t there = min(*a.free_count, a.free_capacity);
    uint64_t v[4] = {0, 0, 0, 0}, total[4];  // tokens, pages taken, pages lacking, tokens left out
    Need own{};
    for (uint32_t b = b0; b < b1; ++b) {
        own = need_of(a, b);
        v[0] += own.add, v[1] += own.take, v[2] += own.wanted, v[3] += a.add[b] - own.add;
    }
    block_scan(v, total, sums);
    for (uint32_t b = b0; b < b1; ++b) {
        if (per > 1u) own = need_of(a, b);
        first[b] = saturate(v[0]), taken[b] = saturate(v[1]);
        if (copies) past_of[b] = own.past, held_of[b] = own.held;
        v[0] += own.add, v[1] += own.take;
    }
    if (threadIdx.x == 0u) first[a.batch] = saturate(total[0]), taken[a.batch] = saturate(total[1]);
    __syncthreads();

    auto past_at = [&](uint32_t b) { return copies ? past_of[b] : a.past[b]; };
    auto held_at = [&](uint32_t b) { return copies ? held_of[b] : min(a.held[b], a.page_stride); };
    if (block < a.tokens) {
        // where the page of an own token is found, once the takes are done: in the table or in the pool's list
        auto page_at = [&](uint32_t b, uint32_t held, uint32_t index) -> const uint32_t* {
            const uint32_t j = index >> a.page_shift;
            if (j >= a.page_stride) return nullptr;
            if (j < held) return a.pages + (uint64_t)b * a.page_stride + j;
            const uint64_t k = (uint64_t)taken[b] + (j - held);
            return k < there ? a.free_pages + (there - 1u - (uint32_t)k) : nullptr;
        };
        auto slot_of = [&](uint32_t page, uint32_t index) {
            return page >> (32u - a.page_shift) ? kNone : (page << a.page_shift) + (index & ((1u << a.page_shift) - 1u));
        };
        if (a.parents) {
            // a wave to a tree, a lane to a node: the ancestors' bits and whether all of them are there, over twice as
            // many generations in every round
            const uint32_t lane = threadIdx.x & 63u;
            if (const uint32_t b = block * kWaves + (threadIdx.x >> 6); b < a.batch) {
                const uint32_t n = first[b + 1u] - first[b], past = past_at(b), held = held_at(b);
                const uint64_t at = (uint64_t)b * a.row_tokens + lane, pos = (uint64_t)past + lane;
                const bool is = lane < n && pos >= a.prefix_len && pos - a.prefix_len <= 0xFFFFFFFFull;
                const uint32_t index = is ? (uint32_t)(pos - a.prefix_len) : 0u;
                const uint32_t* from = is ? page_at(b, held, index) : nullptr;
                int above = lane < a.row_tokens ? a.parents[at] : -2;
                const uint32_t page = from ? *from : kNone;
                int there_too = lane < n && above >= -1 && above < (int)lane;
                if (!there_too) above = -1;
                unsigned long long mask = 1ull << lane;
#pragma unroll
                for (uint32_t round = 0; round < 6u; ++round) {
                    const int up = above < 0 ? (int)lane : above;
                    const unsigned long long bits = __shfl(mask, up);
                    const int ok = __shfl(there_too, up), next = __shfl(above, up);
                    if (above >= 0) mask |= bits, there_too &= ok, above = next;
                }
                const uint32_t depth = there_too ? (uint32_t)__popcll(mask) - 1u : 0u;
                if (a.masks && lane < a.row_tokens) a.masks[at] = there_too ? mask : 0u;
                if (a.positions && lane < a.row_tokens) a.positions[at] = lane < n ? saturate((uint64_t)past + depth) : 0u;
                if (a.slots && lane < a.row_tokens) a.slots[at] = slot_of(page, index);
            }
        } else {
            const uint32_t i0 = block * kTokensPerBlock + threadIdx.x;
            uint32_t seq[kPerThread] = {}, t[kPerThread], past[kPerThread], held[kPerThread], page[kPerThread];
            bool is[kPerThread];
            if (!a.row_tokens)  // the last sequence whose first token is not behind this one, as find()
                for (uint32_t step = a.batch > 1u ? 1u << (31u - (uint32_t)__clz((int)(a.batch - 1u))) : 0u; step; step /= 2u)
#pragma unroll
                    for (uint32_t n = 0; n < kPerThread; ++n) {
                        const uint32_t b = seq[n] + step;
                        if (b < a.batch && first[b] <= i0 + n * kThreads) seq[n] = b;
                    }
#pragma unroll
            for (uint32_t n = 0; n < kPerThread; ++n) {
                const uint32_t i = i0 + n * kThreads;
                const uint32_t b = a.row_tokens ? i / a.row_tokens : seq[n];
                is[n] = i < a.max_tokens && b < a.batch;
                seq[n] = is[n] ? b : 0u;
                t[n] = is[n] ? i - (a.row_tokens ? b * a.row_tokens : first[b]) : 0u;
                is[n] = is[n] && t[n] < first[b + 1u] - first[b];
                past[n] = held[n] = 0u;
                if (is[n]) past[n] = past_at(seq[n]), held[n] = held_at(seq[n]);
            }
#pragma unroll
            for (uint32_t n = 0; n < kPerThread; ++n) {
                const uint64_t pos = (uint64_t)past[n] + t[n];
                const bool lies = is[n] && pos >= a.prefix_len && pos - a.prefix_len <= 0xFFFFFFFFull;
                const uint32_t* from = lies ? page_at(seq[n], held[n], (uint32_t)(pos - a.prefix_len)) : nullptr;
                page[n] = from ? *from : kNone;
            }
#pragma unroll
            for (uint32_t n = 0; n < kPerThread; ++n) {
                const uint32_t i = i0 + n * kThreads;
                if (i >= a.max_tokens) continue;
                const uint64_t pos = (uint64_t)past[n] + t[n];
                if (a.positions) a.positions[i] = is[n] ? saturate(pos) : 0u;
                if (a.slots) a.slots[i] = slot_of(page[n], (uint32_t)(pos - a.prefix_len));
            }
        }
    }
    if (block >= a.pages_from) {
        for (uint64_t k = (uint64_t)(block - a.pages_from) * kThreads + threadIdx.x; k < taken[a.batch]; k += (uint64_t)(gridDim.x - a.pages_from) * kThreads) {
            const uint32_t b = find(taken, a.batch, (uint32_t)k), j = held_at(b) + (uint32_t)k - taken[b];
            a.pages[(uint64_t)b * a.page_stride + j] = k < there ? a.free_pages[there - 1u - (uint32_t)k] : kNone;
        }
    }
    if (!a.state || block != gridDim.x - 1u) return;
    __syncthreads();  // what the tokens read of held and free_count may be overwritten here
    for (uint32_t b = b0; b < b1; ++b) {
        const Need n = per > 1u ? need_of(a, b) : own;
        const uint32_t got = there > taken[b] ? min(n.take, there - taken[b]) : 0u, past = n.past;
        if (a.kv_len) a.kv_len[b] = a.row_tokens ? (n.add ? saturate((uint64_t)past + a.row_tokens) : 0u) : saturate((uint64_t)past + n.add);
        if (a.starts) a.starts[b] = a.row_tokens ? b * a.row_tokens : first[b];
        a.held_out[b] = n.held + got;
    }
    if (threadIdx.x == 0u) {
        if (a.starts) a.starts[a.batch] = a.row_tokens ? a.batch * a.row_tokens : first[a.batch];
        const uint32_t got = total[1] < there ? (uint32_t)total[1] : there;
        *a.free_out = there - got;
        if (a.totals) {
            a.totals[0] = saturate(total[0]);
            a.totals[1] = saturate(total[3] + (!a.row_tokens && total[0] > a.max_tokens ? total[0] - a.max_tokens : 0u));
            a.totals[2] = got;
            a.totals[3] = saturate(total[2] - got);
        }
    }
}

__global__ __launch_bounds__(kThreads) void k_release(const ReleaseArgs a) {
    extern __shared__ uint32_t given[];  // pages given back before each sequence
    __shared__ uint64_t sums[1][kWaves];
    const uint32_t per = (a.batch + kThreads - 1u) / kThreads, b0 = threadIdx.x * per, b1 = min(a.batch, b0 + per);
    auto keep_of = [&](uint32_t b) {
        const uint64_t keep = pages_for(a.keep_len[b], a.prefix_len, a.page_shift);
        const uint32_t held = min(a.held[b], a.page_stride);
        return (uint32_t)(keep < held ? keep : held);
    };
    uint64_t gives[1] = {0}, total[1];
    for (uint32_t b = b0; b < b1; ++b) gives[0] += min(a.held[b], a.page_stride) - keep_of(b);
    block_scan(gives, total, sums);
    for (uint32_t b = b0; b < b1; ++b) {
        given[b] = saturate(gives[0]);
        gives[0] += min(a.held[b], a.page_stride) - keep_of(b);
    }
    const uint32_t there = min(*a.free_count, a.free_capacity);
    const uint32_t room = a.free_capacity - there, n = total[0] < room ? (uint32_t)total[0] : room;
    __syncthreads();
    for (uint32_t k = threadIdx.x; k < n; k += kThreads) {
        const uint32_t b = find(given, a.batch, k);
        a.free_pages[there + k] = a.pages[(uint64_t)b * a.page_stride + keep_of(b) + k - given[b]];
    }
    __syncthreads();  // held and free_count have been read
    for (uint32_t b = threadIdx.x; b < a.batch; b += kThreads) a.held[b] = keep_of(b);
    if (threadIdx.x == 0u) *a.free_count = there + n;
}

// A wave to a sequence, a lane to a node. From node 0 on, the first child whose token is the one that the model
// chose after its parent.
__global__ __launch_bounds__(kThreads) void k_accept(const AcceptArgs a) {
    const uint32_t b = blockIdx.x * kWaves + (threadIdx.x >> 6), lane = threadIdx.x & 63u;
    if (b >= a.batch) return;
    const bool in = lane < a.row_tokens;
    const uint64_t at = (uint64_t)b * a.row_tokens + lane;
    const uint32_t n = min(a.add[b], a.row_tokens);
    const bool node = lane < n;
    const int above = node ? a.parents[at] : -2;
    const uint32_t token = node ? a.tokens[at] : 0u, chosen = node ? a.chosen[at] : kNone, slot = in && a.slots ? a.slots[at] : kNone;
    uint32_t kept = 0, next = kNone, mine = kNone;  // mine: the node that is number `lane` of the path
    unsigned long long found = __ballot(lane == 0u && above == -1);
    while (found) {
        const uint32_t at_node = (uint32_t)__ffsll(found) - 1u;
        if (lane == kept) mine = at_node;
        ++kept;
        next = __shfl(chosen, (int)at_node);
        // a child comes after its parent, so the walk ends
        found = __ballot(next != kNone && above == (int)at_node && lane > at_node && token == next);
    }
    const uint32_t from = __shfl(slot, (int)(mine == kNone ? lane : mine));
    if (in) {
        if (a.path) a.path[at] = mine;
        if (a.source) a.source[at] = mine == kNone ? kNone : from;
        if (a.target) a.target[at] = mine == kNone ? kNone : slot;
    }
    if (lane == 0u) {
        a.kept[b] = kept;
        a.next[b] = next;
        if (a.length) a.length[b] = saturate((uint64_t)a.past[b] + kept);
    }
}

}  // namespace

// Few tokens are one workgroup's. More have workgroups of their own, the new pages others, and the last of these the
// lengths and the pool after the step, or, where these are to be updated in place and all the others read them, a
// launch behind. In one row the three chains of loads took 7.1 us for 24 prompts of 32,762 tokens.
void launch_plan(PlanArgs a, hipStream_t st) {
    const uint32_t lds = (2u * (a.batch + 1u) + (a.batch <= kCopied ? 2u * a.batch : 0u)) * 4u;
    const uint32_t tokens = a.parents ? (a.batch + kWaves - 1u) / kWaves : grid_blocks(((uint64_t)a.max_tokens + kTokensPerBlock - 1u) / kTokensPerBlock);
    const bool apart = a.held_out != a.held && a.free_out != a.free_count && a.kv_len != a.past;
    uint32_t blocks = 1u;
    a.tokens = 1u, a.pages_from = 0u, a.state = 1;
    if (tokens > 1u) {
        const uint32_t pages = (uint32_t)((((uint64_t)a.max_tokens >> a.page_shift) + a.batch + kThreads - 1u) / kThreads);
        a.tokens = a.pages_from = tokens, a.state = apart;
        blocks = tokens + (pages ? pages : 1u);
    }
    hipLaunchKernelGGL(k_plan, dim3(blocks), dim3(kThreads), lds, st, a);
    check_hip(hipGetLastError(), "batch plan");
    if (a.state) return;
    a.tokens = 0u, a.pages_from = 1u, a.state = 1;
    hipLaunchKernelGGL(k_plan, dim3(1), dim3(kThreads), lds, st, a);
    check_hip(hipGetLastError(), "batch plan");
}

void launch_release(const ReleaseArgs& a, hipStream_t st) {
    hipLaunchKernelGGL(k_release, dim3(1), dim3(kThreads), a.batch * 4u, st, a);
    check_hip(hipGetLastError(), "pages release");
}

void launch_accept(const AcceptArgs& a, hipStream_t st) {
    hipLaunchKernelGGL(k_accept, dim3((a.batch + kWaves - 1u) / kWaves), dim3(kThreads), 0, st, a);
    check_hip(hipGetLastError(), "tree accept");
}

}  // namespace tdt

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
constexpr uint32_t kTokensPerBlock = 8u * kThreads;
constexpr uint32_t kNone = 0xFFFFFFFFu;

__device__ inline uint32_t saturate(uint64_t v) { return v < kNone ? (uint32_t)v : kNone; }

// Pages of a sequence's own tokens when it holds `len` tokens.
__device__ inline uint64_t pages_for(uint64_t len, uint32_t prefix, uint32_t shift) {
    return len > prefix ? (len - prefix + (1u << shift) - 1u) >> shift : 0u;
}

// Exclusive sum of v over the workgroup's threads, and the sum of all; `sums` holds one word per wave.
__device__ inline uint64_t block_scan(uint64_t v, uint64_t* sums, uint64_t& total) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    uint64_t upto = v;
#pragma unroll
    for (uint32_t d = 1; d < 64u; d *= 2u) {
        const uint64_t before = __shfl_up((unsigned long long)upto, d);
        if (lane >= d) upto += before;
    }
    __syncthreads();  // the last use of sums is over
    if (lane == 63u) sums[wave] = upto;
    __syncthreads();
    uint64_t before = 0;
    total = 0;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) {
        if (w < wave) before += sums[w];
        total += sums[w];
    }
    return before + upto - v;
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
    uint32_t add, held, take;  // tokens added, pages held, pages taken (a table's end limits both)
    uint64_t wanted;           // pages that it lacks
};
__device__ inline Need need_of(const PlanArgs& a, uint32_t b) {
    Need n;
    const uint32_t add = a.add[b];
    n.add = a.row_tokens ? min(add, a.row_tokens) : add;
    n.held = min(a.held[b], a.page_stride);
    const uint64_t all = pages_for((uint64_t)a.past[b] + n.add, a.prefix_len, a.page_shift);
    n.wanted = all > n.held ? all - n.held : 0u;
    const uint32_t room = (uint32_t)(all < a.page_stride ? all : a.page_stride);
    n.take = room > n.held ? room - n.held : 0u;
    return n;
}

__global__ __launch_bounds__(kThreads) void k_plan(const PlanArgs a) {
    extern __shared__ uint32_t lds[];
    __shared__ uint64_t sums[kWaves];
    uint32_t *first = lds, *taken = lds + a.batch + 1u;  // tokens and taken pages before each sequence
    const uint32_t per = (a.batch + kThreads - 1u) / kThreads, b0 = threadIdx.x * per, b1 = min(a.batch, b0 + per);
    uint64_t add = 0, take = 0, wanted = 0, over = 0;
    for (uint32_t b = b0; b < b1; ++b) {
        const Need n = need_of(a, b);
        add += n.add, take += n.take, wanted += n.wanted, over += a.add[b] - n.add;
    }
    uint64_t tokens, takes, wants, overs;
    uint64_t add_at = block_scan(add, sums, tokens), take_at = block_scan(take, sums, takes);
    block_scan(wanted, sums, wants);
    block_scan(over, sums, overs);
    for (uint32_t b = b0; b < b1; ++b) {
        const Need n = need_of(a, b);
        first[b] = saturate(add_at), taken[b] = saturate(take_at);
        add_at += n.add, take_at += n.take;
    }
    if (threadIdx.x == 0u) first[a.batch] = saturate(tokens), taken[a.batch] = saturate(takes);
    const uint32_t there = min(*a.free_count, a.free_capacity);
    __syncthreads();

    if (a.tokens) {
        auto page_of = [&](uint32_t b, uint32_t index) {  // the page of an own token, once the takes are done
            const uint32_t j = index >> a.page_shift, held = min(a.held[b], a.page_stride);
            if (j >= a.page_stride) return kNone;
            if (j < held) return a.pages[(uint64_t)b * a.page_stride + j];
            const uint64_t k = (uint64_t)taken[b] + (j - held);
            return k < there ? a.free_pages[there - 1u - (uint32_t)k] : kNone;
        };
        auto slot_of = [&](uint32_t b, uint64_t pos) {
            if (pos < a.prefix_len || pos - a.prefix_len > 0xFFFFFFFFull) return kNone;
            const uint32_t index = (uint32_t)(pos - a.prefix_len), page = page_of(b, index);
            return page >> (32u - a.page_shift) ? kNone : (page << a.page_shift) + (index & ((1u << a.page_shift) - 1u));
        };
        if (a.parents) {
            // a wave to a tree, a lane to a node: the ancestors' bits and whether all of them are there, over twice as
            // many generations in every round
            const uint32_t lane = threadIdx.x & 63u;
            for (uint32_t b = blockIdx.x * kWaves + (threadIdx.x >> 6); b < a.batch; b += gridDim.x * kWaves) {
                const uint32_t n = min(a.add[b], a.row_tokens), past = a.past[b];
                const uint64_t at = (uint64_t)b * a.row_tokens + lane;
                int above = lane < a.row_tokens ? a.parents[at] : -2;
                int there_too = lane < n && above >= -1 && above < (int)lane;
                if (!there_too) above = -1;
                unsigned long long mask = 1ull << lane;
#pragma unroll
                for (uint32_t round = 0; round < 6u; ++round) {
                    const int from = above < 0 ? (int)lane : above;
                    const unsigned long long bits = __shfl(mask, from);
                    const int ok = __shfl(there_too, from), next = __shfl(above, from);
                    if (above >= 0) mask |= bits, there_too &= ok, above = next;
                }
                if (lane >= a.row_tokens) continue;
                const uint32_t depth = there_too ? (uint32_t)__popcll(mask) - 1u : 0u;
                if (a.masks) a.masks[at] = there_too ? mask : 0u;
                if (a.positions) a.positions[at] = lane < n ? saturate((uint64_t)past + depth) : 0u;
                if (a.slots) a.slots[at] = lane < n ? slot_of(b, (uint64_t)past + lane) : kNone;
            }
        } else {
            for (uint32_t i = blockIdx.x * kTokensPerBlock + threadIdx.x; i < min(a.max_tokens, (blockIdx.x + 1u) * kTokensPerBlock);
                 i += kThreads) {
                const uint32_t b = a.row_tokens ? i / a.row_tokens : find(first, a.batch, i);
                const uint32_t t = i - (a.row_tokens ? b * a.row_tokens : first[min(b, a.batch - 1u)]);
                const bool is = b < a.batch && t < (a.row_tokens ? min(a.add[b], a.row_tokens) : first[b + 1u] - first[b]);
                const uint64_t pos = is ? (uint64_t)a.past[b] + t : 0u;
                if (a.positions) a.positions[i] = saturate(pos);
                if (a.slots) a.slots[i] = is ? slot_of(b, pos) : kNone;
            }
        }
        for (uint64_t k = (uint64_t)blockIdx.x * kThreads + threadIdx.x; k < taken[a.batch]; k += (uint64_t)gridDim.x * kThreads) {
            const uint32_t b = find(taken, a.batch, (uint32_t)k), j = min(a.held[b], a.page_stride) + (uint32_t)k - taken[b];
            a.pages[(uint64_t)b * a.page_stride + j] = k < there ? a.free_pages[there - 1u - (uint32_t)k] : kNone;
        }
    }
    if (a.state) {
        __syncthreads();  // what the tokens read of held and free_count may be overwritten here
        for (uint32_t b = threadIdx.x; b < a.batch; b += kThreads) {
            const Need n = need_of(a, b);
            const uint32_t got = there > taken[b] ? min(n.take, there - taken[b]) : 0u;
            if (a.kv_len) a.kv_len[b] = a.row_tokens ? (n.add ? saturate((uint64_t)a.past[b] + a.row_tokens) : 0u) : saturate((uint64_t)a.past[b] + n.add);
            if (a.starts) a.starts[b] = a.row_tokens ? b * a.row_tokens : first[b];
            a.held_out[b] = n.held + got;
        }
        if (threadIdx.x == 0u) {
            if (a.starts) a.starts[a.batch] = a.row_tokens ? a.batch * a.row_tokens : first[a.batch];
            const uint32_t got = takes < there ? (uint32_t)takes : there;
            *a.free_out = there - got;
            if (a.totals) {
                a.totals[0] = saturate(tokens);
                a.totals[1] = saturate(overs + (!a.row_tokens && tokens > a.max_tokens ? tokens - a.max_tokens : 0u));
                a.totals[2] = got;
                a.totals[3] = saturate(wants - got);
            }
        }
    }
}

__global__ __launch_bounds__(kThreads) void k_release(const ReleaseArgs a) {
    extern __shared__ uint32_t given[];  // pages given back before each sequence
    __shared__ uint64_t sums[kWaves];
    const uint32_t per = (a.batch + kThreads - 1u) / kThreads, b0 = threadIdx.x * per, b1 = min(a.batch, b0 + per);
    auto keep_of = [&](uint32_t b) {
        const uint64_t keep = pages_for(a.keep_len[b], a.prefix_len, a.page_shift);
        const uint32_t held = min(a.held[b], a.page_stride);
        return (uint32_t)(keep < held ? keep : held);
    };
    uint64_t gives = 0, total;
    for (uint32_t b = b0; b < b1; ++b) gives += min(a.held[b], a.page_stride) - keep_of(b);
    uint64_t at = block_scan(gives, sums, total);
    for (uint32_t b = b0; b < b1; ++b) {
        given[b] = saturate(at);
        at += min(a.held[b], a.page_stride) - keep_of(b);
    }
    const uint32_t there = min(*a.free_count, a.free_capacity);
    const uint32_t room = a.free_capacity - there, n = total < room ? (uint32_t)total : room;
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

// One workgroup writes everything, the state after all else; several, up to 2,048 tokens or four trees each, leave
// the lengths and the pool, which they all read and which may be written in place, to a launch of their own.
void launch_plan(PlanArgs a, hipStream_t st) {
    const uint32_t lds = 2u * (a.batch + 1u) * 4u;
    const uint32_t blocks = a.parents ? (a.batch + kWaves - 1u) / kWaves : grid_blocks(((uint64_t)a.max_tokens + kTokensPerBlock - 1u) / kTokensPerBlock);
    a.tokens = 1, a.state = blocks <= 1u;
    hipLaunchKernelGGL(k_plan, dim3(blocks ? blocks : 1u), dim3(kThreads), lds, st, a);
    check_hip(hipGetLastError(), "batch plan");
    if (a.state) return;
    a.tokens = 0, a.state = 1;
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

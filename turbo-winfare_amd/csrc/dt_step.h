// Arguments of the kernels around a serving step (step_plan.hip, kv_move.hip, prompt_attention.hip).
#pragma once

#include "dt_kv.h"

namespace tdt {

constexpr uint32_t kPlanMaxBatch = 8192;  // a workgroup holds two words for each sequence in LDS
constexpr uint32_t kTreeNodes = 64;       // a node's mask is one 64-bit word

// step_plan.hip
struct PlanArgs {
    uint32_t batch, page_shift, prefix_len, row_tokens, max_tokens, page_stride, free_capacity;
    const uint32_t *past, *add, *held, *free_pages, *free_count;
    const int32_t* parents;
    uint32_t* pages;
    uint32_t *held_out, *free_out, *starts, *kv_len, *positions, *slots, *totals;
    uint64_t* masks;
    uint32_t tokens, pages_from;  // workgroups of the tokens' entries, and the first that writes pages
    int state;                    // the last one writes the lengths and the pool after the step
};
void launch_plan(PlanArgs a, hipStream_t st);

struct ReleaseArgs {
    uint32_t batch, page_shift, prefix_len, page_stride, free_capacity;
    const uint32_t *keep_len, *pages;
    uint32_t *held, *free_pages, *free_count;
};
void launch_release(const ReleaseArgs& a, hipStream_t st);

struct AcceptArgs {
    uint32_t batch, row_tokens;
    const int32_t* parents;
    const uint32_t *add, *tokens, *chosen, *past, *slots;
    uint32_t *kept, *next, *length, *path, *source, *target;
};
void launch_accept(const AcceptArgs& a, hipStream_t st);

// kv_move.hip
struct KvMoveArgs {
    KvView kv;
    const uint32_t *source, *target;
    uint32_t rows, width;
};
void launch_kv_move(const KvMoveArgs& a, hipStream_t st);

// prompt_attention.hip
struct PromptArgs {
    const void *q, *k, *v;
    void* out;
    uint64_t q_stride, k_stride, v_stride, out_stride;  // elements from one token to the next
    const uint32_t* starts;
    uint32_t batch, tokens, q_heads, kv_heads, group, window;
    float scale_log2e;  // of the scores' magnitude; not 0
    uint32_t flip;      // sign bits of a negative scale, which are the queries' then
};
void launch_prompt(const PromptArgs& a, uint32_t head_dim, int dtype, uint32_t cus, hipStream_t st);

}  // namespace tdt

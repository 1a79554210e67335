// Entry points around a serving step (include/turbo_decode_tail.h): page tables and slots from lengths, a tree's
// confirmed path, and attention over whole prompts. They have no handle; the work goes to the device that a call names.
#include <hip/hip_runtime.h>

#include <cfloat>
#include <cmath>
#include <cstring>
#include <string>

#include "dt_checks.h"
#include "dt_internal.h"
#include "dt_step.h"

using namespace tdt;

namespace {

uint32_t page_shift(uint32_t page_tokens) {
    for (uint32_t shift = 5u; shift <= 8u; ++shift)
        if (page_tokens == 1u << shift) return shift;
    fail("page_tokens must be 32, 64, 128 or 256");
}

void check_batch(int batch) {
    if (batch < 0 || batch > (int)kPlanMaxBatch) fail("batch must be in 0.." + std::to_string(kPlanMaxBatch));
}

// The page tables and the pool, as the plan and the release take them.
void check_pool(int batch, uint32_t page_stride, const void* pages, const void* held, const void* free_pages, uint32_t free_capacity,
                const void* free_count, uint32_t prefix_len) {
    if (page_stride > 0x7FFFFFFFu) fail("page_stride is above 2^31 - 1");
    if (prefix_len > 0x7FFFFF00u) fail("prefix_len must be at most 2^31 - 256");
    if (batch && page_stride) check_words("pages", pages);
    if (batch) check_words("held", held);
    if (free_capacity) check_words("free_pages", free_pages);
    check_words("free_count", free_count);
}

uint32_t tree_rows(uint32_t row_tokens) {
    if (row_tokens < 1u || row_tokens > kTreeNodes) fail("row_tokens must be in 1..64 for trees");
    return row_tokens;
}

int compute_units(int device) {
    int cus = 0;
    check_hip(hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device), "device attribute");
    return cus > 0 ? cus : 1;
}

}  // namespace

extern "C" {

TURBO_DT_API int turbo_batch_plan(const TurboBatchPlan* in, void* hip_stream) {
    ATT_TRY
    if (!in) fail("in is NULL");
    PlanArgs a{};
    check_batch(in->batch);
    a.page_shift = page_shift(in->page_tokens);
    if (in->max_tokens > (uint32_t)kMaxTokens) fail("max_tokens must be at most " + std::to_string(kMaxTokens));
    if (in->row_tokens && in->max_tokens != (uint64_t)in->batch * in->row_tokens) fail("max_tokens must be batch * row_tokens");
    if (in->parents) tree_rows(in->row_tokens);
    else if (in->masks) fail("masks need parents");
    if (in->batch) {  // otherwise arrays of no sequences
        check_words("past_len", in->past_len);
        check_words("new_len", in->new_len);
        check_words("held_out", in->held_out);
    }
    check_pool(in->batch, in->page_stride, in->pages, in->held, in->free_pages, in->free_capacity, in->free_count, in->prefix_len);
    check_words("free_count_out", in->free_count_out);
    if (in->masks) check_words("masks", in->masks, 8u);
    for (const void* p : {static_cast<const void*>(in->parents), static_cast<const void*>(in->starts), static_cast<const void*>(in->kv_len),
                          static_cast<const void*>(in->positions), static_cast<const void*>(in->slots), static_cast<const void*>(in->totals)})
        if (reinterpret_cast<uintptr_t>(p) % 4u != 0u) fail("an array of the plan is not 4-byte aligned");
    // what some workgroups read while others write results; held, free_count and past_len may be updated in place
    const uint64_t each = 4u * (uint64_t)in->batch, nodes = (uint64_t)in->batch * in->row_tokens, tokens = 4u * (uint64_t)in->max_tokens;
    const Span past{in->past_len, each}, held{in->held, each}, count{in->free_count, 4u}, pages{in->pages, each * in->page_stride};
    const Span held_out{in->held_out, each}, count_out{in->free_count_out, 4u}, kv_len{in->kv_len, each};
    const Span inputs[] = {past, held, count, pages, {in->new_len, each}, {in->free_pages, 4u * (uint64_t)in->free_capacity}, {in->parents, 4u * nodes}};
    const Span results[] = {held_out, count_out, kv_len, {in->starts, each + 4u}, {in->positions, tokens}, {in->slots, tokens}, {in->totals, 16u},
                            {in->masks, 8u * nodes}};
    for (const Span& r : results) {
        for (const Span& i : inputs)
            if (r.meets(i) && !(r.is(i) && ((r.is(held_out) && i.is(held)) || (r.is(count_out) && i.is(count)) || (r.is(kv_len) && i.is(past)))))
                fail("a result of the plan lies on one of its inputs");
        for (const Span& other : results)
            if (&other != &r && other.meets(r)) fail("two results of the plan lie on each other");
    }
    for (const Span& i : inputs)
        if (&i != &inputs[3] && pages.meets(i)) fail("the page tables lie on another input of the plan");
    check_device(in->device);
    a.batch = (uint32_t)in->batch;
    a.prefix_len = in->prefix_len;
    a.row_tokens = in->row_tokens;
    a.max_tokens = in->max_tokens;
    a.page_stride = in->page_stride;
    a.free_capacity = in->free_capacity;
    a.past = in->past_len;
    a.add = in->new_len;
    a.held = in->held;
    a.free_pages = in->free_pages;
    a.free_count = in->free_count;
    a.parents = in->parents;
    a.pages = in->pages;
    a.held_out = in->held_out;
    a.free_out = in->free_count_out;
    a.starts = in->starts;
    a.kv_len = in->kv_len;
    a.positions = in->positions;
    a.slots = in->slots;
    a.totals = in->totals;
    a.masks = in->masks;
    DeviceGuard dg(in->device);
    launch_plan(a, static_cast<hipStream_t>(hip_stream));
    return 1;
    ATT_CATCH(0)
}

TURBO_DT_API int turbo_pages_release(const TurboPagesRelease* in, void* hip_stream) {
    ATT_TRY
    if (!in) fail("in is NULL");
    ReleaseArgs a{};
    check_batch(in->batch);
    a.page_shift = page_shift(in->page_tokens);
    if (in->batch == 0) return 1;
    check_words("keep_len", in->keep_len);
    check_pool(in->batch, in->page_stride, in->pages, in->held, in->free_pages, in->free_capacity, in->free_count, in->prefix_len);
    const uint64_t each = 4u * (uint64_t)in->batch;
    const Span updated[] = {{in->held, each}, {in->free_pages, 4u * (uint64_t)in->free_capacity}, {in->free_count, 4u}};
    const Span inputs[] = {{in->keep_len, each}, {in->pages, each * in->page_stride}};
    for (const Span& u : updated) {
        for (const Span& i : inputs)
            if (u.meets(i)) fail("held or the pool lies on an input of the release");
        for (const Span& other : updated)
            if (&other != &u && other.meets(u)) fail("two updated arrays of the release lie on each other");
    }
    check_device(in->device);
    a.batch = (uint32_t)in->batch;
    a.prefix_len = in->prefix_len;
    a.page_stride = in->page_stride;
    a.free_capacity = in->free_capacity;
    a.keep_len = in->keep_len;
    a.pages = in->pages;
    a.held = in->held;
    a.free_pages = in->free_pages;
    a.free_count = in->free_count;
    DeviceGuard dg(in->device);
    launch_release(a, static_cast<hipStream_t>(hip_stream));
    return 1;
    ATT_CATCH(0)
}

TURBO_DT_API int turbo_tree_accept(const TurboTreeAccept* in, void* hip_stream) {
    ATT_TRY
    if (!in) fail("in is NULL");
    AcceptArgs a{};
    if (in->batch < 0 || in->batch > (1 << 20)) fail("batch must be in 0..1048576");
    a.row_tokens = tree_rows(in->row_tokens);
    if (in->batch == 0) return 1;
    check_words("parents", in->parents);
    check_words("new_len", in->new_len);
    check_words("tokens", in->tokens);
    check_words("chosen", in->chosen);
    check_words("kept", in->kept);
    check_words("next", in->next);
    if (in->length) check_words("past_len", in->past_len);
    if ((in->source == nullptr) != (in->target == nullptr)) fail("source and target belong together");
    if (in->source) check_words("slots", in->slots);
    for (const void* p : {static_cast<const void*>(in->length), static_cast<const void*>(in->path), static_cast<const void*>(in->source),
                          static_cast<const void*>(in->target)})
        if (reinterpret_cast<uintptr_t>(p) % 4u != 0u) fail("an array of the tree is not 4-byte aligned");
    // a sequence's wave has read it before it writes: a result may be updated in an input's place, of the same size
    const uint64_t each = 4u * (uint64_t)in->batch, nodes = each * in->row_tokens;
    const Span inputs[] = {{in->parents, nodes}, {in->new_len, each}, {in->tokens, nodes}, {in->chosen, nodes}, {in->past_len, each}, {in->slots, nodes}};
    const Span results[] = {{in->kept, each}, {in->next, each}, {in->length, each}, {in->path, nodes}, {in->source, nodes}, {in->target, nodes}};
    for (const Span& r : results) {
        for (const Span& i : inputs)
            if (r.meets(i) && !r.is(i)) fail("a result of the tree lies across one of its inputs");
        for (const Span& other : results)
            if (&other != &r && other.meets(r)) fail("two results of the tree lie on each other");
    }
    check_device(in->device);
    a.batch = (uint32_t)in->batch;
    a.parents = in->parents;
    a.add = in->new_len;
    a.tokens = in->tokens;
    a.chosen = in->chosen;
    a.past = in->past_len;
    a.slots = in->slots;
    a.kept = in->kept;
    a.next = in->next;
    a.length = in->length;
    a.path = in->path;
    a.source = in->source;
    a.target = in->target;
    DeviceGuard dg(in->device);
    launch_accept(a, static_cast<hipStream_t>(hip_stream));
    return 1;
    ATT_CATCH(0)
}

TURBO_DT_API int turbo_prompt_attention(const TurboPromptInputs* in, void* hip_stream) {
    ATT_TRY
    if (!in) fail("in is NULL");
    const size_t size = dtype_size(in->dtype);
    check_tokens(in->tokens);
    check_head_dim(in->head_dim);
    if (in->batch < 0 || in->batch > (1 << 20)) fail("batch must be in 0..1048576");
    if (in->kv_heads < 1 || in->kv_heads > (int)kMaxKvHeads) fail("kv_heads must be in 1.." + std::to_string(kMaxKvHeads));
    if (in->q_heads < 1 || in->q_heads > (int)kMaxQueryHeads || in->q_heads % in->kv_heads != 0)
        fail("q_heads must be a multiple of kv_heads, at most " + std::to_string(kMaxQueryHeads));
    const double scale = (double)in->scale * 1.4426950408889634;
    if (!(std::fabs(scale) <= (double)FLT_MAX)) fail("scale must be finite and below 2^127");
    if ((uint64_t)in->tokens * (uint64_t)(in->q_heads / in->kv_heads) > (1ull << 31) - 65536u) fail("tokens * q_heads / kv_heads is too large for one call");
    if (in->batch == 0 || in->tokens == 0) return 1;
    PromptArgs a{};
    const size_t q_packed = (size_t)in->q_heads * in->head_dim, kv_packed = (size_t)in->kv_heads * in->head_dim;
    auto rows = [&](const char* name, const void* p, size_t stride, size_t packed) {
        const size_t s = check_rows(name, p, stride, packed, size);
        if (s > (size_t{1} << 24)) fail(std::string(name) + "_stride is above 2^24 elements");
        return s;
    };
    a.q_stride = rows("q", in->q, in->q_stride, q_packed);
    a.k_stride = rows("k", in->k, in->k_stride, kv_packed);
    a.v_stride = rows("v", in->v, in->v_stride, kv_packed);
    a.out_stride = rows("out", in->out, in->out_stride, q_packed);
    if (in->out == in->q || in->out == in->k || in->out == in->v) fail("out is q, k or v");
    check_words("starts", in->starts);
    check_device(in->device);
    a.q = in->q;
    a.k = in->k;
    a.v = in->v;
    a.out = in->out;
    a.starts = in->starts;
    a.batch = (uint32_t)in->batch;
    a.tokens = (uint32_t)in->tokens;
    a.q_heads = (uint32_t)in->q_heads;
    a.kv_heads = (uint32_t)in->kv_heads;
    a.group = a.q_heads / a.kv_heads;
    a.window = in->window;
    // of 0 the least number there is, 2^-149: every finite score then weighs 1 to 2^-21, and a hidden one's -infinity stays
    a.scale_log2e = std::fmax((float)std::fabs(scale), FLT_TRUE_MIN);
    a.flip = in->scale >= 0.0f ? 0u : in->dtype == TURBO_HIDDEN_BF16 ? 0x80008000u : 0x80000000u;
    DeviceGuard dg(in->device);
    launch_prompt(a, in->head_dim, in->dtype, (uint32_t)compute_units(in->device), static_cast<hipStream_t>(hip_stream));
    return 1;
    ATT_CATCH(0)
}

}  // extern "C"

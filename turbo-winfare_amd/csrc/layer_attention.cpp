// Handles and entry points of the layer loop's attention (include/turbo_decode_tail.h): the quantised
// key/value cache, the heads' norms and rotation, and attention over a shared prefix.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstring>
#include <memory>
#include <stdexcept>
#include <string>
#include <vector>

#include "dt_internal.h"
#include "dt_kv.h"

namespace {

constexpr uint32_t kCacheMagic = 0x564B4454u;   // "TDKV"
constexpr uint32_t kRotaryMagic = 0x4F524454u;  // "TDRO"
constexpr int kMaxTokens = 1 << 28;             // a cache read takes 8 threads of one grid dimension to a token
constexpr uint32_t kMaxKvHeads = 1024, kMaxQueryHeads = 8192;

// The streams a handle's calls were enqueued on, waited for before it is freed.
struct Streams {
    static constexpr int kMany = 4;
    hipStream_t used[kMany] = {};
    int n = 0;
    bool many = false;
    void note(hipStream_t st) {
        for (int i = 0; i < n; ++i)
            if (used[i] == st) return;
        if (n < kMany) used[n++] = st;
        else many = true;
    }
    void wait() {
        if (many) (void)hipDeviceSynchronize();
        else for (int i = 0; i < n; ++i) (void)hipStreamSynchronize(used[i]);
    }
};

struct CacheBox {
    uint32_t magic = kCacheMagic;
    int device = 0;
    uint32_t head_dim = 0, page_tokens = 0;
    uint32_t cus = 0;
    tdt::KvView kv{};
    Streams streams;
};

struct RotaryBox {
    uint32_t magic = kRotaryMagic;
    int device = 0;
    uint32_t head_dim = 0, rotary_dim = 0, norms = 0;
    int layout = 0;
    bool still = false;  // some frequency is 0
    float eps = 0.f;
    uint16_t *q_norm = nullptr, *k_norm = nullptr;
    uint64_t* turns = nullptr;
    Streams streams;
};

[[noreturn]] void fail(const std::string& what) { throw std::runtime_error(what); }

CacheBox* cbox(void* p) {
    if (!p) fail("null cache handle");
    auto* c = static_cast<CacheBox*>(p);
    if (c->magic != kCacheMagic) fail("invalid cache handle");
    return c;
}

RotaryBox* rbox(void* p) {
    if (!p) fail("null rotary handle");
    auto* r = static_cast<RotaryBox*>(p);
    if (r->magic != kRotaryMagic) fail("invalid rotary handle");
    return r;
}

void check_head_dim(uint32_t d) {
    if (d != 64u && d != 128u && d != 256u && d != 512u) fail("head_dim must be 64, 128, 256 or 512");
}

void check_device(int device) {
    int ndev = 0;
    tdt::check_hip(hipGetDeviceCount(&ndev), "hipGetDeviceCount");
    if (device < 0 || device >= ndev) fail("no such HIP device");
}

size_t dtype_size(int dtype) {
    if (dtype != TURBO_HIDDEN_F32 && dtype != TURBO_HIDDEN_BF16) fail("dtype must be TURBO_HIDDEN_F32 or TURBO_HIDDEN_BF16");
    return dtype == TURBO_HIDDEN_BF16 ? 2u : 4u;
}

void check_tokens(int tokens) {
    if (tokens < 0 || tokens > kMaxTokens) fail("tokens must be in 0.." + std::to_string(kMaxTokens));
}

// A buffer of rows and its stride in elements (0: packed); the stride it has.
size_t check_rows(const char* name, const void* p, size_t stride, size_t packed, size_t size) {
    if (!p) fail(std::string(name) + " is NULL");
    if (reinterpret_cast<uintptr_t>(p) % 16u != 0u) fail(std::string(name) + " must be 16-byte aligned");
    if (stride == 0u) return packed;
    if (stride < packed) fail(std::string(name) + "_stride is smaller than a token's heads");
    if (stride > (size_t{1} << 32)) fail(std::string(name) + "_stride is above 2^32 elements");
    if (stride * size % 16u != 0u) fail(std::string(name) + "_stride must be a multiple of 16 bytes");
    return stride;
}

// The sizes of an attention call, checked, and how it is split.
tdt::AttnPlan attention_plan(const CacheBox& c, const TurboAttentionInputs& in) {
    dtype_size(in.dtype);
    if (in.batch < 0 || in.batch > (1 << 20)) fail("batch must be in 0..1048576");
    if (in.q_len < 1 || in.q_len > (1 << 20)) fail("q_len must be in 1..1048576");
    if (in.q_heads < 1 || in.q_heads > (int)kMaxQueryHeads || in.q_heads % (int)c.kv.heads != 0)
        fail("q_heads must be a multiple of the cache's kv_heads, at most " + std::to_string(kMaxQueryHeads));
    const uint64_t room = (uint64_t)in.page_stride * c.page_tokens;
    if (in.prefix_len + room > 0x7FFFFF00u) fail("prefix_len + page_stride * page_tokens must be at most 2^31 - 256");
    const uint64_t beyond = in.max_kv_len > in.prefix_len ? in.max_kv_len - in.prefix_len : 0u;
    const tdt::AttnPlan p =
        tdt::plan_attention((uint32_t)in.batch, (uint32_t)in.q_len, (uint32_t)in.q_heads, c.kv.heads, c.head_dim, in.dtype,
                            in.prefix_len, (uint32_t)(room == 0u ? 0u : beyond == 0u ? 1u : beyond < room ? beyond : room),
                            in.window, c.cus);
    if (p.items > (1u << 24) - 1u || p.rows * (c.head_dim / 4u) > 0xFFFFFF00ull) fail("batch * q_len * q_heads is too large for one call");
    return p;
}

}  // namespace

#define ATT_TRY            \
    tdt::set_last_error(""); \
    try {
#define ATT_CATCH(ret)                        \
    }                                         \
    catch (const std::exception& ex) {        \
        tdt::set_last_error(ex.what());       \
        return ret;                           \
    }                                         \
    catch (...) {                             \
        tdt::set_last_error("unknown error"); \
        return ret;                           \
    }

extern "C" {

// ---- the cache ---------------------------------------------------------------------------------

TURBO_DT_API void turbo_kv_cache_desc_default(TurboKvCacheDesc* out) {
    if (!out) return;
    std::memset(out, 0, sizeof(*out));
    out->page_tokens = 64;
    out->kv_heads = 8;
    out->head_dim = 256;
    out->bits = 8;
}

TURBO_DT_API void* turbo_kv_cache_create(const TurboKvCacheDesc* desc) {
    ATT_TRY
    if (!desc) fail("desc is NULL");
    check_head_dim(desc->head_dim);
    if (desc->bits != 4u && desc->bits != 8u) fail("bits must be 4 or 8");
    const uint32_t pt = desc->page_tokens;
    if (pt != 32u && pt != 64u && pt != 128u && pt != 256u) fail("page_tokens must be 32, 64, 128 or 256");
    if (desc->kv_heads == 0u || desc->kv_heads > kMaxKvHeads) fail("kv_heads must be in 1.." + std::to_string(kMaxKvHeads));
    if (desc->pages == 0u) fail("pages must be at least 1");
    if ((uint64_t)desc->pages * pt > 0xFFFFFFFEull) fail("pages * page_tokens must be at most 2^32 - 2");
    check_device(desc->device);
    tdt::DeviceGuard dg(desc->device);
    auto c = std::make_unique<CacheBox>();
    c->device = desc->device;
    c->head_dim = desc->head_dim;
    c->page_tokens = pt;
    int cus = 0;
    tdt::check_hip(hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, desc->device), "device attribute");
    c->cus = cus > 0 ? (uint32_t)cus : 1u;
    tdt::KvView& kv = c->kv;
    kv.pages = desc->pages;
    kv.slots = (uint64_t)desc->pages * pt;
    while ((1u << kv.page_shift) < pt) ++kv.page_shift;
    kv.heads = desc->kv_heads;
    kv.bits = desc->bits;
    kv.groups = desc->head_dim / 64u;
    kv.record = tdt::kv_record_bytes(kv.groups, kv.bits);
    const uint64_t bytes = tdt::kv_record_at(kv, desc->pages, 0u, 0u);
    tdt::check_hip(hipMalloc(&kv.base, bytes), "alloc cache");
    return c.release();
    ATT_CATCH(nullptr)
}

TURBO_DT_API void turbo_kv_cache_destroy(void* handle) {
    if (!handle) return;
    try {
        CacheBox* c = cbox(handle);
        tdt::DeviceGuard dg(c->device);
        c->streams.wait();
        (void)hipFree(c->kv.base);
        c->magic = 0;
        delete c;
    } catch (...) {
    }
}

TURBO_DT_API int turbo_kv_cache_write(void* handle, const void* k, size_t k_stride, const void* v, size_t v_stride, int dtype,
                                      const uint32_t* slots, int tokens, void* hip_stream) {
    ATT_TRY
    CacheBox* c = cbox(handle);
    const size_t size = dtype_size(dtype);
    check_tokens(tokens);
    if (tokens == 0) return 1;
    const size_t packed = (size_t)c->kv.heads * c->head_dim;
    tdt::QkvArgs a{};
    a.k_stride = check_rows("k", k, k_stride, packed, size);
    a.v_stride = check_rows("v", v, v_stride, packed, size);
    if (!slots) fail("slots is NULL");
    a.k = k;
    a.v = v;
    a.slots = slots;
    a.tokens = (uint32_t)tokens;
    a.kv_heads = c->kv.heads;
    a.kv = c->kv;
    tdt::DeviceGuard dg(c->device);
    c->streams.note(static_cast<hipStream_t>(hip_stream));
    tdt::launch_qkv(a, c->head_dim, dtype, static_cast<hipStream_t>(hip_stream));
    return 1;
    ATT_CATCH(0)
}

TURBO_DT_API int turbo_kv_cache_read(void* handle, const uint32_t* slots, int tokens, int dtype, void* k, size_t k_stride, void* v,
                                     size_t v_stride, void* hip_stream) {
    ATT_TRY
    CacheBox* c = cbox(handle);
    const size_t size = dtype_size(dtype);
    check_tokens(tokens);
    if (tokens == 0) return 1;
    const size_t packed = (size_t)c->kv.heads * c->head_dim;
    if (!k && !v) fail("k and v are both NULL");
    if (k && k == v) fail("k and v are the same buffer");
    tdt::KvReadArgs a{};
    if (k) a.k_stride = check_rows("k", k, k_stride, packed, size);
    if (v) a.v_stride = check_rows("v", v, v_stride, packed, size);
    if (!slots) fail("slots is NULL");
    a.kv = c->kv;
    a.slots = slots;
    a.k = k;
    a.v = v;
    a.tokens = (uint32_t)tokens;
    tdt::DeviceGuard dg(c->device);
    c->streams.note(static_cast<hipStream_t>(hip_stream));
    tdt::launch_kv_read(a, c->head_dim, dtype, static_cast<hipStream_t>(hip_stream));
    return 1;
    ATT_CATCH(0)
}

// ---- norms and rotation ---------------------------------------------------------------------------

TURBO_DT_API void turbo_rotary_desc_default(TurboRotaryDesc* out) {
    if (!out) return;
    std::memset(out, 0, sizeof(*out));
    out->head_dim = 256;
    out->rotary_dim = 256;
    out->layout = TURBO_ROPE_HALVES;
    out->norms = TURBO_NORM_Q | TURBO_NORM_K;
    out->eps = 1e-6f;
    out->theta = 10000.0;
}

TURBO_DT_API void turbo_rotary_destroy(void* handle) {
    if (!handle) return;
    try {
        RotaryBox* r = rbox(handle);
        tdt::DeviceGuard dg(r->device);
        r->streams.wait();
        if (r->q_norm) (void)hipFree(r->q_norm);
        if (r->k_norm) (void)hipFree(r->k_norm);
        if (r->turns) (void)hipFree(r->turns);
        r->magic = 0;
        delete r;
    } catch (...) {
    }
}

TURBO_DT_API void* turbo_rotary_create(const TurboRotaryDesc* desc) {
    ATT_TRY
    if (!desc) fail("desc is NULL");
    check_head_dim(desc->head_dim);
    const uint32_t rd = desc->rotary_dim;
    if (desc->layout != TURBO_ROPE_HALVES && desc->layout != TURBO_ROPE_PAIRS) fail("layout must be TURBO_ROPE_HALVES or TURBO_ROPE_PAIRS");
    if (rd > desc->head_dim) fail("rotary_dim is above head_dim");
    if (rd % (desc->layout == TURBO_ROPE_HALVES ? 16u : 2u) != 0u)
        fail("rotary_dim must be even, in halves a multiple of 16");
    if (desc->norms & ~(uint32_t)(TURBO_NORM_Q | TURBO_NORM_K | TURBO_NORM_V)) fail("unknown bit in norms");
    if (!(desc->eps >= 0.0f) || !std::isfinite(desc->eps)) fail("eps must be finite and not negative");
    if (rd && !desc->inv_freq && !(desc->theta > 0.0 && std::isfinite(desc->theta))) fail("theta must be finite and above 0");
    // turns per position, modulo one turn, in 64-bit fixed point
    std::vector<uint64_t> turns(rd / 2u);
    for (uint32_t i = 0; i < rd / 2u; ++i) {
        // 64 bits throughout: a power rounded to double would be off by 2^-25 turns at position 2^32
        const long double f = desc->inv_freq ? (long double)desc->inv_freq[i] : std::pow((long double)desc->theta, -2.0L * i / rd);
        if (!std::isfinite(f)) fail("inv_freq[" + std::to_string(i) + "] is not finite");
        long double t = f / 6.283185307179586476925286766559L;
        t -= std::floor(t);
        t = std::ldexp(t, 64);
        turns[i] = t >= 18446744073709551615.0L ? 0u : (uint64_t)(t + 0.5L);
    }
    check_device(desc->device);
    tdt::DeviceGuard dg(desc->device);
    struct Free {
        void operator()(RotaryBox* r) const { turbo_rotary_destroy(r); }
    };
    std::unique_ptr<RotaryBox, Free> r(new RotaryBox);
    r->device = desc->device;
    r->head_dim = desc->head_dim;
    r->rotary_dim = rd;
    r->layout = desc->layout;
    for (uint64_t t : turns) r->still = r->still || t == 0u;
    r->norms = desc->norms;
    r->eps = desc->eps;
    const hipMemcpyKind kind = desc->weights_on_device ? hipMemcpyDeviceToDevice : hipMemcpyHostToDevice;
    auto weight = [&](uint16_t** to, const uint16_t* from) {
        if (!from) return;
        tdt::check_hip(hipMalloc(to, desc->head_dim * 2u), "alloc norm weight");
        tdt::check_hip(hipMemcpyAsync(*to, from, desc->head_dim * 2u, kind, nullptr), "copy norm weight");
    };
    weight(&r->q_norm, desc->q_norm);
    weight(&r->k_norm, desc->k_norm);
    if (rd) {
        tdt::check_hip(hipMalloc(&r->turns, turns.size() * 8u), "alloc frequencies");
        tdt::check_hip(hipMemcpyAsync(r->turns, turns.data(), turns.size() * 8u, hipMemcpyHostToDevice, nullptr), "copy frequencies");
    }
    tdt::check_hip(hipStreamSynchronize(nullptr), "copy frequencies");
    return r.release();
    ATT_CATCH(nullptr)
}

TURBO_DT_API int turbo_qk_norm_rope(void* handle, const TurboQkvInputs* in, void* hip_stream) {
    ATT_TRY
    RotaryBox* r = rbox(handle);
    if (!in) fail("in is NULL");
    const size_t size = dtype_size(in->dtype);
    check_tokens(in->tokens);
    CacheBox* c = in->cache ? cbox(in->cache) : nullptr;
    if (!in->q && !in->k) fail("q and k are both NULL");
    if (in->q && (in->q_heads < 1 || in->q_heads > (int)kMaxQueryHeads)) fail("q_heads must be in 1.." + std::to_string(kMaxQueryHeads));
    if (in->k && (in->kv_heads < 1 || in->kv_heads > (int)kMaxKvHeads)) fail("kv_heads must be in 1.." + std::to_string(kMaxKvHeads));
    if (in->k && !in->k_out && !c) fail("k has neither k_out nor a cache to go to");
    if (c) {
        if (!in->k || !in->v) fail("a cache needs k and v");
        if (c->device != r->device) fail("the cache is on another device than the rotary handle");
        if (c->head_dim != r->head_dim || (int)c->kv.heads != in->kv_heads) fail("the cache has another head_dim or number of heads");
        if (!in->slots) fail("slots is NULL");
    } else if (in->v) {
        fail("v is given but no cache to take it");
    }
    if (in->tokens == 0) return 1;
    tdt::QkvArgs a{};
    const size_t q_packed = (size_t)(in->q ? in->q_heads : 0) * r->head_dim, kv_packed = (size_t)(in->k ? in->kv_heads : 0) * r->head_dim;
    if (in->q) {
        a.q_stride = check_rows("q", in->q, in->q_stride, q_packed, size);
        a.q_out_stride = check_rows("q_out", in->q_out, in->q_out_stride, q_packed, size);
        if (in->q_out == in->q && a.q_out_stride != a.q_stride) fail("q_out is q with another stride");
    }
    if (in->k) a.k_stride = check_rows("k", in->k, in->k_stride, kv_packed, size);
    if (in->k && in->k_out) {
        a.k_out_stride = check_rows("k_out", in->k_out, in->k_out_stride, kv_packed, size);
        if (in->k_out == in->k && a.k_out_stride != a.k_stride) fail("k_out is k with another stride");
    }
    if (c) a.v_stride = check_rows("v", in->v, in->v_stride, kv_packed, size);
    if (r->rotary_dim && !in->positions) fail("positions is NULL");
    a.q = in->q;
    a.k = in->k;
    a.v = in->v;
    a.q_out = in->q_out;
    a.k_out = in->k_out;
    a.positions = in->positions;
    a.slots = in->slots;
    a.q_norm = r->q_norm;
    a.k_norm = r->k_norm;
    a.turns = r->turns;
    a.tokens = (uint32_t)in->tokens;
    a.q_heads = in->q ? (uint32_t)in->q_heads : 0u;
    a.kv_heads = in->k ? (uint32_t)in->kv_heads : 0u;
    a.rotary_dim = r->rotary_dim;
    a.pairs = r->layout == TURBO_ROPE_PAIRS;
    a.still = r->still;
    a.norms = r->norms;
    a.eps = r->eps;
    if (c) a.kv = c->kv;
    tdt::DeviceGuard dg(r->device);
    r->streams.note(static_cast<hipStream_t>(hip_stream));
    if (c) c->streams.note(static_cast<hipStream_t>(hip_stream));
    tdt::launch_qkv(a, r->head_dim, in->dtype, static_cast<hipStream_t>(hip_stream));
    return 1;
    ATT_CATCH(0)
}

// ---- attention ---------------------------------------------------------------------------------------

TURBO_DT_API int turbo_attention_workspace(void* handle, const TurboAttentionInputs* in, size_t* bytes) {
    ATT_TRY
    CacheBox* c = cbox(handle);
    if (!in || !bytes) fail("in or bytes is NULL");
    *bytes = (size_t)attention_plan(*c, *in).bytes;
    return 1;
    ATT_CATCH(0)
}

TURBO_DT_API int turbo_prefix_attention(void* handle, const TurboAttentionInputs* in, void* hip_stream) {
    ATT_TRY
    CacheBox* c = cbox(handle);
    if (!in) fail("in is NULL");
    const tdt::AttnPlan plan = attention_plan(*c, *in);
    if (!std::isfinite(in->scale)) fail("scale must be finite");
    if (in->batch == 0) return 1;
    const size_t size = dtype_size(in->dtype), packed = (size_t)in->q_heads * c->head_dim;
    tdt::AttnArgs a{};
    a.q_stride = check_rows("q", in->q, in->q_stride, packed, size);
    a.out_stride = check_rows("out", in->out, in->out_stride, packed, size);
    if (in->q == in->out) fail("out is q");
    if (!in->kv_len) fail("kv_len is NULL");
    if (in->prefix_len && !in->prefix_pages) fail("prefix_pages is NULL");
    if (in->page_stride && !in->pages) fail("pages is NULL");
    if (plan.bytes) {
        if (!in->workspace) fail("workspace is NULL");
        if (reinterpret_cast<uintptr_t>(in->workspace) % 16u != 0u) fail("workspace must be 16-byte aligned");
        if (in->workspace_bytes < plan.bytes)
            fail("workspace holds " + std::to_string(in->workspace_bytes) + " bytes, the call needs " + std::to_string(plan.bytes));
    }
    a.kv = c->kv;
    a.q = in->q;
    a.out = in->out;
    a.kv_len = in->kv_len;
    a.prefix_pages = in->prefix_pages;
    a.pages = in->pages;
    a.prefix_len = in->prefix_len;
    a.page_stride = in->page_stride;
    a.batch = (uint32_t)in->batch;
    a.q_len = (uint32_t)in->q_len;
    a.q_heads = (uint32_t)in->q_heads;
    a.group = a.q_heads / c->kv.heads;
    a.window = in->window;
    a.scale_log2e = (float)std::frexp((double)in->scale * 1.4426950408889634, &a.scale_power);
    a.stats = static_cast<float2*>(in->workspace);
    a.sums = reinterpret_cast<float*>(static_cast<uint8_t*>(in->workspace) + plan.stats_bytes);
    tdt::DeviceGuard dg(c->device);
    c->streams.note(static_cast<hipStream_t>(hip_stream));
    tdt::launch_attention(a, plan, c->head_dim, in->dtype, static_cast<hipStream_t>(hip_stream));
    return 1;
    ATT_CATCH(0)
}

}  // extern "C"

// Checks that the layer loop's entry points share, and what turns an exception into a result and a message.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <stdexcept>
#include <string>

#include "dt_internal.h"

namespace tdt {

constexpr int kMaxTokens = 1 << 28;             // a cache read takes 8 threads of one grid dimension to a token
constexpr uint32_t kMaxKvHeads = 1024, kMaxQueryHeads = 8192;

[[noreturn]] inline void fail(const std::string& what) { throw std::runtime_error(what); }

inline void check_head_dim(uint32_t d) {
    if (d != 64u && d != 128u && d != 256u && d != 512u) fail("head_dim must be 64, 128, 256 or 512");
}

inline void check_device(int device) {
    int ndev = 0;
    check_hip(hipGetDeviceCount(&ndev), "hipGetDeviceCount");
    if (device < 0 || device >= ndev) fail("no such HIP device");
}

inline size_t dtype_size(int dtype) {
    if (dtype != TURBO_HIDDEN_F32 && dtype != TURBO_HIDDEN_BF16) fail("dtype must be TURBO_HIDDEN_F32 or TURBO_HIDDEN_BF16");
    return dtype == TURBO_HIDDEN_BF16 ? 2u : 4u;
}

inline void check_tokens(int tokens) {
    if (tokens < 0 || tokens > kMaxTokens) fail("tokens must be in 0.." + std::to_string(kMaxTokens));
}

// A buffer of rows and its stride in elements (0: packed); the stride it has.
inline size_t check_rows(const char* name, const void* p, size_t stride, size_t packed, size_t size) {
    if (!p) fail(std::string(name) + " is NULL");
    if (reinterpret_cast<uintptr_t>(p) % 16u != 0u) fail(std::string(name) + " must be 16-byte aligned");
    if (stride == 0u) return packed;
    if (stride < packed) fail(std::string(name) + "_stride is smaller than a token's heads");
    if (stride > (size_t{1} << 32)) fail(std::string(name) + "_stride is above 2^32 elements");
    if (stride * size % 16u != 0u) fail(std::string(name) + "_stride must be a multiple of 16 bytes");
    return stride;
}

inline void check_words(const char* name, const void* p, uintptr_t align = 4u) {
    if (!p) fail(std::string(name) + " is NULL");
    if (reinterpret_cast<uintptr_t>(p) % align != 0u) fail(std::string(name) + " must be " + std::to_string(align) + "-byte aligned");
}

// An array of a call, and whether two have bytes in common (an absent one has none).
struct Span {
    const void* p;
    uint64_t bytes;
    bool meets(const Span& other) const {
        const uint64_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(other.p);
        return p && other.p && bytes && other.bytes && a < b + other.bytes && b < a + bytes;
    }
    bool is(const Span& other) const { return p == other.p && bytes == other.bytes; }
};

}  // namespace tdt

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

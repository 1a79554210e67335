// Loads from memory to LDS that pass no registers.
#pragma once

#include "dt_internal.h"
#include "dt_mfma.h"

namespace tdt {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Memory that a wave's buffer-to-LDS loads read, 16 bytes to a lane at its byte offset, 1 KB side by side in LDS. They are
// written as assembly because the compiler takes every later LDS read for one of theirs and waits for them there, before
// the tile in hand is begun (4 x 1,000 tokens with heads of 256: 60 us, 55 as assembly). The wait is the caller's, before
// the barrier in front of the tile. A load has no result register; its address register is read at issue.
struct TileSource {
    u32x4 words;
    __device__ inline TileSource(const void* p, uint32_t bytes) {
        const uint64_t at = reinterpret_cast<uint64_t>(p);
        auto scalar = [](uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); };
        words = u32x4{scalar((uint32_t)at), scalar((uint32_t)(at >> 32)) & 0xFFFFu, scalar(bytes), (uint32_t)kBufDword3};
    }
    __device__ inline void load(void* lds, uint32_t offset) const {
        const uint32_t place = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)lds;
        const uint32_t to = (uint32_t)__builtin_amdgcn_readfirstlane((int)place);
        // five wait states between a scalar register that the vector unit wrote and its use by a buffer load, one behind
        // M0, which nothing else here uses
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                     ::"s"(to), "v"(offset), "s"(words)
                     : "memory", "m0");
    }
};

}  // namespace tdt

// Direct-to-LDS loads of the attention kernels (gfx950).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace llkv {

// S_WAITCNT's operand for at most n vector memory operations left, the other counters free.
constexpr int vmcnt_imm(int n) { return 0x3F70 | (n & 15) | (n >> 4) << 14; }

// Direct-to-LDS load of 16 bytes per lane: lane L's bytes land at LDS address
// lds + 16 L (lds uniform over the wave).  Issued as inline assembly, so that
// the compiler, which cannot tell the two tile buffers apart, does not wait for
// it before every LDS read of the other buffer; the caller waits (vmcnt) before
// the barrier that publishes the tile.  A later load only lengthens the
// compiler's own in-order vmcnt waits.
// la: the LDS byte address (lds_addr), wave-uniform.
__device__ inline uint32_t lds_addr(const void* lds) {
    return __builtin_amdgcn_readfirstlane(
        (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)lds);
}

__device__ inline void dma16(const void* gptr, uint32_t la) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
                 :
                 : "v"(gptr), "s"(la)
                 : "memory", "m0");
}

// 4 bytes per lane, to lds + 4 L.
__device__ inline void dma4(const void* gptr, uint32_t la) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off"
                 :
                 : "v"(gptr), "s"(la)
                 : "memory", "m0");
}

// dma16 with a wave-uniform base (scalar registers) and a 32-bit per-lane
// byte offset (no per-lane 64-bit address arithmetic).
// NT: a streaming (nontemporal) load.
template <bool NT = false>
__device__ inline void dma16_s(const void* sbase, uint32_t voff, uint32_t la) {
    const uint64_t b = (uint64_t)(uintptr_t)sbase;
    // (readfirstlane returns int: widen through uint32_t, not by sign extension)
    const uint64_t bs = ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(b >> 32)) << 32) |
                        (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)b);
    if constexpr (NT)
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 nt"
                     :
                     : "v"(voff), "s"(bs), "s"(la)
                     : "memory", "m0");
    else
        asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                     :
                     : "v"(voff), "s"(bs), "s"(la)
                     : "memory", "m0");
}

}  // namespace llkv

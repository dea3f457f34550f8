// lds_dma.hpp -- loads from global memory straight into LDS on gfx950, 16 (4) bytes per
// lane to lds_base + 16 (4) * lane.
//
// In assembly, so that the compiler's LDS bookkeeping does not see them: with such a
// load in flight it cannot count the ordinary LDS reads and drains them all before every
// use.  The kernels wait for these loads themselves (vmcnt, before the barrier that
// publishes the buffer), and the "memory" clobber keeps LDS reads and writes on their
// side of it.
//
// The load takes its LDS address from M0, and the hardware does not hold it back for a
// scalar write of M0 just before it: one wait state has to stand between the two, which
// the compiler adds for its own loads and cannot add inside of an asm statement.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace kc {

#define KC_LDS_DMA(load, address, base) "s_mov_b32 m0, " base "\n\ts_nop 0\n\t" load " " address

// From a lane's own address.
__device__ __forceinline__ void lds_dma16(const void* g, uint32_t lds_base) {
    asm volatile(KC_LDS_DMA("global_load_lds_dwordx4", "%0, off", "%1") ::"v"(g), "s"(lds_base) : "memory", "m0");
}

// From a scalar base and a 32-bit lane offset.
__device__ __forceinline__ void lds_dma16(uint32_t voff, const void* sbase, uint32_t lds_base) {
    asm volatile(KC_LDS_DMA("global_load_lds_dwordx4", "%0, %1", "%2") ::"v"(voff), "s"(sbase), "s"(lds_base)
                 : "memory", "m0");
}
__device__ __forceinline__ void lds_dma4(uint32_t voff, const void* sbase, uint32_t lds_base) {
    asm volatile(KC_LDS_DMA("global_load_lds_dword", "%0, %1", "%2") ::"v"(voff), "s"(sbase), "s"(lds_base)
                 : "memory", "m0");
}

// The same, made to depend on `after` (a value computed from the last LDS read of the
// slot that it overwrites), so that it is issued after that read has returned.
__device__ __forceinline__ void lds_dma16_after(uint32_t voff, const void* sbase, uint32_t lds_base, uint32_t after) {
    asm volatile(KC_LDS_DMA("global_load_lds_dwordx4", "%0, %1", "%2") ::"v"(voff), "s"(sbase), "s"(lds_base),
                 "v"(after)
                 : "memory", "m0");
}

#undef KC_LDS_DMA

}  // namespace kc

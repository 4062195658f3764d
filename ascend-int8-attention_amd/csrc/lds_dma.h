// LDS DMA for gfx950 kernels: global memory to LDS without registers, not
// tracked by the compiler.  Callers order the copies with vm_wait_all and
// lds_barrier.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

// 16 bytes per lane from a scalar base and a 32-bit lane offset: lane l's bytes
// land at LDS byte address lds + 16 l.  M0 carries the LDS address (the
// compiler keeps nothing live in it); the ISA asks for one wait state between
// its scalar write and the DMA, which the compiler does not add inside inline
// assembly.  The compiler's own waits count only the loads it knows, and
// vector-memory operations complete in order, so these copies make them longer,
// never shorter.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void lds_dma16(uint64_t base, uint32_t offset, uint32_t lds)
{
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
                 :: "v"(offset), "s"(base), "s"(lds) : "memory", "m0");
}
#pragma clang diagnostic pop

// Every vector-memory operation of this wave has completed.
__device__ __forceinline__ void vm_wait_all() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// This wave's LDS accesses have completed, and the work-group's waves meet;
// copies in flight stay in flight.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

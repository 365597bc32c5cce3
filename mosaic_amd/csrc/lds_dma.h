// lds_dma.h -- direct-to-LDS loads issued as inline assembly, and the waits and barriers that go
// with them.  The compiler's wait insertion does not see them: across the joins of a ring loop its
// tracking of which LDS object a direct-to-LDS load writes becomes conservative, and it waited for
// the loads just requested for a later step before the current step's LDS reads.  The caller waits
// for these loads (s_waitcnt vmcnt) and synchronises the workgroup itself.  M0 is declared
// clobbered; the compiler sets M0 again before each of its own uses, so nothing it holds is lost.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mosaic {
namespace {

__device__ __forceinline__ void wait_vmem() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
// Workgroup barrier for LDS data whose direct-to-LDS loads each wave has already waited for
// itself: __syncthreads() would also wait for every load still in flight (its release fence
// covers the loads' LDS writes), which takes the prefetch of the next step out of the overlap.
// The memory clobber keeps the compiler from moving LDS accesses across it; lgkmcnt(0) retires
// this wave's LDS reads of the slot that is refilled after the barrier.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ uint32_t lds_addr(const void* ptr) {
    return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)ptr;
}
// address = base (uniform) + voff (per lane), LDS destination M0 + 16 l (dwordx4) or M0 + 4 l
// (dword) for lane l
__device__ __forceinline__ void dma16(const void* base, uint32_t voff, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(base), "s"(lds)
                 : "memory", "m0");
}
__device__ __forceinline__ void dma4(const void* base, uint32_t voff, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(voff), "s"(base), "s"(lds)
                 : "memory", "m0");
}
// the same from an address of each lane's own
__device__ __forceinline__ void dma16_at(const void* from, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ void dma4_at(const void* from, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(from), "s"(lds) : "memory", "m0");
}
#pragma clang diagnostic pop

}  // namespace
}  // namespace mosaic

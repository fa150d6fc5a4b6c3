// tbh_dma.h -- loads that go from memory to LDS without passing a register.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace tbh {
namespace dma {

typedef int i32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ i32x4 make_rsrc(const void *p, int bytes) {
    const uint64_t a = (uint64_t)p;
    const int n = max(bytes, 0);
    // base (48 bits, stride 0: raw buffer), size, 32-bit data format
    return i32x4{__builtin_amdgcn_readfirstlane((int)(uint32_t)a),
                 __builtin_amdgcn_readfirstlane((int)((uint32_t)(a >> 32) & 0xFFFFu)),
                 __builtin_amdgcn_readfirstlane(n), 0x00020000};
}

// 16 (or 4) bytes per active lane from buffer offset `off` + `soff` to LDS
// byte lds + 16 (4) * lane; offsets past the buffer's size write zeros.  No
// register receives the load; completion is waited for by dma_wait.  (One
// wait state between the write of M0 and the load that reads it.  M0 is a
// reserved register, which the compiler neither allocates nor takes as a
// clobber; the built kernels use it in these statements only.)
__device__ __forceinline__ void dma16(uint32_t lds, i32x4 r, uint32_t off, uint32_t soff) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(lds), "v"(off), "s"(r),
                 "s"(soff) : "memory");
}
__device__ __forceinline__ uint32_t lds_addr(const void *p) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char *)p;
}

}  // namespace dma
}  // namespace tbh

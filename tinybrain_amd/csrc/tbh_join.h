// tbh_join.h -- the last block of several that work on one result finds out
// that it is the last, and finishes it: no second launch (3.5 to 5 us each).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace tbh {

// What such blocks hand each other goes past the caches of their XCDs, a word at a
// time: a release of all a cache holds, as a fence makes it, cost 5 to 60 us a launch.
template <class T>
__device__ __forceinline__ void hand_over(T *p, T v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <class T>
__device__ __forceinline__ T handed_over(const T *p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Called by every thread of `n` blocks after what they hand over; true in all threads
// of the block that arrives last.  Nothing waits for another block.  The counter is 0
// before the launch and again after it.  seen: a word of LDS that no other use overlaps.
__device__ __forceinline__ bool last_to_arrive(uint32_t *counter, uint32_t n, uint32_t *seen) {
    // every wave's stores have arrived before the block counts
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
        *seen = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (*seen == n - 1) hand_over(counter, 0u);
    }
    __syncthreads();
    return *seen == n - 1;
}

}  // namespace tbh

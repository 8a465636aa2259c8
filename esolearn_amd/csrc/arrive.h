// Hand-over between the workgroups of one launch: what each leaves for the last
// one to arrive.
#pragma once

#include <hip/hip_runtime.h>

namespace scry {
namespace dev {

// Values that other workgroups, on other XCDs, read in this launch: device-scope
// accesses go past the XCD's own L2.
template <class T>
__device__ __forceinline__ void put(T *p, T v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <class T>
__device__ __forceinline__ T get(const T *p) {
    return __hip_atomic_load(const_cast<T *>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// With every thread of the workgroup: whether it is the last of n to arrive.
// What the others put before they arrived, it gets: each wave waits until its
// device-scope stores are complete, then the barrier, then the count.  (A
// release fence would write back the XCD's whole L2, once a workgroup: 16
// sequences at V = 128256 took 91 us with it.)
__device__ __forceinline__ bool last_to_arrive(unsigned *ctr, unsigned n) {
    __shared__ int s_last;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
        s_last = __hip_atomic_fetch_add(ctr, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == n - 1;
        if (s_last) put(ctr, 0u);  // for the next launch
    }
    __syncthreads();
    return s_last;
}

}  // namespace dev
}  // namespace scry

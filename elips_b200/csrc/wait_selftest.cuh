// The bounded wait that must expire (elips_b200_wait_selftest and its
// counterpart for the 8-bit operators), compiled into each translation unit
// that has an error word.
#pragma once

#include "ptx.cuh"

namespace eb {

// One thread waits on an mbarrier that nothing arrives on, for `budget`
// cycles: the bounded wait expires, records the device error word and raises
// the CTA's abort flag, the path every pipeline wait takes when a producer or
// consumer is lost. Nothing asynchronous is in flight, so returning with the
// barrier pending is safe.
static __global__ void wait_selftest_kernel(long long budget) {
    __shared__ __align__(8) uint64_t bar;
    __shared__ int abort_flag;
    if (threadIdx.x != 0) return;
    mbar_init(smem_u32(&bar), 1);
    abort_flag = 0;
    fence_mbarrier_init();
    mbar_wait_for(smem_u32(&bar), 0, &abort_flag, budget);
}

}  // namespace eb

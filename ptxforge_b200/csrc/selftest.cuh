// selftest.cuh -- a bounded wait that runs out: one block waits on an mbarrier that nothing arrives at, then returns.
#pragma once

#include "gemm_tc.cuh"

namespace pf {

static __global__ void selftest_wait_kernel(unsigned *status, unsigned long long timeout_ns) {
  __shared__ uint64_t bar;
  __shared__ int abort_flag;
  if (threadIdx.x == 0) {
    mbar_init(&bar, 1);
    abort_flag = 0;
    fence_mbar_init();
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    if (!mbar_wait(&bar, 0, timeout_ns, &abort_flag)) atomicOr(status, kErrEpilogueWait);
  }
  __syncthreads();
}

constexpr unsigned long long kSelftestMostNs = 10000000000ull;

}  // namespace pf

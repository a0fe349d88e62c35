// Waits of whole warps and at the end of a product, for the dense FP8 kernels.
#pragma once

#include "common.cuh"

namespace asap {
namespace lin {

// A bounded wait of a whole warp: one lane polls, every lane gets its answer and the warp is converged after it.  (With
// 32 lanes polling, the folding and scale warps filled the shared-memory pipe: a wait on a barrier that had long
// completed then took the MMA issuer 210 cycles, three of them per K block.)  It looks at no clock, as a deadline would hold
// two registers that the folding warps do not have: it ends when another warp's wait has run out, and what it waits for
// hangs on warps that do watch the clock (the producer, the MMA issuer and its drain_mmas) or on a warp that gave up with
// *abort raised.  The count, some minutes of tries, is the last resort.
constexpr uint32_t kSpins = 1u << 27;
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
  int ok = 1;
  if ((threadIdx.x & 31) == 0) {
    for (uint32_t it = 0; ok && !mbar_try_wait(bar, parity);) {
      ++it;
      if ((it & 255u) == 0 && (*abort || it > kSpins)) {
        *abort = 1;
        ok = 0;
      }
    }
  }
  const bool all = __shfl_sync(0xffffffffu, ok, 0) != 0;
  __syncwarp();  // what lane 0 acquired is every lane's
  return all;
}

// The MMA issuer's last wait: every MMA issued has completed (`bar`) before tensor memory is released.  Another warp's
// failure does not end it; it has until the deadline and at least 0.2 s, and raises *abort when it runs out, without which
// warps that wait for those MMAs would go on.
__device__ __forceinline__ void drain_mmas(uint64_t* bar, uint64_t deadline, volatile int* abort) {
  const uint64_t least = globaltimer_ns() + 200000000ull;
  volatile int never = 0;
  if (!mbar_wait(bar, 0, deadline > least ? deadline : least, &never)) *abort = 1;
}

}  // namespace lin
}  // namespace asap

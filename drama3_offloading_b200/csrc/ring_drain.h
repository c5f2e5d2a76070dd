// How a loading thread leaves its ring after a wait has run out: what it has
// asked for must have landed before the block's shared memory goes.  No CUDA in
// here, so that the host can test it.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define D3_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define D3_HOST_DEVICE inline
#endif

namespace d3 {

// Waits until the slots [0, n) of a ring hold what was last asked for, but not
// longer than budget_ns in all: a slot that another thread gave up before never
// fills, and what is in flight lands within microseconds.  `slot` and `phase`
// are the place of the next load, which has not been asked for: slots before it
// were filled in this turn of the ring, the others in the one before.
// filled(i, parity): whether slot i's phase of that parity is over (a try that
// may block for some microseconds); now(): a clock in ns.
template <typename Filled, typename Now>
D3_HOST_DEVICE bool drain_ring(int n, int slot, uint32_t phase, uint64_t budget_ns, Filled filled, Now now) {
  const uint64_t t0 = now();
  bool all = true;
#ifdef __CUDACC__
#pragma unroll 1
#endif
  for (int i = 0; i < n; ++i) {
    const uint32_t parity = phase ^ (i < slot ? 0u : 1u);
    bool there = filled(i, parity);
    while (!there && now() - t0 <= budget_ns) there = filled(i, parity);
    all = all && there;
  }
  return all;
}

}  // namespace d3

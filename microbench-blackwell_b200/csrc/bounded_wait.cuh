// bounded_wait.cuh -- mbarrier waits with a time budget, shared by the GEMM
// kernels: on expiry a wait records a status word, tells the CTA's (and a
// pair peer's) other roles to stop, and returns false.
#pragma once
#include <cstdint>

#include "sm100_ptx.cuh"

namespace {

using namespace sm100;

enum Role : uint32_t { ROLE_PRODUCER = 1, ROLE_MMA = 2, ROLE_EPILOGUE = 3, ROLE_DRAIN = 4 };

struct SharedCtl {
  uint32_t abort_addr;     // local abort flag (shared::cta address)
  uint32_t abort_peer;     // the pair peer's abort flag (shared::cluster), 0 if none
  uint64_t timeout_ns;
  int32_t* status;
};

__device__ __noinline__ void raise_abort(const SharedCtl& c, uint32_t role, uint32_t idx) {
  if (c.status) {
    const int32_t code = (int32_t)(0x3u | (role << 8) | ((idx & 0xFFu) << 12) | ((blockIdx.x & 0x7FFu) << 20));
    atomicCAS(c.status, 0, code);
  }
  st_shared_u32(c.abort_addr, 1u);
  if (c.abort_peer) st_shared_cluster_u32(c.abort_peer, 1u);
}

// Bounded wait for phase `parity` of mbarrier `bar`; false when aborted.
// The probes are plain try_wait (no suspend-time hint: resuming a suspended
// thread added latency to every pipeline round trip); the abort flag is
// checked after every probe and the timer every 8 probes.
template <bool kCluster>
__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, const SharedCtl& c,
                                         uint32_t role, uint32_t idx) {
  if (kCluster ? mbar_test_wait_cluster(bar, parity) : mbar_test_wait(bar, parity)) return true;
  uint64_t t0 = 0;
  for (uint32_t probe = 1;; ++probe) {
    if (kCluster ? mbar_try_wait_cluster(bar, parity) : mbar_try_wait(bar, parity))
      return true;
    if (ld_shared_volatile_u32(c.abort_addr)) return false;
    if ((probe & 7u) == 1u) {
      const uint64_t now = globaltimer_ns();
      if (t0 == 0) {
        t0 = now;
      } else if (now - t0 > c.timeout_ns) {
        raise_abort(c, role, idx);
        return false;
      }
    }
  }
}

// Wait with a short fixed budget during abort drains; never raises.
__device__ __forceinline__ void drain_wait(uint32_t bar, uint32_t parity, uint64_t budget_ns) {
  const uint64_t t0 = globaltimer_ns();
  while (!mbar_try_wait(bar, parity)) {
    if (globaltimer_ns() - t0 > budget_ns) break;
  }
}

}  // namespace

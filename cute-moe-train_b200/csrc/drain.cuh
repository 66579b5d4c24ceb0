// What a CTA still waits for when it stops early (a pipeline wait ran out): its own copies and products in flight.
// Shared memory that a bulk copy still writes, or tensor memory that a product still writes, must not be given back.
// Run once all roles have stopped, so nothing new is issued; the abort flag is set by then, so these waits do not look at
// it: they end with what they wait for, or at their own limit.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#include "moe_gemm.h"
#include "ptx.cuh"
#define MGF_INLINE __host__ __device__ __forceinline__
#else
#define MGF_INLINE inline
#endif

namespace mgf {
namespace drain {

constexpr uint64_t kLimitNs = 100ull * 1000ull * 1000ull;  // a copy or a product takes microseconds

// Polls until done() is true, or the clock is past the deadline (false).
template <typename Done, typename Now>
MGF_INLINE bool wait_until(Done done, Now now_ns, uint64_t deadline_ns) {
  while (!done())
    if (now_ns() > deadline_ns) return false;
  return true;
}

// Copies whose bytes count on this CTA's barriers: one bit per stage that was armed, and the parity of its last phase.
struct Copies {
  uint32_t armed = 0, parity = 0;
  MGF_INLINE void arm(uint32_t stage, uint32_t phase) {
    armed |= 1u << stage;
    parity = (parity & ~(1u << stage)) | (phase << stage);
  }
};

// Waits for the last copy into every armed stage; landed(stage, parity) polls one.  The deadline is for all together.
template <typename Landed, typename Now>
MGF_INLINE bool wait_copies(const Copies& c, Landed landed, Now now_ns, uint64_t deadline_ns) {
  bool all = true;
  for (uint32_t s = 0; s < 32; ++s)
    if ((c.armed >> s) & 1u)
      all &= wait_until([&] { return landed(s, (c.parity >> s) & 1u); }, now_ns, deadline_ns);
  return all;
}

#ifdef __CUDACC__
// One thread of a CTA, for its copies.  In a pair the copies of both CTAs count on the even one's barriers, and a CTA that
// ran ahead of its peer has copies in flight that complete no phase: both hold for the whole limit, and leave together
// at the cluster barrier that follows.
template <int CG>
__device__ __forceinline__ void copies(const Copies& c, uint64_t* full_bar, unsigned int* status) {
  auto now = [] { return ptx::globaltimer_ns(); };
  const uint64_t deadline = now() + kLimitNs;
  const bool all = wait_copies(c, [&](uint32_t s, uint32_t parity) { return ptx::mbar_try_wait(ptx::smem_u32(&full_bar[s]), parity); },
                               now, deadline);
  if (CG == 2) wait_until([] { return false; }, now, deadline);
  if (!all) atomicOr(status, MGF_DEV_DRAIN_TIMEOUT);
}

// The thread that issued the products (it alone can commit them), for all of them.
template <int CG>
__device__ __forceinline__ void products(uint64_t* drain_bar, unsigned int* status) {
  const uint32_t bar = ptx::smem_u32(drain_bar);
  if constexpr (CG == 2) ptx::umma_commit_pair(bar, 0x1);
  else ptx::umma_commit(bar);
  auto now = [] { return ptx::globaltimer_ns(); };
  if (!wait_until([&] { return ptx::mbar_try_wait(bar, 0); }, now, now() + kLimitNs)) atomicOr(status, MGF_DEV_DRAIN_TIMEOUT);
}
#endif

}  // namespace drain
}  // namespace mgf

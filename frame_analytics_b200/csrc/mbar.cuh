// mbarriers with bounded waits (sm_100a).
#pragma once

#include "common.cuh"

namespace fab {

__device__ __forceinline__ unsigned smem_u32(const void* p) {
  return static_cast<unsigned>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void mbar_init(unsigned long long* bar, unsigned count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(smem_u32(bar)), "r"(count));
}
__device__ __forceinline__ void mbar_expect_tx(unsigned long long* bar, unsigned bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(smem_u32(bar)),
               "r"(bytes)
               : "memory");
}
__device__ __forceinline__ bool mbar_try(unsigned a, unsigned parity) {
  unsigned done;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      " selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(done)
      : "r"(a), "r"(parity)
      : "memory");
  return done != 0;
}
__device__ __forceinline__ unsigned long long globaltimer_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
// Slow path of a bounded wait: polls until the phase completes, `limit_ns`
// of wall time passes, or another wait has already failed (the error word is
// set).  On giving up it records FA_E_TIMEOUT in the error word, which the
// next call of any entry point turns into its return status, and returns so
// that the kernel finishes instead of hanging; its outputs are then garbage
// and reported as such.  `err` is a host-mapped word (it may be null: the
// wait then only gives up).
static __device__ __noinline__ void mbar_wait_slow(unsigned a, unsigned parity, unsigned* err,
                                            unsigned long long limit_ns) {
  const unsigned long long t0 = globaltimer_ns();
  for (unsigned i = 1;; ++i) {
    if (mbar_try(a, parity)) return;
    if ((i & 255u) == 0u) {
      const bool failed = err && *reinterpret_cast<volatile unsigned*>(err) != 0u;
      if (failed || globaltimer_ns() - t0 > limit_ns) {
        if (err) {
          *reinterpret_cast<volatile unsigned*>(err) = (unsigned)FA_E_TIMEOUT;
          __threadfence_system();
        }
        return;
      }
    }
  }
}
// Bounded wait on a phase: a few fast polls, then the timed slow path (two
// seconds: a row copy takes microseconds).
constexpr unsigned long long kWaitLimitNs = 2000000000ull;
__device__ __forceinline__ void mbar_wait(unsigned long long* bar, unsigned parity,
                                          unsigned* err) {
  const unsigned a = smem_u32(bar);
#pragma unroll 1
  for (int i = 0; i < 32; ++i)
    if (mbar_try(a, parity)) return;
  mbar_wait_slow(a, parity, err, kWaitLimitNs);
}
__device__ __forceinline__ void fence_async_smem() {
  asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");
}

}  // namespace fab

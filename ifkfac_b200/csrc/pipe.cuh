// Barriers of copy pipelines (mbarriers in shared memory, by 32-bit address) with bounded waits.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace ifk {

__device__ __forceinline__ uint64_t now_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}

// Bounded wait for the phase of this parity: gives up after two seconds, or when another warp of the block
// has (*failed).
__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, volatile int* failed) {
  uint64_t t0 = 0;
  for (uint32_t it = 0;; ++it) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    if (done) return true;
    if ((it & 63) == 63) {
      if (*failed) return false;
      const uint64_t t = now_ns();
      if (t0 == 0) t0 = t;
      else if (t - t0 > 2000000000ull) {
        *failed = 1;
        return false;
      }
    }
  }
}

// Whether the phase has completed, without waiting.
__device__ __forceinline__ bool test_bar(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done;
}

__device__ __forceinline__ void arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// One arrival, and the bytes of the copies that the barrier's phase also waits for.
__device__ __forceinline__ void expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

// Bulk copy global -> shared (16-byte aligned, a multiple of 16 bytes), completing on the barrier.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// A barrier of `threads` threads of the block (ids 1 .. 15).
__device__ __forceinline__ void named_barrier(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

// After a failed wait: stay until the copies in flight have landed (microseconds).
__device__ __forceinline__ void linger() {
  const uint64_t t0 = now_ns();
  while (now_ns() - t0 < 1000000ull) __nanosleep(1000);
}

}  // namespace ifk

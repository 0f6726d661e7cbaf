// Bounded mbarrier waits and the shared-memory descriptor of the tcgen05 kernels.
#pragma once

#include <cstdint>

namespace im {

constexpr unsigned long long QT_WAIT_NS = 1000000000ull;  // of the drains, and of every other wait unless it is set

__device__ __forceinline__ uint32_t qt_smem(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ bool qt_try_wait(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}

// The same with a suspend-time hint: the thread sleeps (up to 20 us) instead of spinning until the phase completes.
__device__ __forceinline__ bool qt_try_wait_sleep(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(done)
      : "r"(bar), "r"(parity), "r"(20000u)
      : "memory");
  return done != 0;
}

__device__ __forceinline__ unsigned long long qt_clock() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}

// Bounded wait of one thread for the phase of `parity`; false when this CTA has given up (now or earlier).
__device__ __forceinline__ bool qt_wait(unsigned long long* bar, uint32_t parity, volatile int* abort_flag,
                                        unsigned* error, unsigned long long limit) {
  const uint32_t b = qt_smem(bar);
  if (*abort_flag) return false;
  if (qt_try_wait(b, parity)) return true;
  const unsigned long long t0 = qt_clock();
  while (true) {
    if (qt_try_wait_sleep(b, parity)) return true;
    if (*abort_flag) return false;
    if (qt_clock() - t0 > limit) {
      *abort_flag = 1;
      atomicExch(error, 1u);
      return false;
    }
  }
}

// The same of a whole warp. It ends in a vote: the warp leaves it converged and of one mind (a lane that gave up takes
// the others along), as the warp-wide barriers and tcgen05's .aligned instructions that follow require.
__device__ __forceinline__ bool qt_wait_warp(unsigned long long* bar, uint32_t parity, volatile int* abort_flag,
                                             unsigned* error, unsigned long long limit) {
  return __all_sync(0xffffffffu, qt_wait(bar, parity, abort_flag, error, limit));
}

// Up to 64 attempts (each suspends the thread for a microsecond or two at most) in a loop of three instructions.
__device__ __forceinline__ bool qt_try_wait_64(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .u32 n;\n\tmov.u32 n, 64;\n"
      "AGAIN:\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t@p bra OUT;\n\t"
      "sub.u32 n, n, 1;\n\tsetp.ne.u32 q, n, 0;\n\t@q bra AGAIN;\n"
      "OUT:\n\tselp.u32 %0, 1, 0, p;\n\t}\n"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}

// Bounded wait of a whole warp, for pipelines whose stages last a few hundred cycles: few instructions while it is
// short, the abort flag and the timer (whose reads cost more than such a wait) only once it is long. It ends in a vote:
// the warp leaves it converged (tcgen05's .aligned instructions follow, and lanes may see a phase complete at different
// attempts) and of one mind (a lane that gave up takes the others along).
__device__ __forceinline__ bool qt_wait_short(uint32_t bar, uint32_t parity, volatile int* abort_flag,
                                              unsigned* error, unsigned long long limit) {
  bool ok = qt_try_wait_64(bar, parity);
  if (!ok) {
    const unsigned long long t0 = qt_clock();
    while (true) {
      ok = qt_try_wait(bar, parity);
      if (ok || *abort_flag) break;
      if (qt_clock() - t0 > limit) {
        *abort_flag = 1;
        atomicExch(error, 1u);
        break;
      }
    }
  }
  return __all_sync(0xffffffffu, ok);
}

// One lane of a converged warp (the same one every time).
__device__ __forceinline__ bool qt_elect() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(p));
  return p != 0;
}

// Bounded wait that ignores the abort flag (draining copies and MMAs already in flight).
__device__ __forceinline__ void qt_drain(unsigned long long* bar, uint32_t parity) {
  const uint32_t b = qt_smem(bar);
  if (qt_try_wait(b, parity)) return;
  const unsigned long long t0 = qt_clock();
  while (!qt_try_wait(b, parity) && qt_clock() - t0 < QT_WAIT_NS) {
  }
}

__device__ __forceinline__ void qt_arrive(unsigned long long* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(qt_smem(bar)) : "memory");
}

__device__ __forceinline__ void qt_init(unsigned long long* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(qt_smem(bar)), "r"(count));
}

__device__ __forceinline__ uint64_t qt_desc(uint32_t saddr) {
  // K-major, 128-byte swizzle: 8-row groups 1024 bytes apart (SBO), leading offset 1 (unused), version 1
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}

}  // namespace im

// Waits on an mbarrier that give up, and what a kernel whose wait ran out leaves behind: NaN in its results and a word
// that the host reads (hyfft_wait_status). The limit is a kernel argument, so that it can be made short (hyfft_set_wait_clocks).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "umma.cuh"

namespace hyfft {

constexpr unsigned kWaitClocks = 1u << 31;   // about a second; a clock of 32 bits comes round after two
extern std::atomic<unsigned> g_wait_clocks;   // engine.cu

namespace {

__device__ unsigned g_ran_out;  // of the kernels of one source file

__device__ __forceinline__ bool try_phase(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}
// Whether the phase is over already; does not wait.
__device__ __forceinline__ bool test_phase(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n.reg .pred p;\nmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}
// Waits for the phase; false after `patience` clocks (0: without waiting).
// No time hint: with one, try_wait becomes a loop of short sleeps (a scan's pass with outputs took 3% longer).
__device__ __forceinline__ bool wait_phase(uint64_t* bar, uint32_t parity, unsigned patience) {
  const uint32_t a = umma::su32(bar);
  if (patience ? try_phase(a, parity) : test_phase(a, parity)) return true;
  const unsigned t0 = (unsigned)clock64();
  do {
    if ((unsigned)clock64() - t0 >= patience) return false;
  } while (!try_phase(a, parity));
  return true;
}

// Whether a wait has run out in this file's kernels on the current device; the device is idle.
inline cudaError_t read_ran_out(bool clear, unsigned* out) {
  cudaError_t e = cudaMemcpyFromSymbol(out, g_ran_out, sizeof(*out));
  const unsigned zero = 0;
  if (e == cudaSuccess && clear && *out) e = cudaMemcpyToSymbol(g_ran_out, &zero, sizeof(zero));
  return e;
}

}  // namespace
}  // namespace hyfft

// Bounded waits on mbarriers for kernels of one translation unit, and the record of one that ran out.
#pragma once
#include <cuda_runtime.h>

#include "ptx.cuh"

namespace iflb200 {

namespace {

__device__ uint32_t g_record[4];                   // role << 24 | barrier << 16 | low bits of a counter; 0: none
__device__ uint64_t g_budget_ns = 2000000000ull;   // of one wait

// Wait of one thread; false once the CTA gives up.  (Short: a kernel has a dozen copies of it.)
__device__ __forceinline__ bool wait_one(uint32_t bar, uint32_t parity, volatile uint32_t* abort, uint32_t code) {
  uint64_t t0 = 0;
#pragma unroll 1
  for (uint32_t spins = 1; !mbar_try_wait(bar, parity); ++spins) {
    if (spins % 512 == 0) {
      if (*abort) return false;
      const uint64_t now = globaltimer_ns();
      if (t0 == 0) t0 = now;
      if (now - t0 > g_budget_ns) {
        *abort = 1;
        atomicCAS(&g_record[0], 0u, code);
        return false;
      }
    }
  }
  return true;
}
// The same for a converged warp.
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, volatile uint32_t* abort, uint32_t code) {
  if (__all_sync(0xFFFFFFFFu, mbar_try_wait(bar, parity))) return true;
  const bool ok = wait_one(bar, parity, abort, code);
  return __all_sync(0xFFFFFFFFu, ok);
}

inline int set_budget_ns(uint64_t ns) { return (int)cudaMemcpyToSymbol(g_budget_ns, &ns, sizeof(ns)); }

// The record, which is cleared (synchronises the stream).
inline int take_record(uint32_t* record, cudaStream_t s) {
  uint32_t host[4] = {0, 0, 0, 0};
  cudaError_t e = cudaMemcpyFromSymbolAsync(host, g_record, sizeof(host), 0, cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  if (e != cudaSuccess) return (int)e;
  *record = host[0];
  if (host[0] != 0) {
    const uint32_t zero[4] = {0, 0, 0, 0};
    e = cudaMemcpyToSymbolAsync(g_record, zero, sizeof(zero), 0, cudaMemcpyHostToDevice, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  }
  return (int)e;
}

}  // namespace

}  // namespace iflb200

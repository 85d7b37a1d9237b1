// Work-group sums and scans (64-lane waves, shuffles, one LDS word per wave).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace va {

// Exclusive sum of `x` over the threads of a work-group of 64 * WAVES threads, and the total of all
// of them. `buf` (WAVES words of LDS) may be used again after the call's last barrier.
template <int WAVES, typename T>
__device__ inline T block_exclusive_sum(T x, T* buf, T& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  T incl = x;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const T y = __shfl_up(incl, off);
    if (lane >= off) incl += y;
  }
  if (lane == 63) buf[wave] = incl;
  __syncthreads();
  T before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    const T y = buf[w];
    if (w < wave) before += y;
    total += y;
  }
  __syncthreads();
  return before + incl - x;
}

}  // namespace va

// Work-group sums and scans of whole numbers: wave scans in registers (DPP shifts, row broadcasts),
// one LDS word per wave and value, two barriers for any number of values.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace va {

template <int CTRL, int ROWS>
__device__ inline int dpp_add(int x) {  // x + the lane that CTRL names (0 where there is none)
  return x + __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false);
}
__device__ inline int wave_inclusive_sum(int x) {
  x = dpp_add<0x111, 0xf>(x);  // row_shr 1, 2, 4, 8: sums within rows of 16 lanes
  x = dpp_add<0x112, 0xf>(x);
  x = dpp_add<0x114, 0xf>(x);
  x = dpp_add<0x118, 0xf>(x);
  x = dpp_add<0x142, 0xa>(x);  // row_bcast 15: the last lane of a row to the next one (rows 1, 3)
  x = dpp_add<0x143, 0xc>(x);  // row_bcast 31: lane 31 to rows 2, 3
  return x;
}

// Exclusive sums of K values over the threads of a work-group of 64 WAVES threads, and their totals.
// `buf` is LDS of K * WAVES words; it may be used again after the call.
template <int WAVES, int K>
__device__ inline void block_exclusive_sums(int (&x)[K], int (&total)[K], int* buf) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int incl[K];
#pragma unroll
  for (int k = 0; k < K; ++k) incl[k] = wave_inclusive_sum(x[k]);
  if (lane == 63)
#pragma unroll
    for (int k = 0; k < K; ++k) buf[k * WAVES + wave] = incl[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {
    // lane w of every wave holds wave w's sum
    const int sums = lane < WAVES ? buf[k * WAVES + lane] : 0;
    const int upto = wave_inclusive_sum(sums);
    total[k] = __builtin_amdgcn_readlane(upto, WAVES - 1);
    const int before = wave == 0 ? 0 : __shfl(upto, wave - 1);
    x[k] = before + incl[k] - x[k];
  }
  __syncthreads();
}

// Places of the set flags of a work-group among all set ones: flag 0 of every thread in thread order,
// then flag 1 of every thread, ... `buf` is LDS of K * WAVES words (at most 64).
template <int WAVES, int K>
__device__ inline void block_places(const bool (&flag)[K], int (&place)[K], int& total, int* buf) {
  static_assert(K * WAVES <= 64, "one lane per wave and flag");
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint64_t set[K];
#pragma unroll
  for (int k = 0; k < K; ++k) set[k] = __builtin_amdgcn_ballot_w64(flag[k]);
  if (lane == 0)
#pragma unroll
    for (int k = 0; k < K; ++k) buf[k * WAVES + wave] = __builtin_popcountll(set[k]);
  __syncthreads();
  const int sums = lane < K * WAVES ? buf[lane] : 0;
  const int upto = wave_inclusive_sum(sums);
  total = __builtin_amdgcn_readlane(upto, K * WAVES - 1);
#pragma unroll
  for (int k = 0; k < K; ++k)
    place[k] = __shfl(upto - sums, k * WAVES + wave) +
               __builtin_popcountll(set[k] & ((1ull << lane) - 1));
  __syncthreads();
}

}  // namespace va

// Sums over the lanes of a wave.  Every lane of the wave calls them.
#pragma once

#include "alpx_common.h"

namespace alpx {

// x of the lane that DPP control CTRL names, 0 for lanes without one and
// outside the rows of ROWS.
template <int CTRL, int ROWS>
__device__ __forceinline__ int lane_shifted(int x) {
  return __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ int64_t lane_shifted(int64_t x) {
  const uint32_t lo = (uint32_t)lane_shifted<CTRL, ROWS>((int)(uint32_t)x);
  const uint32_t hi = (uint32_t)lane_shifted<CTRL, ROWS>((int)(x >> 32));
  return (int64_t)((uint64_t)hi << 32 | lo);
}

// Inclusive sums: within rows of 16 lanes, then each odd row takes the sum
// of the row before it, then the upper half that of the lower.  DPP moves
// take a few cycles; the same steps as shuffles, each a trip through the LDS
// unit, cost ten times that.
template <typename T>
__device__ __forceinline__ T wave_inclusive(T x) {
  x += lane_shifted<0x111, 0xf>(x);  // from 1 lane below,
  x += lane_shifted<0x112, 0xf>(x);  // 2,
  x += lane_shifted<0x114, 0xf>(x);  // 4
  x += lane_shifted<0x118, 0xf>(x);  // and 8
  x += lane_shifted<0x142, 0xa>(x);  // lane 15 of the row before
  x += lane_shifted<0x143, 0xc>(x);  // lane 31
  return x;
}

__device__ __forceinline__ int wave_total(int x) {
  return __builtin_amdgcn_readlane(wave_inclusive(x), 63);
}

// Exclusive sums.
__device__ __forceinline__ int wave_before(int x) { return wave_inclusive(x) - x; }

}  // namespace alpx

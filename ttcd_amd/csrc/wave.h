// wave.h - sums over the 64 lanes of a wavefront by cross-lane moves, without LDS.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ttcd {

// Lanes of a row of 16 by some before (0 where there is none) or around, as CTRL says.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
  return __builtin_amdgcn_update_dpp(0, x, CTRL, 0xf, 0xf, true);
}
template <int CTRL>
__device__ __forceinline__ double dpp(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint64_t lo = dpp<CTRL>((uint32_t)u), hi = dpp<CTRL>((uint32_t)(u >> 32));
  return __builtin_bit_cast(double, hi << 32 | lo);
}
__device__ __forceinline__ uint32_t lane_of(uint32_t x, int lane) {
  return __builtin_amdgcn_readlane(x, lane);
}
__device__ __forceinline__ double lane_of(double x, int lane) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint64_t lo = lane_of((uint32_t)u, lane), hi = lane_of((uint32_t)(u >> 32), lane);
  return __builtin_bit_cast(double, hi << 32 | lo);
}

// Sums over the lanes before this one (all: over all of them).
template <typename V>
__device__ __forceinline__ V scan_before(V x, int lane, V* all = nullptr) {
  x += dpp<0x111>(x);  // row_shr:1, 2, 4, 8
  x += dpp<0x112>(x);
  x += dpp<0x114>(x);
  x += dpp<0x118>(x);
  const V a = lane_of(x, 15), b = a + lane_of(x, 31), c = b + lane_of(x, 47);
  if (all != nullptr) *all = c + lane_of(x, 63);
  return dpp<0x111>(x) + (lane < 16 ? V(0) : lane < 32 ? a : lane < 48 ? b : c);
}
// The sum over a row of 16 lanes, in each of them, and over all.
template <typename V>
__device__ __forceinline__ V sum_of_row(V x) {
  x += dpp<0x121>(x);  // row_ror:1, 2, 4, 8
  x += dpp<0x122>(x);
  x += dpp<0x124>(x);
  x += dpp<0x128>(x);
  return x;
}
template <typename V>
__device__ __forceinline__ V sum_of(V x) {
  x = sum_of_row(x);
  return lane_of(x, 0) + lane_of(x, 16) + (lane_of(x, 32) + lane_of(x, 48));
}
__device__ __forceinline__ uint32_t max_of(uint32_t x) {
  x = max(x, dpp<0x121>(x));
  x = max(x, dpp<0x122>(x));
  x = max(x, dpp<0x124>(x));
  x = max(x, dpp<0x128>(x));
  return max(max(lane_of(x, 0), lane_of(x, 16)), max(lane_of(x, 32), lane_of(x, 48)));
}

}  // namespace ttcd

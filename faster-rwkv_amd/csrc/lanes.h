// Sums over groups of lanes of a wave, in fp32: every lane of the group gets the sum, whose order is fixed.
#pragma once

#include "device_utils.h"

#pragma clang fp contract(off)

namespace frhip {

// v of the lane and of the one 16 or 32 lanes away: the instruction swaps the odd rows (of 16 or 32 lanes) of its first operand with the even
// ones of its second, so of a value and itself the results are the even rows twice and the odd rows twice
__device__ __forceinline__ float add_across_16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float add_across_32(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Over the LANES lanes that share lane / LANES
template <int LANES>
__device__ __forceinline__ float lane_sum(float v) {
  if constexpr (LANES >= 2) v += dpp_mov<0xB1>(v);   // quad_perm [1,0,3,2]
  if constexpr (LANES >= 4) v += dpp_mov<0x4E>(v);   // quad_perm [2,3,0,1]
  if constexpr (LANES >= 8) v += dpp_mov<0x141>(v);  // row_half_mirror
  if constexpr (LANES >= 16) v += dpp_mov<0x140>(v);  // row_mirror
  if constexpr (LANES >= 32) v = add_across_16(v);
  if constexpr (LANES >= 64) v = add_across_32(v);
  return v;
}

}  // namespace frhip

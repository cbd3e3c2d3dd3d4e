// Sums over groups of neighbouring lanes of a wave, in registers: cross-lane operands of VALU instructions up to 16
// lanes, the row swaps of gfx950 for 32 and 64.  Every lane of the group gets the sum, added in the same order.
#pragma once

#include <hip/hip_runtime.h>

namespace tsplat {

template <int CTRL>
__device__ __forceinline__ float lane_moved(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}

template <int G>
__device__ __forceinline__ float group_sum(float v) {
  static_assert(G >= 1 && G <= 64 && (G & (G - 1)) == 0, "a power of two of lanes");
  if constexpr (G >= 2) v += lane_moved<0xb1>(v);    // quad_perm 1 0 3 2
  if constexpr (G >= 4) v += lane_moved<0x4e>(v);    // quad_perm 2 3 0 1
  if constexpr (G >= 8) v += lane_moved<0x141>(v);   // row_half_mirror: the other quad of 8
  if constexpr (G >= 16) v += lane_moved<0x140>(v);  // row_mirror: the other 8 of 16
  if constexpr (G >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if constexpr (G >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return v;
}

}  // namespace tsplat

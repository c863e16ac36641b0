// Values handed from lane to lane of a wavefront through the data-parallel paths of the vector unit (no LDS, no wait).
#ifndef PSKV_LANES_H_
#define PSKV_LANES_H_
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace pskv {

// The lane below's `v`; lane 0 gets `first`.
__device__ __forceinline__ float from_below(float v, float first) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, first), __builtin_bit_cast(int, v),
                                                               0x138 /* wave_shr:1 */, 0xf, 0xf, false));
}

// What the lane that CONTROL names has, 0 where there is none or the lane's row of 16 is not in ROWS.
template <int CONTROL, int ROWS>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CONTROL, ROWS, 0xf, false);
}

// One step of a sum along the lanes that starts anew where `starts` is set: what has been summed up to the lane that CONTROL names
// comes in, unless a start lies between.
template <int CONTROL, int ROWS>
__device__ __forceinline__ void sum_step(float& sum, uint32_t& starts) {
  const float up = __builtin_bit_cast(float, dpp<CONTROL, ROWS>(__builtin_bit_cast(uint32_t, sum)));
  const uint32_t there = dpp<CONTROL, ROWS>(starts);
  sum = starts ? sum : sum + up;
  starts |= there;
}
__device__ __forceinline__ float sum_along(float sum, uint32_t starts) {
  sum_step<0x111 /* row_shr:1 */, 0xf>(sum, starts);
  sum_step<0x112, 0xf>(sum, starts);
  sum_step<0x114, 0xf>(sum, starts);
  sum_step<0x118, 0xf>(sum, starts);
  sum_step<0x142 /* row_bcast:15 */, 0xa>(sum, starts);
  sum_step<0x143 /* row_bcast:31 */, 0xc>(sum, starts);
  return sum;
}

}  // namespace pskv
#endif  // PSKV_LANES_H_

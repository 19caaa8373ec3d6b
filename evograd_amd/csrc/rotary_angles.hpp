// The angles of rotary positions, shared by the kernels that turn heads by them.
#pragma once

#include "eg_common.hpp"

namespace eg {

// (amp cos, amp sign sin) of position * freq. A position of a long context times a frequency
// leaves few bits of an fp32 product behind its whole turns (at position 131072 an fp32 angle is
// off by 0.004), so the turns pos * freq / 2 pi are formed in fp64 and reduced there to an eighth
// of a turn; only that remainder is rounded to fp32 for the sine and cosine.
__device__ __forceinline__ float2 rotary_turn(double pos, double freq, float amp, float sign) {
  // explicit fma: the same bits wherever it is inlined
  const double f = freq * 0.15915494309189533577;
  const double rest = __builtin_fma(pos, f, -rint(pos * f)), quarter = rint(4.0 * rest);
  float s0, c0;
  sincospif(2.f * (float)__builtin_fma(-0.25, quarter, rest), &s0, &c0);
  const int n = (int)quarter & 3;  // s0, c0 turned by n quarters
  const float s1 = n & 1 ? c0 : s0, c1 = n & 1 ? s0 : c0;
  return make_float2(amp * ((n + 1) & 2 ? -c1 : c1), amp * sign * (n & 2 ? -s1 : s1));
}

__device__ __forceinline__ double rotary_position(const void* pos, int pos64, int64_t token) {
  return pos64 ? (double)((const int64_t*)pos)[token] : (double)((const int*)pos)[token];
}

}  // namespace eg

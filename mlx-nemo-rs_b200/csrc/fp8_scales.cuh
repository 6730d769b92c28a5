// fp8_scales.cuh -- the two scales of a 128-block's sum of code products.
#pragma once

#include <cfloat>

namespace nrp {

// Whether a product of scales is a normal number.
__device__ __forceinline__ bool scale_in_range(float s) {
  return (__float_as_uint(s) & 0x7fffffffu) - 0x00800000u < 0x7f000000u;
}

// Factors with which v * a * b is (v * p) * q, for a sum v of products of e4m3
// codes (0, or 2^-18 to 2^25 in magnitude).  The scales' product as one factor
// (p = 1) is right while it is a normal number; where it passes f32's range,
// v * a * b may still lie in it.  Returns whether p is another factor than 1.
// Above the range both scales are at least 1 in magnitude, and v times the smaller
// overflows only if all does; below it v times the larger, which is under 2^23,
// neither overflows nor loses digits that the result has.  A zero, infinite or NaN
// scale acts as in a * b.
__device__ __forceinline__ bool scale_factors(float a, float b, float& p, float& q) {
  p = 1.f;
  q = a * b;
  if (scale_in_range(q)) return false;
  const float x = fabsf(a), y = fabsf(b);
  if (!(x > 0.f && y > 0.f && x <= FLT_MAX && y <= FLT_MAX)) return false;
  const bool a_first = (fabsf(q) > 1.f) == (x < y);
  p = a_first ? a : b;
  q = a_first ? b : a;
  return true;
}

}  // namespace nrp

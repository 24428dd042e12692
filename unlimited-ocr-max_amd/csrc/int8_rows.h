// A head's row of 128 fp32 values as int8 and one scale (the weights' form per 128 values, tools/quantize_int8.py:54-70):
// the scale is the largest magnitude times the fp32 number next to 1 / 127, 1 for a row of zeros, and a value q stands for
// q * scale.  A row with a value that is not finite has the scale NaN, so that it stands for NaN.  The product and the
// division are IEEE's: the bits are those of the same steps anywhere.
#pragma once

#include "uocr_device.h"

namespace uocr {

namespace {

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
// bits: the row's largest magnitude, as abs_bits (which order as the magnitudes do, what is not finite above).
__device__ __forceinline__ float row_scale(uint32_t bits) {
  if (bits >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  const float s = __uint_as_float(bits) * (1.0f / 127.0f);
  return s == 0.0f ? 1.0f : s;
}
// x / scale rounded to the nearest whole number, ties to even, as a byte; 0 where the scale is NaN.
__device__ __forceinline__ uint32_t to_int8(float x, float scale) {
  const float q = fminf(fmaxf(__builtin_rintf(x / scale), -127.0f), 127.0f);
  return scale != scale ? 0u : (uint32_t)(int)q & 0xffu;
}
// Four of them.  Divisions take a dozen instructions each: the products with the reciprocal, off by 127 2^-22 at most, round
// to the same numbers but where they are that near to a tie (or none: a reciprocal that overflows), and then the wave divides.
__device__ __forceinline__ uint32_t to_int8x4(float x, float y, float z, float w, float scale) {
  const float r = __builtin_amdgcn_rcpf(scale);
  const float v[4] = {x * r, y * r, z * r, w * r};
  uint32_t q = 0;
  bool far = true;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float n = __builtin_rintf(v[e]);
    far = far && __builtin_fabsf(v[e] - n) < 0.4999f;
    q |= ((uint32_t)(int)n & 0xffu) << (8 * e);
  }
  if (__ballot(!far) == 0) return q;
  return to_int8(x, scale) | to_int8(y, scale) << 8 | to_int8(z, scale) << 16 | to_int8(w, scale) << 24;
}

}  // namespace

}  // namespace uocr

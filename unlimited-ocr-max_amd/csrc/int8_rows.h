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

}  // namespace

}  // namespace uocr

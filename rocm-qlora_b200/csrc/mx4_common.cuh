// mx4_common.cuh -- the microscaled 4-bit form: e2m1 codes, and scales that are
// powers of two, a byte e + 127 for 2^e, in the pieces of 128 rows x 128
// columns that the tensor cores take.
#pragma once

#include "linear_common.cuh"

namespace rq {

// The value of the low 4 bits of c: sign, 2 exponent bits, 1 mantissa bit.
__device__ __forceinline__ float e2m1_to_f32(int c) {
  const int e = (c >> 1) & 3, m = c & 1;
  const float v = e == 0 ? 0.5f * m : (float)((2 + m) << (e - 1)) * 0.5f;
  return (c & 8) ? -v : v;
}

// 2^(byte - base), NaN for byte 255.  byte - base is -127 at least and 127 at
// most, or the result is 0 (a scale 2^-128 or less of the largest).
__device__ __forceinline__ float pow2_scale(int byte, int base) {
  const int e = byte - base + 127;
  if (byte == 255) return __uint_as_float(0x7fc00000u);
  return __uint_as_float(e > 0 ? (uint32_t)e << 23 : e == 0 ? 0x00400000u : 0u);
}

// Place of the scale byte of row r, block b among scales of `tiles` pieces a row.
__device__ __forceinline__ int64_t mx4_scale_at(int64_t r, int b, int tiles) {
  return ((r / 128) * tiles + b / 4) * 512 + (r % 32) * 16 + (r % 128) / 32 * 4 + b % 4;
}

}  // namespace rq

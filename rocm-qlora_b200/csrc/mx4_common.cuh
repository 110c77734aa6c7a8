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

// A lane's 8 values at columns col .. col + 7, 0 past K.  VEC: whole 16-byte
// pieces, so all 8 exist or none does.
template <int DT, bool VEC>
__device__ __forceinline__ void m4_load(const typename DType<DT>::T* row, int col, int K, float (&v)[8]) {
  if constexpr (!VEC) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = col + i < K ? DType<DT>::to_f32(row[col + i]) : 0.0f;
  } else if constexpr (DT == RQ_F32) {
    const float4 z = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    *reinterpret_cast<float4*>(v) = col < K ? *reinterpret_cast<const float4*>(row + col) : z;
    *reinterpret_cast<float4*>(v + 4) = col < K ? *reinterpret_cast<const float4*>(row + col + 4) : z;
  } else {
    const uint4 w = col < K ? *reinterpret_cast<const uint4*>(row + col) : make_uint4(0u, 0u, 0u, 0u);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == RQ_BF16) {
        v[2 * i] = __uint_as_float(u[i] << 16);
        v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    }
  }
}

// Eight e2m1 codes (nearest, ties to even, saturating), the first in the low bits.
__device__ __forceinline__ uint32_t e2m1x8(const float (&v)[8], float by) {
  uint32_t w;
  asm("{\n .reg .b8 a, b, c, d;\n"
      " cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
      " cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
      " mov.b32 %0, {a, b, c, d};\n}\n"
      : "=r"(w)
      : "f"(v[0] * by), "f"(v[1] * by), "f"(v[2] * by), "f"(v[3] * by), "f"(v[4] * by), "f"(v[5] * by), "f"(v[6] * by),
        "f"(v[7] * by));
  return w;
}

// The scale byte of a block whose largest magnitude has these bits.
__device__ __forceinline__ uint32_t m4_scale(uint32_t top) {
  const uint32_t e = top >> 23;  // 127 + floor(log2 top), 0 below 2^-126
  return e == 255u ? 255u : e > 2u ? e - 2u : 0u;
}

// 2^(127 - byte), the factor that takes values to codes.
__device__ __forceinline__ float m4_factor(uint32_t byte) { return __uint_as_float((254u - min(byte, 253u)) << 23); }

}  // namespace rq

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

// A lane's values as they are in memory (16-bit types two to a word), at columns
// col .. col + W - 1, 0 past K.  ALIGN: bytes at which all pieces of a row lie, of
// which all values exist or none does; 0: none.
template <int DT, int W = 8> struct M4Raw { uint32_t w[DT == RQ_F32 ? W : W / 2]; };

template <int DT, int ALIGN, int W = 8>
__device__ __forceinline__ M4Raw<DT, W> m4_load(const typename DType<DT>::T* row, int col, int K) {
  M4Raw<DT, W> r = {};
  constexpr int words = DT == RQ_F32 ? W : W / 2;
  if constexpr (ALIGN == 32 && words == 8) {
    if (col < K) load32(row + col, r.w);
  } else if constexpr (ALIGN) {
    if (col < K) {
#pragma unroll
      for (int h = 0; h < words / 4; ++h)
        *reinterpret_cast<uint4*>(r.w + 4 * h) = reinterpret_cast<const uint4*>(row + col)[h];
    }
  } else {
    static_assert(W == 8, "");
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (DT == RQ_F32) {
        r.w[i] = col + i < K ? __float_as_uint(row[col + i]) : 0u;
      } else {
        const uint32_t v = col + i < K ? reinterpret_cast<const uint16_t*>(row)[col + i] : 0u;
        r.w[i / 2] |= v << (16 * (i & 1));
      }
    }
  }
  return r;
}

template <int DT, int W>
__device__ __forceinline__ void m4_values(const M4Raw<DT, W>& r, float (&v)[W]) {
#pragma unroll
  for (int i = 0; i < (DT == RQ_F32 ? W : W / 2); ++i) {
    if constexpr (DT == RQ_F32) {
      v[i] = __uint_as_float(r.w[i]);
    } else if constexpr (DT == RQ_BF16) {
      v[2 * i] = __uint_as_float(r.w[i] << 16);
      v[2 * i + 1] = __uint_as_float(r.w[i] & 0xffff0000u);
    } else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r.w[i]));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
}

// Largest magnitudes of blocks, of which each of 32 / W neighbouring lanes has W
// values, as fp32 bits, in which an infinity or NaN is the largest.  16-bit magnitudes are
// compared two at a time, and two blocks share a word on their way.
template <int DT, int W, int N>
__device__ __forceinline__ void m4_top(const M4Raw<DT, W> (&r)[N], uint32_t (&top)[N]) {
  if constexpr (DT == RQ_F32) {
    static_assert(DT != RQ_F32 || W == 8, "");
#pragma unroll
    for (int n = 0; n < N; ++n) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max(m, r[n].w[i] & 0x7fffffffu);
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
      top[n] = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    }
  } else {
    uint32_t m[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      m[n] = 0;
#pragma unroll
      for (int i = 0; i < W / 2; ++i) m[n] = __vmaxs2(m[n], r[n].w[i] & 0x7fff7fffu);
    }
#pragma unroll
    for (int n = 0; n < N; n += 2) {
      const uint32_t other = n + 1 < N ? m[n + 1 < N ? n + 1 : n] : 0u;
      uint32_t both = __vmaxs2(__byte_perm(m[n], other, 0x5410), __byte_perm(m[n], other, 0x7632));
      both = __vmaxs2(both, __shfl_xor_sync(0xffffffffu, both, 1));
      if constexpr (W == 8) both = __vmaxs2(both, __shfl_xor_sync(0xffffffffu, both, 2));
#pragma unroll
      for (int h = 0; h < 2 && n + h < N; ++h) {
        const uint16_t bits = (uint16_t)(h ? both >> 16 : both);
        top[n + h] = __float_as_uint(DType<DT>::to_f32(*reinterpret_cast<const typename DType<DT>::T*>(&bits)));
      }
    }
  }
}

// Eight e2m1 codes (nearest, ties to even, saturating), the first in the low bits.
__device__ __forceinline__ uint32_t e2m1x8(const float* v, float by) {
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

// act8.cu -- activations kept in 8 bits between forward and backward.
//
// Format: a row of K values is cut into blocks of 128 (the last one short).
// A block keeps scale = max|x| / 127 (fp32) and codes rint(x * (127 / max|x|))
// (int8); the code rows are padded with zeros to whole blocks, so every row
// starts on a 128-byte boundary.  A block whose largest magnitude is below
// 2^-100 (where 127 / max|x| could overflow) is stored as zeros; one that
// holds an infinity or a NaN keeps scale NaN, so it stays visible.
//
// Everything here is one pass over the data.  16 lanes hold a block (8 values
// a lane: one 16-byte load of a 16-bit type), so the block's maximum is four
// shuffles.  Measured (bf16, 8192 x 11008): swiglu8 forward with three copies
// 149 us, 5.4 TB/s (issue bound, 76 % of the slots: the encoding), backward
// 115 us, 6.3 TB/s, and unpack 49 us, 5.5 TB/s (HBM); pack of 8192 x 4096 21
// us, 4.7 TB/s; fp32, 4096 x 11008, forward 108 us, 6.3 TB/s, backward 94, 6.7.
#include <cuda_runtime.h>

#include "linear_common.cuh"

namespace rq {

constexpr int kA8Block = 128, kA8Threads = 256, kA8Lanes = 16;
constexpr int kA8PerCta = kA8Threads / kA8Lanes;  // blocks a CTA holds at once

// Where lane l of a block's 16 has its 8 values: side by side where rows are
// 16-byte aligned (VEC: one load of a 16-bit type), else every 16th, so that
// the lanes' single values are side by side.
template <bool VEC>
__device__ __forceinline__ int lane_at(int i) {
  const int l = threadIdx.x % kA8Lanes;
  return VEC ? l * 8 + i : i * kA8Lanes + l;
}

// Division of n < 2^31 by a number known at launch: (n * mul) >> shift.
struct Divide {
  uint32_t mul;
  int shift;
  uint32_t by;
};
static Divide divide_by(uint32_t d) {
  int s = 0;
  while ((1ull << s) < d) ++s;
  return Divide{(uint32_t)((1ull << (31 + s)) / d + 1), 31 + s, d};
}

// A lane's block: its number, row, first column and how many columns of the
// row are left from there (0 or less: none).
struct Place8 {
  int64_t row, block;
  int col, left;
};

template <bool VEC>
__device__ __forceinline__ bool place8(Place8& p, uint32_t blocks, int K, const Divide& nb) {
  const uint32_t at = blockIdx.x * kA8PerCta + threadIdx.x / kA8Lanes;
  const bool any = at < blocks;
  p.block = any ? at : 0;
  const uint32_t row = (uint32_t)(((uint64_t)p.block * nb.mul) >> nb.shift);
  p.row = row;
  p.col = (int)((uint32_t)p.block - row * nb.by) * kA8Block;
  p.left = any ? K - p.col : 0;
  return any;
}

// A lane's 8 values as they are in memory: 16-bit types packed in 4 words.
template <int DT> struct Raw8 { uint32_t w[DT == RQ_F32 ? 8 : 4]; };

// VEC: whole 16-byte pieces (the row's length is a multiple of a piece).
template <int DT, bool VEC>
__device__ __forceinline__ Raw8<DT> load8(const typename DType<DT>::T* block, int left) {
  Raw8<DT> r = {};
  if constexpr (VEC) {
    constexpr int N = DT == RQ_F32 ? 2 : 1;
#pragma unroll
    for (int h = 0; h < N; ++h) {
      const int at = lane_at<true>(0) + h * 4;
      if (at < left) *reinterpret_cast<uint4*>(r.w + 4 * h) = *reinterpret_cast<const uint4*>(block + at);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int at = lane_at<false>(i);
      if constexpr (DT == RQ_F32) {
        r.w[i] = at < left ? __float_as_uint(block[at]) : 0u;
      } else {
        const uint32_t v = at < left ? reinterpret_cast<const uint16_t*>(block)[at] : 0u;
        r.w[i / 2] |= v << (16 * (i & 1));
      }
    }
  }
  return r;
}

template <int DT, bool VEC>
__device__ __forceinline__ void store8(typename DType<DT>::T* block, int left, const Raw8<DT>& r) {
  if constexpr (VEC) {
    constexpr int N = DT == RQ_F32 ? 2 : 1;
#pragma unroll
    for (int h = 0; h < N; ++h) {
      const int at = lane_at<true>(0) + h * 4;
      if (at < left) *reinterpret_cast<uint4*>(block + at) = *reinterpret_cast<const uint4*>(r.w + 4 * h);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int at = lane_at<false>(i);
      if (at >= left) continue;
      if constexpr (DT == RQ_F32) block[at] = __uint_as_float(r.w[i]);
      else reinterpret_cast<uint16_t*>(block)[at] = (uint16_t)(r.w[i / 2] >> (16 * (i & 1)));
    }
  }
}

template <int DT>
__device__ __forceinline__ void to_floats(const Raw8<DT>& r, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < (DT == RQ_F32 ? 8 : 4); ++i) {
    if constexpr (DT == RQ_F32) v[i] = __uint_as_float(r.w[i]);
    else if constexpr (DT == RQ_BF16) v[2 * i] = __uint_as_float(r.w[i] << 16), v[2 * i + 1] = __uint_as_float(r.w[i] & 0xffff0000u);
    else {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r.w[i]));
      v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
  }
}

template <int DT>
__device__ __forceinline__ Raw8<DT> from_floats(const float (&v)[8]) {
  Raw8<DT> r;
#pragma unroll
  for (int i = 0; i < (DT == RQ_F32 ? 8 : 4); ++i) {
    if constexpr (DT == RQ_F32) {
      r.w[i] = __float_as_uint(v[i]);
    } else if constexpr (DT == RQ_BF16) {
      const __nv_bfloat162 q = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      r.w[i] = *reinterpret_cast<const uint32_t*>(&q);
    } else {
      const __half2 q = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
      r.w[i] = *reinterpret_cast<const uint32_t*>(&q);
    }
  }
  return r;
}

// The largest magnitudes of the blocks of N tensors, as fp32.  Magnitudes are
// compared as bit patterns, in which an infinity or NaN is the largest; of
// 16-bit types two at a time, and two tensors share a word on their way
// through the lanes.
template <int DT, int N>
__device__ __forceinline__ void block_max(const Raw8<DT> (&r)[N], float (&most)[N]) {
  if constexpr (DT == RQ_F32) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      unsigned top = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, r[n].w[i] & 0x7fffffffu);
#pragma unroll
      for (int o = kA8Lanes / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      most[n] = __uint_as_float(top);
    }
  } else {
    unsigned top[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const unsigned m = __vmaxs2(__vmaxs2(r[n].w[0] & 0x7fff7fffu, r[n].w[1] & 0x7fff7fffu),
                                  __vmaxs2(r[n].w[2] & 0x7fff7fffu, r[n].w[3] & 0x7fff7fffu));
      top[n] = max(m & 0xffffu, m >> 16);
    }
#pragma unroll
    for (int n = 0; n < N; n += 2) {
      unsigned m = top[n] | (n + 1 < N ? top[n + 1] << 16 : 0u);
#pragma unroll
      for (int o = kA8Lanes / 2; o > 0; o >>= 1) m = __vmaxs2(m, __shfl_xor_sync(0xffffffffu, m, o));
#pragma unroll
      for (int h = 0; h < 2 && n + h < N; ++h) {
        const uint16_t bits = (uint16_t)(h ? m >> 16 : m);
        most[n + h] = DType<DT>::to_f32(*reinterpret_cast<const typename DType<DT>::T*>(&bits));
      }
    }
  }
}

// Codes and scales of the blocks of N tensors, copy n at codes + n * plane
// blocks.  Every block needs two divisions; the lanes share them out: lane n
// has max / 127, lane N + n has 127 / max, and passes it on.  Adding 1.5 * 2^23
// rounds a product to the nearest whole (ties to even) and leaves the code in
// the low byte: two fp32 operations instead of a conversion, whose pipe is
// eight times narrower.
template <int DT, bool VEC, int N>
__device__ __forceinline__ void encode8(const Raw8<DT> (&r)[N], const Place8& p, bool any, int64_t plane,
                                        int8_t* __restrict__ codes, float* __restrict__ scales) {
  const int l = threadIdx.x % kA8Lanes;
  float most[N];
  block_max<DT, N>(r, most);
  float mine = most[0];
#pragma unroll
  for (int n = 1; n < N; ++n) mine = l == n || l == N + n ? most[n] : mine;
  const bool live = mine >= 0x1p-100f && mine < INFINITY;
  const float quotient = ieee_div(l < N ? mine : 127.0f, l < N ? 127.0f : (live ? mine : 1.0f));
  if (any && l < N) scales[l * plane + p.block] = live ? quotient : (mine < INFINITY ? 0.0f : __uint_as_float(0x7fc00000u));
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const float by = __shfl_sync(0xffffffffu, quotient, N + n, kA8Lanes);
    const bool on = most[n] >= 0x1p-100f && most[n] < INFINITY;
    float v[8];
    to_floats<DT>(r[n], v);
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(__fadd_rn(__fmul_rn(v[i], by), 12582912.0f));
    if (!any) continue;
    int8_t* to = codes + (n * plane + p.block) * kA8Block;
    if constexpr (VEC) {
      const uint32_t a = __byte_perm(__byte_perm(w[0], w[1], 0x0040), __byte_perm(w[2], w[3], 0x0040), 0x5410);
      const uint32_t b = __byte_perm(__byte_perm(w[4], w[5], 0x0040), __byte_perm(w[6], w[7], 0x0040), 0x5410);
      *reinterpret_cast<uint2*>(to + lane_at<true>(0)) = on ? make_uint2(a, b) : make_uint2(0u, 0u);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) to[lane_at<false>(i)] = on ? (int8_t)w[i] : (int8_t)0;
    }
  }
}

template <bool VEC>
__device__ __forceinline__ void decode8(const int8_t* __restrict__ codes, const float* __restrict__ scales,
                                        int64_t block, float (&v)[8]) {
  const float scale = scales[block];
  const int8_t* from = codes + block * kA8Block;
  if constexpr (VEC) {
    const uint2 q = *reinterpret_cast<const uint2*>(from + lane_at<true>(0));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)(int)(int8_t)((i < 4 ? q.x : q.y) >> (8 * (i & 3))) * scale;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)(int)from[lane_at<false>(i)] * scale;
  }
}

template <int DT, bool VEC>
__global__ void __launch_bounds__(kA8Threads) act8_pack_k(const void* __restrict__ x, int64_t ld, uint32_t blocks,
                                                          int K, Divide nb, int8_t* __restrict__ codes,
                                                          float* __restrict__ scales) {
  grid_begin();
  using T = typename DType<DT>::T;
  Place8 p;
  const bool any = place8<VEC>(p, blocks, K, nb);
  const Raw8<DT> r[1] = {load8<DT, VEC>(static_cast<const T*>(x) + p.row * ld + p.col, p.left)};
  encode8<DT, VEC, 1>(r, p, any, blocks, codes, scales);
}

template <int DT, bool VEC>
__global__ void __launch_bounds__(kA8Threads) act8_unpack_k(const int8_t* __restrict__ codes,
                                                            const float* __restrict__ scales, uint32_t blocks, int K,
                                                            Divide nb, void* __restrict__ out) {
  grid_begin();
  using T = typename DType<DT>::T;
  Place8 p;
  if (!place8<VEC>(p, blocks, K, nb)) return;
  float v[8];
  decode8<VEC>(codes, scales, p.block, v);
  store8<DT, VEC>(static_cast<T*>(out) + p.row * K + p.col, p.left, from_floats<DT>(v));
}

// 1 / (1 + e^-g).  For 16-bit tensors the approximate exponential and
// reciprocal, which err by 2^-22 of their value, and by the rounding of
// g log2(e) in the exponent's argument (|g| 2^-24): far below a 16-bit
// result's rounding.  They have no denormal results, but a bf16 product of a
// gate down to -96 and such a sigmoid can be a normal number: both work 2^24
// times up, in 2^-24 + e^-g 2^-24, and one multiplication takes that back.
// 32-bit tensors take the accurate functions.
template <int DT>
__device__ __forceinline__ float sigmoid(float g) {
  if constexpr (DT == RQ_F32) return ieee_div(1.0f, 1.0f + expf(-g));
  constexpr float up = DT == RQ_BF16 ? 24.0f : 0.0f, down = DT == RQ_BF16 ? 0x1p-24f : 1.0f;
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fmaf(g, -1.4426950408889634f, -up)));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(down + e));
  return r * down;
}

// h = silu(g) u, with g and u (and h as it was rounded) packed in the same pass.
// Six CTAs an SM, 40 registers (16-bit 149 us; 155 with the 44 that it would
// take), fewer where fp32 values need more.
template <int DT, bool VEC, int COPIES>
__global__ void __launch_bounds__(kA8Threads, DT != RQ_F32 || (VEC && COPIES == 2) ? 6 : VEC ? 5 : 4)
    swiglu8_forward_k(const void* __restrict__ g, int64_t ldg, const void* __restrict__ u, int64_t ldu,
                      uint32_t blocks, int K, Divide nb, void* __restrict__ h, int8_t* __restrict__ codes,
                      float* __restrict__ scales) {
  grid_begin();
  using T = typename DType<DT>::T;
  Place8 p;
  const bool any = place8<VEC>(p, blocks, K, nb);
  Raw8<DT> r[COPIES];
  r[0] = load8<DT, VEC>(static_cast<const T*>(g) + p.row * ldg + p.col, p.left);
  r[1] = load8<DT, VEC>(static_cast<const T*>(u) + p.row * ldu + p.col, p.left);
  float a[8], b[8];
  to_floats<DT>(r[0], a);
  to_floats<DT>(r[1], b);
#pragma unroll
  for (int i = 0; i < 8; ++i) b[i] = a[i] * sigmoid<DT>(a[i]) * b[i];
  const Raw8<DT> y = from_floats<DT>(b);
  store8<DT, VEC>(static_cast<T*>(h) + p.row * K + p.col, p.left, y);
  if constexpr (COPIES == 3) r[2] = y;
  encode8<DT, VEC, COPIES>(r, p, any, blocks, codes, scales);
}

// With p = 1 / (1 + e^-g): dg = dh u p (1 + g (1 - p)), du = dh g p.
template <int DT, bool VEC>
__global__ void __launch_bounds__(kA8Threads) swiglu8_backward_k(const void* __restrict__ dh, int64_t ldh,
                                                                 const int8_t* __restrict__ codes,
                                                                 const float* __restrict__ scales, uint32_t blocks,
                                                                 int K, Divide nb, void* __restrict__ dg,
                                                                 void* __restrict__ du) {
  grid_begin();
  using T = typename DType<DT>::T;
  Place8 p;
  if (!place8<VEC>(p, blocks, K, nb)) return;
  float a[8], b[8], d[8];
  to_floats<DT>(load8<DT, VEC>(static_cast<const T*>(dh) + p.row * ldh + p.col, p.left), d);
  decode8<VEC>(codes, scales, p.block, a);
  decode8<VEC>(codes, scales, (int64_t)blocks + p.block, b);
  float x[8], y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float e = sigmoid<DT>(a[i]);
    x[i] = d[i] * b[i] * e * (1.0f + a[i] * (1.0f - e));
    y[i] = d[i] * a[i] * e;
  }
  store8<DT, VEC>(static_cast<T*>(dg) + p.row * K + p.col, p.left, from_floats<DT>(x));
  store8<DT, VEC>(static_cast<T*>(du) + p.row * K + p.col, p.left, from_floats<DT>(y));
}

// Rows of K columns that are made of whole aligned 16-byte pieces.
static bool rows16(const void* p, int64_t ld, int64_t K, int dt) {
  const int e = dt == RQ_F32 ? 4 : 2;
  return (uintptr_t)p % 16 == 0 && ld * e % 16 == 0 && K * e % 16 == 0;
}

static uint32_t a8_row_blocks(int64_t K) { return (uint32_t)((K + kA8Block - 1) / kA8Block); }

#define RQ_A8_LAUNCH(kern, vec, ...)                                                                         \
  do {                                                                                                       \
    const unsigned grid = (blocks + kA8PerCta - 1) / kA8PerCta;                                              \
    auto* k = dt == RQ_F32 ? ((vec) ? kern<RQ_F32, true> : kern<RQ_F32, false>)                              \
              : dt == RQ_BF16 ? ((vec) ? kern<RQ_BF16, true> : kern<RQ_BF16, false>)                         \
                              : ((vec) ? kern<RQ_F16, true> : kern<RQ_F16, false>);                          \
    return launch_dependent(k, grid, kA8Threads, st, __VA_ARGS__);                                           \
  } while (0)

int act8_pack(const void* x, int dt, int64_t ld, int64_t M, int64_t K, int8_t* codes, float* scales, cudaStream_t st) {
  const Divide nb = divide_by(a8_row_blocks(K));
  const uint32_t blocks = (uint32_t)M * nb.by;
  RQ_A8_LAUNCH(act8_pack_k, rows16(x, ld, K, dt), x, ld, blocks, (int)K, nb, codes, scales);
}

int act8_unpack(const int8_t* codes, const float* scales, int64_t M, int64_t K, void* out, int dt, cudaStream_t st) {
  const Divide nb = divide_by(a8_row_blocks(K));
  const uint32_t blocks = (uint32_t)M * nb.by;
  RQ_A8_LAUNCH(act8_unpack_k, rows16(out, K, K, dt), codes, scales, blocks, (int)K, nb, out);
}

template <int DT, bool VEC>
static int launch_swiglu8(const void* g, int64_t ldg, const void* u, int64_t ldu, uint32_t blocks, int K,
                           const Divide& nb, void* h, int8_t* codes, float* scales, int copies, cudaStream_t st) {
  auto* kern = copies == 3 ? swiglu8_forward_k<DT, VEC, 3> : swiglu8_forward_k<DT, VEC, 2>;
  return launch_dependent(kern, (blocks + kA8PerCta - 1) / kA8PerCta, kA8Threads, st, g, ldg, u, ldu, blocks, K, nb, h,
                          codes, scales);
}

int swiglu8_forward(const void* g, int64_t ldg, const void* u, int64_t ldu, int dt, int64_t M, int64_t K, void* h,
                    int8_t* codes, float* scales, int copies, cudaStream_t st) {
  const Divide nb = divide_by(a8_row_blocks(K));
  const uint32_t blocks = (uint32_t)M * nb.by;
  const bool vec = rows16(g, ldg, K, dt) && rows16(u, ldu, K, dt) && rows16(h, K, K, dt);
  auto* launch = dt == RQ_F32 ? (vec ? launch_swiglu8<RQ_F32, true> : launch_swiglu8<RQ_F32, false>)
                 : dt == RQ_BF16 ? (vec ? launch_swiglu8<RQ_BF16, true> : launch_swiglu8<RQ_BF16, false>)
                                 : (vec ? launch_swiglu8<RQ_F16, true> : launch_swiglu8<RQ_F16, false>);
  return launch(g, ldg, u, ldu, blocks, (int)K, nb, h, codes, scales, copies, st);
}

int swiglu8_backward(const void* dh, int64_t ldh, int dt, int64_t M, int64_t K, const int8_t* codes,
                     const float* scales, void* dg, void* du, cudaStream_t st) {
  const Divide nb = divide_by(a8_row_blocks(K));
  const uint32_t blocks = (uint32_t)M * nb.by;
  const bool vec = rows16(dh, ldh, K, dt) && rows16(dg, K, K, dt) && rows16(du, K, K, dt);
  RQ_A8_LAUNCH(swiglu8_backward_k, vec, dh, ldh, codes, scales, blocks, (int)K, nb, dg, du);
}

}  // namespace rq

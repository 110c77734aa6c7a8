// act8.cu -- activations kept in 8 bits between forward and backward.
//
// Format: a row of K values is cut into blocks of 128 (the last one short).
// A block keeps scale = max|x| / 127 (fp32) and codes rint(x * (127 / max|x|))
// (int8); the code rows are padded with zeros to whole blocks, so every row
// starts on a 128-byte boundary.  A block whose largest magnitude is below
// 2^-100 (where 127 / max|x| could overflow) is stored as zeros; one that
// holds an infinity or a NaN keeps scale NaN, so it stays visible.
//
// Everything here is one pass over the data, bound by HBM.  16 lanes hold a
// block (8 values a lane: one 16-byte load of a 16-bit type), so the block's
// maximum is four shuffles.
#include <cuda_runtime.h>

#include "linear_common.cuh"

namespace rq {

constexpr int kA8Block = 128, kA8Threads = 256, kA8Lanes = 16;
constexpr int kA8PerCta = kA8Threads / kA8Lanes;  // blocks a CTA holds at once

template <int DT, bool VEC>
__device__ __forceinline__ void load8(const typename DType<DT>::T* p, int n, float (&v)[8]) {
  if (VEC && n == 8) {
    if constexpr (DT == RQ_F32) {
      const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
      const uint4 q = *reinterpret_cast<const uint4*>(p);
      const typename DType<DT>::T* e = reinterpret_cast<const typename DType<DT>::T*>(&q);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = DType<DT>::to_f32(e[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? DType<DT>::to_f32(p[i]) : 0.0f;
  }
}

template <int DT, bool VEC>
__device__ __forceinline__ void store8(typename DType<DT>::T* p, int n, const float (&v)[8]) {
  if (VEC && n == 8) {
    if constexpr (DT == RQ_F32) {
      reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      *reinterpret_cast<uint4*>(p) =
          make_uint4(pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3]), pack2<DT>(v[4], v[5]), pack2<DT>(v[6], v[7]));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = DType<DT>::from_f32(v[i]);
  }
}

// The block's scale and this lane's 8 codes.  The maximum is taken over the
// magnitudes' bit patterns, in which an infinity or NaN is the largest.
// Adding 1.5 * 2^23 rounds the product to the nearest whole (ties to even) and
// leaves the code in the low byte: two fp32 operations instead of a
// conversion, whose pipe is eight times narrower.
__device__ __forceinline__ uint2 encode8(const float (&v)[8], float* scale) {
  unsigned top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
#pragma unroll
  for (int o = kA8Lanes / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float most = __uint_as_float(top);
  const bool live = top < 0x7f800000u && most >= 0x1p-100f;
  *scale = live ? ieee_div(most, 127.0f) : (top < 0x7f800000u ? 0.0f : __uint_as_float(0x7fc00000u));
  const float by = ieee_div(127.0f, live ? most : 1.0f);
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(__fadd_rn(__fmul_rn(v[i], by), 12582912.0f));
  const uint32_t a = __byte_perm(__byte_perm(w[0], w[1], 0x0040), __byte_perm(w[2], w[3], 0x0040), 0x5410);
  const uint32_t b = __byte_perm(__byte_perm(w[4], w[5], 0x0040), __byte_perm(w[6], w[7], 0x0040), 0x5410);
  return live ? make_uint2(a, b) : make_uint2(0u, 0u);
}

__device__ __forceinline__ void decode8(uint2 q, float scale, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t w = i < 4 ? q.x : q.y;
    v[i] = (float)(int)(int8_t)(w >> (8 * (i & 3))) * scale;
  }
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

// Where a lane's 8 values are: row, column, how many of them exist.
struct Place8 {
  int64_t row, block;
  int col, n;
  bool any;
};

__device__ __forceinline__ Place8 place8(uint32_t at, uint32_t blocks, int K, const Divide& nb) {
  Place8 p;
  p.any = at < blocks;
  at = p.any ? at : 0;
  const uint32_t row = (uint32_t)(((uint64_t)at * nb.mul) >> nb.shift);
  p.row = row;
  p.block = at;
  p.col = (int)(at - row * nb.by) * kA8Block + (threadIdx.x % kA8Lanes) * 8;
  p.n = p.any ? max(0, min(8, K - p.col)) : 0;
  return p;
}

template <int DT, bool VEC>
__global__ void __launch_bounds__(kA8Threads) act8_pack_k(const void* __restrict__ x, int64_t ld, uint32_t blocks, int K,
                                                          Divide nb, int8_t* __restrict__ codes,
                                                          float* __restrict__ scales) {
  using T = typename DType<DT>::T;
  const Place8 p = place8(blockIdx.x * kA8PerCta + threadIdx.x / kA8Lanes, blocks, K, nb);
  float v[8], s;
  load8<DT, VEC>(static_cast<const T*>(x) + p.row * ld + p.col, p.n, v);
  const uint2 q = encode8(v, &s);
  if (!p.any) return;
  *reinterpret_cast<uint2*>(codes + p.block * kA8Block + (threadIdx.x % kA8Lanes) * 8) = q;
  if (threadIdx.x % kA8Lanes == 0) scales[p.block] = s;
}

template <int DT, bool VEC>
__global__ void __launch_bounds__(kA8Threads) act8_unpack_k(const int8_t* __restrict__ codes,
                                                            const float* __restrict__ scales, uint32_t blocks, int K, Divide nb,
                                                            void* __restrict__ out) {
  using T = typename DType<DT>::T;
  const Place8 p = place8(blockIdx.x * kA8PerCta + threadIdx.x / kA8Lanes, blocks, K, nb);
  if (!p.any) return;
  float v[8];
  decode8(*reinterpret_cast<const uint2*>(codes + p.block * kA8Block + (threadIdx.x % kA8Lanes) * 8), scales[p.block],
          v);
  store8<DT, VEC>(static_cast<T*>(out) + p.row * K + p.col, p.n, v);
}

// 1 / (1 + e^-g).  The fast exponential and reciprocal err by a few units in
// the last place of 32 bits, far below a 16-bit result's rounding; 32-bit
// tensors take the accurate ones.
template <int DT>
__device__ __forceinline__ float sigmoid(float g) {
  if constexpr (DT == RQ_F32) return ieee_div(1.0f, 1.0f + expf(-g));
  return __fdividef(1.0f, 1.0f + __expf(-g));
}

// h = silu(g) u, with g and u (and h as it was rounded) packed in the same pass.
template <int DT, bool VEC>
__global__ void __launch_bounds__(kA8Threads) swiglu8_forward_k(const void* __restrict__ g, int64_t ldg,
                                                                const void* __restrict__ u, int64_t ldu, uint32_t blocks, int K, Divide nb, void* __restrict__ h,
                                                                int8_t* __restrict__ codes, float* __restrict__ scales,
                                                                int copies) {
  using T = typename DType<DT>::T;
  const Place8 p = place8(blockIdx.x * kA8PerCta + threadIdx.x / kA8Lanes, blocks, K, nb);
  const int lane8 = (threadIdx.x % kA8Lanes) * 8;
  const int64_t plane = blocks;  // of one packed copy
  float a[8], b[8], s;
  load8<DT, VEC>(static_cast<const T*>(g) + p.row * ldg + p.col, p.n, a);
  load8<DT, VEC>(static_cast<const T*>(u) + p.row * ldu + p.col, p.n, b);
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = round_to<DT>(a[i] * sigmoid<DT>(a[i]) * b[i]);
  uint2 q = encode8(a, &s);
  if (p.any) {
    *reinterpret_cast<uint2*>(codes + p.block * kA8Block + lane8) = q;
    if (lane8 == 0) scales[p.block] = s;
  }
  q = encode8(b, &s);
  if (p.any) {
    *reinterpret_cast<uint2*>(codes + (plane + p.block) * kA8Block + lane8) = q;
    if (lane8 == 0) scales[plane + p.block] = s;
    store8<DT, VEC>(static_cast<T*>(h) + p.row * K + p.col, p.n, y);
  }
  if (copies < 3) return;
  q = encode8(y, &s);
  if (p.any) {
    *reinterpret_cast<uint2*>(codes + (2 * plane + p.block) * kA8Block + lane8) = q;
    if (lane8 == 0) scales[2 * plane + p.block] = s;
  }
}

// With p = 1 / (1 + e^-g): dg = dh u p (1 + g (1 - p)), du = dh g p.
template <int DT, bool VEC>
__global__ void __launch_bounds__(kA8Threads) swiglu8_backward_k(const void* __restrict__ dh, int64_t ldh,
                                                                 const int8_t* __restrict__ codes,
                                                                 const float* __restrict__ scales, uint32_t blocks, int K, Divide nb, void* __restrict__ dg, void* __restrict__ du) {
  using T = typename DType<DT>::T;
  const Place8 p = place8(blockIdx.x * kA8PerCta + threadIdx.x / kA8Lanes, blocks, K, nb);
  if (!p.any) return;
  const int lane8 = (threadIdx.x % kA8Lanes) * 8;
  const int64_t plane = blocks;
  float a[8], b[8], d[8];
  load8<DT, VEC>(static_cast<const T*>(dh) + p.row * ldh + p.col, p.n, d);
  decode8(*reinterpret_cast<const uint2*>(codes + p.block * kA8Block + lane8), scales[p.block], a);
  decode8(*reinterpret_cast<const uint2*>(codes + (plane + p.block) * kA8Block + lane8), scales[plane + p.block], b);
  float x[8], y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float e = sigmoid<DT>(a[i]);
    x[i] = d[i] * b[i] * e * (1.0f + a[i] * (1.0f - e));
    y[i] = d[i] * a[i] * e;
  }
  store8<DT, VEC>(static_cast<T*>(dg) + p.row * K + p.col, p.n, x);
  store8<DT, VEC>(static_cast<T*>(du) + p.row * K + p.col, p.n, y);
}

static bool rows16(const void* p, int64_t ld, int dt) {
  return (uintptr_t)p % 16 == 0 && ld * (dt == RQ_F32 ? 4 : 2) % 16 == 0;
}

static uint32_t a8_row_blocks(int64_t K) { return (uint32_t)((K + kA8Block - 1) / kA8Block); }

#define RQ_A8_LAUNCH(kern, vec, ...)                                                              \
  do {                                                                                            \
    const unsigned grid = (blocks + kA8PerCta - 1) / kA8PerCta;                                   \
    if (vec) {                                                                                    \
      if (dt == RQ_F32) kern<RQ_F32, true><<<grid, kA8Threads, 0, st>>>(__VA_ARGS__);             \
      else if (dt == RQ_BF16) kern<RQ_BF16, true><<<grid, kA8Threads, 0, st>>>(__VA_ARGS__);      \
      else kern<RQ_F16, true><<<grid, kA8Threads, 0, st>>>(__VA_ARGS__);                          \
    } else {                                                                                      \
      if (dt == RQ_F32) kern<RQ_F32, false><<<grid, kA8Threads, 0, st>>>(__VA_ARGS__);            \
      else if (dt == RQ_BF16) kern<RQ_BF16, false><<<grid, kA8Threads, 0, st>>>(__VA_ARGS__);     \
      else kern<RQ_F16, false><<<grid, kA8Threads, 0, st>>>(__VA_ARGS__);                         \
    }                                                                                             \
    return check_launch();                                                                        \
  } while (0)

int act8_pack(const void* x, int dt, int64_t ld, int64_t M, int64_t K, int8_t* codes, float* scales, cudaStream_t st) {
  const Divide nb = divide_by(a8_row_blocks(K));
  const uint32_t blocks = (uint32_t)M * nb.by;
  RQ_A8_LAUNCH(act8_pack_k, rows16(x, ld, dt), x, ld, blocks, (int)K, nb, codes, scales);
}

int act8_unpack(const int8_t* codes, const float* scales, int64_t M, int64_t K, void* out, int dt, cudaStream_t st) {
  const Divide nb = divide_by(a8_row_blocks(K));
  const uint32_t blocks = (uint32_t)M * nb.by;
  RQ_A8_LAUNCH(act8_unpack_k, rows16(out, K, dt), codes, scales, blocks, (int)K, nb, out);
}

int swiglu8_forward(const void* g, int64_t ldg, const void* u, int64_t ldu, int dt, int64_t M, int64_t K, void* h,
                    int8_t* codes, float* scales, int copies, cudaStream_t st) {
  const Divide nb = divide_by(a8_row_blocks(K));
  const uint32_t blocks = (uint32_t)M * nb.by;
  const bool vec = rows16(g, ldg, dt) && rows16(u, ldu, dt) && rows16(h, K, dt);
  RQ_A8_LAUNCH(swiglu8_forward_k, vec, g, ldg, u, ldu, blocks, (int)K, nb, h, codes, scales, copies);
}

int swiglu8_backward(const void* dh, int64_t ldh, int dt, int64_t M, int64_t K, const int8_t* codes,
                     const float* scales, void* dg, void* du, cudaStream_t st) {
  const Divide nb = divide_by(a8_row_blocks(K));
  const uint32_t blocks = (uint32_t)M * nb.by;
  const bool vec = rows16(dh, ldh, dt) && rows16(dg, K, dt) && rows16(du, K, dt);
  RQ_A8_LAUNCH(swiglu8_backward_k, vec, dh, ldh, codes, scales, blocks, (int)K, nb, dg, du);
}

}  // namespace rq

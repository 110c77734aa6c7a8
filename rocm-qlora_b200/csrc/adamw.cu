// adamw.cu -- an AdamW step over many tensors in one launch, with the gradient
// norm that clips it, and moments held in 32 or in 8 bits.
//
//   g = c grad                       c = min(1, max_norm / (norm + 1e-6)), or 1
//   m = b1 m + (1 - b1) g            v = b2 v + (1 - b2) g g
//   p = p (1 - lr wd) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// A tensor's values are cut into blocks of 256 (the last one short); the
// moments of all tensors lie in one arena of whole blocks.  A warp takes a
// block, 8 values a lane.  One launch, and one before it, whose programmatic
// dependent it is, for the norm's partial sums where it clips: every CTA adds
// those up for itself, and the last one to end counts the tensors' steps.
//
// Moments in 8 bits, per block:
//   m          e4m3 codes of m (448 / max|m|), scale max|m| / 448
//   sqrt(v)    codes of 4 exponent and 4 mantissa bits (the whole numbers up to
//              31, then 16 steps to a power of two, up to 31 2^14) of
//              r (507904 / max r), scale max r / 507904; r > 0 never becomes 0,
//              which would make the next quotient unbounded.
// The root has half of v's range, and no sign bit is spent on it.  Maxima
// below 2^-100 are stored as zeros, an infinity or NaN makes the scale NaN.
// The parameters are updated with the moments as they were before rounding.
// Products and sums of the moments are rounded one by one (no fused
// multiply-add), so that a code is what the formula in 32 bits gives.
//
// With 32-bit moments a step is bound by memory (40 M values in fp32, 448 tensors,
// clipped, 32 bytes a value: 208 us, 6.1 TB/s), with 8-bit ones by issue slots
// and memory (160 M values in bf16, 448 tensors, clipped, 12 bytes a value: 379 us,
// 5.1 TB/s; 202 M with remainders, 14 bytes: 498 us, 5.7 TB/s).
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <float.h>
#include <math.h>

#include "gemv_common.cuh"
#include "linear_common.cuh"

namespace rq {

constexpr int kAdBlock = RQ_ADAM_BLOCK, kAdThreads = 256, kAdWarps = kAdThreads / 32;
constexpr float kMTop = 448.0f, kRTop = 507904.0f;

// The tensors of a launch, as kernel parameters (32 KB at most): nothing is
// copied to the device beforehand, and a captured launch keeps them.
template <int MAX>
struct AdTensors {
  void* p[MAX];
  const void* g[MAX];
  uint32_t first[MAX + 1];  // launch-wide number of a tensor's first block; [count]: blocks in all
  uint32_t block[MAX];      // its first block in the arena
  uint16_t slot[MAX];       // its place among the steps
  uint16_t tail[MAX];       // values of its last block
  int count;
};
constexpr int kAdSmall = 64, kAdLarge = RQ_ADAM_TENSORS;
static_assert(sizeof(AdTensors<kAdLarge>) <= 31 * 1024, "kernel parameters end at 32764 bytes");

// The tensor that holds launch-wide block b.
template <int MAX>
__device__ __forceinline__ int tensor_of(const AdTensors<MAX>& t, uint32_t b) {
  int lo = 0, hi = t.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (t.first[mid] <= b) lo = mid;
    else hi = mid;
  }
  return lo;
}

// A CTA's share of the blocks: side by side, so that one search finds the
// first tensor and the next ones follow.
__device__ __forceinline__ void share(uint32_t blocks, uint32_t& b, uint32_t& end) {
  b = (uint32_t)((uint64_t)blocks * blockIdx.x / gridDim.x);
  end = (uint32_t)((uint64_t)blocks * (blockIdx.x + 1) / gridDim.x);
}

// A lane's 8 values as they are in memory: 16-bit types packed in 4 words.
template <int DT> struct Raw { uint32_t w[DT == RQ_F32 ? 8 : 4]; };

template <int DT>
__device__ __forceinline__ void put(Raw<DT>& r, int i, float x, float y);

// 8 values at `at`, of which the first `n` exist (the others 0); VEC: all, and aligned.
template <int DT, bool VEC>
__device__ __forceinline__ Raw<DT> load_raw(const void* p, int64_t at, int n) {
  using T = typename DType<DT>::T;
  const T* from = static_cast<const T*>(p) + at;
  Raw<DT> r;
  if constexpr (VEC) {
#pragma unroll
    for (int h = 0; h < (DT == RQ_F32 ? 2 : 1); ++h)
      *reinterpret_cast<uint4*>(r.w + 4 * h) = reinterpret_cast<const uint4*>(from)[h];
  } else {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? DType<DT>::to_f32(from[i]) : 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) put(r, i, v[2 * i], v[2 * i + 1]);
  }
  return r;
}

// Values 2 i and 2 i + 1.
template <int DT>
__device__ __forceinline__ float2 pair_of(const Raw<DT>& r, int i) {
  if constexpr (DT == RQ_F32) return make_float2(__uint_as_float(r.w[2 * i]), __uint_as_float(r.w[2 * i + 1]));
  else if constexpr (DT == RQ_BF16) return make_float2(__uint_as_float(r.w[i] << 16), __uint_as_float(r.w[i] & 0xffff0000u));
  else return __half22float2(*reinterpret_cast<const __half2*>(&r.w[i]));
}
template <int DT>
__device__ __forceinline__ void put(Raw<DT>& r, int i, float x, float y) {
  if constexpr (DT == RQ_F32) r.w[2 * i] = __float_as_uint(x), r.w[2 * i + 1] = __float_as_uint(y);
  else r.w[i] = pack2<DT>(x, y);
}

template <int DT, bool VEC>
__device__ __forceinline__ void store_raw(void* p, int64_t at, int n, const Raw<DT>& r) {
  using T = typename DType<DT>::T;
  T* to = static_cast<T*>(p) + at;
  if constexpr (VEC) {
#pragma unroll
    for (int h = 0; h < (DT == RQ_F32 ? 2 : 1); ++h)
      reinterpret_cast<uint4*>(to)[h] = *reinterpret_cast<const uint4*>(r.w + 4 * h);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = pair_of<DT>(r, i);
      if (2 * i < n) to[2 * i] = DType<DT>::from_f32(v.x);
      if (2 * i + 1 < n) to[2 * i + 1] = DType<DT>::from_f32(v.y);
    }
  }
}

// 8 fp32 moments of a lane, in one access: with two of 16 bytes a warp's accesses
// leave every second 16 bytes out (reading 202 M moments back 365 us, now 301).
__device__ __forceinline__ void load_moments(const float* from, float (&v)[8]) {
  uint32_t w[8];
  load32(from, w);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
}
__device__ __forceinline__ void store_moments(float* to, const float (&v)[8]) {
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = __float_as_uint(v[i]);
  store32(to, w);
}

// ------------------------------------------------------------------ norm

// Adds the squares of a lane's 8 values in 64 bits.  Widening takes a
// conversion, whose pipe does 8 values a cycle; for normal numbers the bits are
// moved instead (the exponent grows by 896), in bf16 from the packed words, where
// two values share the test for others.
template <int DT>
__device__ __forceinline__ void add_squares(const Raw<DT>& r, double& s) {
  constexpr uint32_t up = 896u << 20;
  if constexpr (DT == RQ_BF16) {
    uint32_t least = 0x7f807f80u, most = 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t e = r.w[i] & 0x7f807f80u;
      least = __vminu2(least, e);
      most = __vmaxu2(most, e);
    }
    if ((least & 0xffffu) != 0u && least > 0xffffu && (most & 0xffffu) != 0x7f80u && most < 0x7f800000u) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const double x = __hiloint2double((int)((r.w[i] & 0x7fffu) * 8192u + up), 0);
        const double y = __hiloint2double((int)(((r.w[i] & 0x7fff0000u) >> 3) + up), 0);
        s = fma(x, x, s);
        s = fma(y, y, s);
      }
      return;
    }
  }
  float v[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = pair_of<DT>(r, i);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
  uint32_t least = 0x7f800000u, most = 0u;
  if constexpr (DT != RQ_BF16) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t e = __float_as_uint(v[i]) & 0x7f800000u;
      least = min(least, e);
      most = max(most, e);
    }
  }
  if (DT != RQ_BF16 && least != 0u && most != 0x7f800000u) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t b = __float_as_uint(v[i]) & 0x7fffffffu;
      const double d = __hiloint2double((int)(__umulhi(b, 1u << 29) + up), (int)(b << 29));
      s = fma(d, d, s);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) s = fma((double)v[i], (double)v[i], s);
  }
}

template <int DT, int MAX>
__global__ void __launch_bounds__(kAdThreads) norm_partial_k(const __grid_constant__ AdTensors<MAX> t,
                                                             double* __restrict__ partials) {
  grid_begin();
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  uint32_t b, end;
  share(t.first[t.count], b, end);
  b += warp;
  double sum = 0.0;
  int i = b < end ? tensor_of(t, b) : 0;
  while (b < end) {
    while (b >= t.first[i + 1]) ++i;
    const int64_t at = (int64_t)(b - t.first[i]) * kAdBlock + lane * 8;
    const bool aligned = (uintptr_t)t.g[i] % 16 == 0;
    // four blocks of one tensor at once, so that their loads are on the way together
    constexpr int N = 4;
    const uint32_t whole = min(end, t.first[i + 1] - 1);
    if (aligned && b + (N - 1) * kAdWarps < whole) {
      Raw<DT> v[N];
#pragma unroll
      for (int k = 0; k < N; ++k) v[k] = load_raw<DT, true>(t.g[i], at + k * kAdWarps * kAdBlock, 8);
#pragma unroll
      for (int k = 0; k < N; ++k) add_squares<DT>(v[k], sum);
      b += N * kAdWarps;
      continue;
    }
    const bool last = b + 1 == t.first[i + 1];
    const int n = (last ? t.tail[i] : kAdBlock) - lane * 8;
    if (aligned && (!last || t.tail[i] == kAdBlock)) add_squares<DT>(load_raw<DT, true>(t.g[i], at, 8), sum);
    else add_squares<DT>(load_raw<DT, false>(t.g[i], at, n), sum);
    b += kAdWarps;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  __shared__ double part[kAdWarps];
  if (lane == 0) part[warp] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double s = 0.0;
    for (int w = 0; w < kAdWarps; ++w) s += part[w];
    partials[blockIdx.x] = s;
  }
  // what the caller sums has RQ_NORM_PARTIALS values whatever the grid
  if (blockIdx.x == 0)
    for (int j = gridDim.x + threadIdx.x; j < RQ_NORM_PARTIALS; j += kAdThreads) partials[j] = 0.0;
}

// Sum of the partial sums, by one CTA in a fixed order; every thread gets it.
__device__ __forceinline__ double sum_partials(const double* partials, int n) {
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += kAdThreads) s += partials[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  __shared__ double part[kAdWarps];
  if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = s;
  __syncthreads();
  s = 0.0;
  for (int w = 0; w < kAdWarps; ++w) s += part[w];
  return s;
}

__global__ void __launch_bounds__(kAdThreads) norm_end_k(const double* __restrict__ partials, int n,
                                                         float* __restrict__ norm) {
  grid_begin();
  const double s = sum_partials(partials, n);
  if (threadIdx.x == 0) *norm = (float)sqrt(s);
}

// ------------------------------------------------------- moments in 8 bits

// Two values in one instruction, each rounded as by itself.
__device__ __forceinline__ uint64_t pair64(float2 a) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a.x), "f"(a.y));
  return d;
}
__device__ __forceinline__ float2 float2_of(uint64_t a) {
  float2 d;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(d.x), "=f"(d.y) : "l"(a));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(pair64(a)), "l"(pair64(b)));
  return float2_of(d);
}
__device__ __forceinline__ float2 mul2(float2 a, float b) { return mul2(a, make_float2(b, b)); }
// One by one: the compiler makes a product of pairs and their addition one rounding.
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return make_float2(__fadd_rn(a.x, b.x), __fadd_rn(a.y, b.y)); }
__device__ __forceinline__ float2 fma2(float2 a, float b, float2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(pair64(a)), "l"(pair64(make_float2(b, b))), "l"(pair64(c)));
  return float2_of(d);
}

// Largest magnitude, which a NaN wins; smallest value.
__device__ __forceinline__ float max_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float min3(float a, float b, float c) {
  float d;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// The root's code of a value t in [0, kRTop], in the low byte: a float of 4
// exponent and 4 mantissa bits, whose first 16 codes are the numbers 0 to 15.
// Adding 1.5 2^(23 + e) rounds t to q 2^e, ties to even, with e = 0 below 32 and
// 16 <= q <= 32 from there; the code is q + 16 e, and the sum holds q in its low
// bits and e in its exponent.
__device__ __forceinline__ uint32_t root_code(float t) {
  // 2^(4 + e) is the power of two in t, at least 2^4
  const uint32_t at = __viaddmax_u32(__float_as_uint(t) & 0x7f800000u, 19u << 23 | 0x400000u, 150u << 23 | 0x400000u);
  const uint32_t sum = __float_as_uint(__fadd_rn(t, __uint_as_float(at)));
  return sum + (sum >> 19) - ((150u << 4) + 8u);
}
// Values 2 i and 2 i + 1 of m and v from a lane's code words.  A root's code at the
// lowest exponent and highest mantissa bits of a half is the value times 2^-18,
// subnormals included.
__device__ __forceinline__ void decode2(const uint2& cm, const uint2& cr, const float2& scale, int i, float2& m, float2& v) {
  const uint32_t w = (i < 2 ? cm.x : cm.y) >> (16 * (i & 1));
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3);
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
  m = mul2(f, scale.x);
  const uint32_t c = __byte_perm(i < 2 ? cr.x : cr.y, 0u, i & 1 ? 0x3424u : 0x1404u) >> 2;
  const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&c));
  const float2 a = mul2(r, scale.y * 0x1p18f);
  v = mul2(a, a);
}

// m and r = sqrt(v) of a whole warp's block to codes and scales.  Of the four
// quotients a block needs, lanes 0 to 3 have one each: most / max (what values
// are multiplied by on the way to codes) and max / most, of m and of r.
__device__ __forceinline__ void encode_moments(const float (&m)[8], const float (&r)[8], int64_t block, int lane,
                                               uint8_t* codes_m, uint8_t* codes_r, float2* scales) {
  const float tm = max_nan(max_nan(m[0], m[1], m[2]), max_nan(m[3], m[4], m[5]), max_nan(m[6], m[7], 0.0f));
  const float tr = max_nan(max_nan(r[0], r[1], r[2]), max_nan(r[3], r[4], r[5]), max_nan(r[6], r[7], 0.0f));
  // as bit patterns, in which an infinity or NaN is the largest
  const uint32_t bm = __reduce_max_sync(0xffffffffu, __float_as_uint(tm) & 0x7fffffffu);
  const uint32_t br = __reduce_max_sync(0xffffffffu, __float_as_uint(tr) & 0x7fffffffu);
  const uint32_t bits = lane & 1 ? br : bm;
  const float top = __uint_as_float(bits), most = lane & 1 ? kRTop : kMTop;
  const bool bad = bits >= 0x7f800000u, live = top >= 0x1p-100f && !bad;
  float q = ieee_div(lane & 2 ? top : most, lane & 2 ? most : live ? top : 1.0f);
  q = live ? q : bad && (lane & 2) ? __uint_as_float(0x7fc00000u) : 0.0f;
  const float to_m = __shfl_sync(0xffffffffu, q, 0), to_r = __shfl_sync(0xffffffffu, q, 1);
  if (lane == 2 || lane == 3) reinterpret_cast<float*>(scales + block)[lane - 2] = q;
  uint32_t cm[4], c[8];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    cm[i] = __nv_cvt_float2_to_fp8x2(mul2(make_float2(m[2 * i], m[2 * i + 1]), to_m), __NV_SATFINITE, __NV_E4M3);
  float t[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 x = mul2(make_float2(r[2 * i], r[2 * i + 1]), to_r);
    t[2 * i] = x.x;
    t[2 * i + 1] = x.y;
  }
  // what is not 0 is at least 1: seldom less before
  if (min3(min3(t[0], t[1], t[2]), min3(t[3], t[4], t[5]), fminf(t[6], t[7])) < 1.0f && to_r > 0.0f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = r[i] > 0.0f ? fmaxf(t[i], 1.0f) : t[i];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) c[i] = root_code(t[i]);
  const int64_t at = block * kAdBlock + lane * 8;
  *reinterpret_cast<uint2*>(codes_m + at) = make_uint2(cm[0] | cm[1] << 16, cm[2] | cm[3] << 16);
  *reinterpret_cast<uint2*>(codes_r + at) =
      make_uint2(__byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410),
                 __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410));
}

// ------------------------------------------------------------------ update

struct AdState {
  void* m;           // fp32 [blocks * 256], or codes
  void* v;
  float2* scales;    // 8 bits: [blocks] (m, root)
  int16_t* low;      // what bf16 parameters leave of a 32-bit value, or null
  float beta1, rest1, beta2, rest2, eps;
  // the step
  double lr, decay, log_beta1, log_beta2;  // log 0 = -inf: the first moment is the gradient itself
  const float* lr_at;                      // learning rate on the device, or null
  const double* partials;
  int n_partials;
  float max_norm;
  float* norm;
  int32_t* steps;
  uint32_t* ticket;
};

// What a step number t and the norm make of the formula:
//   x = lr / (1 - b1^t), y = 1 / sqrt(1 - b2^t), z = 1 - lr wd, w = c.
// 1 - b^t is -expm1(t log b), in 64 bits.
__device__ __forceinline__ float4 factors_of(const AdState& a, int t, float c) {
  const double lr = a.lr_at ? (double)*a.lr_at : a.lr;
  const double c1 = -expm1(t * a.log_beta1), c2 = -expm1(t * a.log_beta2);
  return make_float4((float)(lr / c1), (float)(1.0 / sqrt(c2)), (float)(1.0 - lr * a.decay), c);
}

// What bf16 parameters leave: the 32-bit value of a bf16 and its 16 bits, and
// back, rounded half away from zero so that what is left fits 16 bits with its
// sign.
// A parameter that was written from outside comes with the remainder of the
// value before, which is less than a unit in its last place.  Two kinds of pair do
// not count, since rounding leaves none: a negative remainder at 0, where one
// step down in the bits is a NaN, and any at an infinity (a value above the
// largest bf16 becomes one for good).
__device__ __forceinline__ float join_low(float p, uint32_t low16) {
  const uint32_t sum = __float_as_uint(p) + (uint32_t)(int32_t)(int16_t)low16;
  const bool other_sign = (int32_t)(sum ^ __float_as_uint(p)) < 0;  // only a step down from 0
  return other_sign || !(fabsf(p) < __uint_as_float(0x7f800000u)) ? p : __uint_as_float(sum);
}
__device__ __forceinline__ float split_low(float p, uint32_t& low16) {
  const uint32_t bits = __float_as_uint(p);
  const bool finite = (bits & 0x7f800000u) != 0x7f800000u;
  const uint32_t top = finite ? (bits + 0x8000u) & 0xffff0000u : (bits & 0x7fffffu) ? 0x7fc00000u : bits;
  low16 = (finite ? bits - top : 0u) & 0xffffu;
  return __uint_as_float(top);
}

// Two values: m, v and p after the step, and r = sqrt(v).
template <bool EIGHT>
__device__ __forceinline__ float2 update(float2 g, float2& m, float2& v, float2 p, const float4& f, const AdState& a) {
  const float2 x = mul2(g, f.w);
  m = add2(mul2(m, a.beta1), mul2(x, a.rest1));
  v = add2(mul2(v, a.beta2), mul2(mul2(x, x), a.rest2));
  // in 8 bits the root is the state (and takes v's place); elsewhere it only divides the step
  float2 r, q;
  if constexpr (EIGHT) {
    v = r = make_float2(__fsqrt_rn(v.x), __fsqrt_rn(v.y));
  } else {
    asm("sqrt.approx.f32 %0, %1;" : "=f"(r.x) : "f"(v.x));
    asm("sqrt.approx.f32 %0, %1;" : "=f"(r.y) : "f"(v.y));
  }
  // The approximate root and reciprocal are off by 2^-23 at most, twice what a
  // rounding leaves: next to the step's ten roundings that makes 14 of 2^-24 at worst,
  // for a parameter that begins at 0 too.  Correctly rounded ones make a small step 30 %
  // longer (one projection's adapters 5.2 us and 6.7) and one with 8-bit moments 11 %
  // (160 M values in bf16 379 us and 421).  The divisor is at least eps or 2^-75.
  const float2 d = fma2(r, f.y, make_float2(a.eps, a.eps));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q.x) : "f"(d.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(q.y) : "f"(d.y));
  return fma2(p, f.z, mul2(mul2(m, -f.x), q));
}

// What a lane reads of a block.
template <int DT, bool EIGHT, bool LOW>
struct In {
  Raw<DT> g, p;
  Raw<RQ_BF16> low;
  uint2 cm, cr;  // 8 bits
  float2 scale;
  float m[8], v[8];  // 32 bits
};

template <int DT, bool VEC, bool EIGHT, bool LOW>
__device__ __forceinline__ void fetch(In<DT, EIGHT, LOW>& d, const void* p, const void* g, int64_t at, int n,
                                      int64_t block, int lane, const AdState& a) {
  const int64_t sat = block * kAdBlock + lane * 8;
  d.g = load_raw<DT, VEC>(g, at, n);
  d.p = load_raw<DT, VEC>(p, at, n);
  if constexpr (LOW) d.low = load_raw<RQ_BF16, true>(a.low, sat, 8);
  if constexpr (EIGHT) {
    d.cm = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.m) + sat);
    d.cr = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.v) + sat);
    d.scale = a.scales[block];
  } else {
    load_moments(static_cast<const float*>(a.m) + sat, d.m);
    load_moments(static_cast<const float*>(a.v) + sat, d.v);
  }
}

template <int DT, bool VEC, bool EIGHT, bool LOW>
__device__ __forceinline__ void update8(const In<DT, EIGHT, LOW>& d, void* p, int64_t at, int n, int64_t block,
                                        int lane, const float4& f, const AdState& a) {
  const int64_t sat = block * kAdBlock + lane * 8;
  Raw<DT> pr;
  Raw<RQ_BF16> low;
  float m[8], v[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 mv, vv;
    if constexpr (EIGHT) {
      decode2(d.cm, d.cr, d.scale, i, mv, vv);
    } else {
      mv = make_float2(d.m[2 * i], d.m[2 * i + 1]);
      vv = make_float2(d.v[2 * i], d.v[2 * i + 1]);
    }
    const float2 gv = pair_of<DT>(d.g, i);
    float2 pv = pair_of<DT>(d.p, i);
    if constexpr (LOW) pv = make_float2(join_low(pv.x, d.low.w[i]), join_low(pv.y, d.low.w[i] >> 16));
    pv = update<EIGHT>(gv, mv, vv, pv, f, a);
    m[2 * i] = mv.x, m[2 * i + 1] = mv.y;
    v[2 * i] = vv.x, v[2 * i + 1] = vv.y;
    if constexpr (LOW) {
      uint32_t x, y;
      pv = make_float2(split_low(pv.x, x), split_low(pv.y, y));
      low.w[i] = x | y << 16;
    }
    put<DT>(pr, i, pv.x, pv.y);
  }
  store_raw<DT, VEC>(p, at, n, pr);
  if constexpr (LOW) store_raw<RQ_BF16, true>(a.low, sat, 8, low);
  if constexpr (EIGHT) {
    encode_moments(m, v, block, lane, static_cast<uint8_t*>(a.m), static_cast<uint8_t*>(a.v), a.scales);
  } else {
    store_moments(static_cast<float*>(a.m) + sat, m);
    store_moments(static_cast<float*>(a.v) + sat, v);
  }
}

// CTAs an SM.  Four would leave 64 registers a thread, too few for the next block's
// inputs (8 bits, 202 M values with remainders: 498 us with three, 541 with four).
constexpr int kAdResident = 3;

template <int DT, bool EIGHT, bool LOW, int MAX>
__global__ void __launch_bounds__(kAdThreads, kAdResident) adam_update_k(const __grid_constant__ AdTensors<MAX> t,
                                                                        const AdState a) {
  grid_begin();
  const int lane = threadIdx.x % 32;
  float c = 1.0f;
  if (a.n_partials > 0) {
    const float total = (float)sqrt(sum_partials(a.partials, a.n_partials));
    if (blockIdx.x == 0 && threadIdx.x == 0) *a.norm = total;
    const float quotient = __fmul_rn(ieee_div(1.0f, __fadd_rn(total, 1e-6f)), a.max_norm);
    c = quotient > 1.0f ? 1.0f : quotient;  // a NaN stays one
  }
  uint32_t b, end;
  share(t.first[t.count], b, end);
  b += threadIdx.x / 32;
  int i = b < end ? tensor_of(t, b) : 0, step = 0;
  float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  while (b < end) {
    while (b >= t.first[i + 1]) ++i;
    const int now = a.steps[t.slot[i]] + 1;
    if (now != step) f = factors_of(a, step = now, c);
    void* const p = t.p[i];
    const void* const g = t.g[i];
    const uint32_t next = t.first[i + 1];
    uint32_t in = b - t.first[i];
    // whole blocks of an aligned tensor, then what is left one by one
    if (((uintptr_t)g | (uintptr_t)p) % 16 == 0) {
      const uint32_t whole = min(end, next - (t.tail[i] != kAdBlock));
      int64_t at = (int64_t)in * kAdBlock + lane * 8, block = (int64_t)t.block[i] + in;
      // with 8-bit moments the next block is on its way while this one is computed
      // (160 M values in bf16 419 us without, 379 with)
      In<DT, EIGHT, LOW> d;
      if (EIGHT && b < whole) fetch<DT, true, EIGHT, LOW>(d, p, g, at, 8, block, lane, a);
#pragma unroll 1
      for (; b < whole; b += kAdWarps, at += kAdWarps * kAdBlock, block += kAdWarps) {
        if constexpr (!EIGHT) fetch<DT, true, EIGHT, LOW>(d, p, g, at, 8, block, lane, a);
        const In<DT, EIGHT, LOW> now_in = d;
        if (EIGHT && b + kAdWarps < whole)
          fetch<DT, true, EIGHT, LOW>(d, p, g, at + kAdWarps * kAdBlock, 8, block + kAdWarps, lane, a);
        update8<DT, true, EIGHT, LOW>(now_in, p, at, 8, block, lane, f, a);
      }
      in = b - t.first[i];
    }
    if (b < end && b < next) {
      const int n = (b + 1 == next ? t.tail[i] : kAdBlock) - lane * 8;
      In<DT, EIGHT, LOW> d;
      fetch<DT, false, EIGHT, LOW>(d, p, g, (int64_t)in * kAdBlock + lane * 8, n, (int64_t)t.block[i] + in, lane, a);
      update8<DT, false, EIGHT, LOW>(d, p, (int64_t)in * kAdBlock + lane * 8, n, (int64_t)t.block[i] + in, lane, f, a);
      b += kAdWarps;
    }
  }
  // every CTA has read the steps before it takes a ticket; the last one counts
  __shared__ bool last;
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(a.ticket, 1u) + 1 == gridDim.x;
  __syncthreads();
  if (last) {
    for (int k = threadIdx.x; k < t.count; k += kAdThreads) ++a.steps[t.slot[k]];
    if (threadIdx.x == 0) *a.ticket = 0u;
  }
}

// Values of 8-bit moments, and codes of values (v is squared, not the root).
__global__ void __launch_bounds__(kAdThreads) adam_unpack_k(const uint8_t* codes_m, const uint8_t* codes_r,
                                                            const float2* scales, uint32_t blocks, float* m, float* v) {
  grid_begin();
  const uint32_t b = blockIdx.x * kAdWarps + threadIdx.x / 32;
  if (b >= blocks) return;
  const int64_t at = (int64_t)b * kAdBlock + threadIdx.x % 32 * 8;
  const uint2 cm = *reinterpret_cast<const uint2*>(codes_m + at), cr = *reinterpret_cast<const uint2*>(codes_r + at);
  const float2 scale = scales[b];
  float x[8], y[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 s, t;
    decode2(cm, cr, scale, i, s, t);
    x[2 * i] = s.x, x[2 * i + 1] = s.y;
    y[2 * i] = t.x, y[2 * i + 1] = t.y;
  }
  store_moments(m + at, x);
  store_moments(v + at, y);
}

__global__ void __launch_bounds__(kAdThreads) adam_pack_k(const float* m, const float* v, uint32_t blocks,
                                                          uint8_t* codes_m, uint8_t* codes_r, float2* scales) {
  grid_begin();
  const uint32_t b = blockIdx.x * kAdWarps + threadIdx.x / 32;
  if (b >= blocks) return;
  const int64_t at = (int64_t)b * kAdBlock + threadIdx.x % 32 * 8;
  float x[8], y[8];
  load_moments(m + at, x);
  load_moments(v + at, y);
#pragma unroll
  for (int i = 0; i < 8; ++i) y[i] = __fsqrt_rn(y[i]);
  encode_moments(x, y, b, threadIdx.x % 32, codes_m, codes_r, scales);
}

// -------------------------------------------------------------- host side

template <int MAX>
static void fill(AdTensors<MAX>& t, const RqAdamTensor* list, int count) {
  uint32_t at = 0;
  t.count = count;
  for (int i = 0; i < count; ++i) {
    const int64_t blocks = (list[i].n + kAdBlock - 1) / kAdBlock;
    t.p[i] = list[i].param;
    t.g[i] = list[i].grad;
    t.first[i] = at;
    t.block[i] = (uint32_t)list[i].block;
    t.slot[i] = (uint16_t)list[i].slot;
    t.tail[i] = (uint16_t)(list[i].n - (blocks - 1) * kAdBlock);
    at += (uint32_t)blocks;
  }
  t.first[count] = at;
}

static unsigned grid_for(uint32_t blocks, int ctas_per_sm) {
  const unsigned want = (blocks + kAdWarps - 1) / kAdWarps, most = (unsigned)(num_sms() * ctas_per_sm);
  return want < 1 ? 1 : want < most ? want : most;
}

template <int DT>
static int norm_t(const RqAdamTensor* list, int count, double* partials, cudaStream_t st) {
  if (count <= kAdSmall) {
    AdTensors<kAdSmall> t;
    fill(t, list, count);
    unsigned grid = grid_for(t.first[count], 8);
    if (grid > RQ_NORM_PARTIALS) grid = RQ_NORM_PARTIALS;
    return launch_dependent(norm_partial_k<DT, kAdSmall>, grid, kAdThreads, st, t, partials);
  }
  AdTensors<kAdLarge> t;
  fill(t, list, count);
  unsigned grid = grid_for(t.first[count], 8);
  if (grid > RQ_NORM_PARTIALS) grid = RQ_NORM_PARTIALS;
  return launch_dependent(norm_partial_k<DT, kAdLarge>, grid, kAdThreads, st, t, partials);
}

int grad_norm_partial(const RqAdamTensor* list, int count, int dt, double* partials, cudaStream_t st) {
  return dt == RQ_F32 ? norm_t<RQ_F32>(list, count, partials, st)
         : dt == RQ_BF16 ? norm_t<RQ_BF16>(list, count, partials, st)
                         : norm_t<RQ_F16>(list, count, partials, st);
}

int grad_norm_end(const double* partials, int n, float* norm, cudaStream_t st) {
  return launch_dependent(norm_end_k, 1, kAdThreads, st, partials, n, norm);
}

template <int DT, bool EIGHT, bool LOW, int MAX>
static int update_t(const RqAdamTensor* list, int count, const AdState& a, cudaStream_t st) {
  AdTensors<MAX> t;
  fill(t, list, count);
  // 32 bits: more than are resident, or the last to end are waited for (208 us with
  // 8 an SM, 222 with 3)
  const unsigned grid = grid_for(t.first[count], EIGHT ? kAdResident : 8);
  return launch_dependent(adam_update_k<DT, EIGHT, LOW, MAX>, grid, kAdThreads, st, t, a);
}

template <bool EIGHT, int MAX>
static int update_d(const RqAdamTensor* list, int count, int dt, const AdState& a, cudaStream_t st) {
  if (a.low) return update_t<RQ_BF16, EIGHT, true, MAX>(list, count, a, st);
  return dt == RQ_F32 ? update_t<RQ_F32, EIGHT, false, MAX>(list, count, a, st)
         : dt == RQ_BF16 ? update_t<RQ_BF16, EIGHT, false, MAX>(list, count, a, st)
                         : update_t<RQ_F16, EIGHT, false, MAX>(list, count, a, st);
}

int adam_update(const RqAdamTensor* list, int count, int dt, int bits, void* m, void* v, float* scales, int16_t* low,
                const RqAdamStep& step, cudaStream_t st) {
  AdState a = {};
  a.m = m;
  a.v = v;
  a.scales = reinterpret_cast<float2*>(scales);
  a.low = low;
  a.beta1 = (float)step.beta1;
  a.rest1 = (float)(1.0 - step.beta1);
  a.beta2 = (float)step.beta2;
  a.rest2 = (float)(1.0 - step.beta2);
  // the quotient takes subnormal divisors as 0
  a.eps = step.eps > 0.0 && step.eps < FLT_MIN ? FLT_MIN : (float)step.eps;
  a.lr = step.lr;
  a.decay = step.decay;
  a.log_beta1 = log(step.beta1);
  a.log_beta2 = log(step.beta2);
  a.lr_at = step.lr_at;
  a.partials = step.partials;
  a.n_partials = step.n_partials;
  a.max_norm = step.max_norm;
  a.norm = step.norm;
  a.steps = step.steps;
  a.ticket = step.ticket;
  if (bits == 8)
    return count <= kAdSmall ? update_d<true, kAdSmall>(list, count, dt, a, st)
                             : update_d<true, kAdLarge>(list, count, dt, a, st);
  return count <= kAdSmall ? update_d<false, kAdSmall>(list, count, dt, a, st)
                           : update_d<false, kAdLarge>(list, count, dt, a, st);
}

int adam_unpack(const uint8_t* m8, const uint8_t* r8, const float* scales, int64_t blocks, float* m, float* v,
                cudaStream_t st) {
  return launch_dependent(adam_unpack_k, (unsigned)((blocks + kAdWarps - 1) / kAdWarps), kAdThreads, st, m8, r8,
                          reinterpret_cast<const float2*>(scales), (uint32_t)blocks, m, v);
}

int adam_pack(const float* m, const float* v, int64_t blocks, uint8_t* m8, uint8_t* r8, float* scales,
              cudaStream_t st) {
  return launch_dependent(adam_pack_k, (unsigned)((blocks + kAdWarps - 1) / kAdWarps), kAdThreads, st, m, v,
                          (uint32_t)blocks, m8, r8, reinterpret_cast<float2*>(scales));
}

}  // namespace rq

// mx4.cu -- rows to and from microscaled 4-bit values: blocks of 32 columns
// with e = max(floor(log2 max|x|) - 2, -127), codes e2m1(x 2^-e), scale byte
// e + 127.  e is read off the maximum's exponent bits and 2^-e is exact, so the
// codes are those of the definition bit for bit.
//
// One pass over the data.  A lane has W = 16 values of a row in 16 bits or 8 in 32,
// one access of 32 bytes; 8 in 16 bits, or in two accesses, where rows lie at
// multiples of 16 bytes only.  128 / W lanes have a piece of 128 columns, and take
// rows r, r + 32, r + 64 and r + 96 of 128: four loads on their way at once, and
// their 16 scale bytes lie side by side.  Rows past M up to whole pieces of 128
// count as zeros.
// Bound by memory: 11008 x 4096 in bf16 is packed in 18.7 us (6.1 TB/s; 22.2 with
// 8 values a lane, whose blocks' scales took twice the instructions) and unpacked
// in 19.4 (5.9 TB/s); 2047 x 11008 in fp16 in 9.6 (10.7 with 8 values a lane).
#include <cuda_runtime.h>

#include "mx4_common.cuh"

namespace rq {

constexpr int kM4Threads = 256, kM4Lanes = 16, kM4PerCta = kM4Threads / kM4Lanes;

// Division of n < 2^31 by a number known at launch: (n * mul) >> shift.
struct M4Divide {
  uint32_t mul;
  int shift;
  uint32_t by;
};
static M4Divide m4_divide(uint32_t d) {
  int s = 0;
  while ((1ull << s) < d) ++s;
  return M4Divide{(uint32_t)((1ull << (31 + s)) / d + 1), 31 + s, d};
}

// Values of a lane, of rows whose pieces lie at ALIGN bytes.
template <int DT, int ALIGN> constexpr int kM4Lane = DT != RQ_F32 && ALIGN == 32 ? 16 : 8;

// A warp has 32 W columns of 4 rows.
template <int DT, int ALIGN>
__global__ void __launch_bounds__(kM4Threads) mx4_pack_k(const void* __restrict__ x, int64_t ld, int64_t M, int K,
                                                         uint32_t warps, M4Divide np, int tiles,
                                                         uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  grid_begin();
  using T = typename DType<DT>::T;
  constexpr int W = kM4Lane<DT, ALIGN>, L = 128 / W;
  const uint32_t p = blockIdx.x * (kM4Threads / 32) + threadIdx.x / 32;
  const uint32_t q = (uint32_t)(((uint64_t)p * np.mul) >> np.shift);  // 32 groups of 4 rows to a tile of 128
  const int l = threadIdx.x % L, tile = (int)(p - q * np.by) * (32 / L) + threadIdx.x % 32 / L;
  const bool in = p < warps && tile < tiles;
  const int64_t row0 = (int64_t)(q / 32) * 128 + q % 32;
  const int col = tile * 128 + l * W;
  M4Raw<DT, W> r[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t row = row0 + 32 * j;
    const bool any = in && row < M;
    r[j] = m4_load<DT, ALIGN, W>(static_cast<const T*>(x) + (any ? row * ld : 0), col, any ? K : 0);
  }
  uint32_t top[4];
  m4_top<DT, W, 4>(r, top);
  uint32_t bytes = 0;  // row j's scale of this lane's block in byte j
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t byte = m4_scale(top[j]);
    bytes |= byte << (8 * j);
    float v[W];
    m4_values<DT, W>(r[j], v);
    const float f = m4_factor(byte);
    const int64_t row = row0 + 32 * j;
    uint8_t* to = codes + (row * tiles + tile) * 64 + l * (W / 2);
    const uint32_t w = e2m1x8(v, f);
    if constexpr (W == 16) {
      const uint32_t high = e2m1x8(v + 8, f);
      if (in && row < M) *reinterpret_cast<uint2*>(to) = make_uint2(w, high);
    } else {
      if (in && row < M) *reinterpret_cast<uint32_t*>(to) = w;
    }
  }
  uint32_t b[4];  // the four blocks' bytes, to be turned into the four rows'
#pragma unroll
  for (int i = 0; i < 4; ++i) b[i] = __shfl_sync(0xffffffffu, bytes, L / 4 * i, L);
  if (in && l == 0) {
    const uint32_t lo01 = __byte_perm(b[0], b[1], 0x5140), hi01 = __byte_perm(b[0], b[1], 0x7362),
                   lo23 = __byte_perm(b[2], b[3], 0x5140), hi23 = __byte_perm(b[2], b[3], 0x7362);
    *reinterpret_cast<uint4*>(scales + ((row0 / 128) * tiles + tile) * 512 + row0 % 32 * 16) =
        make_uint4(__byte_perm(lo01, lo23, 0x5410), __byte_perm(lo01, lo23, 0x7632), __byte_perm(hi01, hi23, 0x5410),
                   __byte_perm(hi01, hi23, 0x7632));
  }
}

// As packing.
template <int DT, int ALIGN>
__global__ void __launch_bounds__(kM4Threads) mx4_unpack_k(const uint8_t* __restrict__ codes,
                                                           const uint8_t* __restrict__ scales, int64_t M, int K,
                                                           uint32_t warps, M4Divide np, int tiles,
                                                           void* __restrict__ out) {
  grid_begin();
  using T = typename DType<DT>::T;
  constexpr int W = kM4Lane<DT, ALIGN>, L = 128 / W;
  const uint32_t p = blockIdx.x * (kM4Threads / 32) + threadIdx.x / 32;
  const uint32_t q = (uint32_t)(((uint64_t)p * np.mul) >> np.shift);
  const int l = threadIdx.x % L, tile = (int)(p - q * np.by) * (32 / L) + threadIdx.x % 32 / L;
  const int64_t row0 = (int64_t)(q / 32) * 128 + q % 32;
  const int col = tile * 128 + l * W;
  if (p >= warps || col >= K) return;
  // byte l W / 32 of word j: row j's scale of this lane's block
  const uint4 s4 = *reinterpret_cast<const uint4*>(scales + ((row0 / 128) * tiles + tile) * 512 + row0 % 32 * 16);
  const uint32_t s[4] = {s4.x, s4.y, s4.z, s4.w};
  uint2 w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t row = row0 + 32 * j;
    const uint8_t* from = codes + (row * tiles + tile) * 64 + l * (W / 2);
    w[j] = make_uint2(0u, 0u);
    if constexpr (W == 16) {
      if (row < M) w[j] = *reinterpret_cast<const uint2*>(from);
    } else {
      if (row < M) w[j].x = *reinterpret_cast<const uint32_t*>(from);
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t row = row0 + 32 * j;
    if (row >= M) break;
    const float f = pow2_scale((int)(s[j] >> (8 * (l * W / 32)) & 255u), 127);
    float v[W];
#pragma unroll
    for (int i = 0; i < W / 2; ++i) {
      uint32_t h;
      asm("{\n .reg .b8 b;\n cvt.u8.u32 b, %1;\n cvt.rn.f16x2.e2m1x2 %0, b;\n}\n" : "=r"(h) : "r"(((i < 4 ? w[j].x : w[j].y) >> (8 * (i % 4))) & 0xffu));
      const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&h));
      v[2 * i] = x.x * f;
      v[2 * i + 1] = x.y * f;
    }
    T* to = static_cast<T*>(out) + row * K + col;
    constexpr int words = DT == RQ_F32 ? W : W / 2;
    uint32_t o[words];
#pragma unroll
    for (int i = 0; i < words; ++i) {
      if constexpr (DT == RQ_F32) o[i] = __float_as_uint(v[i]);
      else o[i] = pack2<DT>(v[2 * i], v[2 * i + 1]);
    }
    if constexpr (ALIGN == 32) {
      store32(to, o);
    } else {
#pragma unroll
      for (int h = 0; h < words / 4; ++h) reinterpret_cast<uint4*>(to)[h] = *reinterpret_cast<const uint4*>(o + 4 * h);
    }
  }
}

// Rows that are not 16-byte aligned: a lane has every 16th value of a piece, so
// that the lanes' single values are side by side.
template <int DT>
__global__ void __launch_bounds__(kM4Threads) mx4_unpack_odd_k(const uint8_t* __restrict__ codes,
                                                               const uint8_t* __restrict__ scales, uint32_t pieces,
                                                               int K, M4Divide nt, void* __restrict__ out) {
  grid_begin();
  using T = typename DType<DT>::T;
  const uint32_t p = blockIdx.x * kM4PerCta + threadIdx.x / kM4Lanes;
  if (p >= pieces) return;
  const int l = threadIdx.x % kM4Lanes;
  const uint32_t row = (uint32_t)(((uint64_t)p * nt.mul) >> nt.shift), tile = p - row * nt.by;
  const uint32_t bytes = *reinterpret_cast<const uint32_t*>(scales + mx4_scale_at(row, (int)tile * 4, (int)nt.by));
  const uint8_t* from = codes + ((int64_t)row * nt.by + tile) * 64;
  T* to = static_cast<T*>(out) + (int64_t)row * K + (int)tile * 128;
  const int left = K - (int)tile * 128;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int at = i * kM4Lanes + l;
    const float s = pow2_scale((int)(bytes >> (8 * (i / 2)) & 255u), 127);
    const float v = e2m1_to_f32(from[at / 2] >> (4 * (at & 1))) * s;
    if (at < left) to[at] = DType<DT>::from_f32(v);
  }
}

// Bytes at which all of a lane's pieces of rows of K columns lie.
static int m4_align(const void* p, int64_t ld, int64_t K, int dt) {
  const int e = dt == RQ_F32 ? 4 : 2;
  const uint64_t all = (uintptr_t)p | (uint64_t)(ld * e);
  return all % 32 == 0 && K * e % 32 == 0 ? 32 : all % 16 == 0 && K % 8 == 0 ? 16 : 0;
}

// Warps, and how many to a group of 4 rows.
static uint32_t m4_warps(int64_t M, int tiles, int dt, int align, M4Divide& np) {
  const int pieces = dt != RQ_F32 && align == 32 ? 4 : 2;
  np = m4_divide((uint32_t)((tiles + pieces - 1) / pieces));
  return (uint32_t)((M + 127) / 128 * 32) * np.by;
}

int mx4_pack(const void* x, int dt, int64_t ld, int64_t M, int64_t K, uint8_t* codes, uint8_t* scales, cudaStream_t st) {
  const int tiles = (int)(mx4_pitch(K) / 128);
  const int align = m4_align(x, ld, K, dt);
  M4Divide np;
  const uint32_t warps = m4_warps(M, tiles, dt, align, np);
#define RQ_BY_ALIGN(k, DT) (align == 32 ? k<DT, 32> : align == 16 ? k<DT, 16> : k<DT, 0>)
  auto* k = dt == RQ_F32    ? RQ_BY_ALIGN(mx4_pack_k, RQ_F32)
            : dt == RQ_BF16 ? RQ_BY_ALIGN(mx4_pack_k, RQ_BF16)
                            : RQ_BY_ALIGN(mx4_pack_k, RQ_F16);
#undef RQ_BY_ALIGN
  return launch_dependent(k, (warps + kM4Threads / 32 - 1) / (kM4Threads / 32), kM4Threads, st, x, ld, M, (int)K, warps, np,
                          tiles, codes, scales);
}

int mx4_unpack(const uint8_t* codes, const uint8_t* scales, int64_t M, int64_t K, void* out, int dt, cudaStream_t st) {
  const int tiles = (int)(mx4_pitch(K) / 128);
  if (const int align = m4_align(out, K, K, dt)) {
    M4Divide np;
    const uint32_t warps = m4_warps(M, tiles, dt, align, np);
#define RQ_BY_ALIGN(k, DT) (align == 32 ? k<DT, 32> : k<DT, 16>)
    auto* k = dt == RQ_F32    ? RQ_BY_ALIGN(mx4_unpack_k, RQ_F32)
              : dt == RQ_BF16 ? RQ_BY_ALIGN(mx4_unpack_k, RQ_BF16)
                              : RQ_BY_ALIGN(mx4_unpack_k, RQ_F16);
#undef RQ_BY_ALIGN
    return launch_dependent(k, (warps + kM4Threads / 32 - 1) / (kM4Threads / 32), kM4Threads, st, codes, scales, M, (int)K,
                            warps, np, tiles, out);
  }
  const M4Divide nt = m4_divide((uint32_t)tiles);
  const uint32_t pieces = (uint32_t)M * nt.by;
  auto* k = dt == RQ_F32    ? mx4_unpack_odd_k<RQ_F32>
            : dt == RQ_BF16 ? mx4_unpack_odd_k<RQ_BF16>
                            : mx4_unpack_odd_k<RQ_F16>;
  return launch_dependent(k, (pieces + kM4PerCta - 1) / kM4PerCta, kM4Threads, st, codes, scales, pieces, (int)K, nt, out);
}

// Rows of 16-bit values to rows that begin at 16 bytes: a thread writes 8 values.
// Inside a row it reads the two aligned 16-byte pieces that hold them and shifts
// (by as much for the whole row); at its ends value by value, so that nothing
// outside the row is read.
__global__ void __launch_bounds__(128) align_rows_k(const uint16_t* __restrict__ x, int64_t ld, int N, uint32_t per,
                                                    uint16_t* __restrict__ out, int64_t ldo) {
  grid_begin();
  const uint32_t m = blockIdx.x / per;
  const int c = (int)((blockIdx.x - m * per) * 128 + threadIdx.x) * 8;
  if (c >= N) return;
  const uint16_t* from = x + (int64_t)m * ld + c;
  const uint32_t off = (uint32_t)((uintptr_t)from & 15);
  uint32_t w[4];
  if (c >= 8 && c + 16 <= N) {
    const uint4* p = reinterpret_cast<const uint4*>((uintptr_t)from & ~(uintptr_t)15);
    const uint4 a = __ldg(p), b = off ? __ldg(p + 1) : a;
    const uint32_t v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    const uint32_t k = off / 4, bits = off % 4 * 8;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t lo = k == 0 ? v[i] : k == 1 ? v[i + 1] : k == 2 ? v[i + 2] : v[i + 3];
      const uint32_t hi = k == 0 ? v[i + 1] : k == 1 ? v[i + 2] : k == 2 ? v[i + 3] : v[i + 4 < 8 ? i + 4 : 7];
      w[i] = __funnelshift_r(lo, hi, bits);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[i] = (c + 2 * i < N ? from[2 * i] : 0u) | (c + 2 * i + 1 < N ? from[2 * i + 1] : 0u) << 16;
  }
  *reinterpret_cast<uint4*>(out + (int64_t)m * ldo + c) = make_uint4(w[0], w[1], w[2], w[3]);
}

int align_rows(const void* x, int64_t ld, int64_t M, int64_t N, void* out, int64_t ldo, cudaStream_t st) {
  const uint32_t per = (uint32_t)((N + 1023) / 1024);
  return launch_dependent(align_rows_k, (unsigned)(M * per), 128, st, static_cast<const uint16_t*>(x), ld, (int)N, per,
                          static_cast<uint16_t*>(out), ldo);
}

}  // namespace rq

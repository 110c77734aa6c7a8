// mx4_dx.cu -- the input gradient of a projection in microscaled 4 bits:
//   dx[m, k] = sum_n dy[m, n] w[n, k],  dy in 16 bits, w [N, K] packed.
//
// The scales go along k, which the sum does not run over, so the block-scaled
// tensor cores cannot take w; it is widened to dy's type in shared memory and
// multiplied by tcgen05.mma kind::f16.  In bf16 every value of w is exact.  In
// fp16 w is taken times 2^(127 - top) with its largest scale byte `top`, which a
// small kernel before finds (what is then below 2^-24 rounds to a multiple of
// that), and the epilogue multiplies that back.
//
// CTA pairs stay and take tiles of 256 tokens x BN columns in turn, as 2-SM
// MMAs (M = 256): each CTA holds its 128 tokens of dy and widens half of the
// columns.  A stage of the ring holds 128 rows of w (a wait or a commit costs
// the tensor pipe about 100 cycles, next to the 1024 of a stage's 8 MMAs).
//   warp 0      producer: dy [128 x 128] as two K-major tiles whose bytes count
//               on the leader's barrier, and this CTA's codes of the stage
//   warp 1      tensor memory; the leader's issues the MMAs
//   8 or 16     widen: a thread has BN / 4 columns of a row, stores 16-byte units
//   warps       of an MN-major tile (w's own row layout, 128-byte swizzle)
//   4 warps     epilogue, from one of two accumulators while the MMAs fill the
//               other
// Widening without a table: the 3 bits of a code's magnitude, put at the lowest
// exponent bits and the highest mantissa bit of the 16-bit type, are the value
// times 2^-126 (fp16: 2^-14), subnormals included, and one or two packed
// multiplications take that and the scale in.  A word's 8 codes come out as
// (0, 4), (1, 5), (2, 6), (3, 7); they are stored so, and the epilogue puts the
// columns right.
// Bound by the tensor cores, whose pipe is 67 % active: dy 8192 x 11008 to dx 8192 x
// 4096 in bf16 takes 533 us, 1386 TFLOP/s, and reads 235 MB (operands 204); once the
// power limit is reached 580 to 600.
#include <cuda.h>
#include <cuda_runtime.h>

#include "gemv_common.cuh"
#include "mx4_common.cuh"
#include "rq_internal.h"
#include "tcgen05_common.cuh"

namespace rq {

__device__ unsigned int g_mx4_dx_timeouts;

int mx4_dx_take_timeouts(unsigned int* v) {
  unsigned int zero = 0;
  cudaError_t e = cudaMemcpyFromSymbol(v, g_mx4_dx_timeouts, sizeof(*v));
  if (e == cudaSuccess) e = cudaMemcpyToSymbol(g_mx4_dx_timeouts, &zero, sizeof(zero));
  if (e != cudaSuccess) {
    set_cuda_error(e);
    return RQ_ERR_CUDA;
  }
  return RQ_OK;
}

namespace {

constexpr int kWiden = 8, kEpi = 4;                      // warps
constexpr int kRows = 128;                               // rows of w (columns of dy) a stage
constexpr uint32_t kA = 128 * 128;                       // 64 columns of dy of a CTA's 128 tokens

template <int DT, int BN>
struct Plan {
  // Teams of 8 widening warps that take the stages in turn.  Two hide the waits
  // and fences between stages, but take issue slots and shared memory from each
  // other: dy 8192 x 11008 to 4096 columns in bf16 613 us with one and 531 with two,
  // 4096 x 4096 to 4096 140 and 119; 2047 x 4096 to 11008 in fp16 (whose widening is
  // shorter) 149 and 157, 512 x 4096 to 4096 (tiles of 128 columns) 26.7 and 28.7.
  static constexpr int kTeams = DT == RQ_BF16 && BN == 256 ? 2 : 1;
  static constexpr int kEpi0 = 2 + kTeams * kWiden;      // first epilogue warp
  static constexpr int kThreads = 32 * (kEpi0 + kEpi);
  static constexpr int BNH = BN / 2;                     // columns of a CTA
  static constexpr uint32_t kChunk = kRows * 128;        // 64 widened columns of a stage
  static constexpr uint32_t kB = 2 * kA, kC = kB + BNH / 64 * kChunk;
  static constexpr uint32_t kCodes = kRows * BNH / 2;
  static constexpr uint32_t kStage = kC + kCodes;
  static constexpr int S = BN == 256 ? 3 : 4;
  static constexpr uint32_t kOut = S * kStage;           // staged: a warp's 32 rows of 32 columns
  static constexpr uint32_t kSmem = kOut + kEpi * 2048 + 1024;
  static constexpr uint32_t kCols = 2 * BN;              // tensor memory: two accumulators
  static_assert(kStage % 1024 == 0 && kSmem <= 226 * 1024, "");
};

struct Args {
  CUtensorMap amap;   // dy [M][N], box 64 x 128, 128-byte swizzle
  CUtensorMap cmap;   // codes [N][pitch / 2], box BN / 4 bytes x 128
  const uint8_t* scales;
  const int32_t* tops;  // fp16: kTops maxima of scale bytes
  void* out;          // [M][K]
  int M, N, K, pieces;  // pieces of 128 columns
};

// Codes k and k + 4 of a word, at the low exponent bits.
template <int DT, int K4>
__device__ __forceinline__ uint32_t spread(uint32_t w) {
  constexpr int up = DT == RQ_BF16 ? 6 : 9;
  constexpr uint32_t magnitude = 0x00070007u << up;
  const uint32_t a = up > 4 * K4 ? w << (up - 4 * K4) : w >> (4 * K4 - up), s = K4 < 3 ? w << (12 - 4 * K4) : w;
  return (a & magnitude) | (s & 0x80008000u);
}

template <int DT>
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
  uint32_t d;
  if constexpr (DT == RQ_BF16) asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  else asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// What takes spread codes to values: in bf16 2^(byte - 1), in two steps (2^126
// first) where that leaves the range, in fp16 2^(14 + byte - top).
template <int DT>
__device__ __forceinline__ uint32_t factor(uint32_t byte, int top) {
  uint32_t f;
  if constexpr (DT == RQ_BF16) f = pack_rn<DT>(pow2_scale((int)byte, byte > 128u ? 127 : 1), 0.0f);
  else f = pack_rn<DT>(pow2_scale((int)byte, top) * 16384.0f, 0.0f);
  return f << 16 | f;
}

template <int DT, bool FAR>
__device__ __forceinline__ uint4 widen8(uint32_t w, uint32_t by) {
  uint4 v = make_uint4(spread<DT, 0>(w), spread<DT, 1>(w), spread<DT, 2>(w), spread<DT, 3>(w));
  if constexpr (FAR) {
    const uint32_t up = 0x7e807e80u;  // 2^126
    v = make_uint4(mul2<DT>(v.x, up), mul2<DT>(v.y, up), mul2<DT>(v.z, up), mul2<DT>(v.w, up));
  }
  return make_uint4(mul2<DT>(v.x, by), mul2<DT>(v.y, by), mul2<DT>(v.z, by), mul2<DT>(v.w, by));
}

// wait_pair by a warp: one try of all lanes where the phase is over already.
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, const PairAbort& ab, int lane) {
  if (__all_sync(0xffffffffu, mbar_test<false>(bar, parity))) return true;
  bool ok = true;
  if (lane == 0) ok = wait_pair(bar, parity, ab);
  return __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
}

// Largest scale byte but 255 of a CTA's share of n 16-byte pieces.
constexpr int kTops = 148;
static_assert(kTops * 4 <= RQ_MX4_DX_WORKSPACE, "");
__global__ void __launch_bounds__(512) mx4_tops_k(const uint4* __restrict__ scales, int64_t n, int32_t* __restrict__ tops) {
  grid_begin();
  uint32_t top = 0;
  for (int64_t i = (int64_t)blockIdx.x * 512 + threadIdx.x; i < n; i += kTops * 512) {
    const uint4 v = scales[i];
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) top = __vmaxu4(top, w[j] & ~__vcmpeq4(w[j], 0xffffffffu));
  }
  top = max(max(top & 255u, top >> 8 & 255u), max(top >> 16 & 255u, top >> 24));
  top = __reduce_max_sync(0xffffffffu, top);
  __shared__ uint32_t part[16];
  if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int i = 1; i < 16; ++i) top = max(top, part[i]);
    tops[blockIdx.x] = (int32_t)top;
  }
}
// The largest of them, by a warp.
__device__ __forceinline__ int top_of(const int32_t* tops, int lane) {
  int top = 0;
  for (int i = lane; i < kTops; i += 32) top = max(top, tops[i]);
  return __reduce_max_sync(0xffffffffu, top);
}

template <int DT, int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Plan<DT, BN>::kThreads, 1) mx4_dx_k(const __grid_constant__ Args g) {
  using PL = Plan<DT, BN>;
  using T = typename DType<DT>::T;
  constexpr int S = PL::S;
  extern __shared__ __align__(1024) unsigned char dsm[];
  // dy[S] (leader's: both CTAs' dy), codes[S] (own), read[S] (own codes are
  // widened), wide[S] (leader's: its widening warps, and a signal of the peer's
  // for each), empty[S], acc[2], taken[2] (leader's)
  __shared__ __align__(8) uint64_t bars[5 * S + 5];
  __shared__ uint32_t tmem_sh;
  __shared__ int abort_flag;
  __shared__ __align__(16) uint32_t sig_src[4], sig_dst[4];  // of the 16-byte signals (contents unused)
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const uint32_t rank = cluster_rank();
  const uint32_t sraw = smem_u32(dsm), sbase = (sraw + 1023u) & ~1023u;
  unsigned char* sm = dsm + (sbase - sraw);
  const uint32_t dy0 = smem_u32(bars), codes0 = dy0 + 8 * S, read0 = codes0 + 8 * S, wide0 = read0 + 8 * S,
                 empty0 = wide0 + 8 * S, acc0 = empty0 + 8 * S, taken0 = acc0 + 16, drainbar = taken0 + 16;
  const PairAbort ab{&abort_flag, mapa(smem_u32(&abort_flag), rank ^ 1u), &g_mx4_dx_timeouts};
  const int steps = (g.N + kRows - 1) / kRows;
  // tiles of the same tokens follow one another: dy, the larger operand, is read
  // from HBM once
  const int ct = (g.K + BN - 1) / BN, ntile = (g.M + 255) / 256 * ct;
  const int first = blockIdx.x / 2, stride = gridDim.x / 2;
  const int tiles = first < ntile ? (ntile - 1 - first) / stride + 1 : 0, total = tiles * steps;

  if (tid == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(dy0 + 8 * i, 1);
      mbar_init(codes0 + 8 * i, 1);
      mbar_init(read0 + 8 * i, kWiden);
      mbar_init(wide0 + 8 * i, kWiden);
      mbar_init(empty0 + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(acc0 + 8 * i, 1);
      mbar_init(taken0 + 8 * i, 2 * kEpi);
    }
    mbar_init(drainbar, 1);
    abort_flag = 0;
    for (int i = 0; i < 4; ++i) sig_src[i] = sig_dst[i] = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_sh)),
                 "r"(PL::kCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  cluster_sync();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmem_sh;
  grid_begin();

  if (warp == 0) {
    if (lane == 0) {
      // dy waits for the MMAs of its slot's stage before, the codes only for the
      // widening: they are loaded ahead
      const uint32_t lead = mapa(dy0, 0);
      int ahead = 0;
      bool ok = true;
      auto load_codes = [&](int i) {
        const int t = first + i / steps * stride, slot = i % S;
        mbar_expect_tx(codes0 + 8 * slot, PL::kCodes);
        tma_2d(sbase + slot * PL::kStage + PL::kC, &g.cmap, (t % ct * BN + (int)rank * PL::BNH) / 2, i % steps * kRows,
               codes0 + 8 * slot);
      };
      for (; ahead < S && ahead < total; ++ahead) load_codes(ahead);
      for (int i = 0; i < total && ok; ++i) {
        const int t = first + i / steps * stride, st = i % steps, slot = i % S;
        if (i >= S) ok = wait_pair(empty0 + 8 * slot, ((i / S) - 1) & 1, ab);
        if (!ok) break;
        const uint32_t at = sbase + slot * PL::kStage;
        const int m0 = t / ct * 256 + (int)rank * 128;
        if (rank == 0) mbar_expect_tx(dy0 + 8 * slot, 4 * kA);
        tma_pair(at, &g.amap, st * kRows, m0, lead + 8 * slot);
        tma_pair(at + kA, &g.amap, st * kRows + 64, m0, lead + 8 * slot);
        // the codes S stages after those that have been widened by now, or are
        // about to be: at most one stage ahead of dy's round
        if (ahead < total && ahead <= i + S) {
          ok = wait_pair(read0 + 8 * (ahead % S), ((ahead / S) - 1) & 1, ab);
          if (ok) load_codes(ahead++);
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      const uint32_t idesc = idesc_pair<DT, BN>(true);
      bool ok = true;
      for (int t = 0, i = 0; t < tiles && ok; ++t) {
        const uint32_t d = tmem + (uint32_t)(t & 1) * BN;
        if (t >= 2 && !wait_pair<true>(taken0 + 8 * (t & 1), ((t >> 1) - 1) & 1, ab)) break;
        for (int st = 0; st < steps; ++st, ++i) {
          const int slot = i % S;
          ok = wait_pair(dy0 + 8 * slot, (i / S) & 1, ab) && wait_pair<true>(wide0 + 8 * slot, (i / S) & 1, ab);
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t a = sbase + slot * PL::kStage, b = a + PL::kB;
#pragma unroll
          for (int k = 0; k < kRows / 16; ++k)
            mma_pair(d, sw128_desc(a + k / 4 * kA + k % 4 * 32), sw128_mn_desc(b + k * 2048, PL::kChunk), idesc,
                     (st > 0 || k > 0) ? 1u : 0u);
          mma_commit_pair(empty0 + 8 * slot, 3);
        }
        if (ok) mma_commit_pair(acc0 + 8 * (t & 1), 3);
      }
    }
  } else if (warp < PL::kEpi0) {
    // row 32 (w % 4) + lane of the stage, columns BN / 4 (w / 4) .. of the CTA's
    // half: the lanes of a store have 8 different units of the swizzle
    constexpr int U = BN / 32;  // 16-byte units, of 8 codes each
    constexpr int TM = PL::kTeams;
    const int w = (warp - 2) % kWiden, row = (w & 3) * 32 + lane, col = (w >> 2) * (BN / 4);
    const uint32_t store = PL::kB + col / 64 * PL::kChunk + row * 128;
    const int unit = col % 64 / 8;
    const int top = DT == RQ_F16 ? top_of(g.tops, lane) : 127;
    // codes: 16-byte pieces of a row of BN / 4 bytes, in the swizzle of their TMA box
    const uint32_t load = PL::kC + row * (BN / 4);
    const int swz = BN == 256 ? (row >> 1) & 3 : (row >> 2) & 1, piece = col / 32;
    const uint32_t wide = mapa(wide0, 0), sig_lead = mapa(smem_u32(sig_dst), 0);
    int i = (warp - 2) / kWiden;  // the team's next stage, of all
    bool ok = true;
    for (int n = 0; n < tiles && ok; ++n) {
      const int c = (first + n * stride) % ct * BN + (int)rank * PL::BNH + col;
      const bool any = c < g.pieces * 128;
      const uint8_t* p = g.scales + (int64_t)(c / 128) * 512 + (row % 32) * 16 + row / 32 * 4 + c % 128 / 32;
      auto scale = [&](int st) -> uint32_t {  // the scale bytes of this thread's columns
        if (!any || st >= steps) return 0u;
        const uint8_t* q = p + (int64_t)st * g.pieces * 512;
        return BN == 256 ? __ldg(reinterpret_cast<const uint16_t*>(q)) : __ldg(q);
      };
      int st = i - n * steps, slot = i % S;
      uint32_t round = (uint32_t)(i / S);  // how often the ring has gone round
      uint32_t s0 = scale(st), s1 = scale(st + TM), s2 = scale(st + 2 * TM);  // on their way
      for (; st < steps; st += TM, i += TM) {
        const uint32_t by[2] = {factor<DT>(s0 & 255u, top), BN == 256 ? factor<DT>(s0 >> 8, top) : 0u};
        // a scale above 2 in bf16 takes two steps
        const bool far[2] = {DT == RQ_BF16 && (s0 & 255u) > 128u, DT == RQ_BF16 && BN == 256 && (s0 >> 8) > 128u};
        s0 = s1;
        s1 = s2;
        s2 = scale(st + 3 * TM);
        // In this order: the stage before in this slot may have been another team's,
        // and a test of the codes' parity could take the round before that for this
        // one while its codes are still on their way.  Its MMAs are over, so they
        // are not.
        if (round > 0) ok = wait_warp(empty0 + 8 * slot, (round - 1) & 1, ab, lane);
        if (!ok) break;
        ok = wait_warp(codes0 + 8 * slot, round & 1, ab, lane);
        if (!ok) break;
        unsigned char* at = sm + slot * PL::kStage;
        uint4 cw[U / 4];
#pragma unroll
        for (int h = 0; h < U / 4; ++h) cw[h] = *reinterpret_cast<const uint4*>(at + load + (((piece + h) ^ swz) << 4));
#pragma unroll
        for (int h = 0; h < U / 4; ++h) {  // 32 columns, one scale
          const uint32_t word[4] = {cw[h].x, cw[h].y, cw[h].z, cw[h].w};
#pragma unroll
          for (int u = 0; u < 4; ++u)
            *reinterpret_cast<uint4*>(at + store + (((unit + 4 * h + u) ^ (row & 7)) << 4)) =
                far[h] ? widen8<DT, true>(word[u], by[h]) : widen8<DT, false>(word[u], by[h]);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // visible to the tensor cores
        __syncwarp();
        if (lane == 0) {
          // The leader's warps arrive and each expect the 16 bytes of a signal from one
          // of the peer's, whose values its MMAs read too.  A signal is a copy in the
          // proxy that the values were just made visible to, and its completion is
          // ordered for the cluster.  An arrival from the other CTA would need a release
          // at cluster scope, which waits for everything remote (dy 8192 x 11008 641
          // us with that, 533 with signals; one token's 4096 to 4096 43 and 25).
          if (rank == 0) mbar_expect_tx(wide0 + 8 * slot, 16);
          else bulk_signal(sig_lead, smem_u32(sig_src), wide + 8 * slot);
          // Only now: the values have been used, so the loads of the codes are over.
          // Said right after them, the next TMA copy overtook loads still in the
          // queue (an arrival waits for neither those nor for the other proxy).
          mbar_arrive(read0 + 8 * slot);
        }
        slot += TM;
        if (slot >= S) slot -= S, ++round;
      }
    }
  } else {
    const int quad = warp & 3;
    unsigned char* stage = sm + PL::kOut + (warp - PL::kEpi0) * 2048;
    const uint32_t took = mapa(taken0, 0);
    T* out = static_cast<T*>(g.out);
    const float back = DT == RQ_F16 ? pow2_scale(top_of(g.tops, lane), 127) : 1.0f;
    const bool rows16 = (uintptr_t)out % 16 == 0 && g.K % 8 == 0;
    for (int n = 0; n < tiles; ++n) {
      const int t = first + n * stride, m0 = t / ct * 256 + (int)rank * 128 + quad * 32, c0 = t % ct * BN;
      bool ok = true;
      if (lane == 0) ok = wait_pair(acc0 + 8 * (n & 1), (n >> 1) & 1, ab) && !ab.raised();
      if (!__shfl_sync(0xffffffffu, (int)ok, 0)) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
      for (int c = 0; c < BN; c += 32) {
        float acc[32];
        tmem_ld32(tmem + ((uint32_t)(quad * 32) << 16) + (uint32_t)(n & 1) * BN + c, acc);
        uint4 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const float* a = acc + 8 * u;  // columns 0, 4, 1, 5, 2, 6, 3, 7
          if constexpr (DT == RQ_F16) {
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[8 * u + j] *= back;
          }
          v[u] = make_uint4(pack_rn<DT>(a[0], a[2]), pack_rn<DT>(a[4], a[6]), pack_rn<DT>(a[1], a[3]), pack_rn<DT>(a[5], a[7]));
        }
        const int k = c0 + c;
        if (rows16) {
          if (m0 + lane < g.M) {
            T* to = out + (int64_t)(m0 + lane) * g.K + k;
#pragma unroll
            for (int u = 0; u < 4; ++u)
              if (k + 8 * u < g.K) reinterpret_cast<uint4*>(to)[u] = v[u];
          }
        } else {
          // rows that are not 16-byte aligned: a row a time, one column a lane
#pragma unroll
          for (int u = 0; u < 4; ++u)
            *reinterpret_cast<uint4*>(stage + lane * 64 + ((u ^ (lane >> 1 & 3)) << 4)) = v[u];
          __syncwarp();
#pragma unroll 1
          for (int r0 = 0; r0 < 32; r0 += 16) {
            T x[16];
#pragma unroll
            for (int r = 0; r < 16; ++r)
              x[r] = *reinterpret_cast<const T*>(stage + (r0 + r) * 64 + ((lane / 8 ^ (r >> 1 & 3)) << 4) + lane % 8 * 2);
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if (m0 + r0 + r < g.M && k + lane < g.K) out[(int64_t)(m0 + r0 + r) * g.K + k + lane] = x[r];
          }
          __syncwarp();
        }
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) arrive_cluster(took + 8 * (n & 1));
    }
  }

  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  cluster_sync();  // no copy, commit or arrive can reach a CTA that has left
  if (tid == 0 && ab.raised()) {
    // after a wait that ran out: this pair's MMAs (bounded), and time for
    // copies and arrives under way to land
    if (rank == 0) {
      mma_commit_pair(drainbar, 1);
      drain(drainbar, 0);
    }
    const uint64_t t0 = gtimer_ns();
    while (gtimer_ns() - t0 < 200000) __nanosleep(1000);
  }
  __syncthreads();
  cluster_sync();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(PL::kCols) : "memory");
}

template <int DT, int BN>
int run(const void* dy, int64_t ld, int64_t M, const Mx4& w, int64_t K, void* dx, void* ws, cudaStream_t st) {
  Args g;
  const int64_t pitch = mx4_pitch(K);
  {
    const uint64_t d[3] = {(uint64_t)w.rows, (uint64_t)M, 1}, s[2] = {(uint64_t)ld * 2, 0};
    const uint32_t b[3] = {64, 128, 1};
    const int rc = tensor_map_encode(CU_TENSOR_MAP_DATA_TYPE_UINT16, CU_TENSOR_MAP_SWIZZLE_128B, 2, dy, d, s, b, &g.amap);
    if (rc != RQ_OK) return rc;
  }
  {
    const uint64_t d[3] = {(uint64_t)pitch / 2, (uint64_t)w.rows, 1}, s[2] = {(uint64_t)pitch / 2, 0};
    const uint32_t b[3] = {BN / 4, kRows, 1};
    const int rc = tensor_map_encode(CU_TENSOR_MAP_DATA_TYPE_UINT8,
                                     BN == 256 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B, 2, w.codes, d, s,
                                     b, &g.cmap);
    if (rc != RQ_OK) return rc;
  }
  g.scales = w.scales;
  g.tops = static_cast<const int32_t*>(ws);
  g.out = dx;
  g.M = (int)M;
  g.N = (int)w.rows;
  g.K = (int)K;
  g.pieces = (int)(pitch / 128);
  const void* kern = (const void*)mx4_dx_k<DT, BN>;
  const int rc = ensure_smem_limit(kern, Plan<DT, BN>::kSmem);
  if (rc != RQ_OK) return rc;
  const int64_t ntile = ((M + 255) / 256) * ((K + BN - 1) / BN), pairs = num_sms() / 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * (ntile < pairs ? ntile : pairs)));
  cfg.blockDim = dim3(Plan<DT, BN>::kThreads);
  cfg.dynamicSmemBytes = Plan<DT, BN>::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = 2;
  at[1].val.clusterDim.y = 1;
  at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  void* params[] = {&g};
  const cudaError_t e = cudaLaunchKernelExC(&cfg, kern, params);
  if (e != cudaSuccess) {
    set_cuda_error(e);
    return RQ_ERR_CUDA;
  }
  return check_launch();
}

}  // namespace

// 256 columns a tile, or 128 where twice the tiles still fit one round: an MMA of
// 128 columns takes about as long (it reads as much of dy), so a second round of
// them costs more than idle SMs.
int mx4_dx(const void* dy, int dt, int64_t ld, int64_t M, const Mx4& w, int64_t K, void* dx, void* ws, cudaStream_t st) {
  const bool wide = 2 * ((M + 255) / 256) * ((K + 255) / 256) > num_sms() / 2;
  if (dt == RQ_BF16)
    return wide ? run<RQ_BF16, 256>(dy, ld, M, w, K, dx, ws, st) : run<RQ_BF16, 128>(dy, ld, M, w, K, dx, ws, st);
  const int64_t pieces = (w.rows + 127) / 128 * (mx4_pitch(K) / 128) * 32;
  const int rc = launch_dependent(mx4_tops_k, kTops, 512, st, reinterpret_cast<const uint4*>(w.scales), pieces,
                                  static_cast<int32_t*>(ws));
  if (rc != RQ_OK) return rc;
  return wide ? run<RQ_F16, 256>(dy, ld, M, w, K, dx, ws, st) : run<RQ_F16, 128>(dy, ld, M, w, K, dx, ws, st);
}

}  // namespace rq

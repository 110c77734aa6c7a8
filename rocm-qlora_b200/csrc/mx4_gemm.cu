// mx4_gemm.cu -- products of two operands in microscaled 4 bits on the
// block-scaled tensor cores:  out[m, n] = sum_k a[m, k] b[n, k] (+ bias[n]).
//
// tcgen05.mma kind::mxf4 multiplies e2m1 codes of two K-major tiles from shared
// memory, each block of 32 codes with its power-of-two scale from tensor
// memory, and sums in fp32 in tensor memory: 4 times the rate of 16-bit
// operands, and no value is ever unpacked.
//
// Codes come to a ring of stages by TMA, 128 bytes (256 columns) of a row with
// 128-byte swizzle; scales are pieces of 512 bytes (128 rows x 128 columns,
// stored in the order that tensor memory takes), 4 columns of tensor memory each.
// Every slot of the ring has scale columns of its own, so none is overwritten in
// use.  Warp 0 loads (one thread), warp 1 has the tensor memory and issues the
// MMAs (one thread), 8 epilogue warps share the 32 rows of a lane quarter by twos.
// Two kernels:
//   mx4_pair_k   many tiles.  CTA pairs stay and take tiles of 256 tokens x 256
//                outputs in turn (2-SM MMAs; a CTA loads its 128 tokens and half
//                of the outputs).  The epilogue empties the accumulator into
//                registers, and the next tile's MMAs run while it stores.  Bound
//                by the tensor cores: 8192 x 4096 -> 11008 in bf16 takes 145 us,
//                5.1 PFLOP/s (MMA pipe 66 % active; 4096 x 4096 -> 4096, whose
//                3.5 rounds of tiles take four, 32 us).
//   mx4_split_k  few tiles.  P are outputs, Q up to 128 tokens, and a cluster
//                splits the columns: each CTA parks its sums in shared memory,
//                and all add up a share in rank order (fixed order: deterministic).
//                Bound by latency: 64 x 4096 -> 11008 takes 11.0 us, 3.4 of
//                them the weight's bytes at the copy bandwidth; one token x
//                4096 -> 4096 6.3.
// Waits are bounded: one that runs out counts a kernel timeout, the CTAs drain
// their copies, and mx4_pair_k stores nothing more, mx4_split_k NaNs (other CTAs
// of the cluster add up what this one should have had).
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>

#include "gemv_common.cuh"
#include "mx4_common.cuh"
#include "rq_internal.h"
#include "tcgen05_common.cuh"

namespace rq {

__device__ unsigned int g_mx4_timeouts;

int mx4_take_timeouts(unsigned int* v) {
  unsigned int zero = 0;
  cudaError_t e = cudaMemcpyFromSymbol(v, g_mx4_timeouts, sizeof(*v));
  if (e == cudaSuccess) e = cudaMemcpyToSymbol(g_mx4_timeouts, &zero, sizeof(zero));
  if (e != cudaSuccess) {
    set_cuda_error(e);
    return RQ_ERR_CUDA;
  }
  return RQ_OK;
}

namespace {

constexpr int kEpiWarps = 8;
constexpr int kThreads = 64 + 32 * kEpiWarps;
constexpr uint32_t kP = 128;                  // rows of P a tile
constexpr uint32_t kPBytes = kP * 128;        // codes of a stage: 256 columns
constexpr uint32_t kPiece = 512;

constexpr int kPark = 132;                    // floats of a token's parked sums

// PACK: Q's rows come in 16 bits and are packed by the epilogue warps, for all of
// the CTA's stages (beside the ring), while the first of P's are on their way.
template <int BN, bool PACK>
struct Plan {
  static constexpr int NB = (BN + 127) / 128;                       // scale pieces of Q a 128 columns
  static constexpr uint32_t kQCodes = BN * 128, kQScales = 2 * NB * kPiece;  // [piece][128 columns]
  static constexpr uint32_t kQStage = kQCodes + kQScales;
  static constexpr uint32_t kSP = kPBytes;                          // P's scale pieces in a stage
  static constexpr uint32_t kQ = kSP + 2 * kPiece;                  // Q's codes, then scales
  static constexpr uint32_t kStage = kQ + (PACK ? 0 : kQStage);
  // two CTAs an SM
  static constexpr int kStages = BN == 128 ? 3 : 4;
  static constexpr uint32_t kRed = BN * kPark * 4;                  // parked sums, in the ring's place
  static constexpr uint32_t kRing = kStages * kStage;
  static constexpr uint32_t kSmem = (kRing > kRed ? kRing : kRed) + 1024;
  static constexpr uint32_t kAcc = BN < 32 ? 32 : BN;               // accumulator columns
  static constexpr uint32_t kSlotCols = 2 * (4 + 4 * NB);           // scale columns of a slot
  static constexpr uint32_t kNeed = kAcc + kStages * kSlotCols;
  static constexpr uint32_t kCols = kNeed <= 128 ? 128 : 256;
  static_assert(kNeed <= 256 && kStage % 1024 == 0 && kQStage % 1024 == 0 && kRed <= kRing && kSmem <= 113 * 1024, "");
};

struct Args {
  CUtensorMap pmap, qmap;   // codes [rows][pitch / 2], boxes 128 bytes x 128 and x BN
  const uint8_t* pscales;
  const uint8_t* qscales;
  const void* bias;
  void* out;
  int prows, qrows, tiles;  // tiles: pieces of 128 columns
  int64_t ld;
  const void* x;            // PACK: Q's rows [qrows, K]
  int64_t ldx;
  int K;
  uint64_t limit;           // of a wait, in ns; 0: has run out before it begins
  bool vec;
  bool early;               // the kernel before this one is the packing of Q's rows, which has itself waited for
                            // all before it: P is there already
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// 32 rows of 16 bytes (8-row groups 128 bytes apart, no swizzle) to 4 columns
// of all four lane quarters.
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint32_t saddr) {
  const uint64_t d = (uint64_t)((saddr >> 4) & 0x3FFF) | (uint64_t)1 << 16 | (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46;
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(d) : "memory");
}

// e2m1 operands, power-of-two scales; `half`: which two of a word's
// four scale bytes the 64 columns take.
template <int M, int N>
__device__ __forceinline__ uint32_t idesc_mx4(uint32_t half) {
  return (1u << 7) | (1u << 10) | ((uint32_t)(N >> 3) << 17) | (1u << 23) | ((uint32_t)(M >> 7) << 27) | (2 * half) << 4 |
         (2 * half) << 29;
}
#define RQ_MMA_MX4(group)                                                                                          \
  asm volatile(                                                                                                    \
      "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"                                                               \
      " tcgen05.mma.cta_group::" group ".kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}\n" \
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accum)                                           \
      : "memory")
template <int CTAS>
__device__ __forceinline__ void mma_mx4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb,
                                        uint32_t accum) {
  if constexpr (CTAS == 1) RQ_MMA_MX4("1");
  else RQ_MMA_MX4("2");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile int* abort, uint64_t limit) {
  if (mbar_try<false>(bar, parity)) return true;
  const uint64_t t0 = gtimer_ns();
  while (!*abort) {
    if (mbar_try<false>(bar, parity)) return true;
    if (gtimer_ns() - t0 > limit) {
      *abort = 1;
      atomicAdd(&g_mx4_timeouts, 1u);
      return false;
    }
  }
  return false;
}
// out[q, p] (tokens Q, outputs P): sums of its share of the columns.
template <int DT, int BN, bool PACK>
__global__ void __launch_bounds__(kThreads, 2) mx4_split_k(const __grid_constant__ Args g) {
  using PL = Plan<BN, PACK>;
  using T = typename DType<DT>::T;
  constexpr int S = PL::kStages, NB = PL::NB;
  extern __shared__ __align__(1024) unsigned char dsm[];
  __shared__ __align__(8) uint64_t bars[2 * S + 2];
  __shared__ uint32_t tmem_sh;
  __shared__ int abort_flag, issued, consumed;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const uint32_t sraw = smem_u32(dsm), sbase = (sraw + 1023u) & ~1023u;
  unsigned char* sm = dsm + (sbase - sraw);
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * S, accbar = empty0 + 8 * S, qbar = accbar + 8;
  volatile int* abort = &abort_flag;
  const int q0 = blockIdx.x * BN, p0 = blockIdx.y * (int)kP;
  const int sk = gridDim.z, rank = blockIdx.z;
  const int steps = (g.tiles + 1) / 2;
  const int s0 = steps * rank / sk, s1 = steps * (rank + 1) / sk;

  if (tid == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(full0 + 8 * i, 1);
      mbar_init(empty0 + 8 * i, 1);
    }
    mbar_init(accbar, 2);
    mbar_init(qbar, kEpiWarps);
    issued = consumed = 0;
    abort_flag = g.limit == 0;
    if (g.limit == 0) atomicAdd(&g_mx4_timeouts, 1u);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_sh)),
                 "r"(PL::kCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = tmem_sh;
  if (warp > 0 || !g.early) grid_begin();

  if (warp == 0) {
    const uint8_t* ps = g.pscales + (int64_t)(p0 / 128) * g.tiles * kPiece;
    const uint8_t* qs = g.qscales + (int64_t)(q0 / 128) * g.tiles * kPiece;
    const int qpieces = min(NB, (g.qrows + 127) / 128 - q0 / 128);  // pieces past the last row do not exist
    auto load_p = [&](int st, int slot) {
      const uint32_t at = sbase + slot * PL::kStage, bar = full0 + 8 * slot;
      const uint32_t bytes = (uint32_t)min(2, g.tiles - 2 * st) * kPiece;
      mbar_expect_tx(bar, PACK ? kPBytes + bytes : kPBytes + PL::kQCodes + (1 + qpieces) * bytes);
      tma_2d(at, &g.pmap, st * 128, p0, bar);
      bulk_load(at + PL::kSP, ps + (int64_t)st * 2 * kPiece, bytes, bar);
    };
    const int early = g.early ? min(S, s1 - s0) : 0;
    if (g.early) {
      if (lane == 0)
        for (int i = 0; i < early; ++i) load_p(s0 + i, i);
      __syncwarp();
      grid_begin();
    }
    if (lane == 0) {
      for (int st = s0; st < s1; ++st) {
        const int i = st - s0, slot = i % S;
        if (i >= S && !wait(empty0 + 8 * slot, ((i / S) - 1) & 1, abort, g.limit)) break;
        if (i >= early) load_p(st, slot);
        if constexpr (!PACK) {
          const uint32_t at = sbase + slot * PL::kStage, bar = full0 + 8 * slot;
          const uint32_t bytes = (uint32_t)min(2, g.tiles - 2 * st) * kPiece;
          tma_2d(at + PL::kQ, &g.qmap, st * 128, q0, bar);
          for (int j = 0; j < qpieces; ++j)
            bulk_load(at + PL::kQ + PL::kQCodes + j * 2 * kPiece, qs + ((int64_t)j * g.tiles + st * 2) * kPiece, bytes, bar);
        }
        *reinterpret_cast<volatile int*>(&issued) = i + 1;
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const bool packed = !PACK || wait(qbar, 0, abort, g.limit);
      for (int st = s0; st < s1 && packed; ++st) {
        const int i = st - s0, slot = i % S;
        if (!wait(full0 + 8 * slot, (i / S) & 1, abort, g.limit)) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t at = sbase + slot * PL::kStage, q = PACK ? sbase + PL::kRing + i * PL::kQStage : at + PL::kQ, tsc = tmem + PL::kAcc + slot * PL::kSlotCols;
        const int nt = min(2, g.tiles - 2 * st);
        for (int t = 0; t < nt; ++t) {
          const uint32_t tp = tsc + t * (PL::kSlotCols / 2), tq = tp + 4;
          copy_scales(tp, at + PL::kSP + t * kPiece);
#pragma unroll
          for (int j = 0; j < NB; ++j) copy_scales(tq + 4 * j, q + PL::kQCodes + (2 * j + t) * kPiece);
#pragma unroll
          for (int h = 0; h < 2; ++h)
            mma_mx4<1>(tmem, sw128_desc(at + (2 * t + h) * 32), sw128_desc(q + (2 * t + h) * 32),
                       idesc_mx4<128, BN>(h), tp, tq, (i > 0 || t > 0 || h > 0) ? 1u : 0u);
        }
        mma_commit(empty0 + 8 * slot);
        *reinterpret_cast<volatile int*>(&consumed) = i + 1;
      }
      mma_commit(accbar);
      mbar_arrive(accbar);  // whoever sees the barrier sees an abort before it too
    }
  } else if constexpr (PACK) {
    // a warp packs the 256 columns of a token's stage: 8 values a lane, a code
    // row of 128 bytes in the swizzle of the TMA tiles
    const T* x = static_cast<const T*>(g.x);
    const int rows = min(BN, g.qrows - q0);
    for (int e = warp - 2; e < (s1 - s0) * rows; e += kEpiWarps) {
      const int i = e / rows, r = e % rows;
      unsigned char* q = sm + PL::kRing + i * PL::kQStage;
      const T* row = x + (int64_t)(q0 + r) * g.ldx;
      const int col = (s0 + i) * 256 + lane * 8;
      const M4Raw<DT> raw[1] = {g.vec ? m4_load<DT, 16>(row, col, g.K) : m4_load<DT, 0>(row, col, g.K)};
      uint32_t top[1];
      m4_top<DT, 8, 1>(raw, top);
      const uint32_t byte = m4_scale(top[0]);
      float v[8];
      m4_values<DT, 8>(raw[0], v);
      *reinterpret_cast<uint32_t*>(q + r * 128 + ((lane / 4 ^ (r & 7)) << 4) + lane % 4 * 4) = e2m1x8(v, m4_factor(byte));
      uint32_t word = byte << (lane % 16 / 4 * 8);
      word |= __shfl_xor_sync(0xffffffffu, word, 4);
      word |= __shfl_xor_sync(0xffffffffu, word, 8);
      if (lane % 16 == 0)
        *reinterpret_cast<uint32_t*>(q + PL::kQCodes + lane / 16 * kPiece + r / 128 * 2 * kPiece + r % 32 * 16 + r % 128 / 32 * 4) = word;
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // visible to the tensor cores
    __syncwarp();
    if (lane == 0) mbar_arrive(qbar);
  }
  __syncwarp();

  const int quad = warp & 3, row = quad * 32 + lane;  // of the tile, epilogue warps
  const int c_lo = BN >= 64 ? ((warp - 2) >> 2) * (BN / 2) : 0, c_hi = BN >= 64 ? c_lo + BN / 2 : BN;
  const bool has_bias = g.bias != nullptr;
  T* out = static_cast<T*>(g.out);
  bool ok = false;
  if (warp >= 2) {
    if (lane == 0) ok = wait(accbar, 0, abort, g.limit) && !*abort;
    ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  }
  if (warp >= 2 && (BN >= 64 || warp < 6)) {
    float* red = reinterpret_cast<float*>(sm);
    const int n = p0 + row;
    const float bv = has_bias && n < g.prows ? DType<DT>::to_f32(static_cast<const T*>(g.bias)[n]) : 0.0f;
    for (int c = c_lo; c < c_hi; c += 32) {
      float acc[32];
      tmem_ld32(tmem + ((uint32_t)(quad * 32) << 16) + c, acc);
      if (sk > 1) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (c + j < BN && ok) red[(c + j) * kPark + row] = acc[j];
      } else {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (c + j < BN && q0 + c + j < g.qrows && n < g.prows)
            out[(int64_t)(q0 + c + j) * g.ld + n] = DType<DT>::from_f32(ok ? acc[j] + bv : __uint_as_float(0x7fc00000u));
      }
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (warp == 1) {
    if (lane == 0 && *abort) {
      drain(accbar, 0);
      const int done = *reinterpret_cast<volatile int*>(&consumed), n = *reinterpret_cast<volatile int*>(&issued);
      for (int i = done; i < n; ++i) drain(full0 + 8 * (i % S), (i / S) & 1);
    }
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(PL::kCols) : "memory");
  }
  if (sk > 1) {
    if (*abort) {  // the same for all threads since their last barrier
      __syncthreads();  // copies under way have been drained
      for (int i = tid; i < BN * kPark; i += kThreads) reinterpret_cast<uint32_t*>(sm)[i] = 0x7fc00000u;
    }
    __syncwarp();
    cluster_sync();  // all sums are parked
    // this CTA's share: groups of 4 outputs of a token, the loads of all ranks at once
    const uint32_t red = smem_u32(sm);
    const int groups = min(BN, g.qrows - q0) * 32;
    for (int e = groups * rank / sk + tid; e < groups * (rank + 1) / sk; e += kThreads) {
      const int t = e / 32, o = e % 32 * 4, n = p0 + o;
      if (n >= g.prows) continue;
      float4 v[8];
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (r < sk)
          asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                       : "=f"(v[r].x), "=f"(v[r].y), "=f"(v[r].z), "=f"(v[r].w)
                       : "r"(mapa(red + (t * kPark + o) * 4, (uint32_t)r)));
      float sum[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
#pragma unroll
      for (int r = 1; r < 8; ++r)
        if (r < sk) sum[0] += v[r].x, sum[1] += v[r].y, sum[2] += v[r].z, sum[3] += v[r].w;
      if (has_bias) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n + j < g.prows) sum[j] += DType<DT>::to_f32(static_cast<const T*>(g.bias)[n + j]);
      }
      T* to = out + (int64_t)(q0 + t) * g.ld + n;
      if (n + 4 <= g.prows && (uintptr_t)to % 8 == 0) {
        *reinterpret_cast<uint2*>(to) = make_uint2(pack_rn<DT>(sum[0], sum[1]), pack_rn<DT>(sum[2], sum[3]));
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n + j < g.prows) to[j] = DType<DT>::from_f32(sum[j]);
      }
    }
    __syncwarp();
    cluster_sync();  // shared memory stays until the others have read it
  }
}

// ------------------------------------------------------------- CTA pairs

namespace pair {
// A stage holds 512 columns here: a wait or a commit costs the tensor pipe about
// 100 cycles, next to the 1082 of a stage's 8 MMAs.  Four warps store the scales
// to tensor memory, from registers: as copies (tcgen05.cp) between the MMAs a
// stage's 12 pieces cost the pipe about 960 cycles more, since one copy at a time
// overlaps an MMA (8192 x 4096 -> 11008: 214 us with copies, 188 with stores,
// both with stages of 256 columns; 145 with stages of 512).
constexpr int S = 3;
constexpr uint32_t kCodes = 128 * 128;                      // 256 columns of P's or of half of Q's rows
constexpr uint32_t kStage = 4 * kCodes;                     // P's two, Q's two
constexpr uint32_t kOutWarp = 32 * 128;                     // staged: 32 rows of 64 outputs
constexpr uint32_t kSmem = S * kStage + kEpiWarps * kOutWarp + 1024;
constexpr uint32_t kSlotCols = 4 * 12;                      // scales: for each 128 columns P's 4 and Q's 8
constexpr int kScaleWarps = 4, kEpi0 = 2 + kScaleWarps;     // first epilogue warp
constexpr int kThreads = 32 * (kEpi0 + kEpiWarps);
constexpr int kAhead = 2;                                   // stages of scales on their way in registers
static_assert(kSmem <= 226 * 1024 && 256 + S * kSlotCols <= 512, "");
}  // namespace pair

struct PairArgs {
  CUtensorMap pmap, qmap;    // codes, boxes 128 bytes x 128 rows
  const uint8_t* pscales;
  const uint8_t* qscales;
  const void* bias;
  void* out;
  int prows, qrows, tiles;
  int64_t ld;
};

// 12 columns of this thread's lane
__device__ __forceinline__ void tmem_st12(uint32_t taddr, const uint4 (&v)[3]) {
#pragma unroll
  for (int i = 0; i < 3; ++i)
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr + 4 * i), "r"(v[i].x),
                 "r"(v[i].y), "r"(v[i].z), "r"(v[i].w)
                 : "memory");
}

// out[p, q]: P tokens, Q outputs.
template <int DT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(pair::kThreads, 1) mx4_pair_k(const __grid_constant__ PairArgs g) {
  using namespace pair;
  using T = typename DType<DT>::T;
  extern __shared__ __align__(1024) unsigned char dsm[];
  // full[S] (leader's: both CTAs' codes have landed and scales are in both
  // tensor memories), empty[S], acc (sums complete), taken (leader's: both
  // CTAs' epilogues have read them)
  __shared__ __align__(8) uint64_t bars[2 * S + 3];
  __shared__ uint32_t tmem_sh;
  __shared__ int abort_flag;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const uint32_t rank = cluster_rank();
  const uint32_t sraw = smem_u32(dsm), sbase = (sraw + 1023u) & ~1023u;
  unsigned char* sm = dsm + (sbase - sraw);
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * S, accbar = empty0 + 8 * S, taken = accbar + 8,
                 drainbar = taken + 8, lead = mapa(full0, 0);
  const PairAbort ab{&abort_flag, mapa(smem_u32(&abort_flag), rank ^ 1u), &g_mx4_timeouts};
  const int steps = (g.tiles + 3) / 4;
  const int pt = (g.prows + 255) / 256, qt = (g.qrows + 255) / 256, ntile = pt * qt;
  const int first = blockIdx.x / 2, stride = gridDim.x / 2;
  const int total = first < ntile ? ((ntile - 1 - first) / stride + 1) * steps : 0;  // stages

  if (tid == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(full0 + 8 * i, 1 + 2 * kScaleWarps);
      mbar_init(empty0 + 8 * i, 1);
    }
    mbar_init(accbar, 1);
    mbar_init(taken, 2 * kEpiWarps);
    mbar_init(drainbar, 1);
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_sh)), "r"(512)
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
      int i = 0;
      bool ok = true;
      for (int t = first; t < ntile && ok; t += stride) {
        const int p0 = t % pt * 256 + (int)rank * 128, qh = t / pt * 256 + (int)rank * 128;
        for (int st = 0; st < steps; ++st, ++i) {
          const int slot = i % S;
          if (i >= S && !wait_pair(empty0 + 8 * slot, ((i / S) - 1) & 1, ab)) {
            ok = false;
            break;
          }
          const uint32_t at = sbase + slot * kStage, bar = lead + 8 * slot;
          if (rank == 0) mbar_expect_tx(full0 + 8 * slot, 2 * kStage);
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            tma_pair(at + j * kCodes, &g.pmap, st * 256 + j * 128, p0, bar);
            tma_pair(at + (2 + j) * kCodes, &g.qmap, st * 256 + j * 128, qh, bar);
          }
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      int i = 0, done = 0;  // stages, tiles
      bool ok = true;
      for (int t = first; t < ntile && ok; t += stride, ++done) {
        if (done > 0 && !wait_pair<true>(taken, (done - 1) & 1, ab)) break;
        for (int st = 0; st < steps; ++st, ++i) {
          const int slot = i % S;
          if (!wait_pair<true>(full0 + 8 * slot, (i / S) & 1, ab)) {
            ok = false;
            break;
          }
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t at = sbase + slot * kStage, tsc = tmem + 256 + slot * kSlotCols;
          const int nt = min(4, g.tiles - 4 * st);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (k < nt)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint32_t a = at + (k / 2) * kCodes + (k % 2 * 2 + h) * 32;
                mma_mx4<2>(tmem, sw128_desc(a), sw128_desc(a + 2 * kCodes), idesc_mx4<256, 256>(h), tsc + k * 12,
                           tsc + k * 12 + 4, (st > 0 || k > 0 || h > 0) ? 1u : 0u);
              }
          mma_commit_pair(empty0 + 8 * slot, 3);
        }
        if (ok) mma_commit_pair(accbar, 3);
      }
    }
  } else if (warp < kEpi0) {
    // ------------------------- scales to this warp's quarter of the lanes:
    // lane l has 4 bytes of row l of each group of 32 rows.  Pieces past the
    // last row or column are not read; what they would scale is 0 or not stored.
    const uint32_t quarter = (uint32_t)((warp & 3) * 32) << 16;
    struct Scales {
      uint4 v[4][3];
    };
    int ft = first, fs = 0;  // tile and stage of the next load
    auto fetch = [&](Scales& x) {
      if (ft >= ntile) return;
      const int p0 = ft % pt * 256 + (int)rank * 128, q0 = ft / pt * 256;
      const int rows[3] = {p0, q0, q0 + 128}, most[3] = {g.prows, g.qrows, g.qrows};
#pragma unroll
      for (int j = 0; j < 3; ++j) {
        const uint8_t* from = (j == 0 ? g.pscales : g.qscales) + ((int64_t)(rows[j] / 128) * g.tiles + 4 * fs) * kPiece +
                              lane * 16;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          x.v[k][j] = rows[j] < most[j] && 4 * fs + k < g.tiles ? __ldg(reinterpret_cast<const uint4*>(from + k * kPiece))
                                                                 : make_uint4(0u, 0u, 0u, 0u);
      }
      if (++fs == steps) fs = 0, ft += stride;
    };
    Scales ring[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) fetch(ring[j]);
    bool ok = true;
    for (int i0 = 0; i0 < total && ok; i0 += kAhead) {
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int i = i0 + j, slot = i % S;
        if (!ok || i >= total) break;
        if (i >= S) {
          if (lane == 0) ok = wait_pair(empty0 + 8 * slot, ((i / S) - 1) & 1, ab);
          ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        }
        const uint32_t to = tmem + quarter + 256 + slot * kSlotCols;
#pragma unroll
        for (int k = 0; k < 4; ++k) tmem_st12(to + 12 * k, ring[j].v[k]);
        fetch(ring[j]);
        asm volatile("tcgen05.wait::st.sync.aligned;\n\ttcgen05.fence::before_thread_sync;" ::: "memory");
        if (lane == 0) arrive_cluster(lead + 8 * slot);
      }
    }
  } else {
    const int quad = warp & 3, half = (warp - kEpi0) >> 2;
    unsigned char* stage = sm + S * kStage + (warp - kEpi0) * kOutWarp;
    const uint32_t took = mapa(taken, 0);
    T* out = static_cast<T*>(g.out);
    const bool rows16 = (uintptr_t)out % 16 == 0 && g.ld % 8 == 0;
    int done = 0;
    for (int t = first; t < ntile; t += stride, ++done) {
      const int p0 = t % pt * 256 + (int)rank * 128 + quad * 32, q0 = t / pt * 256 + half * 128;
      // 128 outputs' bias in this warp's staging, while it waits: as shuffles of a lane's
      // values they held up the next tile's MMAs (8192 x 4096 -> 11008 with bias 164 us,
      // now 150; without 145)
      if (g.bias) {
#pragma unroll
        for (int j = 0; j < 128; j += 32) {
          const int q = q0 + j + lane;
          reinterpret_cast<float*>(stage)[j + lane] =
              q < g.qrows ? DType<DT>::to_f32(static_cast<const T*>(g.bias)[q]) : 0.0f;
        }
        __syncwarp();
      }
      bool ok = true;
      if (lane == 0) ok = wait_pair(accbar, done & 1, ab) && !ab.raised();
      if (!__shfl_sync(0xffffffffu, (int)ok, 0)) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      uint4 w[16];  // this lane's row: 128 outputs, 8 a piece
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float acc[32];
        tmem_ld32(tmem + ((uint32_t)(quad * 32) << 16) + half * 128 + c * 32, acc);
        if (g.bias) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float4 b = reinterpret_cast<const float4*>(stage)[c * 8 + j];
            acc[4 * j] += b.x, acc[4 * j + 1] += b.y, acc[4 * j + 2] += b.z, acc[4 * j + 3] += b.w;
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
          w[4 * c + j] =
              make_uint4(pack_rn<DT>(acc[8 * j], acc[8 * j + 1]), pack_rn<DT>(acc[8 * j + 2], acc[8 * j + 3]),
                         pack_rn<DT>(acc[8 * j + 4], acc[8 * j + 5]), pack_rn<DT>(acc[8 * j + 6], acc[8 * j + 7]));
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) arrive_cluster(took);  // the accumulator is free for the next tile
      // through shared memory, 64 outputs at a time, to stores of whole 128-byte
      // row pieces; piece j of row r is at j ^ (r % 8)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
          *reinterpret_cast<uint4*>(stage + lane * 128 + ((j ^ (lane & 7)) << 4)) = w[8 * h + j];
        __syncwarp();
        if (rows16) {
          const int q = q0 + h * 64 + lane % 8 * 8;
#pragma unroll
          for (int r0 = 0; r0 < 32; r0 += 4) {
            const int r = r0 + lane / 8;
            const uint4 v = *reinterpret_cast<const uint4*>(stage + r * 128 + ((lane % 8 ^ (r & 7)) << 4));
            if (p0 + r < g.prows && q < g.qrows) *reinterpret_cast<uint4*>(out + (int64_t)(p0 + r) * g.ld + q) = v;
          }
        } else {
          // one output a lane, 8 rows' loads before their stores
          const int q = q0 + h * 64 + lane;
#pragma unroll 1
          for (int r0 = 0; r0 < 32; r0 += 8) {
            T v[8][2];
#pragma unroll
            for (int r = 0; r < 8; ++r)
#pragma unroll
              for (int j = 0; j < 2; ++j)
                v[r][j] = *reinterpret_cast<const T*>(stage + (r0 + r) * 128 + ((j * 4 + lane / 8 ^ r) << 4) + lane % 8 * 2);
#pragma unroll
            for (int r = 0; r < 8; ++r)
#pragma unroll
              for (int j = 0; j < 2; ++j)
                if (p0 + r0 + r < g.prows && q + 32 * j < g.qrows) out[(int64_t)(p0 + r0 + r) * g.ld + q + 32 * j] = v[r][j];
          }
        }
        __syncwarp();  // the staged rows are read before the next ones are written
      }
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
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// ------------------------------------------------------------------- host

int launch(const void* kern, uint32_t smem, dim3 grid, int threads, dim3 cluster, const void* args, cudaStream_t st) {
  const int rc = ensure_smem_limit(kern, smem);
  if (rc != RQ_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = cluster.x;
  at[1].val.clusterDim.y = cluster.y;
  at[1].val.clusterDim.z = cluster.z;
  cfg.attrs = at;
  cfg.numAttrs = cluster.x * cluster.z > 1 ? 2 : 1;
  void* params[] = {const_cast<void*>(args)};
  const cudaError_t e = cudaLaunchKernelExC(&cfg, kern, params);
  if (e != cudaSuccess) {
    set_cuda_error(e);
    return RQ_ERR_CUDA;
  }
  return check_launch();
}

int code_map(const Mx4& x, int64_t pitch, uint32_t rows, CUtensorMap* map) {
  const uint64_t d[3] = {(uint64_t)pitch / 2, (uint64_t)x.rows, 1}, s[2] = {(uint64_t)pitch / 2, 0};
  const uint32_t b[3] = {128, rows, 1};
  return tensor_map_encode(CU_TENSOR_MAP_DATA_TYPE_UINT8, CU_TENSOR_MAP_SWIZZLE_128B, 2, x.codes, d, s, b, map);
}

// Few tokens: the columns are split until two CTAs an SM have work, with at least
// two stages each of 16 or 32 tokens, four of 64, eight of 128: more sums to add
// up cost more than they save (1111 x 1093 -> 1089, 5 stages of 128 tokens: 7.8
// us whole and 8.7 in halves; 64 x 4096 -> 11008, 16 stages: 12.6 whole, 11.0 in
// thirds; 16 tokens 11.7 and 9.5).
int split_for(int64_t tiles, int64_t steps, int bn) {
  const int64_t room = 2 * num_sms() / tiles, most = steps / (bn <= 32 ? 2 : bn / 16);
  const int64_t sk = room < most ? room : most;
  return sk < 1 ? 1 : sk > 8 ? 8 : (int)sk;
}

std::atomic<uint64_t> g_limit{kPairWaitNs};

struct Rows {  // tokens in 16 bits
  const void* x;
  int64_t ld;
};

template <int DT, int BN, bool PACK>
int split_t(const Mx4& a, const Rows& x, const Mx4& b, int64_t K, const void* bias, void* out, bool early, cudaStream_t st) {
  using PL = Plan<BN, PACK>;
  const int64_t pitch = mx4_pitch(K), steps = (pitch / 128 + 1) / 2;
  Args g;
  int rc = code_map(b, pitch, kP, &g.pmap);
  if (rc != RQ_OK) return rc;
  if constexpr (PACK) g.qmap = g.pmap;
  else rc = code_map(a, pitch, BN, &g.qmap);
  if (rc != RQ_OK) return rc;
  g.pscales = b.scales;
  g.qscales = a.scales;
  g.bias = bias;
  g.out = out;
  g.prows = (int)b.rows;
  g.qrows = (int)a.rows;
  g.tiles = (int)(pitch / 128);
  g.ld = b.rows;
  g.x = x.x;
  g.ldx = x.ld;
  g.K = (int)K;
  g.early = early;
  g.limit = g_limit.load(std::memory_order_relaxed);
  g.vec = (uintptr_t)x.x % 16 == 0 && x.ld % 8 == 0 && K % 8 == 0;
  const int64_t tiles = ((b.rows + kP - 1) / kP) * ((a.rows + BN - 1) / BN);
  const int sk = split_for(tiles, steps, BN);
  const uint32_t smem = PL::kSmem + (PACK ? (uint32_t)((steps + sk - 1) / sk) * PL::kQStage : 0);
  if (smem > 226 * 1024) return RQ_ERR_UNSUPPORTED;
  const dim3 grid((unsigned)((a.rows + BN - 1) / BN), (unsigned)((b.rows + kP - 1) / kP), (unsigned)sk);
  return launch((const void*)mx4_split_k<DT, BN, PACK>, smem, grid, kThreads, dim3(1, 1, (unsigned)sk), &g, st);
}

template <int DT>
int pair_t(const Mx4& a, const Mx4& b, int64_t K, const void* bias, void* out, cudaStream_t st) {
  const int64_t pitch = mx4_pitch(K);
  PairArgs g;
  int rc = code_map(a, pitch, 128, &g.pmap);
  if (rc == RQ_OK) rc = code_map(b, pitch, 128, &g.qmap);
  if (rc != RQ_OK) return rc;
  g.pscales = a.scales;
  g.qscales = b.scales;
  g.bias = bias;
  g.out = out;
  g.prows = (int)a.rows;
  g.qrows = (int)b.rows;
  g.tiles = (int)(pitch / 128);
  g.ld = b.rows;
  const int64_t ntile = ((a.rows + 255) / 256) * ((b.rows + 255) / 256), pairs = num_sms() / 2;
  return launch((const void*)mx4_pair_k<DT>, pair::kSmem, dim3((unsigned)(2 * (ntile < pairs ? ntile : pairs))),
                pair::kThreads, dim3(2, 1, 1), &g, st);
}

template <int DT>
int matmul_t(const Mx4& a, const Mx4& b, int64_t K, const void* bias, void* out, bool early, cudaStream_t st) {
  if (a.rows > 256 && ((a.rows + 255) / 256) * ((b.rows + 255) / 256) * 4 >= num_sms()) return pair_t<DT>(a, b, K, bias, out, st);
  // the narrowest tile that holds the tokens, or 128 of them
  const Rows x{nullptr, 0};
  if (a.rows <= 16) return split_t<DT, 16, false>(a, x, b, K, bias, out, early, st);
  if (a.rows <= 32) return split_t<DT, 32, false>(a, x, b, K, bias, out, early, st);
  if (a.rows <= 64) return split_t<DT, 64, false>(a, x, b, K, bias, out, early, st);
  return split_t<DT, 128, false>(a, x, b, K, bias, out, early, st);
}

}  // namespace

void mx4_set_wait(int64_t ns) { g_limit.store(ns < 0 ? kPairWaitNs : (uint64_t)ns, std::memory_order_relaxed); }

int mx4_matmul(const Mx4& a, const Mx4& b, int64_t K, const void* bias, void* out, int dt, cudaStream_t st) {
  return dt == RQ_BF16 ? matmul_t<RQ_BF16>(a, b, K, bias, out, false, st) : matmul_t<RQ_F16>(a, b, K, bias, out, false, st);
}

// Up to 8 tokens are packed by the product's own CTAs, unless a row is so long that
// a CTA's share does not fit its shared memory.  4096 -> 11008: one token 9.4 us where
// the packing in a launch of its own makes 10.9; 8 tokens 11.7 and 11.1, but a call
// takes 6.7 us of the host's time instead of 10.4, which is what an eager step of few
// tokens waits for (captured, 8 tokens are 0.6 us better off with two launches).
constexpr int64_t kPackRows = 8, kPackColumns = 12800;  // 50 stages
static bool packs(int64_t M, int64_t K) { return M <= kPackRows && K <= kPackColumns; }

// Codes of x, then their scales.
static int64_t code_bytes(int64_t M, int64_t K) { return (M * mx4_pitch(K) / 2 + 255) / 256 * 256; }
int64_t mx4_linear_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  (void)N;
  return packs(M, K) ? 0 : code_bytes(M, K) + (M + 127) / 128 * (mx4_pitch(K) / 128) * 512;
}

int mx4_linear(const void* x, int dt, int64_t ld, int64_t M, const Mx4& w, int64_t K, const void* bias, void* out,
               void* ws, cudaStream_t st) {
  if (packs(M, K)) {
    const Mx4 a{nullptr, nullptr, M};
    const Rows rows{x, ld};
    return dt == RQ_BF16 ? split_t<RQ_BF16, 16, true>(a, rows, w, K, bias, out, false, st)
                         : split_t<RQ_F16, 16, true>(a, rows, w, K, bias, out, false, st);
  }
  uint8_t* codes = static_cast<uint8_t*>(ws);
  uint8_t* scales = codes + code_bytes(M, K);
  const int rc = mx4_pack(x, dt, ld, M, K, codes, scales, st);
  if (rc != RQ_OK) return rc;
  const Mx4 a{codes, scales, M};
  return dt == RQ_BF16 ? matmul_t<RQ_BF16>(a, w, K, bias, out, true, st) : matmul_t<RQ_F16>(a, w, K, bias, out, true, st);
}

}  // namespace rq

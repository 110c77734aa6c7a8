// mx4_gemm.cu -- products of two operands in microscaled 4 bits on the
// block-scaled tensor cores:  out[m, n] = sum_k a[m, k] b[n, k] (+ bias[n]).
//
// tcgen05.mma kind::mxf4 multiplies e2m1 codes of two K-major tiles from shared
// memory, each block of 32 codes with its power-of-two scale from tensor
// memory, and sums in fp32 in tensor memory: 4 times the rate of 16-bit
// operands, and no value is ever unpacked.
//
// A CTA computes 128 rows of operand P times BN rows of operand Q.  A stage of
// its ring holds 256 columns: P's codes [128 x 128 bytes] and Q's [BN x 128
// bytes] by TMA (128-byte swizzle), and both scales' pieces of 512 bytes (128
// rows x 128 columns, stored in the order that tensor memory takes) by bulk
// copies.  tcgen05.cp spreads a piece over 4 columns of tensor memory; every
// slot has columns of its own, so a copy never overwrites scales in use.
//   warp 0     producer (one thread)
//   warp 1     tensor memory; one thread copies scales and issues the MMAs
//   warps 2-9  epilogue: warps w and w + 4 share the 32 rows of lane quarter w % 4
// P are rows of a (tokens) and Q rows of b (outputs), or, with SWAP, the other
// way round: few tokens then fill the narrow side.  With few tiles a cluster
// splits the columns: each CTA parks its sums in shared memory, and all add up
// a share in rank order (fixed order: deterministic).
// Waits are bounded: one that runs out counts a kernel timeout, the CTA drains
// its copies and stores nothing.
#include <cuda.h>
#include <cuda_runtime.h>

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
constexpr uint64_t kWaitNs = 2000000000ull;   // a bounded wait gives up after about 2 s

template <int BN>
struct Plan {
  static constexpr int NB = (BN + 127) / 128;                       // scale pieces of Q a 128 columns
  static constexpr uint32_t kQBytes = BN * 128;
  static constexpr uint32_t kSP = kPBytes + kQBytes;                // P's scale pieces in a stage
  static constexpr uint32_t kSQ = kSP + 2 * kPiece;                 // Q's: [piece][128 columns]
  static constexpr uint32_t kStage = kSQ + 2 * NB * kPiece;
  static constexpr int kStages = BN == 256 ? 4 : BN == 128 ? 5 : 6;
  static constexpr uint32_t kRed = BN * 129 * 4;                    // parked sums, in the ring's place
  static constexpr uint32_t kRing = kStages * kStage;
  static constexpr uint32_t kSmem = (kRing > kRed ? kRing : kRed) + 1024;
  static constexpr uint32_t kAcc = BN < 32 ? 32 : BN;               // accumulator columns
  static constexpr uint32_t kSlotCols = 2 * (4 + 4 * NB);           // scale columns of a slot
  static constexpr uint32_t kNeed = kAcc + kStages * kSlotCols;
  static constexpr uint32_t kCols = kNeed <= 128 ? 128 : kNeed <= 256 ? 256 : 512;
  static_assert(kNeed <= 512 && kStage % 1024 == 0 && kSmem <= 226 * 1024, "");
};

struct Args {
  CUtensorMap pmap, qmap;   // codes [rows][pitch / 2], boxes 128 bytes x 128 and x BN
  const uint8_t* pscales;
  const uint8_t* qscales;
  const void* bias;
  void* out;
  int prows, qrows, tiles;  // tiles: pieces of 128 columns
  int64_t ld;
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

// e2m1 operands, power-of-two scales, M = 128; `half`: which two of a word's
// four scale bytes the 64 columns take.
template <int BN>
__device__ __forceinline__ uint32_t idesc_mx4(uint32_t half) {
  return (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) | (1u << 23) | (1u << 27) | (2 * half) << 4 | (2 * half) << 29;
}
__device__ __forceinline__ void mma_mx4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb,
                                        uint32_t accum) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
      " tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accum)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile int* abort) {
  if (mbar_try<false>(bar, parity)) return true;
  const uint64_t t0 = gtimer_ns();
  while (!*abort) {
    if (mbar_try<false>(bar, parity)) return true;
    if (gtimer_ns() - t0 > kWaitNs) {
      *abort = 1;
      atomicAdd(&g_mx4_timeouts, 1u);
      return false;
    }
  }
  return false;
}
__device__ __forceinline__ void drain(uint32_t bar, uint32_t parity) {
  const uint64_t t0 = gtimer_ns();
  while (!mbar_test<false>(bar, parity) && gtimer_ns() - t0 < kWaitNs) __nanosleep(100);
}

template <int DT, int BN, bool SWAP>
__global__ void __launch_bounds__(kThreads, 1) mx4_gemm_k(const __grid_constant__ Args g) {
  using PL = Plan<BN>;
  using T = typename DType<DT>::T;
  constexpr int S = PL::kStages, NB = PL::NB;
  extern __shared__ __align__(1024) unsigned char dsm[];
  __shared__ __align__(8) uint64_t bars[2 * S + 1];
  __shared__ uint32_t tmem_sh;
  __shared__ int abort_flag, issued, consumed;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const uint32_t sraw = smem_u32(dsm), sbase = (sraw + 1023u) & ~1023u;
  unsigned char* sm = dsm + (sbase - sraw);
  const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * S, accbar = empty0 + 8 * S;
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
    mbar_init(accbar, 1);
    abort_flag = issued = consumed = 0;
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
  grid_begin();

  if (warp == 0) {
    if (lane == 0) {
      const uint8_t* ps = g.pscales + (int64_t)(p0 / 128) * g.tiles * kPiece;
      const uint8_t* qs = g.qscales + (int64_t)(q0 / 128) * g.tiles * kPiece;
      const int qpieces = min(NB, (g.qrows + 127) / 128 - q0 / 128);  // pieces past the last row do not exist
      for (int st = s0; st < s1; ++st) {
        const int i = st - s0, slot = i % S;
        if (i >= S && !wait(empty0 + 8 * slot, ((i / S) - 1) & 1, abort)) break;
        const uint32_t at = sbase + slot * PL::kStage, bar = full0 + 8 * slot;
        const uint32_t bytes = (uint32_t)min(2, g.tiles - 2 * st) * kPiece;
        mbar_expect_tx(bar, kPBytes + PL::kQBytes + (1 + qpieces) * bytes);
        tma_2d(at, &g.pmap, st * 128, p0, bar);
        tma_2d(at + kPBytes, &g.qmap, st * 128, q0, bar);
        bulk_load(at + PL::kSP, ps + (int64_t)st * 2 * kPiece, bytes, bar);
        for (int j = 0; j < qpieces; ++j)
          bulk_load(at + PL::kSQ + j * 2 * kPiece, qs + ((int64_t)j * g.tiles + st * 2) * kPiece, bytes, bar);
        *reinterpret_cast<volatile int*>(&issued) = i + 1;
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      for (int st = s0; st < s1; ++st) {
        const int i = st - s0, slot = i % S;
        if (!wait(full0 + 8 * slot, (i / S) & 1, abort)) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t at = sbase + slot * PL::kStage, tsc = tmem + PL::kAcc + slot * PL::kSlotCols;
        const int nt = min(2, g.tiles - 2 * st);
        for (int t = 0; t < nt; ++t) {
          const uint32_t tp = tsc + t * (PL::kSlotCols / 2), tq = tp + 4;
          copy_scales(tp, at + PL::kSP + t * kPiece);
#pragma unroll
          for (int j = 0; j < NB; ++j) copy_scales(tq + 4 * j, at + PL::kSQ + (2 * j + t) * kPiece);
#pragma unroll
          for (int h = 0; h < 2; ++h)
            mma_mx4(tmem, sw128_desc(at + (2 * t + h) * 32), sw128_desc(at + kPBytes + (2 * t + h) * 32),
                    idesc_mx4<BN>(h), tp, tq, (i > 0 || t > 0 || h > 0) ? 1u : 0u);
        }
        mma_commit(empty0 + 8 * slot);
        *reinterpret_cast<volatile int*>(&consumed) = i + 1;
      }
      mma_commit(accbar);
    }
  }
  __syncwarp();

  const int quad = warp & 3, row = quad * 32 + lane;  // of the tile, epilogue warps
  const int c_lo = BN >= 64 ? ((warp - 2) >> 2) * (BN / 2) : 0, c_hi = BN >= 64 ? c_lo + BN / 2 : BN;
  const bool has_bias = g.bias != nullptr;
  T* out = static_cast<T*>(g.out);
  bool ok = false;
  if (warp >= 2) {
    if (lane == 0) ok = wait(accbar, 0, abort) && !*abort;
    ok = __shfl_sync(0xffffffffu, (int)ok, 0) != 0;
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  }
  if (warp >= 2 && (BN >= 64 || warp < 6)) {
    float* red = reinterpret_cast<float*>(sm);
    for (int c = c_lo; c < c_hi; c += 32) {
      float acc[32];
      tmem_ld32(tmem + ((uint32_t)(quad * 32) << 16) + c, acc);
      if (sk > 1) {
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (c + j < BN) red[(c + j) * 129 + row] = ok && s1 > s0 ? acc[j] : 0.0f;
      } else if (!ok) {
        continue;
      } else if constexpr (SWAP) {
        // rows of P are outputs, one a lane; columns are tokens
        const int n = p0 + row;
        const float bv = has_bias && n < g.prows ? DType<DT>::to_f32(static_cast<const T*>(g.bias)[n]) : 0.0f;
#pragma unroll
        for (int j = 0; j < 32; ++j)
          if (c + j < BN && q0 + c + j < g.qrows && n < g.prows)
            out[(int64_t)(q0 + c + j) * g.ld + n] = DType<DT>::from_f32(acc[j] + bv);
      } else {
        const int m = p0 + row;
        if (m >= g.prows) continue;
        T* to = out + (int64_t)m * g.ld + q0 + c;
        if (has_bias) {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            acc[j] += q0 + c + j < g.qrows ? DType<DT>::to_f32(static_cast<const T*>(g.bias)[q0 + c + j]) : 0.0f;
        }
        if (q0 + c + 32 <= g.qrows && (uintptr_t)to % 16 == 0) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            reinterpret_cast<uint4*>(to)[j] =
                make_uint4(pack_rn<DT>(acc[8 * j], acc[8 * j + 1]), pack_rn<DT>(acc[8 * j + 2], acc[8 * j + 3]),
                           pack_rn<DT>(acc[8 * j + 4], acc[8 * j + 5]), pack_rn<DT>(acc[8 * j + 6], acc[8 * j + 7]));
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (q0 + c + j < g.qrows) to[j] = DType<DT>::from_f32(acc[j]);
        }
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
    __syncwarp();
    cluster_sync();  // all sums are parked
    const uint32_t red = smem_u32(sm);
    // this CTA's share of the Q rows (SWAP: tokens) or of the P rows (tokens): a warp a token
    constexpr int kTokens = SWAP ? BN : (int)kP, kOut = SWAP ? (int)kP : BN;
    const int t0 = kTokens * rank / sk, t1 = kTokens * (rank + 1) / sk;
    for (int t = t0 + warp; t < t1; t += kThreads / 32) {
      const int m = (SWAP ? q0 : p0) + t, rows = SWAP ? g.qrows : g.prows;
      if (m >= rows) continue;
      for (int o = lane; o < kOut; o += 32) {
        const int n = (SWAP ? p0 : q0) + o;
        if (n >= (SWAP ? g.prows : g.qrows)) continue;
        const uint32_t at = red + (SWAP ? t * 129 + o : o * 129 + t) * 4;
        float sum = 0.0f;
        for (int r = 0; r < sk; ++r) {
          float v;
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(mapa(at, (uint32_t)r)));
          sum += v;
        }
        if (has_bias) sum += DType<DT>::to_f32(static_cast<const T*>(g.bias)[n]);
        out[(int64_t)m * g.ld + n] = DType<DT>::from_f32(sum);
      }
    }
    __syncwarp();
    cluster_sync();  // shared memory stays until the others have read it
  }
}

template <int DT, int BN, bool SWAP>
int run(const Args& g, int sk, cudaStream_t st) {
  const void* kern = (const void*)mx4_gemm_k<DT, BN, SWAP>;
  const int rc = ensure_smem_limit(kern, Plan<BN>::kSmem);
  if (rc != RQ_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((g.qrows + BN - 1) / BN), (unsigned)((g.prows + kP - 1) / kP), (unsigned)sk);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Plan<BN>::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = 1;
  at[1].val.clusterDim.y = 1;
  at[1].val.clusterDim.z = (unsigned)sk;
  cfg.attrs = at;
  cfg.numAttrs = sk > 1 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, mx4_gemm_k<DT, BN, SWAP>, g);
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

// How often the columns are split: until the grid fills the GPU, with at least
// two stages a CTA.
int split_for(int64_t tiles, int64_t steps) {
  int sk = 1;
  while (sk < 8 && tiles * sk * 2 <= num_sms() && steps >= 4 * sk) sk *= 2;
  return sk;
}

template <int DT>
int matmul_t(const Mx4& a, const Mx4& b, int64_t K, const void* bias, void* out, cudaStream_t st) {
  const int64_t pitch = mx4_pitch(K), steps = (pitch / 128 + 1) / 2;
  const bool swap = a.rows <= 256;
  const Mx4 &p = swap ? b : a, &q = swap ? a : b;
  const int bn = !swap ? 256 : a.rows <= 16 ? 16 : a.rows <= 32 ? 32 : a.rows <= 64 ? 64 : a.rows <= 128 ? 128 : 256;
  Args g;
  int rc = code_map(p, pitch, kP, &g.pmap);
  if (rc == RQ_OK) rc = code_map(q, pitch, (uint32_t)bn, &g.qmap);
  if (rc != RQ_OK) return rc;
  g.pscales = p.scales;
  g.qscales = q.scales;
  g.bias = bias;
  g.out = out;
  g.prows = (int)p.rows;
  g.qrows = (int)q.rows;
  g.tiles = (int)(pitch / 128);
  g.ld = b.rows;
  const int sk = split_for(((p.rows + kP - 1) / kP) * ((q.rows + bn - 1) / bn), steps);
  if (!swap) return run<DT, 256, false>(g, sk, st);
  switch (bn) {
    case 16: return run<DT, 16, true>(g, sk, st);
    case 32: return run<DT, 32, true>(g, sk, st);
    case 64: return run<DT, 64, true>(g, sk, st);
    case 128: return run<DT, 128, true>(g, sk, st);
    default: return run<DT, 256, true>(g, sk, st);
  }
}

}  // namespace

int mx4_matmul(const Mx4& a, const Mx4& b, int64_t K, const void* bias, void* out, int dt, cudaStream_t st) {
  return dt == RQ_BF16 ? matmul_t<RQ_BF16>(a, b, K, bias, out, st) : matmul_t<RQ_F16>(a, b, K, bias, out, st);
}

// Codes of x, then their scales.
static int64_t code_bytes(int64_t M, int64_t K) { return (M * mx4_pitch(K) / 2 + 255) / 256 * 256; }
int64_t mx4_linear_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  (void)N;
  return code_bytes(M, K) + (M + 127) / 128 * (mx4_pitch(K) / 128) * 512;
}

int mx4_linear(const void* x, int dt, int64_t ld, int64_t M, const Mx4& w, int64_t K, const void* bias, void* out,
               void* ws, cudaStream_t st) {
  uint8_t* codes = static_cast<uint8_t*>(ws);
  uint8_t* scales = codes + code_bytes(M, K);
  const int rc = mx4_pack(x, dt, ld, M, K, codes, scales, nullptr, st);
  if (rc != RQ_OK) return rc;
  return mx4_matmul(Mx4{codes, scales, M}, w, K, bias, out, dt, st);
}

}  // namespace rq

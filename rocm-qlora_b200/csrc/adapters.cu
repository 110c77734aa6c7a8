// adapters.cu -- the low-rank adapters of many requests beside one shared
// projection, forward and backward.
//
// A bank holds `count` adapters as A [count, K, r] and B [count, N, r] (both
// with the rank innermost), and each row m of a batch names its adapter a:
//   forward   t_m = s_a (x_m A_a)          y_m  = base_m + t_m B_a^T
//   backward  g_m = s_a (dy_m B_a)         dx_m = dxbase_m + g_m A_a^T
//             dA_a = sum_m x_m^T g_m       dB_a = sum_m dy_m^T t_m
// The backward's row products are the forward's with A and B exchanged, and
// the two gradients are one sum over the rows of an adapter, so there are
// two operators: apply (U = A, V = B or the other way round) and grad.
//
// The plan orders the rows by adapter (stable: equal inputs give equal sums)
// and cuts them into tiles of at most tile_rows rows of one adapter.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <mutex>

#include "gemv_common.cuh"

namespace cg = cooperative_groups;

namespace rq {

// Plan layout, int32 words: groups are the adapters 0..count-1, then the rows
// without an adapter (id -1), then the rows whose id names none (their
// outputs are NaN).
//   [0]                    tiles in the table
//   [1, count + 4)         first row (in plan order) of each group, and rows
//   [align4, + 4 * max)    tiles: group, first row, rows, 0
//   [.., + rows)           the batch row at each place of the plan order
__host__ __device__ inline int64_t plan_tiles_at(int count) { return ((int64_t)count + 4 + 3) / 4 * 4; }
__host__ __device__ inline int64_t plan_max_tiles(int64_t rows, int count, int tile) {
  const int64_t t = rows / tile + count + 2;
  return t < rows ? t : rows;
}
__host__ __device__ inline int64_t plan_rows_at(int64_t rows, int count, int tile) {
  return plan_tiles_at(count) + 4 * plan_max_tiles(rows, count, tile);
}

int64_t adapter_plan_words(int64_t rows, int count, int tile) { return plan_rows_at(rows, count, tile) + rows; }

constexpr int kPlanThreads = 256;

__device__ __forceinline__ int plan_group(const void* ids, int wide, int64_t m, int count) {
  const int64_t v = wide ? static_cast<const int64_t*>(ids)[m] : (int64_t)static_cast<const int*>(ids)[m];
  return v >= 0 && v < count ? (int)v : (v == -1 ? count : count + 1);
}

// One CTA a group: counts the rows of the groups before it, then writes its
// rows in batch order.
__global__ void __launch_bounds__(kPlanThreads) plan_rows_k(const void* __restrict__ ids, int wide, int rows, int count,
                                                            int rows_at, int* __restrict__ plan) {
  const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  __shared__ int sums[kPlanThreads / 32];
  __shared__ int sums2[kPlanThreads / 32];
  int less = 0;
  for (int m = tid; m < rows; m += kPlanThreads) less += plan_group(ids, wide, m, count) < g;
  less = __reduce_add_sync(0xffffffffu, less);
  if (lane == 0) sums[warp] = less;
  __syncthreads();
  int at = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 32; ++w) at += sums[w];
  if (tid == 0) {
    plan[1 + g] = at;
    if (g == count + 1) plan[1 + count + 2] = rows;
  }
  for (int m0 = 0; m0 < rows; m0 += kPlanThreads) {
    const int m = m0 + tid;
    const bool mine = m < rows && plan_group(ids, wide, m, count) == g;
    const unsigned votes = __ballot_sync(0xffffffffu, mine);
    if (lane == 0) sums2[warp] = __popc(votes);
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / 32; ++w) {
      before += w < warp ? sums2[w] : 0;
      all += sums2[w];
    }
    if (mine) plan[rows_at + at + before + __popc(votes & ((1u << lane) - 1u))] = m;
    at += all;
    __syncthreads();
  }
}

// One CTA: the tile table from the groups' row ranges.  `firsts` (dynamic
// shared memory, groups + 1 ints) is each group's first tile.
__global__ void __launch_bounds__(1024) plan_tiles_k(int count, int tile, int tiles_at, int* __restrict__ plan) {
  extern __shared__ int firsts[];
  __shared__ int part[32];
  __shared__ int carry;
  const int groups = count + 2, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) carry = 0;
  __syncthreads();
  for (int g0 = 0; g0 < groups; g0 += 1024) {
    const int g = g0 + tid;
    const int n = g < groups ? (plan[2 + g] - plan[1 + g] + tile - 1) / tile : 0;
    int v = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    if (lane == 31) part[warp] = v;
    __syncthreads();
    int before = carry;
    for (int w = 0; w < warp; ++w) before += part[w];
    if (g < groups) firsts[g] = before + v - n;
    __syncthreads();
    if (tid == 1023) carry = before + v;
    __syncthreads();
  }
  const int total = carry;
  if (tid == 0) {
    plan[0] = total;
    firsts[groups] = total;
  }
  __syncthreads();
  for (int t = tid; t < total; t += 1024) {
    int lo = 0, hi = groups;  // the group with firsts[g] <= t < firsts[g + 1]
    while (hi - lo > 1) {
      const int mid = (lo + hi) / 2;
      if (firsts[mid] <= t) lo = mid;
      else hi = mid;
    }
    const int first = plan[1 + lo] + (t - firsts[lo]) * tile, end = plan[2 + lo];
    reinterpret_cast<int4*>(plan + tiles_at)[t] = make_int4(lo, first, min(tile, end - first), 0);
  }
}

int adapter_plan(const void* ids, int wide, int64_t rows, int count, int tile, int* plan, cudaStream_t st) {
  plan_rows_k<<<count + 2, kPlanThreads, 0, st>>>(ids, wide, (int)rows, count, (int)plan_rows_at(rows, count, tile),
                                                  plan);
  plan_tiles_k<<<1, 1024, (count + 3) * sizeof(int), st>>>(count, tile, (int)plan_tiles_at(count), plan);
  return check_launch();
}

// ------------------------------------------------------------------ apply

constexpr int kApThreads = 256, kApWarps = kApThreads / 32;
constexpr int kApWin = 32;  // columns of a window: one 16-byte load of each lane of a quad

// Bytes between rows of the staged U (conflict-free ldmatrix) and of the
// intermediate's pieces (a quarter warp's loads on distinct banks).
__host__ __device__ constexpr int ap_pitch_u(int R) { return R * 2 + 16; }
__host__ __device__ constexpr int ap_pitch_m(int R) { return R <= 32 ? R * 2 : R * 2 + 64; }

// Steps of the first product under way at once, and their shared memory: a
// step is NW windows of each warp, with U's rows for them.
__host__ __device__ constexpr int ap_steps(int R, int NW) {
  return NW == 1 ? (R <= 32 ? 3 : 2) : (R == 64 ? 3 : 4);
}
// A lane's piece of a row is 16 bytes, or 5 words where rows are not 16-byte
// aligned (its 8 values and what shares their first or last word).
__host__ __device__ constexpr int ap_x_bytes(int NW, bool words) { return kApWarps * NW * 2 * 32 * (words ? 20 : 16); }

struct ApplyArgs {
  AdapterRows a;
  const void* in;
  int64_t ldin;
  const void* U;
  const void* V;
  const float* scaling;
  const void* base;
  int64_t ldb;
  float* mid;
  void* out;
  int64_t ldo;
  bool vec_in;  // rows of `in` are whole aligned 16-byte pieces
};

// A tile's rows: batch row, where its base and output are and, for fp16, the
// power of two that its intermediate was scaled down by.
struct ApplyRows {
  const uint16_t* base[128];
  uint16_t* out[128];
  int row[128];
  float mul[128];
};

__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool take) {
  const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(d), "l"(src), "r"(take ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(void* dst, const void* src, bool take) {
  const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(d), "l"(src), "r"(take ? 4 : 0) : "memory");
}
// The 4-byte word of values e and e + 1 of a row (e may be -1: the row's first
// value sits in the word's upper half), as far as they lie before `end`.
__device__ __forceinline__ void cp_async_word(void* dst, const uint16_t* row, int64_t e, int64_t end) {
  const uint32_t d = (uint32_t)__cvta_generic_to_shared(dst);
  const int64_t left = end - e;
  const uint32_t bytes = left >= 2 ? 4u : left == 1 ? 2u : 0u;
  // no bytes: any address will do, as long as it is aligned
  const uint16_t* src = bytes ? row + e : reinterpret_cast<const uint16_t*>((uintptr_t)row & ~(uintptr_t)3);
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"(d), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&d)[4], const void* p) {
  const uint32_t a = (uint32_t)__cvta_generic_to_shared(p);
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
               : "r"(a)
               : "memory");
}

// 8 consecutive 16-bit values of a row from column c (a multiple of 8), zero
// past `cols`.  VEC: the row is 16-byte aligned and cols a multiple of 8.
// Other rows are read in aligned 4-byte words and shifted into place; a row at
// an odd 2-byte address then reads the two bytes before its first value, which
// share that value's word.
template <bool VEC>
__device__ __forceinline__ uint4 load_row8(const uint16_t* row, int64_t c, int64_t cols) {
  if constexpr (VEC) return c < cols ? *reinterpret_cast<const uint4*>(row + c) : make_uint4(0u, 0u, 0u, 0u);
  const uint32_t odd = ((uintptr_t)row >> 1) & 1;
  uint32_t w[5];
#pragma unroll
  for (int j = 0; j < 5; ++j) {
    const int64_t e = c - odd + 2 * j;  // the word's first value
    w[j] = 0;
    if (j < 4 || odd) {
      if (e + 1 < cols) w[j] = *reinterpret_cast<const uint32_t*>(row + e);
      else if (e < cols) w[j] = row[e];
    }
  }
  return make_uint4(__funnelshift_r(w[0], w[1], 16 * odd), __funnelshift_r(w[1], w[2], 16 * odd),
                    __funnelshift_r(w[2], w[3], 16 * odd), __funnelshift_r(w[3], w[4], 16 * odd));
}

// The first `n` of 8 packed values to a row that is only 2-byte aligned.
__device__ __forceinline__ void store_row8(uint16_t* p, const uint32_t (&w)[4], int64_t n) {
  if (n >= 8 && ((uintptr_t)p & 2) == 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) reinterpret_cast<uint32_t*>(p)[i] = w[i];
  } else if (n >= 8) {
    p[0] = (uint16_t)w[0];
#pragma unroll
    for (int i = 0; i < 3; ++i) *reinterpret_cast<uint32_t*>(p + 1 + 2 * i) = __funnelshift_r(w[i], w[i + 1], 16);
    p[7] = (uint16_t)(w[3] >> 16);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
  }
}

// Two fp32 values rounded to 16 bits, packed (low, high): one conversion.
template <int DT>
__device__ __forceinline__ uint32_t pair16(float lo, float hi) {
  if constexpr (DT == RQ_BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
template <int DT>
__device__ __forceinline__ float2 unpair16(uint32_t w) {
  if constexpr (DT == RQ_BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// Two values as sums of 16-bit pieces: three for bf16, the upper halves of the
// value and of what is left twice, which are its 24 bits; two for fp16, rounded,
// which are 22 bits.  An infinity keeps zero remainders, so that it stays an
// infinity; NaN is in one of the first two pieces.
template <int DT> constexpr int kPieces = DT == RQ_BF16 ? 3 : 2;
template <int DT>
__device__ __forceinline__ void split16(float x, float y, uint32_t (&p)[kPieces<DT>]) {
  if constexpr (DT == RQ_BF16) {
    auto upper = [](float v) { return __uint_as_float(__float_as_uint(v) & 0xffff0000u); };
    p[0] = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
    x = fabsf(x) == INFINITY ? 0.0f : x - upper(x), y = fabsf(y) == INFINITY ? 0.0f : y - upper(y);
    p[1] = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
    p[2] = __byte_perm(__float_as_uint(x - upper(x)), __float_as_uint(y - upper(y)), 0x7632);
  } else {
    p[0] = pair16<DT>(x, y);
    const float2 h = unpair16<DT>(p[0]);
    p[1] = pair16<DT>(fabsf(x) < INFINITY ? x - h.x : 0.0f, fabsf(y) < INFINITY ? y - h.y : 0.0f);
  }
}

__device__ __forceinline__ bool any_nan(float x, float y) { return !(x == x && y == y); }

// sum + 0 w, for both 16-bit values of a word.
template <int DT>
__device__ __forceinline__ uint32_t add_zeros(uint32_t w, uint32_t sum) {
  if constexpr (DT == RQ_BF16) {
    const __nv_bfloat162 v = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&w), __float2bfloat162_rn(0.0f),
                                     *reinterpret_cast<const __nv_bfloat162*>(&sum));
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __hfma2(*reinterpret_cast<const __half2*>(&w), __float2half2_rn(0.0f),
                              *reinterpret_cast<const __half2*>(&sum));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}

// The values that are not finite as zeros.
template <int DT>
__device__ __forceinline__ uint32_t finite16(uint32_t w) {
  constexpr uint32_t top = DT == RQ_BF16 ? 0x7f807f80u : 0x7c007c00u;
  return w & ~__vcmpeq2(w & top, top);
}

template <int N>
__device__ __forceinline__ void store_words(void* p, const uint32_t (&w)[N]) {
  if constexpr (N == 1) *static_cast<uint32_t*>(p) = w[0];
  if constexpr (N == 2) *static_cast<uint2*>(p) = make_uint2(w[0], w[1]);
  if constexpr (N == 4) *static_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// The sum over the cluster's CTAs, in rank order, of what each has at p.  All
// loads are issued before the first add.
template <class V>
__device__ __forceinline__ V cluster_sum(cg::cluster_group& cluster, float* p, int csize) {
  constexpr int E = sizeof(V) / 4;
  V q[8], s;
#pragma unroll
  for (int c = 0; c < 8; ++c)
    if (c < csize) q[c] = *reinterpret_cast<const V*>(cluster.map_shared_rank(p, c));
  float* f = reinterpret_cast<float*>(&s);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    f[e] = 0.0f;
#pragma unroll
    for (int c = 0; c < 8; ++c) f[e] += c < csize ? reinterpret_cast<const float*>(&q[c])[e] : 0.0f;
  }
  return s;
}

template <class P>
struct ClusterLaunch {  // a kernel of one argument, its cluster size chosen at launch
  void (*kern)(P);
  int threads;
  size_t smem;

  cudaLaunchConfig_t config(dim3 grid, int csize, cudaLaunchAttribute (&at)[2], cudaStream_t st) const {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = csize;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;  // the kernels begin with grid_begin()
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    return cfg;
  }

  // Clusters of each size 1..8 that the GPU holds at once (their CTAs have to
  // share a GPC, so not simply its CTA slots over the size).
  const int* resident() const {
    struct Entry {
      const void* k;
      int dev;
      size_t smem;
      int n[9];
    };
    // one entry a kernel, shared-memory size (by tile) and device; a full table
    // (more devices than it is made for) only means asking again
    static std::mutex mu;
    static Entry known[512];
    static int count = 0;
    thread_local Entry e;
    int dev = 0;
    cudaGetDevice(&dev);
    std::lock_guard<std::mutex> lock(mu);
    for (int i = 0; i < count; ++i)
      if (known[i].k == (const void*)kern && known[i].dev == dev && known[i].smem == smem) return known[i].n;
    e = Entry{(const void*)kern, dev, smem, {}};
    for (int c = 1; c <= 8; ++c) {
      cudaLaunchAttribute at[2];
      cudaLaunchConfig_t cfg = config(dim3(c), c, at, nullptr);
      cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&e.n[c], kern, &cfg) != cudaSuccess || e.n[c] < 1) {
        cudaGetLastError();
        e.n[c] = std::max(1, num_sms() / c);
      }
    }
    if (count < 512) known[count++] = e;
    return e.n;
  }

  int prepare() const { return ensure_smem_limit((const void*)kern, smem); }

  int launch(const P& args, dim3 grid, int csize, cudaStream_t st) const {
    cudaLaunchAttribute at[2];
    const cudaLaunchConfig_t cfg = config(grid, csize, at, st);
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args);
    if (e != cudaSuccess) {
      set_cuda_error(e);
      return RQ_ERR_CUDA;
    }
    return check_launch();
  }
};

// The rows of a tile without an adapter: out = base (or zero), mid = 0; NaN
// for both where the id named no adapter.
template <bool VEC>
__device__ __noinline__ void rows_without(const ApplyArgs& p, const int* order, int first, int rows, bool bad,
                                          int crank, int csize) {
  const AdapterRows& a = p.a;
  const float fill = bad ? __uint_as_float(0x7fc00000u) : 0.0f;
  const uint32_t bits = bad ? 0x7fff7fffu : 0u;  // NaN in both 16-bit types
  const uint16_t* base = static_cast<const uint16_t*>(p.base);
  uint16_t* out = static_cast<uint16_t*>(p.out);
  for (int i = crank; i < rows; i += csize) {
    const int64_t m = order ? min(max(order[first + i], 0), (int)a.M - 1) : first + i;
    if (p.mid)
      for (int j = threadIdx.x; j < a.r; j += kApThreads) p.mid[m * a.r + j] = fill;
    if (p.out == p.base && !bad) continue;
    if constexpr (VEC) {
      for (int64_t d = threadIdx.x * 8; d < a.D2; d += kApThreads * 8)
        *reinterpret_cast<uint4*>(out + m * p.ldo + d) =
            base && !bad ? *reinterpret_cast<const uint4*>(base + m * p.ldb + d) : make_uint4(bits, bits, bits, bits);
    } else {
      for (int64_t d = threadIdx.x; d < a.D2; d += kApThreads)
        out[m * p.ldo + d] = base && !bad ? base[m * p.ldb + d] : (uint16_t)bits;
    }
  }
}

// A lane's outputs of an m-tile and 32-column chunks, value by value: for
// chunks of V that hold an infinity (times a piece of mid that is zero it would
// be NaN; times their sum it is not, unless that is zero) or a NaN.
template <int DT, int R, int CW>
__device__ __noinline__ void tile_by_value(const ApplyRows& at, const unsigned char* mids, int piece_bytes,
                                           const uint16_t* V, int r, bool has_base, int row0, int rows, int64_t col,
                                           int64_t end) {
  using T = typename DType<DT>::T;
  for (int h = 0; h < 2; ++h) {
    const int row = row0 + 8 * h;
    if (row >= rows) continue;
    const float mul = DT == RQ_F16 ? at.mul[row] : 1.0f;
    for (int w = 0; w < CW * 32; w += w % 32 == 7 ? 25 : 1) {
      const int64_t n = col + w;
      if (n >= end) break;
      float s = 0.0f;
      for (int j = 0; j < r; ++j) {
        float t = 0.0f;
        for (int k = 0; k < kPieces<DT>; ++k)
          t += DType<DT>::to_f32(reinterpret_cast<const T*>(mids + k * piece_bytes + row * ap_pitch_m(R))[j]);
        s = fmaf(t, DType<DT>::to_f32(reinterpret_cast<const T*>(V + n * r)[j]), s);
      }
      const float old = has_base ? DType<DT>::to_f32(reinterpret_cast<const T*>(at.base[row])[n]) : 0.0f;
      reinterpret_cast<T*>(at.out[row])[n] = DType<DT>::from_f32(fmaf(s, mul, old));
    }
  }
}

// One cluster computes one tile: `tile` rows (16 to 128) of one adapter.
//
// Mathematics.  mid = s (in U) and out = base + mid V^T, both on tensor cores
// (mma m16n8k16, fp32 accumulation).  U and V enter as they are; mid is fp32
// and is multiplied as the sum of 16-bit pieces, so that it keeps its 24 bits
// (bf16, three pieces; with two, 16 bits, one result in a thousand rounds the
// other way) or 22 (fp16, two pieces).  For fp16, whose exponent range a small
// gradient would leave, each row of mid is first brought near 2^14 by a power
// of two that the output row takes back.
//
// What bounds it: in and base are read and out written once (HBM), while U
// and V are shared by the tile's rows (L2).  The sum over all input columns
// has to be complete before the first output, so with one launch the split
// is by columns inside a cluster: each CTA sums its share of the input
// columns, the partial sums meet through distributed shared memory in rank
// order (equal inputs give equal bits), and each CTA writes its share of the
// output columns.  A decode row costs one launch, no workspace and no second
// kernel.
//
// Loads.  A quad's four lanes hold 32 consecutive columns of a row, 8 each, in
// one 16-byte piece that the lane fetches for itself by cp.async several steps
// ahead; the MMA's order of the reduction index follows that, and U's rows are
// put into shared memory in the order that ldmatrix then needs.  V's columns
// are permuted the same way among the MMA's n index, so that a lane ends with
// 8 consecutive output columns: one 16-byte load of base and one store.
//
// Measured (bf16): one row of 4096 to 4096, rank 16, 6.1 us (a launch and a
// chain of five dependent loads); 8192 rows, 46 us, 4.3 TB/s of the 201 MB
// (31 us at the copy bandwidth; launch, plan, meeting and sums are the rest);
// rank 64, 74 us, the tensor pipe 40 % active: the three pieces of mid.  fp16 rows of 1093 to
// 1088, rank 64, 1111 of them: 14 us.
template <int DT, int R, int NW, bool VEC>
__global__ void __launch_bounds__(kApThreads, R <= 64 ? 2 : 1) adapters_apply_k(const __grid_constant__ ApplyArgs p) {
  constexpr int NT = R / 8;               // n-tiles of the first product
  constexpr int KS = R / 16;              // k-steps of the second
  constexpr int PU = ap_pitch_u(R), PM = ap_pitch_m(R), S = ap_steps(R, NW);
  constexpr int P = kPieces<DT>;
  constexpr int CW = R <= 32 ? 2 : 1, AHEAD = 2;  // second product: 32-column chunks of a warp, m-tiles under way
  extern __shared__ __align__(16) unsigned char smem[];
  const AdapterRows& a = p.a;
  cg::cluster_group cluster = cg::this_cluster();
  const int crank = (int)cluster.block_rank(), csize = (int)cluster.num_blocks();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  grid_begin();

  // ---- the tile
  const int tile_id = (int)(blockIdx.x / csize);
  int group, first, rows;
  const int* order = nullptr;
  if (a.plan) {
    const int tiles = a.plan[0];  // the table has room for every tile of the grid: both loads at once
    const int4 e = reinterpret_cast<const int4*>(a.plan + plan_tiles_at(a.count))[tile_id];
    if (tile_id >= tiles) return;
    // held inside the batch, so that a plan that is not one cannot reach outside it
    group = min(max(e.x, 0), a.count + 1), first = min(max(e.y, 0), (int)a.M - 1);
    rows = min(max(e.z, 1), min(a.tile, (int)a.M - first));
    order = a.plan + plan_rows_at(a.M, a.count, a.tile);
  } else {
    group = 0, first = tile_id * a.tile;
    rows = min(a.tile, (int)a.M - first);
  }
  const int WM = a.tile / 16, WK = kApWarps / WM;  // warps along rows, along columns
  if (group >= a.count) {  // no adapter: base as it is; an id that names none: NaN
    rows_without<VEC>(p, order, first, rows, group > a.count, crank, csize);
    return;
  }

  const int KC = NW * WK * kApWin, step_bytes = KC * PU + ap_x_bytes(NW, !p.vec_in);  // columns of a step
  ApplyRows& at = *reinterpret_cast<ApplyRows*>(smem);
  unsigned char* ring = smem + sizeof(ApplyRows);
  float* part = reinterpret_cast<float*>(ring);  // [128][R], over the ring
  unsigned char* mids = ring + 128 * R * 4;      // pieces of mid: [P][tile][PM], over the ring
  const uint16_t* in = static_cast<const uint16_t*>(p.in);
  const uint16_t* base = static_cast<const uint16_t*>(p.base);
  const int chunks2 = (int)((a.D2 + 31) / 32), per2 = (chunks2 + csize - 1) / csize;
  const int ch_begin = min(chunks2, crank * per2), ch_end = min(chunks2, ch_begin + per2);
  const int wins = (int)((a.D1 + kApWin - 1) / kApWin), per = (wins + csize - 1) / csize;
  const int w_begin = min(wins, crank * per), w_end = min(wins, w_begin + per);
  // ---- partial sums over this CTA's input columns
  const uint16_t* U = static_cast<const uint16_t*>(p.U) + (int64_t)group * a.D1 * a.r;
  const int step = NW * WK, chunks = (w_end - w_begin + step - 1) / step;
  const int wm = warp % WM, wk = warp / WM;

  // What a thread stages of U is an arithmetic sequence: piece q of every
  // ROWS-th row from k0 on, each row at the place its window's order gives it.
  constexpr int ROWS = kApThreads / NT;
  const int q = tid % NT, k0 = tid / NT;
  auto slot_of = [](int k) { return (k & ~31) | ((k & 6) << 2) | (((k & 31) >> 3) << 1) | (k & 1); };
  const bool rank = q * 8 < a.r;
  const uint16_t* u_src = U + ((int64_t)w_begin * kApWin + k0) * a.r + (rank ? q * 8 : 0);
  // rows from u_src on that are this CTA's: x is zero past them, which an infinity of U would make a NaN
  int u_left = (int)(min((int64_t)w_end * kApWin, a.D1) - (int64_t)w_begin * kApWin) - k0;
  const uint32_t u_dst = slot_of(k0) * PU + q * 16;
  auto stage_u = [&](int c) {
    if (c >= chunks) return;
    unsigned char* dst = ring + (c % S) * step_bytes + u_dst;
#pragma unroll 4
    for (int i = 0; i * ROWS + k0 < KC; ++i) {
      // of 32 rows a window's order keeps multiples of 16 apart: 16 rows on are 4 places on
      const uint32_t to = ROWS == 16 ? (i >> 1) * 32 * PU + (i & 1) * 4 * PU : i * ROWS * PU;
      const bool ok = rank && i * ROWS < u_left;
      cp_async16(dst + to, ok ? u_src + (int64_t)i * ROWS * a.r : U, ok);
    }
    u_src += (int64_t)KC * a.r;
    u_left -= KC;
  };
  // The first steps of U need no row number: they are on their way while the
  // plan's rows are looked up.
  for (int c = 0; c < S - 1; ++c) stage_u(c);
  const uint16_t* V = static_cast<const uint16_t*>(p.V) + (int64_t)group * a.D2 * a.r;
  if (tid < a.tile) {
    const int place = first + min(tid, rows - 1);
    const int m = order ? min(max(order[place], 0), (int)a.M - 1) : place;
    at.row[tid] = m;
    at.base[tid] = base + (int64_t)m * p.ldb;
    at.out[tid] = static_cast<uint16_t*>(p.out) + (int64_t)m * p.ldo;
  }
  __syncthreads();
  const uint16_t* xa = in + (int64_t)at.row[wm * 16 + g] * p.ldin;
  const uint16_t* xb = in + (int64_t)at.row[wm * 16 + g + 8] * p.ldin;
  // this lane's part of the rows: what it multiplies it also fetches
  const uint32_t x_dst = KC * PU + warp * NW * 64 * (p.vec_in ? 16 : 20) + lane * (p.vec_in ? 16 : 4);
  const uint32_t odd_a = ((uintptr_t)xa >> 1) & 1, odd_b = ((uintptr_t)xb >> 1) & 1;
  int64_t x_col = (int64_t)(w_begin + wk * NW) * kApWin + t * 8;
  const int64_t x_end = min((int64_t)w_end * kApWin, a.D1);
  auto stage_x = [&](int c) {
    if (c < chunks) {
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const int64_t col = x_col + w * kApWin;
        unsigned char* x = ring + (c % S) * step_bytes + x_dst;
        if (p.vec_in) {
          const bool ok = col < x_end;
          cp_async16(x + w * 1024, xa + (ok ? col : 0), ok);
          cp_async16(x + w * 1024 + 512, xb + (ok ? col : 0), ok);
        } else {
#pragma unroll
          for (int j = 0; j < 5; ++j) {
            cp_async_word(x + w * 1280 + j * 128, xa, col - odd_a + 2 * j, col < x_end ? x_end : 0);
            cp_async_word(x + w * 1280 + 640 + j * 128, xb, col - odd_b + 2 * j, col < x_end ? x_end : 0);
          }
        }
      }
      x_col += step * kApWin;
    }
    cp_async_commit();
  };
  auto piece = [&](const unsigned char* x, int w, int h) {
    if (p.vec_in) return *reinterpret_cast<const uint4*>(x + w * 1024 + h * 512);
    uint32_t q[5];
#pragma unroll
    for (int j = 0; j < 5; ++j) q[j] = *reinterpret_cast<const uint32_t*>(x + w * 1280 + h * 640 + j * 128);
    const uint32_t by = 16 * (h ? odd_b : odd_a);
    return make_uint4(__funnelshift_r(q[0], q[1], by), __funnelshift_r(q[1], q[2], by), __funnelshift_r(q[2], q[3], by),
                      __funnelshift_r(q[3], q[4], by));
  };
  float acc[NT][4], sum[NT][4];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[i][e] = sum[i][e] = 0.0f;
  for (int c = 0; c < S - 1; ++c) stage_x(c);
  for (int c = 0; c < chunks; ++c) {
    cp_async_wait<S - 2>();
    __syncthreads();  // step c is here, and step c - 1, whose place comes next, has been read
    stage_u(c + S - 1);
    stage_x(c + S - 1);
    const unsigned char* u = ring + (c % S) * step_bytes + wk * NW * kApWin * PU;
    const unsigned char* mine = ring + (c % S) * step_bytes + x_dst;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const uint4 x = piece(mine, w, 0), y = piece(mine, w, 1);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const unsigned char* row = u + (w * 32 + s * 16 + (lane & 15)) * PU + (lane >> 4) * 16;
#pragma unroll
        for (int j = 0; j < NT; j += 2) {
          uint32_t b[4];
          ldmatrix4_trans(b, row + j * 16);
          Mma16816<DT>::run(acc[j], s ? x.z : x.x, s ? y.z : y.x, s ? x.w : x.y, s ? y.w : y.y, b[0], b[1]);
          Mma16816<DT>::run(acc[j + 1], s ? x.z : x.x, s ? y.z : y.x, s ? x.w : x.y, s ? y.w : y.y, b[2], b[3]);
        }
      }
    }
    // The MMA's sum is cut off, not rounded, at each of its steps, which shifts
    // that of a long row (22016 positive products: by 2e-5 in bf16, 3.5e-5 in
    // fp16).  After every 8 steps it is added to one that is rounded (5e-7).
    if ((c + 1) % (4 / NW) == 0 || c + 1 == chunks) {
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[i][e] += acc[i][e], acc[i][e] = 0.0f;
    }
  }
  cp_async_wait<0>();
  __syncthreads();  // the sums lie over the ring

  // ---- the sums meet: warps of the CTA in order, then the cluster's CTAs in rank order
  float* mine = part + (wk * a.tile + wm * 16) * R;
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    *reinterpret_cast<float2*>(mine + g * R + j * 8 + 2 * t) = make_float2(sum[j][0], sum[j][1]);
    *reinterpret_cast<float2*>(mine + (g + 8) * R + j * 8 + 2 * t) = make_float2(sum[j][2], sum[j][3]);
  }
  __syncthreads();
  if (WK > 1) {
    for (int i = tid; i < a.tile * R; i += kApThreads) {
      float v = part[i];
      for (int w = 1; w < WK; ++w) v += part[w * a.tile * R + i];
      part[i] = v;
    }
  }
  // ---- this warp's output columns, CW x 32 at a time, all rows of the tile, as
  // one sequence of (chunk, m-tile): base is fetched AHEAD of them in advance,
  // the first before the sums meet.
  const int n_tiles = (rows + 15) / 16, ch_step = kApWarps * CW;
  const int64_t end = min((int64_t)ch_end * 32, a.D2);  // columns this CTA writes
  int f_ch = ch_begin + warp * CW, f_mt = 0;            // next to be fetched
  uint4 ahead[AHEAD][CW][2] = {};
  auto fetch = [&](uint4 (&old)[CW][2]) {
    if (f_ch < ch_end) {
      if (base) {
        const uint16_t* ra = at.base[f_mt * 16 + g];
        const uint16_t* rb = at.base[f_mt * 16 + g + 8];
        const int64_t col = (int64_t)f_ch * 32 + 8 * t;
#pragma unroll
        for (int w = 0; w < CW; ++w) {
          old[w][0] = load_row8<VEC>(ra, col + 32 * w, end);
          old[w][1] = load_row8<VEC>(rb, col + 32 * w, end);
        }
      }
      if (++f_mt == n_tiles) f_mt = 0, f_ch += ch_step;
    }
  };
  // B fragments: for n-tile j the lane's column is 8 (g / 2) + 2 j + g % 2
  uint32_t b[CW][4][KS][2];
  auto load_b = [&](int ch) {
#pragma unroll
    for (int j = 0; j < 4 * CW; ++j) {
      const int64_t n = (int64_t)ch * 32 + 32 * (j / 4) + 8 * (g >> 1) + 2 * (j % 4) + (g & 1);
      const uint16_t* v = V + n * a.r;
      const bool ok = n < end;
      if constexpr (R == 16) {
        const uint2 q = ok && 4 * t < a.r ? *reinterpret_cast<const uint2*>(v + 4 * t) : make_uint2(0u, 0u);
        b[j / 4][j % 4][0][0] = q.x, b[j / 4][j % 4][0][1] = q.y;
      } else {
#pragma unroll
        for (int w = 0; w < KS / 2; ++w) {
          const uint4 q = ok && 32 * w + 8 * t < a.r ? *reinterpret_cast<const uint4*>(v + 32 * w + 8 * t)
                                                     : make_uint4(0u, 0u, 0u, 0u);
          uint32_t(&f)[KS][2] = b[j / 4][j % 4];
          f[2 * w][0] = q.x, f[2 * w][1] = q.y, f[2 * w + 1][0] = q.z, f[2 * w + 1][1] = q.w;
        }
      }
    }
  };
  // Whether all of the chunk's V is finite: a sum of zeros times it is NaN else.
  // Of the first chunk it is asked after the sums have met, so that V is on its
  // way until then.
  auto finite_b = [&] {
    uint32_t sum = 0;
#pragma unroll
    for (int j = 0; j < 4 * CW; ++j)
#pragma unroll
      for (int k = 0; k < KS; ++k) sum = add_zeros<DT>(b[j / 4][j % 4][k][1], add_zeros<DT>(b[j / 4][j % 4][k][0], sum));
    const float2 zero = unpair16<DT>(sum);
    return !__any_sync(0xffffffffu, any_nan(zero.x, zero.y));
  };
  if (f_ch < ch_end) load_b(f_ch);
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) fetch(ahead[i]);
  cluster.sync();
  // LR lanes a row, this CTA's share of the rows; the result goes to every CTA
  constexpr int LR = R == 16 ? 8 : 16, E = R / LR;
  const int share = (a.tile + csize - 1) / csize, l = tid % LR;
  const float s = p.scaling[group];
  for (int i0 = 0; i0 < share; i0 += kApThreads / LR) {
    const int i = i0 + tid / LR, row = crank * share + i;
    const bool on = i < share && row < a.tile;
    __align__(16) float v[E];
    float* src = part + (on ? row : 0) * R + l * E;
    if constexpr (E == 2) *reinterpret_cast<float2*>(v) = cluster_sum<float2>(cluster, src, csize);
#pragma unroll
    for (int e = 0; e + 4 <= E; e += 4) *reinterpret_cast<float4*>(v + e) = cluster_sum<float4>(cluster, src + e, csize);
    float top = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      v[e] = l * E + e < a.r ? v[e] * s : 0.0f;  // an infinity of x times the padding is NaN
      top = fmaxf(top, fabsf(v[e]) < INFINITY ? fabsf(v[e]) : 0.0f);
      if (p.mid && on && row < rows && l * E + e < a.r) p.mid[(int64_t)at.row[row] * a.r + l * E + e] = v[e];
    }
    float mul = 1.0f, back = 1.0f;
    if constexpr (DT == RQ_F16) {
#pragma unroll
      for (int o = LR / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const int ex = (int)(__float_as_uint(top) >> 23);  // biased exponent; 255: not finite, small: leave
      if (ex > 30 && ex < 255) {
        mul = __uint_as_float((uint32_t)(268 - ex) << 23);
        back = __uint_as_float((uint32_t)(ex - 14) << 23);
      }
    }
    if (on) {
      __align__(16) uint32_t w[P][E / 2];
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        uint32_t q[P];
        split16<DT>(v[e] * mul, v[e + 1] * mul, q);
#pragma unroll
        for (int k = 0; k < P; ++k) w[k][e / 2] = q[k];
      }
      unsigned char* to = mids + row * PM + l * E * 2;
      for (int c = 0; c < csize; ++c) {
        unsigned char* m = cluster.map_shared_rank(to, c);
#pragma unroll
        for (int k = 0; k < P; ++k) store_words<E / 2>(m + k * a.tile * PM, w[k]);
        if (DT == RQ_F16 && l == 0) cluster.map_shared_rank(at.mul, c)[row] = back;
      }
    }
  }
  cluster.sync();

  // base starts the accumulators, so the sum costs no instruction of its own
  auto tile = [&](int64_t col, int mt, uint4 (&old)[CW][2]) {
    const int ra = mt * 16 + g;
    // fp16: the row's power of two, taken off base here and put back below
    float off_a = 1.0f, off_b = 1.0f, mul_a = 1.0f, mul_b = 1.0f;
    if constexpr (DT == RQ_F16) {
      mul_a = at.mul[ra], mul_b = at.mul[ra + 8];
      off_a = __uint_as_float((254u << 23) - __float_as_uint(mul_a));
      off_b = __uint_as_float((254u << 23) - __float_as_uint(mul_b));
    }
    float acc[CW][4][4];
#pragma unroll
    for (int w = 0; w < CW; ++w) {
      const uint32_t qa[4] = {old[w][0].x, old[w][0].y, old[w][0].z, old[w][0].w};
      const uint32_t qb[4] = {old[w][1].x, old[w][1].y, old[w][1].z, old[w][1].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 x = unpair16<DT>(qa[j]), y = unpair16<DT>(qb[j]);
        if constexpr (DT == RQ_F16) {
          acc[w][j][0] = x.x * off_a, acc[w][j][1] = x.y * off_a, acc[w][j][2] = y.x * off_b, acc[w][j][3] = y.y * off_b;
        } else {
          acc[w][j][0] = x.x, acc[w][j][1] = x.y, acc[w][j][2] = y.x, acc[w][j][3] = y.y;
        }
      }
    }
    fetch(old);
#pragma unroll
    for (int piece = 0; piece < P; ++piece) {
      const unsigned char* ma = mids + (piece * a.tile + ra) * PM;
      const unsigned char* mb = ma + 8 * PM;
      if constexpr (R == 16) {
        const uint2 qa = *reinterpret_cast<const uint2*>(ma + 8 * t), qb = *reinterpret_cast<const uint2*>(mb + 8 * t);
#pragma unroll
        for (int w = 0; w < CW; ++w)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            Mma16816<DT>::run(acc[w][j], qa.x, qb.x, qa.y, qb.y, b[w][j][0][0], b[w][j][0][1]);
      } else {
#pragma unroll
        for (int k = 0; k < KS / 2; ++k) {
          const uint4 qa = *reinterpret_cast<const uint4*>(ma + 64 * k + 16 * t);
          const uint4 qb = *reinterpret_cast<const uint4*>(mb + 64 * k + 16 * t);
#pragma unroll
          for (int w = 0; w < CW; ++w)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              Mma16816<DT>::run(acc[w][j], qa.x, qb.x, qa.y, qb.y, b[w][j][2 * k][0], b[w][j][2 * k][1]);
              Mma16816<DT>::run(acc[w][j], qa.z, qb.z, qa.w, qb.w, b[w][j][2 * k + 1][0], b[w][j][2 * k + 1][1]);
            }
        }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (ra + 8 * h >= rows) continue;
      uint16_t* dst = at.out[ra + 8 * h] + col;
      const float mul = h ? mul_b : mul_a;
#pragma unroll
      for (int w = 0; w < CW; ++w) {
        uint32_t res[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float x = acc[w][j][2 * h], y = acc[w][j][2 * h + 1];
          if constexpr (DT == RQ_F16) x *= mul, y *= mul;
          res[j] = pair16<DT>(x, y);
        }
        if constexpr (VEC) {
          if (col + 32 * w < end)
            *reinterpret_cast<uint4*>(dst + 32 * w) = make_uint4(res[0], res[1], res[2], res[3]);
        } else {
          store_row8(dst + 32 * w, res, end - col - 32 * w);
        }
      }
    }
  };
  int ch = ch_begin + warp * CW, mt = 0;
  bool by_value = ch < ch_end && !finite_b();
  while (ch < ch_end) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (ch >= ch_end) break;
      if (by_value) {
        tile_by_value<DT, R, CW>(at, mids, a.tile * PM, V, a.r, base != nullptr, mt * 16 + g, rows,
                                 (int64_t)ch * 32 + 8 * t, end);
        fetch(ahead[i]);
      } else {
        tile((int64_t)ch * 32 + 8 * t, mt, ahead[i]);
      }
      if (++mt == n_tiles) {
        mt = 0, ch += ch_step;
        if (ch < ch_end) {
          load_b(ch);
          by_value = !finite_b();
        }
      }
    }
  }
}

static bool rows16b(const void* p, int64_t ld) { return (uintptr_t)p % 16 == 0 && ld % 8 == 0; }

template <int DT, int R, int NW>
static int launch_apply(const ApplyArgs& p, bool vec, int64_t tiles, cudaStream_t st) {
  const int columns = NW * (kApWarps / (p.a.tile / 16)) * kApWin;  // of a step
  const size_t ring = (size_t)ap_steps(R, NW) * (columns * ap_pitch_u(R) + ap_x_bytes(NW, !p.vec_in));
  const size_t after = (size_t)128 * R * 4 + (size_t)kPieces<DT> * p.a.tile * ap_pitch_m(R);
  const size_t smem = sizeof(ApplyRows) + std::max(ring, after);
  const ClusterLaunch<ApplyArgs> l{vec ? adapters_apply_k<DT, R, NW, true> : adapters_apply_k<DT, R, NW, false>,
                                   kApThreads, smem};
  const int rc = l.prepare();
  if (rc != RQ_OK) return rc;
  // The cluster size of the least time: rounds of the GPU, each about 6 us of
  // fixed cost and 1e-4 us a value of a CTA's share of in, base and out (8192
  // rows, 4096 x 4096, rank 16, tiles of 128: 46 us with 4, 53 with 8, 58
  // with 2; rank 64 74, 85 and 91).
  const int* resident = l.resident();
  const double expected = (double)p.a.M / p.a.tile + (p.a.plan ? 0.5 * p.a.count : 0.0);
  const double work = 1e-4 * p.a.tile * ((double)p.a.D1 + 2.0 * p.a.D2);
  int csize = 8;
  double best = 1e30;
  for (int c = 8; c >= 1; --c) {
    const double rounds = std::ceil(std::min(expected, (double)tiles) / resident[c]);
    if (rounds * (6.0 + work / c) < best) best = rounds * (6.0 + work / c), csize = c;
  }
  return l.launch(p, dim3((unsigned)(tiles * csize)), csize, st);
}

template <int DT, int NW>
static int launch_apply_r(const ApplyArgs& p, bool vec, int64_t tiles, cudaStream_t st) {
  if (p.a.r <= 16) return launch_apply<DT, 16, NW>(p, vec, tiles, st);
  if (p.a.r <= 32) return launch_apply<DT, 32, NW>(p, vec, tiles, st);
  if (p.a.r <= 64) return launch_apply<DT, 64, NW>(p, vec, tiles, st);
  return launch_apply<DT, 128, NW>(p, vec, tiles, st);
}

int adapters_apply(const AdapterRows& a0, const void* in, int64_t ldin, const void* U, const void* V,
                   const float* scaling, const void* base, int64_t ldb, float* mid, void* out, int64_t ldo,
                   cudaStream_t st) {
  AdapterRows a = a0;
  if (!a.plan) a.tile = a.M <= 16 ? 16 : a.M <= 32 ? 32 : a.M <= 4096 ? 64 : 128;  // as plans are made
  const int64_t tiles = a.plan ? plan_max_tiles(a.M, a.count, a.tile) : (a.M + a.tile - 1) / a.tile;
  const ApplyArgs p{a, in, ldin, U, V, scaling, base, ldb, mid, out, ldo, a.D1 % 8 == 0 && rows16b(in, ldin)};
  const bool vec = a.D2 % 8 == 0 && rows16b(out, ldo) && (!base || rows16b(base, ldb));  // base and out
  if (a.dt == RQ_BF16)
    return a.tile >= 64 ? launch_apply_r<RQ_BF16, 2>(p, vec, tiles, st)
                        : launch_apply_r<RQ_BF16, 1>(p, vec, tiles, st);
  return a.tile >= 64 ? launch_apply_r<RQ_F16, 2>(p, vec, tiles, st)
                      : launch_apply_r<RQ_F16, 1>(p, vec, tiles, st);
}

// ------------------------------------------------------------------- grad

constexpr int kGrWarps = 8;                                  // of a CTA whose groups split the rows
constexpr int kGrCols = 128;                                 // columns of a CTA: one block of 8-bit codes
constexpr int kGrSums = kGrCols * 16 * 4;                    // a warp's 128 x 16 sums
// One step in a ring: 16 rows of z (swizzled 16-byte pieces) and of mid (16
// ranks a warp, padded so that fragment loads use distinct banks), and the
// scales of codes.  RG warps, 16 ranks each, share a ring and its rows.
__host__ __device__ constexpr int gr_row_bytes(bool codes) { return codes ? kGrCols : kGrCols * 2; }
__host__ __device__ constexpr int gr_mid_pitch(int RG) { return (16 * RG + 4) * 4; }
__host__ __device__ constexpr int gr_step_bytes(bool codes, int RG) {
  return 16 * (gr_row_bytes(codes) + gr_mid_pitch(RG) + (codes ? 4 : 0));
}
// steps of a ring: about 100 KB of rings a CTA, so that two share an SM
__host__ __device__ constexpr int gr_steps(bool codes, bool vec, int RG) {
  return !vec ? 2 : (codes ? 3 : 2) + (RG == 1 ? 0 : RG == 2 ? 2 : RG == 4 ? 4 : 6);
}

struct GradArgs {
  AdapterRows a;
  const void* z;
  int64_t ldz;
  const float* zscale;
  int64_t lds;
  const float* mid;
  void* G;
  int beside;  // the adapters of more than `most` rows are summed by the launch before
  int most;
};

// Rows of an adapter: places [first, last) of the plan's order; without a plan
// the whole batch is adapter 0's.
__device__ __forceinline__ int2 grad_rows(const AdapterRows& a, int adapter) {
  if (!a.plan) return make_int2(0, adapter == 0 ? (int)a.M : 0);
  const int first = max(a.plan[1 + adapter], 0);
  return make_int2(first, max(first, min(a.plan[2 + adapter], (int)a.M)));
}

// The nth adapter of more than `most` rows; -1: there are not so many.
template <int THREADS>
__device__ int nth_large(const GradArgs& p, int nth) {
  __shared__ uint32_t votes[THREADS / 32];
  for (int i0 = 0; i0 < p.a.count; i0 += THREADS) {
    const int i = i0 + (int)threadIdx.x;
    const int2 rows = i < p.a.count ? grad_rows(p.a, i) : make_int2(0, 0);
    const uint32_t vote = __ballot_sync(0xffffffffu, rows.y - rows.x > p.most);
    if (threadIdx.x % 32 == 0) votes[threadIdx.x / 32] = vote;
    __syncthreads();
    for (int w = 0; w < THREADS / 32; ++w) {
      uint32_t v = votes[w];
      const int n = __popc(v);
      if (nth < n) {
        for (; nth > 0; --nth) v &= v - 1;
        return i0 + 32 * w + __ffs(v) - 1;
      }
      nth -= n;
    }
    __syncthreads();  // all have read the votes
  }
  return -1;
}

// Two codes in the low bytes of a word's halves as 16-bit values, exact.  bf16:
// 0x4300 with the code's lower 7 bits is 128 + (q mod 128), and with its sign
// bit alone 128 for q >= 0 and 256 for q < 0; their difference is q.  fp16:
// 0x64uu with u = q + 128 is 1024 + u.
template <int DT>
__device__ __forceinline__ uint32_t codes2(uint32_t w) {
  if constexpr (DT == RQ_BF16) {
    const uint32_t x = (w & 0x007f007fu) | 0x43004300u, y = (w & 0x00800080u) | 0x43004300u;
    const __nv_bfloat162 d =
        __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&y));
    return *reinterpret_cast<const uint32_t*>(&d);
  } else {
    const uint32_t x = ((w & 0x00ff00ffu) ^ 0x64806480u), y = 0x64806480u;
    const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&y));
    return *reinterpret_cast<const uint32_t*>(&d);
  }
}

// The sums of one warp: 128 columns from block * 128 on, 16 ranks, over the
// rows of its group; acc[m-tile][rank of a pair][].  Gives, for fp16, the
// biased exponent that they are scaled down by.  AGAIN: what is not finite in z
// meets only the first piece of mid (a piece that is zero would make an
// infinity NaN).
template <int DT, bool CODES, bool VEC, int RG, int MW, bool AGAIN>
__device__ __forceinline__ int sum_rows(const GradArgs& p, int2 places, int block, int crank, int csize,
                                        float (&acc)[8][2][4]) {
  constexpr int ROW = gr_row_bytes(CODES), PITCH = gr_mid_pitch(RG), STEP = gr_step_bytes(CODES, RG);
  constexpr int S = gr_steps(CODES, VEC, RG);
  constexpr bool CONV = CODES && RG > 1;        // codes become 16-bit once for all warps of a group
  constexpr int PAIR = 2;                       // m-tiles at a time: four sums between two products of one sum
  constexpr int TR = 2 * RG;                    // threads of a group that fetch one row
  constexpr int PIECES = (ROW / 16 + TR - 1) / TR;  // 16-byte pieces of it each
  extern __shared__ __align__(16) unsigned char smem[];
  const AdapterRows& a = p.a;
  const int first = places.x, last = places.y;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int rg = warp % RG, mw = warp / RG;
  const int* order = a.plan ? a.plan + plan_rows_at(a.M, a.count, a.tile) : nullptr;
  const int64_t c0 = (int64_t)block * kGrCols;
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int n = 0; n < 2; ++n) acc[i][n][0] = acc[i][n][1] = acc[i][n][2] = acc[i][n][3] = 0.0f;
  int ex_now = 0;          // fp16: biased exponent that mid is scaled down by
  float mul = 1.0f;

  // fetching: a thread's row of a step and every TR-th of its pieces
  const int gt = rg * 32 + lane, frow = gt / TR, fpart = gt % TR;
  const int begin = first + (crank * MW + mw) * 16, stride = csize * MW * 16;
  const int steps = begin < last ? (last - begin + stride - 1) / stride : 0;
  unsigned char* ring = smem + mw * S * STEP;
  unsigned char* wide = smem + MW * S * STEP + mw * 16 * 2 * kGrCols;
  auto row_of = [&](int s) {  // batch row of this thread's row in step s; -1: none
    const int place = begin + s * stride + frow;
    if (s >= steps || place >= last) return -1;
    return order ? min(max(order[place], 0), (int)a.M - 1) : place;
  };
  int next = row_of(0);
  auto fetch = [&](int s) {
    unsigned char* dst = ring + (s % S) * STEP;
    const bool on = next >= 0;
    const int64_t m = on ? next : 0;
    if constexpr (CODES) {
      const uint8_t* row = static_cast<const uint8_t*>(p.z) + m * p.ldz + c0 + 16 * fpart;
#pragma unroll
      for (int i = 0; i < PIECES; ++i)
        if (TR * i + fpart < ROW / 16)
          cp_async16(dst + frow * ROW + (((TR * i + fpart) ^ (frow & 7)) << 4), row + 16 * TR * i, on);
    } else {
      const uint16_t* row = static_cast<const uint16_t*>(p.z) + m * p.ldz;
      const int64_t left = a.D1 - c0 - 8 * fpart;  // columns from this thread's first piece
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        unsigned char* to = dst + frow * ROW + (((TR * i + fpart) ^ (frow & 7)) << 4);
        if constexpr (VEC)
          cp_async16(to, row + (8 * TR * i < left ? c0 + 8 * fpart + 8 * TR * i : 0), on && 8 * TR * i < left);
        else
          *reinterpret_cast<uint4*>(to) = load_row8<false>(row, c0 + 8 * fpart + 8 * TR * i, on ? a.D1 : 0);
      }
    }
    // 8 ranks of mid, and the row's scale
    unsigned char* to = dst + 16 * ROW + frow * PITCH + 32 * fpart;
    const bool some = on && 8 * fpart < a.r;
    const float* mid = p.mid + (some ? m * a.r + 8 * fpart : 0);
    cp_async16(to, mid, some);
    cp_async16(to + 16, mid + 4, some);
    if (CODES && fpart == 0)
      cp_async4(dst + 16 * (ROW + PITCH) + frow * 4, p.zscale + m * p.lds + block, on);
    cp_async_commit();
    next = row_of(s + 1);
  };
  auto meet = [&] {  // the group's warps
    if constexpr (RG == 1) __syncwarp();
    else if constexpr (MW == 1) __syncthreads();  // a barrier by number counts as all 16: 4 CTAs an SM
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + mw), "n"(32 * RG) : "memory");
  };
  for (int s = 0; s < S - 1; ++s) fetch(s);
  for (int s = 0; s < steps; ++s) {
    // one warp alone may fetch before it waits (its lanes have met after step
    // s - 1); warps that share a ring meet once, when step s is here and step
    // s - 1 has been read
    if constexpr (RG == 1) fetch(s + S - 1), cp_async_wait<S - 1>();
    else cp_async_wait<S - 2>();
    meet();
    if constexpr (RG != 1) fetch(s + S - 1);
    const unsigned char* src = ring + (s % S) * STEP;
    if constexpr (CONV) {
      // the group's 16-bit copy of the step: this thread's part of its row
      constexpr int W = ROW / TR / 4;  // words of codes
      uint32_t q[W], w[2 * W];
#pragma unroll
      for (int i = 0; i < W; i += 2) {
        const int k = fpart * W + i;  // word of the row, in piece k / 4
        const uint2 v = *reinterpret_cast<const uint2*>(src + frow * ROW + (((k / 4) ^ (frow & 7)) << 4) + k % 4 * 4);
        q[i] = v.x, q[i + 1] = v.y;
      }
#pragma unroll
      for (int i = 0; i < W; ++i)
        w[2 * i] = codes2<DT>(__byte_perm(q[i], 0, 0x4140)), w[2 * i + 1] = codes2<DT>(__byte_perm(q[i], 0, 0x4342));
#pragma unroll
      for (int i = 0; i < 2 * W / 4; ++i)
        *reinterpret_cast<uint4*>(wide + frow * 2 * kGrCols + (((fpart * (W / 2) + i) ^ (frow & 7)) << 4)) =
            make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
      meet();
    }
    // mid of rows 2t, 2t+1, 2t+8, 2t+9, ranks 2g and 2g+1 (n index g of the two n-tiles)
    float2 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 2 * t + (i & 1) + 4 * (i & 2);
      v[i] = *reinterpret_cast<const float2*>(src + 16 * ROW + row * PITCH + 64 * rg + 8 * g);
      if constexpr (CODES) {
        const float f = *reinterpret_cast<const float*>(src + 16 * (ROW + PITCH) + row * 4);
        v[i].x *= f, v[i].y *= f;
      }
    }
    if constexpr (DT == RQ_F16) {
      // keep mid near 2^14 as fp16: when a step's largest value passes the
      // scale in use, the sums so far are scaled down to the new one
      unsigned top = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        top = max(top, max(__float_as_uint(v[i].x) & 0x7fffffffu, __float_as_uint(v[i].y) & 0x7fffffffu));
      int ex = (int)(__reduce_max_sync(0xffffffffu, top) >> 23);
      if (ex == 255) {  // the largest finite one
        top = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          for (const float x : {fabsf(v[i].x), fabsf(v[i].y)})
            if (x < INFINITY) top = max(top, __float_as_uint(x));
        ex = (int)(__reduce_max_sync(0xffffffffu, top) >> 23);
      }
      if (ex > ex_now && ex > 30 && ex < 255) {
        if (ex_now) {
          const float down = ex - ex_now < 126 ? __uint_as_float((uint32_t)(127 - (ex - ex_now)) << 23) : 0x1p-126f;
#pragma unroll
          for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[i][n][e] *= down;
        }
        ex_now = ex;
        mul = __uint_as_float((uint32_t)(268 - ex) << 23);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i].x *= mul, v[i].y *= mul;
    }
    constexpr int P = kPieces<DT>;
    uint32_t b[P][2][2];  // [piece][n-tile][k pair]
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      uint32_t q[2][P];
      split16<DT>(v[2 * k].x, v[2 * k + 1].x, q[0]);
      split16<DT>(v[2 * k].y, v[2 * k + 1].y, q[1]);
#pragma unroll
      for (int e = 0; e < P; ++e) b[e][0][k] = q[0][e], b[e][1][k] = q[1][e];
    }
    // A fragments: 8 x 8 pieces (rows 0-7 | 8-15) x (a piece | the next), transposed
    const int lrow = (lane & 7) + 8 * (lane >> 4), lpiece = (lane >> 3) & 1;
    const unsigned char* z = (CONV ? wide : src) + lrow * (CONV ? 2 * kGrCols : ROW);
#pragma unroll
    for (int i = 0; i < 8; i += PAIR) {
      uint32_t f[PAIR][4];
      if constexpr (CODES && !CONV) {
        // a piece holds 16 columns as 8 pairs: the even columns (tile i) and the odd ones (tile i + 1) of
        // two pieces
        uint32_t raw[4];
        ldmatrix4_trans(raw, z + (((i + lpiece) ^ (lrow & 7)) << 4));
#pragma unroll
        for (int e = 0; e < 4; ++e) f[0][e] = codes2<DT>(raw[e]), f[PAIR - 1][e] = codes2<DT>(raw[e] >> 8);
      } else {
#pragma unroll
        for (int k = 0; k < PAIR; ++k) ldmatrix4_trans(f[k], z + (((2 * (i + k) + lpiece) ^ (lrow & 7)) << 4));
      }
#pragma unroll
      for (int e = 0; e < P; ++e) {
        if constexpr (AGAIN) {
          if (e == 1)
#pragma unroll
            for (int k = 0; k < PAIR; ++k)
#pragma unroll
              for (int q = 0; q < 4; ++q) f[k][q] = finite16<DT>(f[k][q]);
        }
#pragma unroll
        for (int k = 0; k < PAIR; ++k)
#pragma unroll
          for (int n = 0; n < 2; ++n)
            Mma16816<DT>::run(acc[i + k][n], f[k][0], f[k][1], f[k][2], f[k][3], b[e][n][0], b[e][n][1]);
      }
    }
    if constexpr (RG == 1) meet();  // all lanes have read the step before its place is fetched into
  }
  cp_async_wait<0>();
  return ex_now;
}

template <int DT, bool VEC, int RG, int MW>
__device__ __noinline__ int sum_rows_again(const GradArgs& p, int2 places, int block, int crank, int csize, float* sums) {
  float acc[8][2][4];
  const int ex = sum_rows<DT, false, VEC, RG, MW, true>(p, places, block, crank, csize, acc);
#pragma unroll
  for (int i = 0; i < 64; ++i) sums[i] = acc[i / 8][i / 4 % 2][i % 4];
  return ex;
}

// Whether one of a group's threads says so; its threads meet.
template <int RG, int MW>
__device__ __forceinline__ bool group_any(int mw, bool v) {
  if constexpr (RG == 1) {
    return __any_sync(0xffffffffu, v);
  } else if constexpr (MW == 1) {
    return __syncthreads_or(v);
  } else {
    int any;
    asm volatile("{\n.reg .pred p, q;\nsetp.ne.s32 p, %1, 0;\nbar.red.or.pred q, %2, %3, p;\nselp.s32 %0, 1, 0, q;\n}"
                 : "=r"(any)
                 : "r"((int)v), "r"(1 + mw), "n"(32 * RG)
                 : "memory");
    return any;
  }
}

// G_a[d, j] = sum over the rows m of a of z[m, d] mid[m, j].
//
// One CTA sums 128 columns of one adapter.  RG warps hold 16 ranks each; the
// MW groups of them (8 / RG, or 1) split the rows, and the CTAs of a cluster
// split them again.  Sums meet in shared and distributed shared memory in group and rank
// order, so equal inputs give equal bits, without atomics or a workspace.
//
// The reduction runs over rows, so the MMA's k index is the row and ldmatrix
// transposes z's tile on its way to the registers.  Each group fetches its own
// 16-row steps by cp.async into its own ring, a thread one row a step, and
// only the group waits for them.  z is read once.  Codes become 16-bit values
// exactly; their scale multiplies the other operand, mid, in fp32, which then
// enters as 16-bit pieces as in the row products.
//
// Bound by HBM in the limit; what a CTA costs besides its rows (sums, the
// meetings) is what is seen: 64 MB of z at rank 16 take 24 us, 32 MB of codes
// 22; rank 64 61 and 64 us, where four warps a group share the rows and the
// three pieces of mid are mma.sync's work.
template <int DT, bool CODES, bool VEC, int RG, int MW, bool LARGE>
__device__ __forceinline__ void adapter_gradient(const GradArgs& p) {
  using T = typename DType<DT>::T;
  constexpr int R16 = RG * 16, THREADS = 32 * RG * MW;
  constexpr bool CONV = CODES && RG > 1;
  extern __shared__ __align__(16) unsigned char smem[];
  float* sums = reinterpret_cast<float*>(smem);
  const AdapterRows& a = p.a;
  cg::cluster_group cluster = cg::this_cluster();
  const int crank = (int)cluster.block_rank(), csize = (int)cluster.num_blocks();
  const int block = (int)(blockIdx.x / csize);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int rg = warp % RG, mw = warp / RG;

  int adapter = blockIdx.y;
  if constexpr (LARGE) {
    adapter = nth_large<THREADS>(p, adapter);
    if (adapter < 0) return;
  }
  const int2 places = grad_rows(a, adapter);
  const int first = places.x, last = places.y;
  if (MW == 1 && p.beside && last - first > p.most) return;
  if (first >= last) {  // the whole cluster: no rows, zero gradient
    const int64_t d0 = (int64_t)block * kGrCols, n = min((int64_t)kGrCols, a.D1 - d0) * a.r / 8;
    uint4* G = reinterpret_cast<uint4*>(static_cast<T*>(p.G) + ((int64_t)adapter * a.D1 + d0) * a.r);
    for (int64_t i = crank * THREADS + tid; i < n; i += csize * THREADS) G[i] = make_uint4(0u, 0u, 0u, 0u);
    return;
  }
  const int64_t c0 = (int64_t)block * kGrCols;
  float acc[8][2][4];
  int ex_now = sum_rows<DT, CODES, VEC, RG, MW, false>(p, places, block, crank, csize, acc);
  if constexpr (!CODES) {  // codes are finite, but for a scale that is NaN
    bool nan = false;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int n = 0; n < 2; ++n) nan |= any_nan(acc[i][n][0], acc[i][n][1]) || any_nan(acc[i][n][2], acc[i][n][3]);
    if (group_any<RG, MW>(mw, nan)) {
      float again[64];
      ex_now = sum_rows_again<DT, VEC, RG, MW>(p, places, block, crank, csize, again);
#pragma unroll
      for (int i = 0; i < 64; ++i) acc[i / 8][i / 4 % 2][i % 4] = again[i];
    }
  }

  // this warp's sums: m-tile i's rows g and g + 8, ranks 4t .. 4t+3
  const float back = DT == RQ_F16 && ex_now ? __uint_as_float((uint32_t)(ex_now - 14) << 23) : 1.0f;
  // codes read as pairs: m-tile i has the even (odd) columns of pieces i and i + 1, i even (odd)
  auto column = [&](int at) { return c0 + (CODES && !CONV ? (at & ~31) + 2 * (at & 15) + ((at >> 4) & 1) : at); };
  auto write = [&](int64_t d, int j, float4 s) {
    if (d < a.D1 && j < a.r)
      *reinterpret_cast<uint2*>(static_cast<T*>(p.G) + ((int64_t)adapter * a.D1 + d) * a.r + j) =
          make_uint2(pair16<DT>(s.x, s.y), pair16<DT>(s.z, s.w));
  };
  if (MW == 1 && csize == 1) {  // nobody to meet
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        write(column(16 * i + g + 8 * h), rg * 16 + 4 * t,
              make_float4(acc[i][0][2 * h] * back, acc[i][1][2 * h] * back, acc[i][0][2 * h + 1] * back,
                          acc[i][1][2 * h + 1] * back));
    return;
  }
  __syncthreads();  // the sums lie over the ring
  // groups without a row have nothing to add
  const int active = min(MW, max(1, (last - first - crank * MW * 16 + 15) / 16));
  float* mine = sums + mw * kGrCols * R16 + rg * 16 + 4 * t;
  if (mw < active) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<float4*>(mine + (16 * i + g + 8 * h) * R16) =
            make_float4(acc[i][0][2 * h] * back, acc[i][1][2 * h] * back, acc[i][0][2 * h + 1] * back,
                        acc[i][1][2 * h + 1] * back);
  }
  __syncthreads();
  for (int i = tid; active > 1 && i < kGrCols * R16 / 4; i += THREADS) {
    float4 s = reinterpret_cast<const float4*>(sums)[i];
    for (int w = 1; w < active; ++w) {
      const float4 q = reinterpret_cast<const float4*>(sums + w * kGrCols * R16)[i];
      s.x += q.x, s.y += q.y, s.z += q.z, s.w += q.w;
    }
    reinterpret_cast<float4*>(sums)[i] = s;
  }
  cluster.sync();
  // 4 ranks of a column at a time, dealt to the cluster's CTAs
  const int units = R16 / 4;
  for (int i = tid * csize + crank; i < kGrCols * units; i += csize * THREADS) {
    const int at = i / units, j = (i - at * units) * 4;
    if (column(at) >= a.D1 || j >= a.r) continue;
    write(column(at), j, cluster_sum<float4>(cluster, sums + at * R16 + j, csize));
  }
  cluster.sync();  // the others have read this CTA's sums
}

// The two launches of a call with LARGE ones run beside one another: the first
// lets its dependent start once everything before it is complete, and the
// second, which reads and writes nothing of the first's, waits for it only at
// its end, so that whatever follows finds both complete.
template <int DT, bool CODES, bool VEC, int RG, int MW, bool LARGE>
__global__ void __launch_bounds__(32 * RG * MW, 16 / (RG * MW)) adapters_grad_k(const __grid_constant__ GradArgs p) {
  if (MW > 1 || !p.beside) grid_begin();
  adapter_gradient<DT, CODES, VEC, RG, MW, LARGE>(p);
  if (MW == 1 && p.beside) grid_begin();
}

template <int DT, bool CODES, bool VEC, int RG, int MW, bool LARGE = false>
static ClusterLaunch<GradArgs> grad_kernel() {
  const size_t wide = CODES && RG > 1 ? 16 * 2 * kGrCols : 0;  // the 16-bit copy of a step
  const size_t ring = (size_t)MW * (gr_steps(CODES, VEC, RG) * gr_step_bytes(CODES, RG) + wide);
  return {adapters_grad_k<DT, CODES, VEC, RG, MW, LARGE>, 32 * RG * MW, std::max(ring, (size_t)RG * MW * kGrSums)};
}

// A CTA costs about as much as 5 steps besides its steps (its sums through
// shared memory, the cluster's meetings): the cluster size that takes the
// fewest steps over all rounds of the GPU for `count` adapters of `each` rows,
// of which a CTA takes per_step a step.  That number of steps is left in best.
static int grad_cluster(const int* resident, int64_t blocks, int64_t count, int64_t each, int64_t per_step,
                        int64_t* best) {
  int csize = 1;
  *best = INT64_MAX;
  for (int c = 1; c <= 8; ++c) {
    const int64_t rounds = (blocks * count + resident[c] - 1) / resident[c];
    const int64_t steps = (each + per_step * c - 1) / (per_step * c);
    if (rounds * (5 + steps) < *best) *best = rounds * (5 + steps), csize = c;
  }
  return csize;
}

// For many adapters of few rows most groups of a CTA of 8 warps have none: they
// take CTAs of one group, of which up to 16 share an SM: 64 rows of 32 adapters,
// 11008 columns, rank 16, 10 us against 43; 8192 rows of 64, 4096
// columns, rank 16 31 against 57, rank 64 55 against 90.  The host does not
// know how the rows are spread, and an adapter of most of them would keep its
// one group for long (all 8192 rows, rank 16: 509 us): those of more than 4
// times the mean and 64 rows, no more than M / most of them, go to CTAs of 8
// warps in a launch beside.  Half of the rows on one adapter, and all: rank 16
// 62 and 90 us (66 and 85 where all adapters have such CTAs), rank 64 142 and
// 218 (164 and 286).
template <int DT, bool CODES, bool VEC, int RG>
static int launch_grad(const GradArgs& p, int64_t blocks, cudaStream_t st) {
  const int64_t M = p.a.M, count = p.a.count, each = (M + count - 1) / count;
  const auto many = grad_kernel<DT, CODES, VEC, RG, kGrWarps / RG>();
  int rc = many.prepare();
  if (rc != RQ_OK) return rc;
  int64_t steps;
  int csize = grad_cluster(many.resident(), blocks, count, each, kGrWarps / RG * 16, &steps);
  if constexpr (RG < kGrWarps) {
    const auto one = grad_kernel<DT, CODES, VEC, RG, 1>();
    if ((rc = one.prepare()) != RQ_OK) return rc;
    GradArgs q = p;
    q.most = (int)std::min<int64_t>(std::max<int64_t>(64, 4 * each), INT32_MAX - 1);
    const int64_t large = std::min(count, M / (q.most + 1));  // no more adapters than that have so many rows
    int64_t one_steps, rest = 0;
    const int one_csize = grad_cluster(one.resident(), blocks, count, each, 16, &one_steps);
    if (large) rest = 3 + (blocks * large + many.resident()[1] - 1) / many.resident()[1];  // a launch, CTAs that find none
    if (one_steps + rest < steps) {
      if (large) {
        const auto first = grad_kernel<DT, CODES, VEC, RG, kGrWarps / RG, true>();
        if ((rc = first.prepare()) != RQ_OK) return rc;
        csize = grad_cluster(first.resident(), blocks, large, M / large, kGrWarps / RG * 16, &steps);
        rc = first.launch(q, dim3((unsigned)(blocks * csize), (unsigned)large), csize, st);
        if (rc != RQ_OK) return rc;
        q.beside = 1;
      }
      return one.launch(q, dim3((unsigned)(blocks * one_csize), (unsigned)count), one_csize, st);
    }
  }
  return many.launch(p, dim3((unsigned)(blocks * csize), (unsigned)count), csize, st);
}

template <int DT, bool CODES, bool VEC>
static int launch_grad_r(const GradArgs& p, int64_t blocks, cudaStream_t st) {
  if (p.a.r <= 16) return launch_grad<DT, CODES, VEC, 1>(p, blocks, st);
  if (p.a.r <= 32) return launch_grad<DT, CODES, VEC, 2>(p, blocks, st);
  if (p.a.r <= 64) return launch_grad<DT, CODES, VEC, 4>(p, blocks, st);
  return launch_grad<DT, CODES, VEC, 8>(p, blocks, st);
}

template <int DT>
static int launch_grad_dt(const GradArgs& p, int64_t blocks, cudaStream_t st) {
  if (p.zscale) return launch_grad_r<DT, true, true>(p, blocks, st);
  return rows16b(p.z, p.ldz) && p.a.D1 % 8 == 0 ? launch_grad_r<DT, false, true>(p, blocks, st)
                                                : launch_grad_r<DT, false, false>(p, blocks, st);
}

int adapters_grad(const AdapterRows& a, const void* z, int64_t ldz, const float* zscale, int64_t lds, const float* mid,
                  void* G, cudaStream_t st) {
  const GradArgs p{a, z, ldz, zscale, lds, mid, G, 0, 0};
  const int64_t blocks = (a.D1 + kGrCols - 1) / kGrCols;
  return a.dt == RQ_BF16 ? launch_grad_dt<RQ_BF16>(p, blocks, st) : launch_grad_dt<RQ_F16>(p, blocks, st);
}

}  // namespace rq

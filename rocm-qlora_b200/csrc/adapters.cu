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
#include <cuda_runtime.h>

#include "linear_common.cuh"

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

__device__ __forceinline__ int row_group(const AdapterRows& a, int place, int64_t* row) {
  if (!a.plan) {
    *row = place;
    return 0;
  }
  *row = a.plan[plan_rows_at(a.M, a.count, a.tile) + place];
  int lo = 0, hi = a.count + 2;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (a.plan[1 + mid] <= place) lo = mid;
    else hi = mid;
  }
  return lo;
}

// mid[m, j] = s_a sum_d in[m, d] U_a[d, j]; one CTA a row.
template <int DT>
__global__ void __launch_bounds__(128) adapter_down_k(AdapterRows a, const void* __restrict__ in, int64_t ld,
                                                      const void* __restrict__ U, const float* __restrict__ scaling,
                                                      float* __restrict__ mid) {
  using T = typename DType<DT>::T;
  int64_t m;
  const int g = row_group(a, blockIdx.x, &m);
  const int j = threadIdx.x;
  if (j >= a.r) return;
  float acc = 0.0f;
  if (g < a.count) {
    const T* x = static_cast<const T*>(in) + m * ld;
    const T* u = static_cast<const T*>(U) + (int64_t)g * a.D1 * a.r + j;
    for (int64_t d = 0; d < a.D1; ++d) acc = fmaf(DType<DT>::to_f32(x[d]), DType<DT>::to_f32(u[d * a.r]), acc);
    acc *= scaling[g];
  } else if (g > a.count) {
    acc = __int_as_float(0x7fc00000);
  }
  mid[m * a.r + j] = acc;
}

// out[m, d] = base[m, d] + sum_j mid[m, j] V_a[d, j].
template <int DT>
__global__ void __launch_bounds__(256) adapter_up_k(AdapterRows a, const void* __restrict__ base, int64_t ldb,
                                                    const float* __restrict__ mid, const void* __restrict__ V,
                                                    void* __restrict__ out, int64_t ldo) {
  using T = typename DType<DT>::T;
  int64_t m;
  const int g = row_group(a, blockIdx.x, &m);
  const int64_t d = (int64_t)blockIdx.y * 256 + threadIdx.x;
  if (d >= a.D2) return;
  float acc = base ? DType<DT>::to_f32(static_cast<const T*>(base)[m * ldb + d]) : 0.0f;
  if (g < a.count) {
    const T* v = static_cast<const T*>(V) + ((int64_t)g * a.D2 + d) * a.r;
    float sum = 0.0f;
    for (int j = 0; j < a.r; ++j) sum = fmaf(mid[m * a.r + j], DType<DT>::to_f32(v[j]), sum);
    acc += sum;
  } else if (g > a.count) {
    acc = __int_as_float(0x7fc00000);
  }
  static_cast<T*>(out)[m * ldo + d] = DType<DT>::from_f32(acc);
}

int adapters_apply(const AdapterRows& a, const void* in, int64_t ldin, const void* U, const void* V,
                   const float* scaling, const void* base, int64_t ldb, float* mid, void* out, int64_t ldo,
                   cudaStream_t st) {
  const dim3 grid((unsigned)a.M, (unsigned)((a.D2 + 255) / 256));
  if (a.dt == RQ_BF16) {
    adapter_down_k<RQ_BF16><<<(unsigned)a.M, 128, 0, st>>>(a, in, ldin, U, scaling, mid);
    adapter_up_k<RQ_BF16><<<grid, 256, 0, st>>>(a, base, ldb, mid, V, out, ldo);
  } else {
    adapter_down_k<RQ_F16><<<(unsigned)a.M, 128, 0, st>>>(a, in, ldin, U, scaling, mid);
    adapter_up_k<RQ_F16><<<grid, 256, 0, st>>>(a, base, ldb, mid, V, out, ldo);
  }
  return check_launch();
}

// ------------------------------------------------------------------- grad

// G_a[d, j] = sum over the rows of a of z[m, d] mid[m, j]; z either 16-bit
// rows or 8-bit codes with one scale a 128 columns.
template <int DT>
__global__ void __launch_bounds__(128) adapter_grad_k(AdapterRows a, const void* __restrict__ z, int64_t ldz,
                                                      const float* __restrict__ zscale, int64_t lds,
                                                      const float* __restrict__ mid, void* __restrict__ G) {
  using T = typename DType<DT>::T;
  const int g = blockIdx.x, j = threadIdx.x;
  const int64_t d = blockIdx.y;
  if (j >= a.r) return;
  const int first = a.plan ? a.plan[1 + g] : 0, last = a.plan ? a.plan[2 + g] : (int)a.M;
  const int* order = a.plan ? a.plan + plan_rows_at(a.M, a.count, a.tile) : nullptr;
  float acc = 0.0f;
  for (int p = first; p < last; ++p) {
    const int64_t m = order ? order[p] : p;
    const float v = zscale ? (float)static_cast<const int8_t*>(z)[m * ldz + d] * zscale[m * lds + d / 128]
                           : DType<DT>::to_f32(static_cast<const T*>(z)[m * ldz + d]);
    acc = fmaf(v, mid[m * a.r + j], acc);
  }
  static_cast<T*>(G)[((int64_t)g * a.D1 + d) * a.r + j] = DType<DT>::from_f32(acc);
}

int adapters_grad(const AdapterRows& a, const void* z, int64_t ldz, const float* zscale, int64_t lds, const float* mid,
                  void* G, cudaStream_t st) {
  const dim3 grid((unsigned)a.count, (unsigned)a.D1);
  if (a.dt == RQ_BF16)
    adapter_grad_k<RQ_BF16><<<grid, 128, 0, st>>>(a, z, ldz, zscale, lds, mid, G);
  else
    adapter_grad_k<RQ_F16><<<grid, 128, 0, st>>>(a, z, ldz, zscale, lds, mid, G);
  return check_launch();
}

}  // namespace rq

// preference.cu -- log-probabilities of the given tokens, the paired
// preference loss on them, and the gradient of both.
//
// With row x = logits[b, l] and y = labels[b, l + 1]:
//   m = max x,  s = sum_v e^(x_v - m),  log p(y) = x_y - m - log s
//   d log p(y) / dx_v = [v = y] - e^(x_v - m) / s
// A pair is sequence i (chosen) and i + P (rejected), P = B / 2; each token's
// advantage over the reference is summed over the sequence,
//   R_b = sum_l (log p - log p_ref),  z_i = beta (R_i - R_{i+P})
//   sigmoid: loss = mean(-(1 - w) log sigma(z) - w log sigma(-z))
//   ipo:     loss = mean((R_i / n_i - R_{i+P} / n_{i+P} - 1 / (2 beta))^2)
// and the gradient of every logit row of a sequence is one slope (dloss / dR)
// times the row's derivative above.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include "gemv_common.cuh"

namespace cg = cooperative_groups;

namespace rq {

constexpr int kTokThreads = 512;  // of a row, in the gradient and where rows are few
constexpr int kTokBatch = 4;      // 16-byte loads of a thread at a time
// log2(e) as the sum of two floats: the first alone is 1.3e-8 of itself off,
// which would shift every log-probability by that much of the row's entropy
constexpr double kLog2eD = 1.4426950408889634;
constexpr float kLog2e = (float)kLog2eD, kLog2eRest = (float)(kLog2eD - (double)(float)kLog2eD);

// The label that scores row `at` of B * L; false where the row does not count.
__device__ __forceinline__ bool row_label(const TokenRows& t, int64_t at, int64_t* y) {
  const int64_t b = at / t.L, l = at - b * t.L;
  if (l + 1 >= t.L) return false;
  *y = t.labels[b * t.L + l + 1];
  return *y != t.ignore;
}

template <int DT>
__device__ __forceinline__ const typename DType<DT>::T* row_of(const TokenRows& t, int64_t at) {
  const int64_t b = at / t.L, l = at - b * t.L;
  return static_cast<const typename DType<DT>::T*>(t.logits) + b * t.sb + l * t.sl;
}

// A row cut at 16-byte boundaries: `head` values, `vecs` loads, `tail` values.
template <int DT>
struct RowCut {
  using T = typename DType<DT>::T;
  static constexpr int E = 16 / (int)sizeof(T);
  int head, vecs, tail;
  __device__ RowCut(const T* x, int V) {
    head = min(V, (int)((16u - ((uint32_t)(uintptr_t)x & 15u)) & 15u) / (int)sizeof(T));
    vecs = (V - head) / E;
    tail = V - head - vecs * E;
  }
};

template <int DT>
__device__ __forceinline__ void unpack16(const uint4& q, float* f) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == RQ_F32) {
      f[i] = __uint_as_float(w[i]);
    } else if constexpr (DT == RQ_BF16) {
      f[2 * i] = __uint_as_float(w[i] << 16), f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      f[2 * i] = v.x, f[2 * i + 1] = v.y;
    }
  }
}

template <int DT>
__device__ __forceinline__ uint32_t pack16x2(float lo, float hi) {
  if constexpr (DT == RQ_BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// e^x / 2^k
__device__ __forceinline__ float exp_over(float x, float k) {
  return exp2_fast(fmaf(x, kLog2eRest, fmaf(x, kLog2e, -k)));
}

// 2^n for a whole n <= 0
__device__ __forceinline__ float whole_exp2(float n) {
  return n < -126.0f ? 0.0f : __int_as_float((127 + (int)n) << 23);
}

// A running sum of e^x as s * 2^k, k whole and never below the largest
// x log2(e) seen.  With a whole k the shift costs no rounding: e^x / 2^k is
// two fused multiply-adds and one exponential a value, and moving k scales s
// by a power of two.  All exponentials are of arguments up to 0, where
// ex2.approx errs by -4.97e-8 of its value on average (measured over 2^22
// fractions; +3.3e-8 above 0): a sum takes that back at its end, since over
// thousands of tokens it would add up.
constexpr double kExp2Low = 4.97e-8;

// The range of k.  Beyond it fp32 no longer holds x log2(e) to a fraction, and
// at the type's ends not at all.  Values further down count as none beside a
// largest one that is not down there itself; values further up make the sum
// infinite.  Rows of either kind are summed again, by wide_row.
constexpr float kWhole = 0x1p20f;

struct ExpSum {
  float k = 0.0f, s = 0.0f;
  __device__ __forceinline__ void raise(float top) {  // top: the largest of the values to come
    const float z = top * kLog2e;
    if ((z > k || s == 0.0f) && fabsf(z) < kWhole) {
      const float to = ceilf(z);
      if (s != 0.0f) s *= whole_exp2(k - to);
      k = to;
    }
  }
  template <int N>
  __device__ __forceinline__ void add(const float (&x)[N]) {
    float top = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i) top = fmaxf(top, x[i]);
    raise(top);
    float e[N];
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = exp_over(x[i], k);
#pragma unroll
    for (int w = N / 2; w > 0; w /= 2)
#pragma unroll
      for (int i = 0; i < w; ++i) e[i] += e[i + w];
    s += e[0];
  }
};

// A row of logits of any magnitude (masked whole with the type's lowest value,
// say), by its definition: the largest value first, then the sum of e^(x - m)
// in 64 bits.  NaN where that is no distribution: an infinity above, a NaN, or
// nothing finite.  Leaves the warps' largest values and sums for their threads to join.
template <int DT, int TH>
__device__ __noinline__ void wide_row(const typename DType<DT>::T* x, int V, float* tops, double* sums) {
  const int tid = threadIdx.x;
  float top = -INFINITY;
  bool none = false;
  for (int v = tid; v < V; v += TH) {
    const float f = DType<DT>::to_f32(x[v]);
    none |= !(f < INFINITY);
    top = fmaxf(top, f);
  }
  none = __syncthreads_or(none);  // and all have read what tops held
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((tid & 31) == 0) tops[tid >> 5] = top;
  __syncthreads();
  for (int w = 0; w < TH / 32; ++w) top = fmaxf(top, tops[w]);
  double s = 0.0;
  for (int v = tid; v < V; v += TH) s += (double)expf(DType<DT>::to_f32(x[v]) - top);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((tid & 31) == 0) sums[tid >> 5] = none ? (double)__uint_as_float(0x7fc00000u) : s;
  __syncthreads();
}

// stats[at] = (k, s, hi, lo) of each row that counts: the normaliser s 2^k (of
// a wide row (m, -s): -s below zero marks it, and the normaliser is s e^m) and
// the label's log-probability hi + lo; logps (optional) has it at the label's
// own place [b, l + 1], and 0 where nothing counts.  One CTA a row, one pass;
// bound by HBM, with the exponentials (16 a clock of an SM) at 72 % of the
// time a bf16 row takes to arrive.  The end of a row is a few serial steps, so
// where rows are many, small CTAs of which eight share an SM hide it: 16384
// rows of 32000 bf16 logits (14792 count) take 159 us with 128 threads (6.0
// TB/s; nine CTAs an SM, with eight 166) and 256 with 512, but 128 rows 6.3
// and 4.9 us.
template <int DT, int TH>
__global__ void __launch_bounds__(TH, TH == 128 ? 9 : 2) token_stats_k(TokenRows t, float4* __restrict__ stats,
                                                             float* __restrict__ logps) {
  grid_begin();
  using T = typename DType<DT>::T;
  constexpr int E = RowCut<DT>::E;
  const int64_t at = blockIdx.x;
  const int tid = threadIdx.x;
  __shared__ float ks[TH / 32];
  __shared__ double sums[TH / 32];
  int64_t y;
  const bool counts = row_label(t, at, &y);
  if (logps && tid == 0) {
    if (at % t.L == 0) logps[at] = 0.0f;
    if (!counts && at % t.L + 1 < t.L) logps[at + 1] = 0.0f;
  }
  if (!counts) return;
  const T* x = row_of<DT>(t, at);
  const RowCut<DT> cut(x, (int)t.V);
  const uint4* body = reinterpret_cast<const uint4*>(x + cut.head);
  ExpSum sum;
  for (int i = tid; i < cut.vecs; i += kTokBatch * TH) {
    uint4 q[kTokBatch];
#pragma unroll
    for (int j = 0; j < kTokBatch; ++j) {
      const uint32_t low = DT == RQ_F32 ? 0xff800000u : DT == RQ_BF16 ? 0xff80ff80u : 0xfc00fc00u;  // -inf
      q[j] = i + j * TH < cut.vecs ? body[i + j * TH] : make_uint4(low, low, low, low);
    }
    float f[kTokBatch * E];
#pragma unroll
    for (int j = 0; j < kTokBatch; ++j) unpack16<DT>(q[j], f + j * E);
    sum.add(f);
  }
  // the ends of a row that does not start or end on a 16-byte boundary
  if (tid < cut.head + cut.tail) {
    const float f[1] = {DType<DT>::to_f32(x[tid < cut.head ? tid : t.V - cut.tail + (tid - cut.head)])};
    sum.add(f);
  }
  // the threads' sums meet at the largest k, in 64 bits
  float k = sum.s == 0.0f ? -INFINITY : sum.k;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) k = fmaxf(k, __shfl_xor_sync(0xffffffffu, k, o));
  if ((tid & 31) == 0) ks[tid >> 5] = k;
  bool wide = __syncthreads_or(!(sum.s < INFINITY));
  k = ks[0];
#pragma unroll
  for (int w = 1; w < TH / 32; ++w) k = fmaxf(k, ks[w]);
  wide |= k < -0.5f * kWhole;
  if (wide) {
    wide_row<DT, TH>(x, (int)t.V, ks, sums);
    k = ks[0];
    for (int w = 1; w < TH / 32; ++w) k = fmaxf(k, ks[w]);
  } else {
    double s = sum.s == 0.0f ? 0.0 : (double)sum.s * (double)whole_exp2(sum.k - k);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if ((tid & 31) == 0) sums[tid >> 5] = s;
    __syncthreads();
  }
  if (tid == 0) {
    double s = sums[0];
    for (int w = 1; w < TH / 32; ++w) s += sums[w];
    if (!wide) s *= 1.0 + kExp2Low;
    // a label outside the vocabulary has no probability: NaN, not a read past the row
    const float xy = y >= 0 && y < t.V ? DType<DT>::to_f32(x[y]) : __uint_as_float(0x7fc00000u);
    const double lp = (double)xy - (wide ? (double)k : (double)k / kLog2eD) - log2(s) / kLog2eD;
    const float hi = (float)lp;
    stats[at] = make_float4(k, wide ? (float)-s : (float)s, hi, fabsf(hi) < INFINITY ? (float)(lp - (double)hi) : 0.0f);
    if (logps) logps[at + 1] = hi;
  }
}

// Sums per sequence in 64 bits (thousands of tokens, of which the loss takes a
// small difference), then the loss and each sequence's slope.  One cluster:
// pairs are dealt to its CTAs, a pair's two sequences to `ws` warps each, and
// the loss's terms meet in rank order.
constexpr int kPrefWarps = 32, kPrefCtas = 8;

struct SequenceSum {
  double lp, d;  // of log p, and of log p - ref
  int n;
};

__global__ void __launch_bounds__(kPrefWarps * 32) __cluster_dims__(kPrefCtas, 1, 1)
    preference_loss_k(TokenRows t, const float4* __restrict__ stats, const float* __restrict__ ref, int form,
                      float beta, float smooth, float* __restrict__ loss, float* __restrict__ logps,
                      float* __restrict__ rewards, float* __restrict__ slopes) {
  constexpr int U = 4;  // rows of a lane under way
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ SequenceSum part[kPrefWarps];
  __shared__ double total[kPrefWarps];
  grid_begin();
  const int P = (int)(t.B / 2);
  int ws = kPrefWarps / 2;  // warps of a sequence: fewer where that leaves lanes without a row
  while (ws > 1 && ws * 32 >= 2 * t.L) ws /= 2;
  const int at_once = kPrefWarps / (2 * ws), slot = warp / ws;  // slot: pair and half
  double mine = 0.0;  // of the first lane of a pair's warps
  for (int i0 = blockIdx.x * at_once; i0 < P; i0 += kPrefCtas * at_once) {
    const int i = i0 + slot / 2, b = i + (slot & 1) * P;
    SequenceSum s{0.0, 0.0, 0};
    if (i < P) {
      const int64_t row0 = (int64_t)b * t.L;
      for (int64_t l0 = (warp % ws) * 32 + lane; l0 + 1 < t.L; l0 += U * ws * 32) {
        int64_t y[U];
        float4 q[U];
        float r[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int64_t l = l0 + u * ws * 32;
          const bool in = l + 1 < t.L;
          y[u] = in ? t.labels[row0 + l + 1] : t.ignore;
          q[u] = in ? stats[row0 + l] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          r[u] = in ? ref[row0 + l + 1] : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (y[u] == t.ignore) continue;
          const double lp = (double)q[u].z + (double)q[u].w;
          s.lp += lp;
          s.d += lp - (double)r[u];
          ++s.n;
        }
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s.lp += __shfl_xor_sync(0xffffffffu, s.lp, o);
      s.d += __shfl_xor_sync(0xffffffffu, s.d, o);
      s.n += __shfl_xor_sync(0xffffffffu, s.n, o);
    }
    if (lane == 0) part[warp] = s;
    __syncthreads();
    if (lane == 0 && warp % (2 * ws) == 0 && i < P) {
      SequenceSum h[2];
      for (int k = 0; k < 2; ++k) {
        h[k] = part[warp + k * ws];
        for (int w = 1; w < ws; ++w) {
          const SequenceSum& q = part[warp + k * ws + w];
          h[k].lp += q.lp, h[k].d += q.d, h[k].n += q.n;
        }
        logps[i + k * P] = (float)h[k].lp;
        rewards[i + k * P] = (float)(beta * h[k].d);
      }
      double s0, s1;
      if (form == RQ_PREF_IPO) {
        const double n0 = max(h[0].n, 1), n1 = max(h[1].n, 1);
        const double off = h[0].d / n0 - h[1].d / n1 - 0.5 / beta;
        mine += off * off;
        s0 = 2.0 * off / P / n0, s1 = -2.0 * off / P / n1;
      } else {
        const double z = beta * (h[0].d - h[1].d), soft = log1p(exp(-fabs(z)));
        mine += (1.0 - smooth) * (soft + fmax(-z, 0.0)) + smooth * (soft + fmax(z, 0.0));
        s0 = beta * (1.0 / (1.0 + exp(-z)) - (1.0 - smooth)) / P;
        s1 = -s0;
      }
      slopes[i] = (float)s0;
      slopes[i + P] = (float)s1;
    }
    __syncthreads();
  }
  if (lane == 0) total[warp] = mine;
  cluster.sync();
  if (blockIdx.x == 0 && warp == 0) {  // lane w: warp w of every CTA
    double all = 0.0;
    for (int c = 0; c < kPrefCtas; ++c) all += *cluster.map_shared_rank(&total[lane], c);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    if (lane == 0) *loss = (float)(all / P);
  }
  cluster.sync();  // the others' terms have been read
}

// dlogits = c ([v = y] - 2^(x log2(e) - k) / s), zero where the row does not
// count; of a wide row e^(x - m) / s.  The approximate exponential errs by
// 2^-22 of a probability: fp32 gradients are 3.8e-7 of their norm off, 3.7e-7
// with torch's 32-bit operations.  One CTA a row, the rows in the reverse of the
// forward's order, so that the last rows it read are still in L2.  HBM bound:
// 301 us for 16384 rows of 32000 bf16 logits of which 14792 count, 6.6 TB/s.
template <int DT>
__global__ void __launch_bounds__(kTokThreads) token_grad_k(TokenRows t, const float4* __restrict__ stats,
                                                            const float* __restrict__ slopes, int per_token,
                                                            const float* __restrict__ upstream, void* __restrict__ out) {
  grid_begin();
  using T = typename DType<DT>::T;
  constexpr int E = RowCut<DT>::E;
  const int64_t at = (int64_t)gridDim.x - 1 - blockIdx.x;
  const int tid = threadIdx.x;
  T* d = static_cast<T*>(out) + at * t.V;
  int64_t y;
  if (!row_label(t, at, &y)) {
    const RowCut<DT> cut(d, (int)t.V);
    uint4* body = reinterpret_cast<uint4*>(d + cut.head);
    for (int i = tid; i < cut.vecs; i += kTokThreads) __stcs(body + i, make_uint4(0u, 0u, 0u, 0u));
    if (tid < cut.head + cut.tail) d[tid < cut.head ? tid : t.V - cut.tail + (tid - cut.head)] = DType<DT>::from_f32(0.0f);
    return;
  }
  const T* x = row_of<DT>(t, at);
  const float4 q = stats[at];
  float c = per_token ? slopes[at + 1] : slopes[at / t.L];
  if (upstream) c *= *upstream;
  if (y < 0 || y >= t.V) c = __uint_as_float(0x7fc00000u);
  const bool wide = q.y < 0.0f;
  const float by = -c / fabsf(q.y), k = wide ? 0.0f : q.x, m = wide ? q.x : 0.0f;
  auto value = [&](float f) { return by * exp_over(f, k); };
  if (!wide && (((uintptr_t)x ^ (uintptr_t)d) & 15) == 0) {
    const RowCut<DT> cut(x, (int)t.V);
    const uint4* src = reinterpret_cast<const uint4*>(x + cut.head);
    uint4* dst = reinterpret_cast<uint4*>(d + cut.head);
    const int hit = y >= cut.head ? (int)(y - cut.head) / E : -1, which = (int)(y - cut.head) % E;  // the label's load
    for (int i = tid; i < cut.vecs; i += kTokBatch * kTokThreads) {
      uint4 v[kTokBatch];
#pragma unroll
      for (int j = 0; j < kTokBatch; ++j)
        if (i + j * kTokThreads < cut.vecs) v[j] = __ldcs(src + i + j * kTokThreads);
#pragma unroll
      for (int j = 0; j < kTokBatch; ++j) {
        const int at_vec = i + j * kTokThreads;
        if (at_vec >= cut.vecs) continue;
        float f[E];
        unpack16<DT>(v[j], f);
#pragma unroll
        for (int e = 0; e < E; ++e) f[e] = value(f[e]);
        if (at_vec == hit) {
#pragma unroll
          for (int e = 0; e < E; ++e) f[e] += e == which ? c : 0.0f;
        }
        uint4 r;
        if constexpr (DT == RQ_F32)
          r = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
        else
          r = make_uint4(pack16x2<DT>(f[0], f[1]), pack16x2<DT>(f[2], f[3]), pack16x2<DT>(f[E - 4], f[E - 3]),
                         pack16x2<DT>(f[E - 2], f[E - 1]));
        __stcs(dst + at_vec, r);
      }
    }
    if (tid < cut.head + cut.tail) {
      const int64_t v = tid < cut.head ? tid : t.V - cut.tail + (tid - cut.head);
      d[v] = DType<DT>::from_f32(value(DType<DT>::to_f32(x[v])) + (v == y ? c : 0.0f));
    }
  } else {  // rows of different alignment, wide rows: value by value
    for (int64_t v = tid; v < t.V; v += kTokThreads)
      d[v] = DType<DT>::from_f32(value(DType<DT>::to_f32(x[v]) - m) + (v == y ? c : 0.0f));
  }
}

template <int DT>
static int launch_stats(const TokenRows& t, float4* stats, float* logps, cudaStream_t st) {
  const unsigned grid = (unsigned)(t.B * t.L);
  if (grid >= 8u * num_sms()) return launch_dependent(token_stats_k<DT, 128>, grid, 128, st, t, stats, logps);
  return launch_dependent(token_stats_k<DT, kTokThreads>, grid, kTokThreads, st, t, stats, logps);
}

int token_logprobs(const TokenRows& t, float* stats, float* logps, cudaStream_t st) {
  auto* launch = t.dt == RQ_F32 ? launch_stats<RQ_F32> : t.dt == RQ_BF16 ? launch_stats<RQ_BF16> : launch_stats<RQ_F16>;
  return launch(t, (float4*)stats, logps, st);
}

int preference_loss(const TokenRows& t, const float* stats, const float* ref, int form, float beta, float smooth,
                    float* loss, float* logps, float* rewards, float* slopes, cudaStream_t st) {
  return launch_dependent(preference_loss_k, kPrefCtas, kPrefWarps * 32, st, t, (const float4*)stats, ref, form, beta,
                          smooth, loss, logps, rewards, slopes);
}

int token_logprobs_grad(const TokenRows& t, const float* stats, const float* slopes, int per_token,
                        const float* upstream, void* dlogits, cudaStream_t st) {
  auto* kern = t.dt == RQ_F32 ? token_grad_k<RQ_F32> : t.dt == RQ_BF16 ? token_grad_k<RQ_BF16> : token_grad_k<RQ_F16>;
  return launch_dependent(kern, (unsigned)(t.B * t.L), kTokThreads, st, t, (const float4*)stats, slopes, per_token,
                          upstream, dlogits);
}

}  // namespace rq

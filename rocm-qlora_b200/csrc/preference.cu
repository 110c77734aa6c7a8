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
#include <cuda_runtime.h>

#include "linear_common.cuh"

namespace rq {

constexpr int kTokThreads = 256;

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

// stats[at] = (m, s, x_y, 0) of each row that counts; logps (optional), at the
// label's own place [b, l + 1], is log p and 0 where nothing counts.
template <int DT>
__global__ void __launch_bounds__(kTokThreads) token_stats_k(TokenRows t, float4* __restrict__ stats,
                                                             float* __restrict__ logps) {
  const int64_t at = blockIdx.x;
  const int tid = threadIdx.x;
  __shared__ float red[kTokThreads / 32];
  int64_t y;
  const bool counts = row_label(t, at, &y);
  if (logps && tid == 0) {
    if (at % t.L == 0) logps[at] = 0.0f;
    if (!counts && at % t.L + 1 < t.L) logps[at + 1] = 0.0f;
  }
  if (!counts) return;
  const typename DType<DT>::T* x = row_of<DT>(t, at);
  float m = -INFINITY;
  bool bad = false;
  for (int64_t v = tid; v < t.V; v += kTokThreads) {
    const float f = DType<DT>::to_f32(x[v]);
    bad |= isnan(f);
    m = fmaxf(m, f);
  }
  if (bad) m = __uint_as_float(0x7fc00000u);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float u = __shfl_xor_sync(0xffffffffu, m, o);
    m = (isnan(u) || isnan(m)) ? __uint_as_float(0x7fc00000u) : fmaxf(m, u);
  }
  if ((tid & 31) == 0) red[tid >> 5] = m;
  __syncthreads();
  for (int w = 0; w < kTokThreads / 32; ++w) m = (isnan(red[w]) || isnan(m)) ? __uint_as_float(0x7fc00000u) : fmaxf(m, red[w]);
  __syncthreads();
  float s = 0.0f;
  for (int64_t v = tid; v < t.V; v += kTokThreads) s += expf(DType<DT>::to_f32(x[v]) - m);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((tid & 31) == 0) red[tid >> 5] = s;
  __syncthreads();
  if (tid == 0) {
    s = 0.0f;
    for (int w = 0; w < kTokThreads / 32; ++w) s += red[w];
    // a label outside the vocabulary has no probability: NaN, not a read past the row
    const float xy = y >= 0 && y < t.V ? DType<DT>::to_f32(x[y]) : __uint_as_float(0x7fc00000u);
    stats[at] = make_float4(m, s, xy, 0.0f);
    if (logps) logps[at + 1] = (float)((double)(xy - m) - log((double)s));
  }
}

// One CTA: sums per sequence in 64 bits (thousands of tokens, of which the
// loss takes a small difference), then the loss and each sequence's slope.
__global__ void __launch_bounds__(1024) preference_loss_k(TokenRows t, const float4* __restrict__ stats,
                                                          const float* __restrict__ ref, int form, float beta,
                                                          float smooth, float* __restrict__ loss,
                                                          float* __restrict__ logps, float* __restrict__ rewards,
                                                          float* __restrict__ slopes) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  __shared__ double part[32];
  const int64_t P = t.B / 2;
  double mine = 0.0;  // warp's pairs, in order
  for (int64_t i = warp; i < P; i += 32) {
    double R[2], n[2];
    for (int h = 0; h < 2; ++h) {
      const int64_t b = i + h * P;
      double lp = 0.0, rf = 0.0;
      int cnt = 0;
      for (int64_t l = lane; l + 1 < t.L; l += 32) {
        int64_t y;
        if (!row_label(t, b * t.L + l, &y)) continue;
        const float4 q = stats[b * t.L + l];
        lp += (double)(q.z - q.x) - log((double)q.y);
        rf += (double)ref[b * t.L + l + 1];
        ++cnt;
      }
      double d = lp - rf;
      for (int o = 16; o > 0; o >>= 1) {
        lp += __shfl_xor_sync(0xffffffffu, lp, o);
        d += __shfl_xor_sync(0xffffffffu, d, o);
        cnt += __shfl_xor_sync(0xffffffffu, cnt, o);
      }
      R[h] = d;
      n[h] = cnt > 0 ? cnt : 1;
      if (lane == 0) {
        logps[b] = (float)lp;
        rewards[b] = (float)(beta * d);
      }
    }
    double slope, s0, s1;
    if (form == RQ_PREF_IPO) {
      const double off = R[0] / n[0] - R[1] / n[1] - 0.5 / beta;
      mine += off * off;
      slope = 2.0 * off / P;
      s0 = slope / n[0], s1 = -slope / n[1];
    } else {
      const double z = beta * (R[0] - R[1]), soft = log1p(exp(-fabs(z)));
      mine += (1.0 - smooth) * (soft + fmax(-z, 0.0)) + smooth * (soft + fmax(z, 0.0));
      slope = beta * (1.0 / (1.0 + exp(-z)) - (1.0 - smooth)) / P;
      s0 = slope, s1 = -slope;
    }
    if (lane == 0) {
      slopes[i] = (float)s0;
      slopes[i + P] = (float)s1;
    }
  }
  if (lane == 0) part[warp] = mine;
  __syncthreads();
  if (tid == 0) {
    double all = 0.0;
    for (int w = 0; w < 32; ++w) all += part[w];
    *loss = (float)(all / P);
  }
}

template <int DT>
__global__ void __launch_bounds__(kTokThreads) token_grad_k(TokenRows t, const float4* __restrict__ stats,
                                                            const float* __restrict__ slopes, int per_token,
                                                            const float* __restrict__ upstream, void* __restrict__ out) {
  using T = typename DType<DT>::T;
  const int64_t at = blockIdx.x;
  T* d = static_cast<T*>(out) + at * t.V;
  int64_t y;
  if (!row_label(t, at, &y)) {
    for (int64_t v = threadIdx.x; v < t.V; v += kTokThreads) d[v] = DType<DT>::from_f32(0.0f);
    return;
  }
  const T* x = row_of<DT>(t, at);
  const float4 q = stats[at];
  float c = per_token ? slopes[at + 1] : slopes[at / t.L];
  if (upstream) c *= *upstream;
  if (y < 0 || y >= t.V) c = __uint_as_float(0x7fc00000u);
  const float k = -c / q.y;
  for (int64_t v = threadIdx.x; v < t.V; v += kTokThreads)
    d[v] = DType<DT>::from_f32(fmaf(k, expf(DType<DT>::to_f32(x[v]) - q.x), v == y ? c : 0.0f));
}

#define RQ_TOK_LAUNCH(kern, ...)                                                                  \
  do {                                                                                            \
    const unsigned grid = (unsigned)(t.B * t.L);                                                  \
    if (t.dt == RQ_F32) kern<RQ_F32><<<grid, kTokThreads, 0, st>>>(__VA_ARGS__);                  \
    else if (t.dt == RQ_BF16) kern<RQ_BF16><<<grid, kTokThreads, 0, st>>>(__VA_ARGS__);           \
    else kern<RQ_F16><<<grid, kTokThreads, 0, st>>>(__VA_ARGS__);                                 \
    return check_launch();                                                                        \
  } while (0)

int token_logprobs(const TokenRows& t, float* stats, float* logps, cudaStream_t st) {
  RQ_TOK_LAUNCH(token_stats_k, t, (float4*)stats, logps);
}

int preference_loss(const TokenRows& t, const float* stats, const float* ref, int form, float beta, float smooth,
                    float* loss, float* logps, float* rewards, float* slopes, cudaStream_t st) {
  preference_loss_k<<<1, 1024, 0, st>>>(t, (const float4*)stats, ref, form, beta, smooth, loss, logps, rewards, slopes);
  return check_launch();
}

int token_logprobs_grad(const TokenRows& t, const float* stats, const float* slopes, int per_token,
                        const float* upstream, void* dlogits, cudaStream_t st) {
  RQ_TOK_LAUNCH(token_grad_k, t, (const float4*)stats, slopes, per_token, upstream, dlogits);
}

}  // namespace rq

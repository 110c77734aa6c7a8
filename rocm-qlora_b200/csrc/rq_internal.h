// rq_internal.h -- internal (C++) interface between the C-ABI layer and the
// kernel translation units.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/rq_b200.h"

namespace rq {

// Kernel family of the last layer call in this thread (RQ_PATH_*).
int last_path();

// Decode GEMV numerics (rq_set_decode_exact; gemv_nf4.cu).
void set_decode_exact(int on);

// Records the CUDA error of the last failing launch in this thread.
void set_cuda_error(cudaError_t e);

// Driver-API failures (tensor-map encoding) are recorded as this base plus
// the CUresult, so that they do not read as runtime error codes.
constexpr int kDriverErrorBase = 10000;

// Raises a kernel's dynamic shared memory limit to `bytes` on the current
// device (once per kernel, device and size; thread-safe).
int ensure_smem_limit(const void* kernel, size_t bytes);

// Maps the launch status of the kernel just issued to an RQ_* status.
inline int check_launch() {
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_cuda_error(e);
    return RQ_ERR_CUDA;
  }
  return RQ_OK;
}

// Launches a kernel that begins with grid_begin() as the programmatic
// dependent of the kernel before it.
template <class... P, class... A>
int launch_dependent(void (*kern)(P...), unsigned grid, unsigned threads, cudaStream_t st, A&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, static_cast<P>(args)...);
  if (e != cudaSuccess) {
    set_cuda_error(e);
    return RQ_ERR_CUDA;
  }
  return check_launch();
}

int nf4_quantize(const void* x, int dtype, int64_t n, int bs, uint8_t* packed, void* scales, cudaStream_t st);
int nf4_dequantize(const uint8_t* p, int64_t nbytes, const void* s, int sdt, int bs, void* out, int odt,
                   cudaStream_t st);
int dq_dequantize(const uint8_t* p, int64_t numel, const uint8_t* c2, const float* c2s, int fp8, int bs, int bs2,
                  void* out, int odt, cudaStream_t st);
int dq_quantize_scales(const float* c1, int64_t nb, int bs2, int fp8, uint8_t* c2, float* c2s, cudaStream_t st);
int int8_quantize(const void* x, int dtype, int64_t n, int bs, int8_t* q, void* scales, cudaStream_t st);
int int8_quantize_rows(const void* x, int dtype, int64_t rows, int64_t cols, int8_t* q, void* scales,
                       cudaStream_t st);
int int8_dequantize(const int8_t* q, int64_t n, const void* s, int sdt, int bs, int64_t cols, void* out, int odt,
                    cudaStream_t st);

__host__ __device__ inline bool is_nf4_fmt(int fmt) {
  return fmt == RQ_W_NF4 || fmt == RQ_W_NF4_DQ_FP8 || fmt == RQ_W_NF4_DQ_INT8;
}

// Weight operand of a quantized linear layer, as the kernels see it.
struct QWeight {
  int fmt;              // RQ_W_*
  const void* q;        // NF4 packed codes or int8 values
  const void* scales;   // per-block / per-row scales (non-DQ formats)
  int sdt;              // dtype of `scales`
  const uint8_t* c2;    // DQ second-level codes
  const float* c2s;     // DQ second-level scales
  int64_t N, K;
  int bs;               // first-level block size
};

struct LinearArgs {
  QWeight w;
  const void* x;        // [M, K] (forward) or dy [M, N] (dx)
  const void* lora_x;   // input of the adapter branch (forward), usually x
  int xdt;
  int64_t M;
  const void* bias;
  int bdt;
  const void* lora_a;   // [r, K]
  const void* lora_b;   // [N, r]
  int r;
  float scaling;
  void* y;              // [M, N] (forward) or dx [M, K]
  void* ws;
  int64_t ws_bytes;
  const RqGather* gather;  // forward only: write the output into every rank's Y (nullptr: local y)
};

// kernel families (linear.cu picks one per call)
int lora_down(int dt, bool w_transposed, const void* X, int64_t M, int64_t Kr, const void* W2, int R, float pre_s,
              bool do_pre, void* out, float* partial, int64_t partial_elems, unsigned* counters, int ncounters,
              cudaStream_t st);
int simt_forward(const LinearArgs& a, const void* tdown, cudaStream_t st);
int simt_dx(const LinearArgs& a, const void* gt, cudaStream_t st);
bool gemv_supported(const LinearArgs& a);
bool gemv_fuse_down(const LinearArgs& a);
// `partial` / `counters` (workspace): the NF4 GEMV computes tdown itself
int gemv_forward(const LinearArgs& a, const void* tdown, cudaStream_t st, float* partial = nullptr,
                 unsigned* counters = nullptr);

int linear_forward(const LinearArgs& a, cudaStream_t st);
int weight_absmax(const QWeight& w, int dt, float* out, cudaStream_t st);
int weight_to_fp8(const QWeight& w, int dt, float s, uint8_t* out, cudaStream_t st);
int merge_weight(const QWeight& w, const float* A, const float* B, int r, float s, int mode, void* out, int odt,
                 cudaStream_t st);
int linear_dx(const LinearArgs& a, cudaStream_t st);
int64_t linear_workspace_bytes(int64_t M, int64_t N, int64_t K, int r);

// Rows of a batch and the adapters they use (adapters.cu).
struct AdapterRows {
  int64_t M;        // rows
  int64_t D1, D2;   // columns of the input and of the output (grad: D1 only)
  int r;            // rank, a multiple of 8
  int count;        // adapters of the bank
  int dt;           // RQ_BF16 / RQ_F16
  int tile;         // rows of a plan tile
  const int* plan;  // nullptr: every row uses adapter 0
};
int64_t adapter_plan_words(int64_t rows, int count, int tile);
int adapter_plan(const void* ids, int wide, int64_t rows, int count, int tile, int* plan, cudaStream_t st);
int adapters_apply(const AdapterRows& a, const void* in, int64_t ldin, const void* U, const void* V,
                   const float* scaling, const void* base, int64_t ldb, float* mid, void* out, int64_t ldo,
                   cudaStream_t st);
int adapters_grad(const AdapterRows& a, const void* z, int64_t ldz, const float* zscale, int64_t lds, const float* mid,
                  void* G, cudaStream_t st);

// Activations in 8 bits (act8.cu).
int act8_pack(const void* x, int dt, int64_t ld, int64_t M, int64_t K, int8_t* codes, float* scales, cudaStream_t st);
int act8_unpack(const int8_t* codes, const float* scales, int64_t M, int64_t K, void* out, int dt, cudaStream_t st);
int swiglu8_forward(const void* g, int64_t ldg, const void* u, int64_t ldu, int dt, int64_t M, int64_t K, void* h,
                    int8_t* codes, float* scales, int copies, cudaStream_t st);
int swiglu8_backward(const void* dh, int64_t ldh, int dt, int64_t M, int64_t K, const int8_t* codes,
                     const float* scales, void* dg, void* du, cudaStream_t st);

// Token log-probabilities and the preference loss on them (preference.cu).
// Position l of sequence b is scored on label [b, l + 1].
struct TokenRows {
  const void* logits;      // [B, L, V], strides in elements, vocabulary innermost
  int64_t sb, sl;
  int dt;
  int64_t B, L, V;
  const int64_t* labels;   // [B, L] contiguous
  int64_t ignore;          // label of a position that does not count
};
int token_logprobs(const TokenRows& t, float* stats, float* logps, cudaStream_t st);
int preference_loss(const TokenRows& t, const float* stats, const float* ref, int form, float beta, float smooth,
                    float* loss, float* logps, float* rewards, float* slopes, cudaStream_t st);
int token_logprobs_grad(const TokenRows& t, const float* stats, const float* slopes, int per_token,
                        const float* upstream, void* dlogits, cudaStream_t st);

// Microscaled 4-bit values (mx4.cu), their product (mx4_gemm.cu) and its
// gradient (mx4_dx.cu).
struct Mx4 {
  const uint8_t* codes;   // [rows, pitch / 2]
  const uint8_t* scales;  // [ceil(rows / 128), pitch / 128, 512]
  int64_t rows;
};
inline int64_t mx4_pitch(int64_t K) { return (K + 127) / 128 * 128; }
int mx4_pack(const void* x, int dt, int64_t ld, int64_t M, int64_t K, uint8_t* codes, uint8_t* scales, cudaStream_t st);
int mx4_unpack(const uint8_t* codes, const uint8_t* scales, int64_t M, int64_t K, void* out, int dt, cudaStream_t st);
int mx4_matmul(const Mx4& a, const Mx4& b, int64_t K, const void* bias, void* out, int dt, cudaStream_t st);
int64_t mx4_linear_workspace_bytes(int64_t M, int64_t N, int64_t K);
int mx4_linear(const void* x, int dt, int64_t ld, int64_t M, const Mx4& w, int64_t K, const void* bias, void* out,
               void* ws, cudaStream_t st);
void mx4_set_wait(int64_t ns);
int mx4_dx(const void* dy, int dt, int64_t ld, int64_t M, const Mx4& w, int64_t K, void* dx, void* ws, cudaStream_t st);

int align_rows(const void* x, int64_t ld, int64_t M, int64_t N, void* out, int64_t ldo, cudaStream_t st);

// AdamW over many tensors (adamw.cu).
int grad_norm_partial(const RqAdamTensor* list, int count, int dt, double* partials, cudaStream_t st);
int grad_norm_end(const double* partials, int n, float* norm, cudaStream_t st);
int adam_update(const RqAdamTensor* list, int count, int dt, int bits, void* m, void* v, float* scales, int16_t* low,
                const RqAdamStep& step, cudaStream_t st);
int adam_unpack(const uint8_t* m8, const uint8_t* r8, const float* scales, int64_t blocks, float* m, float* v,
                cudaStream_t st);
int adam_pack(const float* m, const float* v, int64_t blocks, uint8_t* m8, uint8_t* r8, float* scales,
              cudaStream_t st);

}  // namespace rq

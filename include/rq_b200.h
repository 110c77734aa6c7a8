/*
 * rq_b200.h -- C ABI of the B200 (sm_100a) implementation of rocm-qlora's
 * quantize / dequantize / QuantLinear+LoRA hot path.
 *
 * Conventions (every rq_* entry point):
 *   - plain device pointers and sizes; no framework types;
 *   - `stream` is a cudaStream_t passed as void* (NULL = legacy default);
 *   - nothing is allocated: callers own inputs, outputs and workspace;
 *   - the return value is RQ_OK (0) or a negative RQ_ERR_* status; the
 *     arguments are validated on the host before any launch, and a launch
 *     failure is reported as RQ_ERR_CUDA (rq_last_cuda_error() has the code);
 *   - calls are asynchronous on `stream` and thread-safe for distinct
 *     streams; a workspace must not be shared by calls that may overlap.
 *
 * Dtype codes: RQ_F32, RQ_BF16, RQ_F16.  Weight formats: RQ_W_* below.
 * Layouts follow the reference exactly (rocm_qlora/quantization):
 *   NF4 codes: flat row-major [N*K] elements, padded with zeros to a multiple
 *     of block_size, two codes per byte, byte i = code[2i] | code[2i+1] << 4;
 *   NF4 scales: one absmax per block, in the weight's dtype;
 *   double quant: c2 = one fp8-e4m3fnuz (or int8) byte per block, padded to a
 *     multiple of 256; c2_scales = fp32 absmax per 256 blocks;
 *   INT8 blockwise: int8 [N*K padded], scales per block (weight dtype);
 *   INT8 per-row: int8 [N, K], scales [N] (weight dtype).
 */
#ifndef RQ_B200_H
#define RQ_B200_H

#include <stdint.h>

#if defined(__GNUC__)
#define RQ_API __attribute__((visibility("default")))
#else
#define RQ_API
#endif

#ifdef __cplusplus
extern "C" {
#endif

#define RQ_OK 0
#define RQ_ERR_INVALID (-1)     /* bad size, null pointer, bad parameter */
#define RQ_ERR_ALIGN (-2)       /* pointer not aligned as required */
#define RQ_ERR_DTYPE (-3)       /* unsupported dtype / format code */
#define RQ_ERR_CUDA (-4)        /* CUDA launch or runtime error */
#define RQ_ERR_WORKSPACE (-5)   /* workspace missing or too small */
#define RQ_ERR_DEVICE (-6)      /* current device is not sm_100 */
#define RQ_ERR_SCRATCH (-7)     /* needs more than rq_linear_forward_noalloc's built-in scratch */
#define RQ_ERR_UNSUPPORTED (-8) /* no fused form for these arguments: nothing was launched */

#define RQ_F32 0
#define RQ_BF16 1
#define RQ_F16 2

#define RQ_W_NF4 0          /* NF4 codes + per-block scales */
#define RQ_W_NF4_DQ_FP8 1   /* NF4 codes + fp8-e4m3fnuz c2 + fp32 c2_scales */
#define RQ_W_NF4_DQ_INT8 2  /* NF4 codes + int8 c2 + fp32 c2_scales */
#define RQ_W_INT8 3         /* int8 blockwise */
#define RQ_W_INT8_ROW 4     /* int8 per output row (per_channel=True) */

/* ------------------------------------------------------------ utilities */
RQ_API int rq_abi_version(void);                 /* bumps when an existing entry point changes */
RQ_API const char* rq_status_string(int status);
/* cudaError_t of the last RQ_ERR_CUDA in this thread, or 10000 + the CUresult
 * when a driver call (tensor-map encoding) failed */
RQ_API int rq_last_cuda_error(void);
/* Number of bounded in-kernel waits that ran out on the current device since
 * the last call (and reset it).  Nonzero means a kernel stopped early and its
 * output is not valid; it indicates a bug, never a normal condition.
 * Synchronous. */
RQ_API int rq_take_kernel_timeouts(unsigned int* count);

/* -------------------------------------------------------- quantization */

/* NF4 blockwise quantization of x[numel] (dtype RQ_F32/BF16/F16).
 * packed: ceil(numel/bs)*bs/2 bytes; scales: ceil(numel/bs) values of dtype.
 * block_size must be even and >= 2.
 * Replaces quantize_int4, rocm_qlora/quantization/quant_ops.py:80-126. */
RQ_API int rq_nf4_quantize(const void* x, int dtype, int64_t numel, int block_size,
                    uint8_t* packed, void* scales, void* stream);

/* NF4 dequantization of `nbytes` packed bytes (2*nbytes values) with
 * per-block scales of scale_dtype into out (out_dtype; RQ_F32 gives the
 * reference's fp32 result, RQ_BF16/RQ_F16 that value rounded).
 * Replaces dequantize_int4, quant_ops.py:128-150, and
 * dequantize_nf4_triton, rocm_qlora/kernels/nf4_dequant.py:81-115. */
RQ_API int rq_nf4_dequantize(const uint8_t* packed, int64_t nbytes, const void* scales,
                      int scale_dtype, int block_size, void* out, int out_dtype,
                      void* stream);

/* INT8 blockwise quantization: q[ceil(numel/bs)*bs], scales[ceil(numel/bs)].
 * Replaces quantize_int8(per_channel=False), quant_ops.py:36-53. */
RQ_API int rq_int8_quantize(const void* x, int dtype, int64_t numel, int block_size,
                     int8_t* q, void* scales, void* stream);

/* INT8 per-row quantization of x[rows, cols]: q[rows, cols], scales[rows].
 * Replaces quantize_int8(per_channel=True), quant_ops.py:28-35. */
RQ_API int rq_int8_quantize_rows(const void* x, int dtype, int64_t rows, int64_t cols,
                          int8_t* q, void* scales, void* stream);

/* INT8 dequantization of q[numel]; cols > 0 selects per-row scales (row =
 * i / cols), else blockwise with block_size.
 * Replaces dequantize_int8, quant_ops.py:55-78. */
RQ_API int rq_int8_dequantize(const int8_t* q, int64_t numel, const void* scales,
                       int scale_dtype, int block_size, int64_t cols, void* out,
                       int out_dtype, void* stream);

/* Second-level quantization of nb fp32 first-level scales c1:
 * c2[ceil(nb/block2)*block2] (fp8 e4m3fnuz bytes if fp8 != 0, else int8),
 * c2_scales[ceil(nb/block2)] fp32.
 * Replaces double_quantize lines 58-97, rocm_qlora/quantization/double_quant.py. */
RQ_API int rq_dq_quantize_scales(const float* c1, int64_t nb, int block2, int fp8,
                          uint8_t* c2, float* c2_scales, void* stream);

/* Double-quantized NF4 dequantization of `numel` values:
 * out[i] = T[code_i] * (c2[i/bs] * c2_scales[i/bs/block2]).
 * Replaces double_dequantize, double_quant.py:99-122. */
RQ_API int rq_dq_dequantize(const uint8_t* packed, int64_t numel, const uint8_t* c2,
                     const float* c2_scales, int fp8, int block_size, int block2,
                     void* out, int out_dtype, void* stream);

/* ------------------------------------------------ QuantLinear + LoRA */

/* Bytes of workspace rq_linear_forward / rq_linear_dx need for these sizes
 * (0 is possible).  The first 256 bytes of a workspace are a counter area
 * that must be zero before its first use; the kernels leave it zero. */
RQ_API int64_t rq_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, int r);

/* y[M,N] = base + lora where, in the activation dtype `xdtype`,
 *   base = round(x[M,K] . deq(W)^T + bias)          (fp32 accumulation)
 *   lora = round(round(round(x . A^T) . B^T) * scaling)
 *   y    = round(base + lora)
 * i.e. LoRALinear.forward in eval mode over QuantLinear.forward
 * (rocm_qlora/lora/lora_layer.py:51-70, quantization/quant_linear.py:121-197,
 * kernels/dequant_matmul.py:356-376).  W is [N, K] in format `wfmt`:
 *   qweight  NF4 packed codes / int8 values (layout above);
 *   scales   per-block (or per-row) scales of scale_dtype (unused for DQ);
 *   c2, c2_scales  double-quant second level (DQ formats only).
 * bias [N] (bias_dtype) may be NULL; lora_a [r,K] and lora_b [N,r] are in
 * xdtype and may both be NULL (r = 0).  lora_x [M,K] is the input of the
 * adapter branch when it differs from x (LoRA dropout in training,
 * lora_layer.py:67); NULL means x.  x, y contiguous row-major.
 * xdtype: RQ_BF16 or RQ_F16 (tensor-core paths) or RQ_F32. */
RQ_API int rq_linear_forward(int wfmt, const void* qweight, const void* scales, int scale_dtype,
                      const uint8_t* c2, const float* c2_scales,
                      int64_t N, int64_t K, int block_size,
                      const void* x, int xdtype, int64_t M, const void* lora_x,
                      const void* bias, int bias_dtype,
                      const void* lora_a, const void* lora_b, int r, float scaling,
                      void* y, void* workspace, int64_t workspace_bytes, void* stream);

/* dx[M,K] = round(round(dy . deq(W)) + round(round(round(dy*scaling) . B) . A)),
 * the input gradient of the same layer (autograd of lora_layer.py:67 with a
 * frozen base; kernels/dequant_matmul.py:337-351 for the base term). */
RQ_API int rq_linear_dx(int wfmt, const void* qweight, const void* scales, int scale_dtype,
                 const uint8_t* c2, const float* c2_scales,
                 int64_t N, int64_t K, int block_size,
                 const void* dy, int xdtype, int64_t M,
                 const void* lora_a, const void* lora_b, int r, float scaling,
                 void* dx, void* workspace, int64_t workspace_bytes, void* stream);

/* The merged weight of a LoRA-adapted layer, dequantized and combined with
 * the adapter in one pass over the codes:
 *   out[n, k] = deq(W)[n, k] + scaling * sum_j lora_b[n, j] * lora_a[j, k]
 * with lora_a [r, K] and lora_b [N, r] fp32 (the adapters' parameter dtype)
 * and out [N, K] row-major in out_dtype.  mode RQ_MERGE_FP32_SUM adds in
 * fp32 and rounds once (LoRALinear.merge_lora, rocm_qlora/lora/
 * lora_layer.py:72-113); RQ_MERGE_ROUND_EACH rounds the weight and the delta
 * to out_dtype first and adds them there (_export_dequant_layer,
 * rocm_qlora/export/gguf_export.py:30-80).  r = 0 gives the dequantized
 * weight alone (lora_a / lora_b may then be NULL).  r <= 128. */
#define RQ_MERGE_FP32_SUM 0
#define RQ_MERGE_ROUND_EACH 1
RQ_API int rq_merge_lora(int wfmt, const void* qweight, const void* scales, int scale_dtype,
                  const uint8_t* c2, const float* c2_scales,
                  int64_t N, int64_t K, int block_size,
                  const float* lora_a, const float* lora_b, int r, float scaling, int mode,
                  void* out, int out_dtype, void* stream);

/* The quantized weight as a per-tensor scaled float8_e4m3fn GEMM operand
 * (FP8LinearWrapper's native path, rocm_qlora/fp8/fp8_linear.py:27-39):
 *   rq_weight_absmax: *absmax (device fp32) = max |rnd(deq(W))|, the weight
 *     rounded to `dtype` (the activation dtype, RQ_BF16 / RQ_F16 / RQ_F32);
 *   rq_weight_to_fp8: fp8_out[n*K + k] = e4m3fn(rnd(rnd(deq(W)[n, k]) / rnd(w_scale)))
 *     (as torch divides a `dtype` tensor by a 0-dim fp32 GPU tensor: the
 *     divisor rounded to `dtype`, the division in fp32 rounded to `dtype`;
 *     then round-to-nearest-even to e4m3fn without saturation), N*K bytes
 *     row-major.
 * The reference computes w_scale = absmax / 448 (e4m3fn's largest value). */
RQ_API int rq_weight_absmax(int wfmt, const void* qweight, const void* scales, int scale_dtype,
                     const uint8_t* c2, const float* c2_scales,
                     int64_t N, int64_t K, int block_size, int dtype,
                     float* absmax, void* stream);
RQ_API int rq_weight_to_fp8(int wfmt, const void* qweight, const void* scales, int scale_dtype,
                     const uint8_t* c2, const float* c2_scales,
                     int64_t N, int64_t K, int block_size, int dtype, float w_scale,
                     uint8_t* fp8_out, void* stream);

/* Bytes of device scratch compiled into the library for
 * rq_linear_forward_noalloc (held on every GPU that loads the library). */
#define RQ_NOALLOC_SCRATCH_BYTES (2u << 20)

/* rq_linear_forward for callers that cannot allocate device memory (plugin
 * hosts that own all device memory and hand out no workspace, cgo / JNI /
 * FFI bindings without a CUDA allocator, loops where cudaMalloc would
 * synchronize the device).  Same arguments and result as rq_linear_forward
 * minus the workspace: the scratch is a fixed RQ_NOALLOC_SCRATCH_BYTES
 * device array inside the library, so nothing is allocated.  Calls whose
 * rq_linear_workspace_bytes(M, N, K, r) exceeds that size return
 * RQ_ERR_SCRATCH before touching the GPU.  The first call on a device looks
 * up the array's device address (make it before any stream capture); after
 * cudaDeviceReset the next call looks it up again.  All
 * calls share the array: calls that may overlap on the GPU race and must not
 * be issued.  This entry point has no counterpart in the reference. */
RQ_API int rq_linear_forward_noalloc(int wfmt, const void* qweight, const void* scales, int scale_dtype,
                      const uint8_t* c2, const float* c2_scales,
                      int64_t N, int64_t K, int block_size,
                      const void* x, int xdtype, int64_t M, const void* lora_x,
                      const void* bias, int bias_dtype,
                      const void* lora_a, const void* lora_b, int r, float scaling,
                      void* y, void* stream);

/* Numerics of the decode GEMV (M <= 16, NF4 formats).  0 (the default): the
 * NF4 levels enter the tensor-core multiply rounded once to the activation
 * dtype and the fp32 block scale multiplies each 64-wide partial sum.  The
 * reference instead rounds level x scale to the activation dtype per weight;
 * the two differ by a fixed error per code, within 1e-2 x RMS of the output
 * for centred activations, but adding up over K when the activations share
 * a sign (after a ReLU, say).  1 (exact): the kernel forms the reference's
 * own weights, fp32 level x fp32 scale rounded to the activation dtype, per
 * weight, so only the summation order differs; slower.  The environment
 * variable RQ_DECODE_EXACT=1 selects 1 at the first call.  Applies to
 * launches made after the call; no counterpart in the reference. */
RQ_API void rq_set_decode_exact(int exact);

/* Kernel family the last rq_linear_forward / rq_linear_dx of this thread
 * ran: RQ_PATH_GEMV (decode, M <= 16), RQ_PATH_GEMM (tcgen05 prefill GEMM),
 * RQ_PATH_GEMV_SLABS (the GEMV over 16-row slabs), RQ_PATH_SIMT (exact
 * CUDA-core kernel), RQ_PATH_NONE (nothing launched).  Introspection for
 * tests and tuning; no counterpart in the reference. */
#define RQ_PATH_NONE 0
#define RQ_PATH_GEMV 1
#define RQ_PATH_GEMM 2
#define RQ_PATH_GEMV_SLABS 3
#define RQ_PATH_SIMT 4
RQ_API int rq_last_path(void);

/* ------------------------------- column shards: fused output gather */

/* Device memory shared with the other ranks of one node (one process per
 * GPU, NVLink peers).  rq_peer_alloc returns a zero-filled cudaMalloc
 * allocation of `bytes` on the current device; rq_peer_handle writes its
 * 64-byte IPC handle to `handle` (the caller ships it to the other ranks);
 * rq_peer_open maps another rank's allocation into this process for the
 * current device (peer access enabled) and rq_peer_close unmaps it.
 * Plumbing for rq_linear_forward_gather; no counterpart in the reference,
 * which replicates layers instead of sharding them. */
RQ_API int rq_peer_alloc(int64_t bytes, void** ptr);
RQ_API int rq_peer_free(void* ptr);
RQ_API int rq_peer_handle(const void* ptr, void* handle);
RQ_API int rq_peer_open(const void* handle, void** ptr);
RQ_API int rq_peer_close(void* ptr);

/* The node-wide output of a column-sharded layer: every rank computes the
 * output features [col, col + N) of the full Y[M, ld] and writes them into
 * EVERY rank's copy of Y.  All pointers are device pointers valid on this
 * rank (peer allocations opened with rq_peer_open):
 *   outs[q]      rank q's Y (row stride ld elements of xdtype), q < world
 *   flags[q]     rank q's flag array, 2 * world uint32 (zero before first
 *                use): [0, world) the epoch each rank finished, [world,
 *                2 * world) the epoch each rank entered
 *   my_flags     this rank's flag array (== flags[rank])
 *   ctrl         this rank's 4 uint32 of control state, zero before first
 *                use: [0] arrival counter (kernels leave it zero), [1] epoch
 *                (calls so far), [2] error (set to 1 if a peer did not
 *                arrive within about 2 s; the output is then incomplete)
 * outs and flags are device arrays of `world` pointers. */
typedef struct RqGather {
  void* const* outs;
  uint32_t* const* flags;
  uint32_t* my_flags;
  uint32_t* ctrl;
  int64_t ld;
  int64_t col;
  int world;
  int rank;
} RqGather;

/* rq_linear_forward of this rank's shard (W is [N, K], the shard's rows)
 * whose output is written into every rank's Y[:, col:col+N] instead of a
 * local y; when the kernel has completed on a rank, every rank's shard of
 * this call is in that rank's Y (the ranks meet at the end of the kernel:
 * the last CTA publishes this call's epoch to every rank's flags and waits,
 * bounded, for all of theirs).  Every rank must make the same sequence of
 * calls with the same M.  A rank's Y is rewritten by the next call that
 * names it, so each rank consumes each result (in stream order) before it
 * issues its next call on the same outputs; a rank writes into the other
 * ranks' Y only after every rank has entered the call (each rank announces
 * its entry at the start of the kernel), so a faster rank never overwrites
 * a result a slower rank is still reading.  Only the fused decode GEMV (NF4 formats, bf16/f16,
 * M <= 16) has this form: other arguments return RQ_ERR_UNSUPPORTED before
 * anything is launched, and the caller gathers with a collective instead.
 * Same-node NVLink peers only; one call in flight per RqGather. */
RQ_API int rq_linear_forward_gather(int wfmt, const void* qweight, const void* scales, int scale_dtype,
                      const uint8_t* c2, const float* c2_scales,
                      int64_t N, int64_t K, int block_size,
                      const void* x, int xdtype, int64_t M,
                      const void* bias, int bias_dtype,
                      const void* lora_a, const void* lora_b, int r, float scaling,
                      const RqGather* gather, void* workspace, int64_t workspace_bytes, void* stream);

/* ------------------------------ adapters of many requests at once */

/* A bank holds `count` adapters over one [N, K] projection as A [count, K, r]
 * and B [count, N, r] (rank innermost, contiguous, RQ_BF16 or RQ_F16, r a
 * multiple of 8 up to 128) and a fp32 factor per adapter.  Each of the M rows
 * of a batch names its adapter; the plan, made once per batch and used by
 * every layer, direction and gradient, orders the rows by adapter.
 *
 * rq_adapter_plan_words: int32 words of a plan of `rows` rows (-1: a bad
 * argument; count is at most RQ_ADAPTERS_MAX).  rq_adapter_plan fills it from ids[rows] (int64 if wide != 0,
 * else int32): 0..count-1 is the adapter, -1 is none, and a row with any
 * other id gets NaN outputs.  tile_rows, 16, 32, 64 or 128, is how many rows
 * of one adapter are computed together; choose about the mean number of rows
 * per adapter, 128 only from some thousands of rows on. */
#define RQ_ADAPTERS_MAX 4096
RQ_API int64_t rq_adapter_plan_words(int64_t rows, int count, int tile_rows);
RQ_API int rq_adapter_plan(const void* ids, int wide, int64_t rows, int count, int tile_rows,
                    int32_t* plan, int64_t plan_words, void* stream);

/* out[m, :] = base[m, :] + mid[m, :] . V_a^T,  mid[m, :] = scaling[a] * (in[m, :] . U_a)
 * for in [M, D1], out and base [M, D2] (base may be NULL: zero, or out itself),
 * U [count, D1, r], V [count, D2, r], mid [M, r] fp32 (written for
 * the backward; may be NULL).  Forward: U = A, V = B, in = x.  Input gradient: U = B, V = A,
 * in = dy.  Everything is accumulated in fp32 and rounded once.  plan NULL:
 * every row uses adapter 0.  Row strides (ld*) in elements, columns
 * contiguous; a stride of 0, here and in the functions below, is one input row
 * for all (not for out). */
RQ_API int rq_adapters_apply(const void* in, int64_t ld_in, const void* U, const void* V,
                      const float* scaling, const void* base, int64_t ld_base,
                      int64_t M, int64_t D1, int64_t D2, int r, int count, int dtype,
                      const int32_t* plan, int64_t plan_words, int tile_rows,
                      float* mid, void* out, int64_t ld_out, void* stream);

/* grad[a, d, j] = sum over the rows m of adapter a of z[m, d] * mid[m, j], for
 * z [M, D] (row stride ld_z): the gradient of A with z = x and the backward's
 * mid, of B with z = dy and the forward's mid.  With z_scales not NULL z is
 * the 8-bit packed form (rq_act8_pack): int8 codes [M, ceil(D / 128) * 128]
 * and z_scales [M, ceil(D / 128)].  grad [count, D, r] in dtype; an adapter
 * without rows gets zeros.  plan NULL: every row is adapter 0's. */
RQ_API int rq_adapters_grad(const void* z, int64_t ld_z, const float* z_scales, const float* mid,
                     int64_t M, int64_t D, int r, int count, int dtype,
                     const int32_t* plan, int64_t plan_words, int tile_rows,
                     void* grad, void* stream);

/* ------------------------------------------- activations in 8 bits */

/* Packed form of x [M, K]: blocks of RQ_ACT8_BLOCK columns of a row, codes
 * int8 [M, nb * RQ_ACT8_BLOCK] and scales fp32 [M, nb], nb = ceil(K / block):
 *   scale = max|x| / 127,  code = rint(x * (127 / max|x|))
 * the last block filled with zero codes.  A block whose largest magnitude is
 * below 2^-100 is stored as zeros; one with an infinity or NaN has scale NaN.
 * codes must be 16-byte aligned.  unpack gives code * scale in dtype,
 * [M, K] contiguous. */
#define RQ_ACT8_BLOCK 128
RQ_API int rq_act8_pack(const void* x, int dtype, int64_t ld_x, int64_t M, int64_t K,
                 int8_t* codes, float* scales, void* stream);
RQ_API int rq_act8_unpack(const int8_t* codes, const float* scales, int64_t M, int64_t K,
                   void* out, int dtype, void* stream);

/* h = silu(gate) * up for [M, K] (h contiguous), with `copies` packed forms
 * written in the same pass one after the other (each [M, nb * block] codes
 * and [M, nb] scales): gate, up and, with copies = 3, h as rounded.
 * Backward from the packed gate and up:
 *   p = 1 / (1 + exp(-gate)),  dgate = dh * up * p * (1 + gate * (1 - p)),
 *   dup = dh * gate * p        ([M, K] contiguous). */
RQ_API int rq_swiglu8_forward(const void* gate, int64_t ld_gate, const void* up, int64_t ld_up, int dtype,
                       int64_t M, int64_t K, void* h, int8_t* codes, float* scales, int copies, void* stream);
RQ_API int rq_swiglu8_backward(const void* dh, int64_t ld_dh, int dtype, int64_t M, int64_t K,
                        const int8_t* codes, const float* scales, void* dgate, void* dup, void* stream);

/* ------------------------------ token log-probabilities, preference loss */

/* logits [B, L, V] (strides in elements, V contiguous), labels [B, L] int64
 * contiguous: position l is scored on labels[b, l + 1]; a label equal to
 * `ignore` (and the last position) does not count, and a label outside
 * [0, V) gives NaN.  rq_token_logprobs writes stats [B, L, 4] fp32, 16-byte
 * aligned (k, s, hi, lo: the sum of the row's exponentials is s 2^k or, where
 * s < 0, in rows whose logits leave +-2^19, -s e^k; the label's log-probability
 * is hi + lo; rows that do not count are left as they are) and, unless NULL, logps [B, L]: the log-probability of each label, 0
 * where it does not count. */
RQ_API int rq_token_logprobs(const void* logits, int dtype, int64_t stride_b, int64_t stride_l,
                      int64_t B, int64_t L, int64_t V, const int64_t* labels, int64_t ignore,
                      float* stats, float* logps, void* stream);

/* Sequences i (chosen) and i + B/2 (rejected) are a pair.  With ref [B, L] the
 * reference model's log-probabilities, R_b = sum (log p - ref) over the
 * labels that count, n_b their number (at least 1), z_i = beta (R_i - R_{i+B/2}):
 *   RQ_PREF_SIGMOID: mean(-(1 - smooth) log sigma(z) - smooth log sigma(-z))
 *   RQ_PREF_IPO:     mean((R_i / n_i - R_{i+B/2} / n_{i+B/2} - 1 / (2 beta))^2), smooth unused
 * Writes loss [1], logps [B] (sums of log p), rewards [B] (beta R) and
 * slopes [B] (d loss / d R), all fp32. */
#define RQ_PREF_SIGMOID 0
#define RQ_PREF_IPO 1
RQ_API int rq_preference_loss(int64_t B, int64_t L, const int64_t* labels, int64_t ignore,
                       const float* stats, const float* ref, int form, float beta, float smooth,
                       float* loss, float* logps, float* rewards, float* slopes, void* stream);

/* dlogits [B, L, V] (contiguous) = upstream * slope * ([v = label] - softmax),
 * zero where the position does not count; slope per sequence (slopes [B]) or,
 * with per_token != 0, slopes [B, L] at the label's place.  upstream: one
 * fp32 on the device, NULL for 1. */
RQ_API int rq_token_logprobs_grad(const void* logits, int dtype, int64_t stride_b, int64_t stride_l,
                           int64_t B, int64_t L, int64_t V, const int64_t* labels, int64_t ignore,
                           const float* stats, const float* slopes, int per_token, const float* upstream,
                           void* dlogits, void* stream);

/* ---------------------------------------- microscaled 4-bit values */

/* Packed form of x [M, K]: blocks of RQ_MX4_BLOCK columns of a row,
 *   e = max(floor(log2 max|x|) - 2, -127),  code = e2m1(x 2^-e)
 * (the nearest of +-{0, .5, 1, 1.5, 2, 3, 4, 6}, ties to the even code), scale
 * byte e + 127; a block of zeros has scale byte 0, one with an infinity or
 * NaN scale byte 255 (NaN).  With Kp = K rounded up to 128:
 *   codes  [M, Kp / 2], two a byte, the even column in the low half; 16-byte
 *          aligned; columns past K are 0;
 *   scales [ceil(M / 128), Kp / 128, 512], 16-byte aligned, in the order that
 *          the tensor cores take: row r, block b is byte
 *          (r % 32) * 16 + (r % 128) / 32 * 4 + b % 4 of its piece; rows past M
 *          and blocks past K are 0. */
#define RQ_MX4_BLOCK 32
RQ_API int64_t rq_mx4_scale_bytes(int64_t M, int64_t K);
RQ_API int rq_mx4_pack(const void* x, int dtype, int64_t ld_x, int64_t M, int64_t K,
                uint8_t* codes, uint8_t* scales, void* stream);
RQ_API int rq_mx4_unpack(const uint8_t* codes, const uint8_t* scales, int64_t M, int64_t K,
                  void* out, int dtype, void* stream);

/* out[m, n] = sum_k a[m, k] b[n, k] (+ bias[n]) of two packed operands, summed
 * in 32 bits and rounded once to out's dtype (bf16 or f16); bias in that dtype
 * or NULL; out [M, N] contiguous. */
RQ_API int rq_mx4_matmul(const uint8_t* a_codes, const uint8_t* a_scales, int64_t M,
                  const uint8_t* b_codes, const uint8_t* b_scales, int64_t N, int64_t K,
                  const void* bias, void* out, int dtype, void* stream);

/* The same for rows x [M, K] (bf16 or f16, row stride ld_x) that are packed on
 * the way.  workspace: rq_mx4_linear_workspace_bytes (0: none), 256-byte
 * aligned. */
RQ_API int64_t rq_mx4_linear_workspace_bytes(int64_t M, int64_t N, int64_t K);
RQ_API int rq_mx4_linear(const void* x, int dtype, int64_t ld_x, int64_t M,
                  const uint8_t* w_codes, const uint8_t* w_scales, int64_t N, int64_t K,
                  const void* bias, void* out, void* workspace, int64_t workspace_bytes, void* stream);

/* How long a product of few tokens (rq_mx4_matmul, rq_mx4_linear) waits for its
 * own copies and sums before it gives up, in ns: 2 s unless set; 0: every wait has
 * run out before it begins; below 0: 2 s again.  Outputs whose sums a wait ran out
 * for are NaN, and rq_take_kernel_timeouts counts it.  A captured call keeps the
 * limit of its capture. */
RQ_API int rq_mx4_set_wait(int64_t ns);

/* dx [M, K] (contiguous) = dy [M, N] . w, w the packed weight [N, K] and dy in
 * dtype (bf16 or f16) with row stride ld_dy, a multiple of 8 with dy 16-byte
 * aligned.  w enters in dy's dtype: exact in bf16; in f16 times 2^(127 - top),
 * top being its largest scale byte but 255, which leaves out what is below
 * 2^-24 of that.  workspace: RQ_MX4_DX_WORKSPACE bytes, 16-byte aligned (f16
 * only). */
#define RQ_MX4_DX_WORKSPACE 1024
RQ_API int rq_mx4_dx(const void* dy, int dtype, int64_t ld_dy, int64_t M,
              const uint8_t* w_codes, const uint8_t* w_scales, int64_t N, int64_t K,
              void* dx, void* workspace, int64_t workspace_bytes, void* stream);

/* Copies rows x [M, N] of 16-bit values (row stride ld_x, any alignment) to rows
 * of stride ld_out, a multiple of 8 of at least N, out 16-byte aligned: what
 * rq_mx4_dx takes.  Columns past N are left as they are or 0. */
RQ_API int rq_align_rows(const void* x, int64_t ld_x, int64_t M, int64_t N, void* out, int64_t ld_out, void* stream);

/* ---------------------------------------------- AdamW over many tensors */

/* One tensor of a step: its values, its gradient (both of the call's dtype),
 * how many, its first block in the arenas of the moments, and its place among
 * the steps.  Blocks are of RQ_ADAM_BLOCK values, the last one short;
 * a call takes up to RQ_ADAM_TENSORS tensors. */
typedef struct RqAdamTensor {
  void* param;
  const void* grad;
  int64_t n;
  int64_t block;
  int32_t slot;
} RqAdamTensor;
#define RQ_ADAM_BLOCK 256
#define RQ_ADAM_TENSORS 1024
#define RQ_NORM_PARTIALS 1184

/* Sums of squares (64 bits) of the gradients of up to RQ_ADAM_TENSORS tensors
 * as RQ_NORM_PARTIALS values; rq_grad_norm_end makes *norm = sqrt(sum) of n. */
RQ_API int rq_grad_norm_partial(const RqAdamTensor* tensors, int count, int dtype, double* partials, void* stream);
RQ_API int rq_grad_norm_end(const double* partials, int n, float* norm, void* stream);

/* A step of the tensors, each one's t = steps[slot] + 1, which is counted up:
 *   g = c grad, m = b1 m + (1 - b1) g, v = b2 v + (1 - b2) g g,
 *   p = p (1 - lr decay) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
 * with c = min(1, max_norm / (norm + 1e-6)) of the norm of n_partials values,
 * which is written to *norm; c is 1 if n_partials is 0.  An eps above 0 counts as
 * 2^-126 at least.  lr_at: learning rate on
 * the device (fp32) in lr's place, or NULL.
 * bits 32: m and v are fp32 arenas [blocks * 256].  bits 8: m holds e4m3 codes
 * of m (448 / max|m|) of a block, v codes of sqrt(v) (507904 / max sqrt(v)) with
 * 4 exponent and 4 mantissa bits (the whole numbers to 31, then 16 steps to a
 * power of two, to 31 2^14; not 0 for v > 0), scales [blocks, 2] what the codes
 * are multiplied by.  low (bf16 parameters, or NULL): int16 [blocks * 256], the
 * difference of a 32-bit value and its bf16 as bit patterns.  Arenas 32-byte
 * aligned.  ticket: one zero, which the call leaves zero. */
typedef struct RqAdamStep {
  double lr, beta1, beta2, eps, decay;
  const float* lr_at;
  const double* partials;
  int n_partials;
  float max_norm;
  float* norm;
  int32_t* steps;
  uint32_t* ticket;
} RqAdamStep;
RQ_API int rq_adam_update(const RqAdamTensor* tensors, int count, int dtype, int bits, void* m, void* v,
                   float* scales, int16_t* low, const RqAdamStep* step, void* stream);

/* Moments of `blocks` blocks between their 8-bit form and fp32 (v, not its root;
 * 32-byte aligned). */
RQ_API int rq_adam_unpack(const uint8_t* m8, const uint8_t* r8, const float* scales, int64_t blocks,
                   float* m, float* v, void* stream);
RQ_API int rq_adam_pack(const float* m, const float* v, int64_t blocks, uint8_t* m8, uint8_t* r8, float* scales,
                 void* stream);

/* ------------------------------------- reference launcher drop-ins */

/* Same symbol names, argument order and types as the reference's HIP
 * launchers (rocm_qlora/hip_kernels/int4_matmul.hip:413-458, bound by
 * ctypes in rocm_qlora/hip_kernels/build_utils.py:237-262): x fp16 [M,K],
 * scales fp16 per 64-block as declared there, c fp16 [M,N], no bias.  They
 * return void like the originals; the status of the last call is available
 * from rq_last_status(). */
RQ_API void launch_int4_dequant_matmul(void* stream, void* x, void* w_packed, void* scales,
                                void* c, int M, int N, int K, int block_size);
RQ_API void launch_int8_dequant_matmul(void* stream, void* x, void* w_int8, void* scales,
                                void* c, int M, int N, int K, int block_size);
RQ_API int rq_last_status(void);

#ifdef __cplusplus
}
#endif

#endif /* RQ_B200_H */

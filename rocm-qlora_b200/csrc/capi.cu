// capi.cu -- the extern "C" boundary (include/rq_b200.h).
//
// Every entry point validates its arguments on the host, checks that the
// current device is an sm_100 part, and then launches on the caller's
// stream.  Nothing here allocates device memory.
#include <cuda_runtime.h>

#include <mutex>
#include <vector>

#include "rq_internal.h"

namespace rq {

static thread_local int g_last_cuda_error = 0;
static thread_local int g_last_status = 0;

void set_cuda_error(cudaError_t e) { g_last_cuda_error = (int)e; }

int ensure_smem_limit(const void* kernel, size_t bytes) {
  struct Entry {
    const void* k;
    int dev;
    size_t bytes;
  };
  static std::mutex mu;
  static std::vector<Entry> done;
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lock(mu);
  for (const Entry& e : done)
    if (e.k == kernel && e.dev == dev && e.bytes >= bytes) return RQ_OK;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e != cudaSuccess) {
    set_cuda_error(e);
    return RQ_ERR_CUDA;
  }
  done.push_back({kernel, dev, bytes});
  return RQ_OK;
}

static int device_ok() {
  static int cache[64];  // 0 unknown, 1 ok, -1 not sm_100
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) {
    set_cuda_error(e);
    return RQ_ERR_CUDA;
  }
  if (dev < 0 || dev >= 64) return RQ_ERR_DEVICE;
  if (cache[dev] == 0) {
    int major = 0, minor = 0;
    cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev);
    cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, dev);
    cache[dev] = (major == 10 && minor == 0) ? 1 : -1;
  }
  return cache[dev] == 1 ? RQ_OK : RQ_ERR_DEVICE;
}

static bool dtype_ok(int dt) { return dt == RQ_F32 || dt == RQ_BF16 || dt == RQ_F16; }

static int dtype_size(int dt) { return dt == RQ_F32 ? 4 : 2; }

static int check_weight(int wfmt, const void* q, const void* scales, int sdt, const uint8_t* c2, const float* c2s,
                        int64_t N, int64_t K, int bs) {
  if (N < 0 || K < 0 || !q) return RQ_ERR_INVALID;
  if (wfmt < RQ_W_NF4 || wfmt > RQ_W_INT8_ROW) return RQ_ERR_DTYPE;
  if (wfmt == RQ_W_NF4_DQ_FP8 || wfmt == RQ_W_NF4_DQ_INT8) {
    if (!c2 || !c2s) return RQ_ERR_INVALID;
  } else {
    if (!scales || !dtype_ok(sdt)) return RQ_ERR_INVALID;
  }
  if (wfmt != RQ_W_INT8_ROW && (bs < 2 || (is_nf4_fmt(wfmt) && (bs & 1)))) return RQ_ERR_INVALID;
  return RQ_OK;
}

static int fill_args(LinearArgs* a, int wfmt, const void* q, const void* scales, int sdt, const uint8_t* c2,
                     const float* c2s, int64_t N, int64_t K, int bs, const void* x, int xdt, int64_t M,
                     const void* bias, int bdt, const void* la, const void* lb, int r, float scaling, void* y,
                     void* ws, int64_t ws_bytes) {
  int rc = check_weight(wfmt, q, scales, sdt, c2, c2s, N, K, bs);
  if (rc != RQ_OK) return rc;
  if (!dtype_ok(xdt)) return RQ_ERR_DTYPE;
  if (M < 0 || (M > 0 && (!x || !y))) return RQ_ERR_INVALID;
  if (bias && !dtype_ok(bdt)) return RQ_ERR_DTYPE;
  if (r < 0 || r > 128) return RQ_ERR_INVALID;
  if (r > 0 && (!la || !lb)) return RQ_ERR_INVALID;
  if ((uintptr_t)x % dtype_size(xdt) || (uintptr_t)y % dtype_size(xdt)) return RQ_ERR_ALIGN;
  a->w = QWeight{wfmt, q, scales, sdt, c2, c2s, N, K, bs};
  a->x = x;
  a->xdt = xdt;
  a->M = M;
  a->bias = bias;
  a->bdt = bdt;
  a->lora_a = la;
  a->lora_b = lb;
  a->r = r;
  a->scaling = scaling;
  a->y = y;
  a->ws = ws;
  a->ws_bytes = ws_bytes;
  a->lora_x = x;
  a->gather = nullptr;
  return RQ_OK;
}

static bool half_ok(int dt) { return dt == RQ_BF16 || dt == RQ_F16; }

// Sizes a kernel indexes with 32 bits.
static bool fits(int64_t v) { return v >= 0 && v < (int64_t)1 << 31; }

// Distances between the rows of an input, which is only read: 0 is one row
// broadcast to all.
static bool row_stride(int64_t M, int64_t ld, int64_t columns) { return M <= 1 || ld == 0 || ld >= columns; }

// Rows whose 8-bit blocks are numbered with 32 bits.
static bool fits_act8(int64_t M, int64_t K) {
  return fits(M) && fits(K) && fits(M * ((K + RQ_ACT8_BLOCK - 1) / RQ_ACT8_BLOCK));
}

static int check_plan(int64_t rows, int count, int tile, const int32_t* plan, int64_t words) {
  if (!fits(rows) || count < 1 || count > RQ_ADAPTERS_MAX) return RQ_ERR_INVALID;
  if (!plan) return RQ_OK;
  if (tile != 16 && tile != 32 && tile != 64 && tile != 128) return RQ_ERR_INVALID;
  if (!fits(adapter_plan_words(rows, count, tile))) return RQ_ERR_INVALID;
  if (words < adapter_plan_words(rows, count, tile)) return RQ_ERR_WORKSPACE;
  return (uintptr_t)plan % 16 ? RQ_ERR_ALIGN : RQ_OK;
}

static int check_tokens(const void* logits, int dt, int64_t B, int64_t L, int64_t V, const int64_t* labels,
                        const float* stats) {
  if (!dtype_ok(dt)) return RQ_ERR_DTYPE;
  if (V < 1 || !fits(V) || !fits(B) || !fits(L) || !fits(B * L)) return RQ_ERR_INVALID;
  if (B * L > 0 && (!logits || !labels || !stats)) return RQ_ERR_INVALID;
  if ((uintptr_t)logits % dtype_size(dt) || (uintptr_t)labels % 8 || (uintptr_t)stats % 16) return RQ_ERR_ALIGN;
  return RQ_OK;
}

static int check_mx4(const uint8_t* codes, const uint8_t* scales, int64_t rows, int64_t K) {
  // pieces of 128 columns, of rows padded to 128, are numbered with 32 bits
  if (!fits(rows) || !fits(K) || !fits((rows + 127) / 128 * 128 * (mx4_pitch(K) / 128))) return RQ_ERR_INVALID;
  if (rows * K == 0) return RQ_OK;
  if (!codes || !scales) return RQ_ERR_INVALID;
  return (uintptr_t)codes % 16 || (uintptr_t)scales % 16 ? RQ_ERR_ALIGN : RQ_OK;
}

// The operands of a product [M, K] . [N, K]^T, and grid sizes it can have.
static int check_product(int dtype, int64_t M, int64_t N, int64_t K) {
  if (!half_ok(dtype)) return RQ_ERR_DTYPE;
  if (!fits(M) || !fits(N) || !fits(K) || M > 65535LL * 128 || N > 65535LL * 128) return RQ_ERR_INVALID;
  return RQ_OK;
}

static int check_tensors(const RqAdamTensor* t, int count, int dtype, bool params, bool state) {
  if (!dtype_ok(dtype)) return RQ_ERR_DTYPE;
  if (count < 0 || count > RQ_ADAM_TENSORS || (count > 0 && !t)) return RQ_ERR_INVALID;
  int64_t blocks = 0;
  for (int i = 0; i < count; ++i) {
    if (t[i].n < 0 || (t[i].n > 0 && (!t[i].grad || (params && !t[i].param)))) return RQ_ERR_INVALID;
    const int64_t own = (t[i].n + RQ_ADAM_BLOCK - 1) / RQ_ADAM_BLOCK;
    blocks += own;
    if (!fits(blocks) || (state && (t[i].slot < 0 || t[i].slot > 65535 || t[i].block < 0 || !fits(t[i].block + own))))
      return RQ_ERR_INVALID;
    if ((uintptr_t)t[i].grad % dtype_size(dtype) || (uintptr_t)t[i].param % dtype_size(dtype)) return RQ_ERR_ALIGN;
  }
  return RQ_OK;
}

}  // namespace rq

using namespace rq;

#define RQ_PROLOGUE()               \
  do {                              \
    int _rc = device_ok();          \
    if (_rc != RQ_OK) return _rc;   \
  } while (0)

extern "C" {

int rq_abi_version(void) { return 3; }

const char* rq_status_string(int s) {
  switch (s) {
    case RQ_OK: return "ok";
    case RQ_ERR_INVALID: return "invalid argument";
    case RQ_ERR_ALIGN: return "misaligned pointer";
    case RQ_ERR_DTYPE: return "unsupported dtype or format";
    case RQ_ERR_CUDA: return "CUDA error";
    case RQ_ERR_WORKSPACE: return "workspace missing or too small";
    case RQ_ERR_DEVICE: return "current device is not an sm_100 (B200) GPU";
    case RQ_ERR_SCRATCH: return "request exceeds the built-in scratch of rq_linear_forward_noalloc";
  }
  return "unknown status";
}

int rq_last_cuda_error(void) { return g_last_cuda_error; }
int rq_last_status(void) { return g_last_status; }
int rq_last_path(void) { return rq::last_path(); }
void rq_set_decode_exact(int exact) { rq::set_decode_exact(exact); }

int rq_nf4_quantize(const void* x, int dtype, int64_t numel, int block_size, uint8_t* packed, void* scales,
                    void* stream) {
  RQ_PROLOGUE();
  if (!dtype_ok(dtype)) return RQ_ERR_DTYPE;
  if (numel < 0 || block_size < 2 || (block_size & 1)) return RQ_ERR_INVALID;
  if (numel == 0) return RQ_OK;
  if (!x || !packed || !scales) return RQ_ERR_INVALID;
  if ((uintptr_t)x % dtype_size(dtype) || (uintptr_t)scales % dtype_size(dtype)) return RQ_ERR_ALIGN;
  return nf4_quantize(x, dtype, numel, block_size, packed, scales, (cudaStream_t)stream);
}

int rq_nf4_dequantize(const uint8_t* packed, int64_t nbytes, const void* scales, int scale_dtype, int block_size,
                      void* out, int out_dtype, void* stream) {
  RQ_PROLOGUE();
  if (!dtype_ok(scale_dtype) || !dtype_ok(out_dtype)) return RQ_ERR_DTYPE;
  if (nbytes < 0 || block_size < 2 || (block_size & 1)) return RQ_ERR_INVALID;
  if (nbytes == 0) return RQ_OK;
  if (!packed || !scales || !out) return RQ_ERR_INVALID;
  if ((uintptr_t)out % dtype_size(out_dtype) || (uintptr_t)scales % dtype_size(scale_dtype)) return RQ_ERR_ALIGN;
  return nf4_dequantize(packed, nbytes, scales, scale_dtype, block_size, out, out_dtype, (cudaStream_t)stream);
}

int rq_int8_quantize(const void* x, int dtype, int64_t numel, int block_size, int8_t* q, void* scales,
                     void* stream) {
  RQ_PROLOGUE();
  if (!dtype_ok(dtype)) return RQ_ERR_DTYPE;
  if (numel < 0 || block_size < 1) return RQ_ERR_INVALID;
  if (numel == 0) return RQ_OK;
  if (!x || !q || !scales) return RQ_ERR_INVALID;
  if ((uintptr_t)x % dtype_size(dtype) || (uintptr_t)scales % dtype_size(dtype)) return RQ_ERR_ALIGN;
  return int8_quantize(x, dtype, numel, block_size, q, scales, (cudaStream_t)stream);
}

int rq_int8_quantize_rows(const void* x, int dtype, int64_t rows, int64_t cols, int8_t* q, void* scales,
                          void* stream) {
  RQ_PROLOGUE();
  if (!dtype_ok(dtype)) return RQ_ERR_DTYPE;
  if (rows < 0 || cols < 0) return RQ_ERR_INVALID;
  if (rows == 0) return RQ_OK;
  if (!x || !q || !scales) return RQ_ERR_INVALID;
  if ((uintptr_t)x % dtype_size(dtype) || (uintptr_t)scales % dtype_size(dtype)) return RQ_ERR_ALIGN;
  return int8_quantize_rows(x, dtype, rows, cols, q, scales, (cudaStream_t)stream);
}

int rq_int8_dequantize(const int8_t* q, int64_t numel, const void* scales, int scale_dtype, int block_size,
                       int64_t cols, void* out, int out_dtype, void* stream) {
  RQ_PROLOGUE();
  if (!dtype_ok(scale_dtype) || !dtype_ok(out_dtype)) return RQ_ERR_DTYPE;
  if (numel < 0 || cols < 0 || (cols == 0 && block_size < 1)) return RQ_ERR_INVALID;
  if (numel == 0) return RQ_OK;
  if (!q || !scales || !out) return RQ_ERR_INVALID;
  if ((uintptr_t)out % dtype_size(out_dtype) || (uintptr_t)scales % dtype_size(scale_dtype)) return RQ_ERR_ALIGN;
  return int8_dequantize(q, numel, scales, scale_dtype, block_size, cols, out, out_dtype, (cudaStream_t)stream);
}

int rq_dq_quantize_scales(const float* c1, int64_t nb, int block2, int fp8, uint8_t* c2, float* c2_scales,
                          void* stream) {
  RQ_PROLOGUE();
  if (nb < 0 || block2 < 1) return RQ_ERR_INVALID;
  if (nb == 0) return RQ_OK;
  if (!c1 || !c2 || !c2_scales) return RQ_ERR_INVALID;
  if ((uintptr_t)c1 % 4 || (uintptr_t)c2_scales % 4) return RQ_ERR_ALIGN;
  return dq_quantize_scales(c1, nb, block2, fp8 ? 1 : 0, c2, c2_scales, (cudaStream_t)stream);
}

int rq_dq_dequantize(const uint8_t* packed, int64_t numel, const uint8_t* c2, const float* c2_scales, int fp8,
                     int block_size, int block2, void* out, int out_dtype, void* stream) {
  RQ_PROLOGUE();
  if (!dtype_ok(out_dtype)) return RQ_ERR_DTYPE;
  if (numel < 0 || block_size < 2 || (block_size & 1) || block2 < 1) return RQ_ERR_INVALID;
  if (numel == 0) return RQ_OK;
  if (!packed || !c2 || !c2_scales || !out) return RQ_ERR_INVALID;
  if ((uintptr_t)out % dtype_size(out_dtype) || (uintptr_t)c2_scales % 4) return RQ_ERR_ALIGN;
  return dq_dequantize(packed, numel, c2, c2_scales, fp8 ? 1 : 0, block_size, block2, out, out_dtype,
                       (cudaStream_t)stream);
}

int64_t rq_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, int r) {
  if (M < 0 || N < 0 || K < 0 || r < 0) return -1;
  return linear_workspace_bytes(M, N, K, r);
}

int rq_linear_forward(int wfmt, const void* qweight, const void* scales, int scale_dtype, const uint8_t* c2,
                      const float* c2_scales, int64_t N, int64_t K, int block_size, const void* x, int xdtype,
                      int64_t M, const void* lora_x, const void* bias, int bias_dtype, const void* lora_a,
                      const void* lora_b, int r, float scaling, void* y, void* workspace, int64_t workspace_bytes,
                      void* stream) {
  RQ_PROLOGUE();
  LinearArgs a;
  int rc = fill_args(&a, wfmt, qweight, scales, scale_dtype, c2, c2_scales, N, K, block_size, x, xdtype, M, bias,
                     bias_dtype, lora_a, lora_b, r, scaling, y, workspace, workspace_bytes);
  if (rc != RQ_OK) return rc;
  if (lora_x && (uintptr_t)lora_x % dtype_size(xdtype)) return RQ_ERR_ALIGN;
  a.lora_x = lora_x ? lora_x : x;
  return linear_forward(a, (cudaStream_t)stream);
}

int rq_linear_forward_gather(int wfmt, const void* qweight, const void* scales, int scale_dtype, const uint8_t* c2,
                             const float* c2_scales, int64_t N, int64_t K, int block_size, const void* x, int xdtype,
                             int64_t M, const void* bias, int bias_dtype, const void* lora_a, const void* lora_b, int r,
                             float scaling, const RqGather* gather, void* workspace, int64_t workspace_bytes,
                             void* stream) {
  RQ_PROLOGUE();
  if (!gather) return RQ_ERR_INVALID;
  LinearArgs a;
  // the output is the ranks' Y, not a local y: x stands in for the argument
  // check (it is never written)
  int rc = fill_args(&a, wfmt, qweight, scales, scale_dtype, c2, c2_scales, N, K, block_size, x, xdtype, M, bias,
                     bias_dtype, lora_a, lora_b, r, scaling, const_cast<void*>(x), workspace, workspace_bytes);
  if (rc != RQ_OK) return rc;
  a.y = nullptr;
  a.gather = gather;
  return linear_forward(a, (cudaStream_t)stream);
}

int rq_linear_dx(int wfmt, const void* qweight, const void* scales, int scale_dtype, const uint8_t* c2,
                 const float* c2_scales, int64_t N, int64_t K, int block_size, const void* dy, int xdtype, int64_t M,
                 const void* lora_a, const void* lora_b, int r, float scaling, void* dx, void* workspace,
                 int64_t workspace_bytes, void* stream) {
  RQ_PROLOGUE();
  LinearArgs a;
  int rc = fill_args(&a, wfmt, qweight, scales, scale_dtype, c2, c2_scales, N, K, block_size, dy, xdtype, M,
                     nullptr, 0, lora_a, lora_b, r, scaling, dx, workspace, workspace_bytes);
  if (rc != RQ_OK) return rc;
  return linear_dx(a, (cudaStream_t)stream);
}

int rq_merge_lora(int wfmt, const void* qweight, const void* scales, int scale_dtype, const uint8_t* c2,
                  const float* c2_scales, int64_t N, int64_t K, int block_size, const float* lora_a,
                  const float* lora_b, int r, float scaling, int mode, void* out, int out_dtype, void* stream) {
  RQ_PROLOGUE();
  int rc = check_weight(wfmt, qweight, scales, scale_dtype, c2, c2_scales, N, K, block_size);
  if (rc != RQ_OK) return rc;
  if (!dtype_ok(out_dtype)) return RQ_ERR_DTYPE;
  if (r < 0 || r > 128 || (r > 0 && (!lora_a || !lora_b)) || (N * K > 0 && !out)) return RQ_ERR_INVALID;
  if (mode != RQ_MERGE_FP32_SUM && mode != RQ_MERGE_ROUND_EACH) return RQ_ERR_INVALID;
  if ((uintptr_t)out % dtype_size(out_dtype)) return RQ_ERR_ALIGN;
  const QWeight w{wfmt, qweight, scales, scale_dtype, c2, c2_scales, N, K, block_size};
  return merge_weight(w, lora_a, lora_b, r, scaling, mode, out, out_dtype, (cudaStream_t)stream);
}

int rq_weight_absmax(int wfmt, const void* qweight, const void* scales, int scale_dtype, const uint8_t* c2,
                     const float* c2_scales, int64_t N, int64_t K, int block_size, int dtype, float* absmax,
                     void* stream) {
  RQ_PROLOGUE();
  const int rc = check_weight(wfmt, qweight, scales, scale_dtype, c2, c2_scales, N, K, block_size);
  if (rc != RQ_OK) return rc;
  if (!dtype_ok(dtype)) return RQ_ERR_DTYPE;
  if (!absmax) return RQ_ERR_INVALID;
  if ((uintptr_t)absmax % 4) return RQ_ERR_ALIGN;
  const QWeight w{wfmt, qweight, scales, scale_dtype, c2, c2_scales, N, K, block_size};
  return weight_absmax(w, dtype, absmax, (cudaStream_t)stream);
}

int rq_weight_to_fp8(int wfmt, const void* qweight, const void* scales, int scale_dtype, const uint8_t* c2,
                     const float* c2_scales, int64_t N, int64_t K, int block_size, int dtype, float w_scale,
                     uint8_t* fp8_out, void* stream) {
  RQ_PROLOGUE();
  const int rc = check_weight(wfmt, qweight, scales, scale_dtype, c2, c2_scales, N, K, block_size);
  if (rc != RQ_OK) return rc;
  if (!dtype_ok(dtype)) return RQ_ERR_DTYPE;
  if (N * K > 0 && !fp8_out) return RQ_ERR_INVALID;
  const QWeight w{wfmt, qweight, scales, scale_dtype, c2, c2_scales, N, K, block_size};
  return weight_to_fp8(w, dtype, w_scale, fp8_out, (cudaStream_t)stream);
}

int64_t rq_adapter_plan_words(int64_t rows, int count, int tile_rows) {
  if (!fits(rows) || count < 1 || count > RQ_ADAPTERS_MAX ||
      (tile_rows != 16 && tile_rows != 32 && tile_rows != 64 && tile_rows != 128))
    return -1;
  return adapter_plan_words(rows, count, tile_rows);
}

int rq_adapter_plan(const void* ids, int wide, int64_t rows, int count, int tile_rows, int32_t* plan,
                    int64_t plan_words, void* stream) {
  RQ_PROLOGUE();
  if (!plan || (rows > 0 && !ids)) return RQ_ERR_INVALID;
  const int rc = check_plan(rows, count, tile_rows, plan, plan_words);
  if (rc != RQ_OK) return rc;
  if ((uintptr_t)ids % (wide ? 8 : 4)) return RQ_ERR_ALIGN;
  return adapter_plan(ids, wide ? 1 : 0, rows, count, tile_rows, plan, (cudaStream_t)stream);
}

int rq_adapters_apply(const void* in, int64_t ld_in, const void* U, const void* V, const float* scaling,
                      const void* base, int64_t ld_base, int64_t M, int64_t D1, int64_t D2, int r, int count,
                      int dtype, const int32_t* plan, int64_t plan_words, int tile_rows, float* mid, void* out,
                      int64_t ld_out, void* stream) {
  RQ_PROLOGUE();
  if (!half_ok(dtype)) return RQ_ERR_DTYPE;
  const int rc = check_plan(M, count, tile_rows, plan, plan_words);
  if (rc != RQ_OK) return rc;
  if (!fits(D1) || !fits(D2) || r < 8 || r > 128 || r % 8) return RQ_ERR_INVALID;
  if (M == 0) return RQ_OK;
  if (!scaling || (D1 > 0 && (!in || !U)) || (D2 > 0 && (!V || !out))) return RQ_ERR_INVALID;
  if (!row_stride(M, ld_in, D1) || (base && !row_stride(M, ld_base, D2)) || (M > 1 && ld_out < D2)) return RQ_ERR_INVALID;
  if ((uintptr_t)in % 2 || (uintptr_t)base % 2 || (uintptr_t)out % 2 || (uintptr_t)U % 16 || (uintptr_t)V % 16 ||
      (uintptr_t)mid % 16 || (uintptr_t)scaling % 4)
    return RQ_ERR_ALIGN;
  const AdapterRows a{M, D1, D2, r, count, dtype, tile_rows, plan};
  return adapters_apply(a, in, ld_in, U, V, scaling, base, ld_base, mid, out, ld_out, (cudaStream_t)stream);
}

int rq_adapters_grad(const void* z, int64_t ld_z, const float* z_scales, const float* mid, int64_t M, int64_t D, int r,
                     int count, int dtype, const int32_t* plan, int64_t plan_words, int tile_rows, void* grad,
                     void* stream) {
  RQ_PROLOGUE();
  if (!half_ok(dtype)) return RQ_ERR_DTYPE;
  const int rc = check_plan(M, count, tile_rows, plan, plan_words);
  if (rc != RQ_OK) return rc;
  if (!fits(D) || r < 8 || r > 128 || r % 8) return RQ_ERR_INVALID;
  if (D == 0) return RQ_OK;
  const int64_t nb = (D + RQ_ACT8_BLOCK - 1) / RQ_ACT8_BLOCK;
  if (!grad || (M > 0 && (!z || !mid))) return RQ_ERR_INVALID;
  if (!row_stride(M, ld_z, z_scales ? nb * RQ_ACT8_BLOCK : D)) return RQ_ERR_INVALID;
  if ((uintptr_t)z % (z_scales ? 16 : 2) || (z_scales && (ld_z % 16 || (uintptr_t)z_scales % 4)) || (uintptr_t)mid % 16 || (uintptr_t)grad % 16)
    return RQ_ERR_ALIGN;
  const AdapterRows a{M, D, 0, r, count, dtype, tile_rows, plan};
  return adapters_grad(a, z, ld_z, z_scales, nb, mid, grad, (cudaStream_t)stream);
}

int rq_act8_pack(const void* x, int dtype, int64_t ld_x, int64_t M, int64_t K, int8_t* codes, float* scales,
                 void* stream) {
  RQ_PROLOGUE();
  if (!dtype_ok(dtype)) return RQ_ERR_DTYPE;
  if (!fits_act8(M, K) || !row_stride(M, ld_x, K)) return RQ_ERR_INVALID;
  if (M * K == 0) return RQ_OK;
  if (!x || !codes || !scales) return RQ_ERR_INVALID;
  if ((uintptr_t)x % dtype_size(dtype) || (uintptr_t)codes % 16 || (uintptr_t)scales % 4) return RQ_ERR_ALIGN;
  return act8_pack(x, dtype, ld_x, M, K, codes, scales, (cudaStream_t)stream);
}

int rq_act8_unpack(const int8_t* codes, const float* scales, int64_t M, int64_t K, void* out, int dtype,
                   void* stream) {
  RQ_PROLOGUE();
  if (!dtype_ok(dtype)) return RQ_ERR_DTYPE;
  if (!fits_act8(M, K)) return RQ_ERR_INVALID;
  if (M * K == 0) return RQ_OK;
  if (!codes || !scales || !out) return RQ_ERR_INVALID;
  if ((uintptr_t)out % dtype_size(dtype) || (uintptr_t)codes % 16 || (uintptr_t)scales % 4) return RQ_ERR_ALIGN;
  return act8_unpack(codes, scales, M, K, out, dtype, (cudaStream_t)stream);
}

int rq_swiglu8_forward(const void* gate, int64_t ld_gate, const void* up, int64_t ld_up, int dtype, int64_t M,
                       int64_t K, void* h, int8_t* codes, float* scales, int copies, void* stream) {
  RQ_PROLOGUE();
  if (!dtype_ok(dtype)) return RQ_ERR_DTYPE;
  if (!fits_act8(M, K) || (copies != 2 && copies != 3)) return RQ_ERR_INVALID;
  if (!row_stride(M, ld_gate, K) || !row_stride(M, ld_up, K)) return RQ_ERR_INVALID;
  if (M * K == 0) return RQ_OK;
  if (!gate || !up || !h || !codes || !scales) return RQ_ERR_INVALID;
  const int e = dtype_size(dtype);
  if ((uintptr_t)gate % e || (uintptr_t)up % e || (uintptr_t)h % e || (uintptr_t)codes % 16 || (uintptr_t)scales % 4)
    return RQ_ERR_ALIGN;
  return swiglu8_forward(gate, ld_gate, up, ld_up, dtype, M, K, h, codes, scales, copies, (cudaStream_t)stream);
}

int rq_swiglu8_backward(const void* dh, int64_t ld_dh, int dtype, int64_t M, int64_t K, const int8_t* codes,
                        const float* scales, void* dgate, void* dup, void* stream) {
  RQ_PROLOGUE();
  if (!dtype_ok(dtype)) return RQ_ERR_DTYPE;
  if (!fits_act8(M, K) || !row_stride(M, ld_dh, K)) return RQ_ERR_INVALID;
  if (M * K == 0) return RQ_OK;
  if (!dh || !codes || !scales || !dgate || !dup) return RQ_ERR_INVALID;
  const int e = dtype_size(dtype);
  if ((uintptr_t)dh % e || (uintptr_t)dgate % e || (uintptr_t)dup % e || (uintptr_t)codes % 16 ||
      (uintptr_t)scales % 4)
    return RQ_ERR_ALIGN;
  return swiglu8_backward(dh, ld_dh, dtype, M, K, codes, scales, dgate, dup, (cudaStream_t)stream);
}

int rq_token_logprobs(const void* logits, int dtype, int64_t stride_b, int64_t stride_l, int64_t B, int64_t L,
                      int64_t V, const int64_t* labels, int64_t ignore, float* stats, float* logps, void* stream) {
  RQ_PROLOGUE();
  const int rc = check_tokens(logits, dtype, B, L, V, labels, stats);
  if (rc != RQ_OK) return rc;
  if (B * L == 0) return RQ_OK;
  if ((uintptr_t)logps % 4) return RQ_ERR_ALIGN;
  const TokenRows t{logits, stride_b, stride_l, dtype, B, L, V, labels, ignore};
  return token_logprobs(t, stats, logps, (cudaStream_t)stream);
}

int rq_preference_loss(int64_t B, int64_t L, const int64_t* labels, int64_t ignore, const float* stats,
                       const float* ref, int form, float beta, float smooth, float* loss, float* logps, float* rewards,
                       float* slopes, void* stream) {
  RQ_PROLOGUE();
  const int rc = check_tokens(stats, RQ_F32, B, L, 1, labels, stats);
  if (rc != RQ_OK) return rc;
  if (B < 2 || B % 2 || L < 1 || (form != RQ_PREF_SIGMOID && form != RQ_PREF_IPO)) return RQ_ERR_INVALID;
  if (!(beta > 0.0f) || !(smooth >= 0.0f && smooth <= 0.5f)) return RQ_ERR_INVALID;
  if (!ref || !loss || !logps || !rewards || !slopes) return RQ_ERR_INVALID;
  if ((uintptr_t)ref % 4 || (uintptr_t)loss % 4 || (uintptr_t)logps % 4 || (uintptr_t)rewards % 4 ||
      (uintptr_t)slopes % 4)
    return RQ_ERR_ALIGN;
  const TokenRows t{nullptr, 0, 0, RQ_F32, B, L, 1, labels, ignore};
  return preference_loss(t, stats, ref, form, beta, smooth, loss, logps, rewards, slopes, (cudaStream_t)stream);
}

int rq_token_logprobs_grad(const void* logits, int dtype, int64_t stride_b, int64_t stride_l, int64_t B, int64_t L,
                           int64_t V, const int64_t* labels, int64_t ignore, const float* stats, const float* slopes,
                           int per_token, const float* upstream, void* dlogits, void* stream) {
  RQ_PROLOGUE();
  const int rc = check_tokens(logits, dtype, B, L, V, labels, stats);
  if (rc != RQ_OK) return rc;
  if (B * L == 0) return RQ_OK;
  if (!slopes || !dlogits) return RQ_ERR_INVALID;
  if ((uintptr_t)slopes % 4 || (uintptr_t)upstream % 4 || (uintptr_t)dlogits % dtype_size(dtype)) return RQ_ERR_ALIGN;
  const TokenRows t{logits, stride_b, stride_l, dtype, B, L, V, labels, ignore};
  return token_logprobs_grad(t, stats, slopes, per_token ? 1 : 0, upstream, dlogits, (cudaStream_t)stream);
}

int64_t rq_mx4_scale_bytes(int64_t M, int64_t K) {
  return !fits(M) || !fits(K) ? -1 : (M + 127) / 128 * (mx4_pitch(K) / 128) * 512;
}

int rq_mx4_pack(const void* x, int dtype, int64_t ld_x, int64_t M, int64_t K, uint8_t* codes, uint8_t* scales,
                void* stream) {
  RQ_PROLOGUE();
  if (!dtype_ok(dtype)) return RQ_ERR_DTYPE;
  if (!row_stride(M, ld_x, K)) return RQ_ERR_INVALID;
  const int rc = check_mx4(codes, scales, M, K);
  if (rc != RQ_OK) return rc;
  if (M * K == 0) return RQ_OK;
  if (!x) return RQ_ERR_INVALID;
  if ((uintptr_t)x % dtype_size(dtype)) return RQ_ERR_ALIGN;
  return mx4_pack(x, dtype, ld_x, M, K, codes, scales, (cudaStream_t)stream);
}

int rq_mx4_unpack(const uint8_t* codes, const uint8_t* scales, int64_t M, int64_t K, void* out, int dtype,
                  void* stream) {
  RQ_PROLOGUE();
  if (!dtype_ok(dtype)) return RQ_ERR_DTYPE;
  const int rc = check_mx4(codes, scales, M, K);
  if (rc != RQ_OK) return rc;
  if (M * K == 0) return RQ_OK;
  if (!out) return RQ_ERR_INVALID;
  if ((uintptr_t)out % dtype_size(dtype)) return RQ_ERR_ALIGN;
  return mx4_unpack(codes, scales, M, K, out, dtype, (cudaStream_t)stream);
}

int rq_mx4_matmul(const uint8_t* a_codes, const uint8_t* a_scales, int64_t M, const uint8_t* b_codes,
                  const uint8_t* b_scales, int64_t N, int64_t K, const void* bias, void* out, int dtype,
                  void* stream) {
  RQ_PROLOGUE();
  int rc = check_product(dtype, M, N, K);
  if (rc == RQ_OK) rc = check_mx4(a_codes, a_scales, M, K);
  if (rc == RQ_OK) rc = check_mx4(b_codes, b_scales, N, K);
  if (rc != RQ_OK) return rc;
  if (M * N == 0) return RQ_OK;
  if (K < 1 || !out) return RQ_ERR_INVALID;
  if ((uintptr_t)out % 2 || (uintptr_t)bias % 2) return RQ_ERR_ALIGN;
  return mx4_matmul(Mx4{a_codes, a_scales, M}, Mx4{b_codes, b_scales, N}, K, bias, out, dtype, (cudaStream_t)stream);
}

int rq_mx4_set_wait(int64_t ns) {
  mx4_set_wait(ns);
  return RQ_OK;
}

int64_t rq_mx4_linear_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  return !fits(M) || !fits(N) || !fits(K) ? -1 : mx4_linear_workspace_bytes(M, N, K);
}

int rq_mx4_linear(const void* x, int dtype, int64_t ld_x, int64_t M, const uint8_t* w_codes, const uint8_t* w_scales,
                  int64_t N, int64_t K, const void* bias, void* out, void* workspace, int64_t workspace_bytes,
                  void* stream) {
  RQ_PROLOGUE();
  int rc = check_product(dtype, M, N, K);
  if (rc == RQ_OK) rc = check_mx4(w_codes, w_scales, N, K);
  if (rc != RQ_OK) return rc;
  if (!row_stride(M, ld_x, K) || !fits((M + 127) / 128 * 128 * (mx4_pitch(K) / 128))) return RQ_ERR_INVALID;
  if (M * N == 0) return RQ_OK;
  if (K < 1 || !x || !out) return RQ_ERR_INVALID;
  const int64_t need = mx4_linear_workspace_bytes(M, N, K);
  if (need > 0 && (!workspace || workspace_bytes < need)) return RQ_ERR_WORKSPACE;
  if ((uintptr_t)x % 2 || (uintptr_t)out % 2 || (uintptr_t)bias % 2 || (uintptr_t)workspace % 256) return RQ_ERR_ALIGN;
  return mx4_linear(x, dtype, ld_x, M, Mx4{w_codes, w_scales, N}, K, bias, out, workspace, (cudaStream_t)stream);
}

int rq_mx4_dx(const void* dy, int dtype, int64_t ld_dy, int64_t M, const uint8_t* w_codes, const uint8_t* w_scales,
              int64_t N, int64_t K, void* dx, void* workspace, int64_t workspace_bytes, void* stream) {
  RQ_PROLOGUE();
  int rc = check_product(dtype, M, N, K);
  if (rc == RQ_OK) rc = check_mx4(w_codes, w_scales, N, K);
  if (rc != RQ_OK) return rc;
  if (M * K == 0) return RQ_OK;
  if (N < 1 || !dy || !dx || ld_dy < N || ld_dy % 8) return RQ_ERR_INVALID;
  if (dtype == RQ_F16 && (!workspace || workspace_bytes < RQ_MX4_DX_WORKSPACE)) return RQ_ERR_WORKSPACE;
  if ((uintptr_t)dy % 16 || (uintptr_t)dx % 2 || (uintptr_t)workspace % 16) return RQ_ERR_ALIGN;
  return mx4_dx(dy, dtype, ld_dy, M, Mx4{w_codes, w_scales, N}, K, dx, workspace, (cudaStream_t)stream);
}

int rq_align_rows(const void* x, int64_t ld_x, int64_t M, int64_t N, void* out, int64_t ld_out, void* stream) {
  RQ_PROLOGUE();
  if (!fits(M) || !fits(N) || !fits(M * (N / 1024 + 1)) || !row_stride(M, ld_x, N) || ld_out < N || ld_out % 8)
    return RQ_ERR_INVALID;
  if (M * N == 0) return RQ_OK;
  if (!x || !out) return RQ_ERR_INVALID;
  if ((uintptr_t)x % 2 || (uintptr_t)out % 16) return RQ_ERR_ALIGN;
  return align_rows(x, ld_x, M, N, out, ld_out, (cudaStream_t)stream);
}

int rq_grad_norm_partial(const RqAdamTensor* tensors, int count, int dtype, double* partials, void* stream) {
  RQ_PROLOGUE();
  const int rc = check_tensors(tensors, count, dtype, false, false);
  if (rc != RQ_OK) return rc;
  if (count < 1 || !partials) return RQ_ERR_INVALID;
  if ((uintptr_t)partials % 8) return RQ_ERR_ALIGN;
  return grad_norm_partial(tensors, count, dtype, partials, (cudaStream_t)stream);
}

int rq_grad_norm_end(const double* partials, int n, float* norm, void* stream) {
  RQ_PROLOGUE();
  if (n < 0 || (n > 0 && !partials) || !norm) return RQ_ERR_INVALID;
  if ((uintptr_t)partials % 8 || (uintptr_t)norm % 4) return RQ_ERR_ALIGN;
  return grad_norm_end(partials, n, norm, (cudaStream_t)stream);
}

static bool beta_ok(double b) { return b >= 0.0 && b < 1.0; }

int rq_adam_update(const RqAdamTensor* tensors, int count, int dtype, int bits, void* m, void* v, float* scales,
                   int16_t* low, const RqAdamStep* step, void* stream) {
  RQ_PROLOGUE();
  const int rc = check_tensors(tensors, count, dtype, true, true);
  if (rc != RQ_OK) return rc;
  if (!step || (bits != 8 && bits != 32) || !beta_ok(step->beta1) || !beta_ok(step->beta2) || !(step->eps >= 0.0))
    return RQ_ERR_INVALID;
  if (low && dtype != RQ_BF16) return RQ_ERR_DTYPE;
  if (count == 0) return RQ_OK;
  if (!m || !v || (bits == 8 && !scales) || !step->steps || !step->ticket) return RQ_ERR_INVALID;
  if (step->n_partials < 0 || (step->n_partials > 0 && (!step->partials || !step->norm))) return RQ_ERR_INVALID;
  if ((uintptr_t)m % 32 || (uintptr_t)v % 32 || (uintptr_t)scales % 8 || (uintptr_t)low % 16 ||
      (uintptr_t)step->partials % 8 || (uintptr_t)step->norm % 4 || (uintptr_t)step->steps % 4 ||
      (uintptr_t)step->ticket % 4 || (uintptr_t)step->lr_at % 4)
    return RQ_ERR_ALIGN;
  return adam_update(tensors, count, dtype, bits, m, v, scales, low, *step, (cudaStream_t)stream);
}

int rq_adam_unpack(const uint8_t* m8, const uint8_t* r8, const float* scales, int64_t blocks, float* m, float* v,
                   void* stream) {
  RQ_PROLOGUE();
  if (!fits(blocks)) return RQ_ERR_INVALID;
  if (blocks == 0) return RQ_OK;
  if (!m8 || !r8 || !scales || !m || !v) return RQ_ERR_INVALID;
  if ((uintptr_t)m8 % 8 || (uintptr_t)r8 % 8 || (uintptr_t)scales % 8 || (uintptr_t)m % 32 || (uintptr_t)v % 32)
    return RQ_ERR_ALIGN;
  return adam_unpack(m8, r8, scales, blocks, m, v, (cudaStream_t)stream);
}

int rq_adam_pack(const float* m, const float* v, int64_t blocks, uint8_t* m8, uint8_t* r8, float* scales,
                 void* stream) {
  RQ_PROLOGUE();
  if (!fits(blocks)) return RQ_ERR_INVALID;
  if (blocks == 0) return RQ_OK;
  if (!m8 || !r8 || !scales || !m || !v) return RQ_ERR_INVALID;
  if ((uintptr_t)m8 % 8 || (uintptr_t)r8 % 8 || (uintptr_t)scales % 8 || (uintptr_t)m % 32 || (uintptr_t)v % 32)
    return RQ_ERR_ALIGN;
  return adam_pack(m, v, blocks, m8, r8, scales, (cudaStream_t)stream);
}

void launch_int4_dequant_matmul(void* stream, void* x, void* w_packed, void* scales, void* c, int M, int N, int K,
                                int block_size) {
  g_last_status = rq_linear_forward(RQ_W_NF4, w_packed, scales, RQ_F16, nullptr, nullptr, N, K, block_size, x,
                                    RQ_F16, M, nullptr, nullptr, 0, nullptr, nullptr, 0, 1.0f, c, nullptr, 0, stream);
}

void launch_int8_dequant_matmul(void* stream, void* x, void* w_int8, void* scales, void* c, int M, int N, int K,
                                int block_size) {
  g_last_status = rq_linear_forward(RQ_W_INT8, w_int8, scales, RQ_F16, nullptr, nullptr, N, K, block_size, x,
                                    RQ_F16, M, nullptr, nullptr, 0, nullptr, nullptr, 0, 1.0f, c, nullptr, 0, stream);
}

}  // extern "C"

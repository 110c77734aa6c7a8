// torch_ops.h -- what the torch extension's sources share.
#pragma once

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include <initializer_list>
#include <optional>

#include "../../include/rq_b200.h"

namespace rq_torch {

inline int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return RQ_F32;
    case at::kBFloat16: return RQ_BF16;
    case at::kHalf: return RQ_F16;
    default: TORCH_CHECK(false, "rocm_qlora: unsupported dtype ", t);
  }
  return RQ_F32;
}

inline const void* ptr(const std::optional<at::Tensor>& t) {
  return t.has_value() && t->defined() ? t->data_ptr() : nullptr;
}

inline void check(int rc, const char* what) {
  TORCH_CHECK(rc == RQ_OK, "rocm_qlora: ", what, " failed: ", rq_status_string(rc), " (status ", rc,
              rc == RQ_ERR_CUDA ? ", cuda error " + std::to_string(rq_last_cuda_error()) : std::string(), ")");
}

using at::Tensor;
using std::optional;

inline cudaStream_t stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// The kernels take pointers: every tensor of a call is on the first one's device.
inline void check_device(const Tensor& first, const Tensor& t) {
  TORCH_CHECK(t.device() == first.device(), "rocm_qlora: tensors are on different devices: ", first.device(), " and ",
              t.device());
}
inline void check_device(const Tensor& first, const optional<Tensor>& t) {
  if (t.has_value() && t->defined()) check_device(first, *t);
}
template <class... Rest>
inline void one_device(const Tensor& first, const Rest&... rest) {
  (check_device(first, rest), ...);
}

// The kernels read banks and codes in 16-byte pieces: a view that starts
// between two of them is copied.
inline Tensor aligned(const Tensor& t) {
  return t.is_meta() || (uintptr_t)t.data_ptr() % 16 == 0 ? t : t.clone(at::MemoryFormat::Contiguous);
}

// One of the operators above, through the dispatcher but for its autograd keys:
// the nodes here are the gradients.
template <auto F, class... A>
auto via(const char* name, A&&... args) {
  static const auto op =
      c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<std::remove_pointer_t<decltype(F)>>();
  const at::AutoDispatchBelowAutograd below;
  return op.call(std::forward<A>(args)...);
}
#define RQ_VIA(op, ...) via<&op>("rocm_qlora::" #op, __VA_ARGS__)

inline void once(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), "rocm_qlora: ", what, " is differentiable once only");
}

// t as [rows, columns]: contiguous columns, rows apart or one row for all; a
// copy where its strides are others (rows that overlap among them).
inline Tensor rows_of(const Tensor& t) {
  Tensor r = t.dim() == 2 ? t : t.reshape({c10::multiply_integers(t.sizes().slice(0, t.dim() - 1)), t.size(-1)});
  const bool columns = r.size(1) <= 1 || r.stride(1) == 1;
  const bool rows = r.size(0) <= 1 || r.stride(0) == 0 || r.stride(0) >= r.size(1);
  return columns && rows ? r : r.contiguous();
}

inline void check_float(at::ScalarType t) {
  TORCH_CHECK_TYPE(t == at::kFloat || t == at::kBFloat16 || t == at::kHalf, "unsupported dtype ", t,
                   "; rocm_qlora kernels take float32, bfloat16 or float16");
}

inline void check_gpu(std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors) {
    TORCH_CHECK_NOT_IMPLEMENTED(!t->is_cpu(), "rocm_qlora (B200 build) computes on the GPU only: move the tensors to a CUDA device");
    TORCH_CHECK(t->device() == (*tensors.begin())->device(), "tensors are on different devices: ",
                (*tensors.begin())->device(), " and ", t->device());
  }
}

}  // namespace rq_torch

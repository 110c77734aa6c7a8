// torch_ops.h -- what the torch extension's sources share.
#pragma once

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

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

}  // namespace rq_torch

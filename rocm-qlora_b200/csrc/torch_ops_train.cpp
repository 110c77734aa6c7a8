// torch_ops_train.cpp -- torch operators of the adapters of many requests,
// the 8-bit activations and the token log-probabilities with the preference
// loss (include/rq_b200.h).  As in torch_ops.cpp, outputs are allocated here,
// launches go to torch's current stream of the input's device, a status other
// than RQ_OK raises, and nothing is computed.  On Meta tensors the operators
// only give shapes; the public ones, at the end, call the others through the
// dispatcher, so that tracing (FakeTensor, make_fx) sees those.
#include "torch_ops.h"

#include <torch/csrc/autograd/VariableTypeUtils.h>
#include <torch/csrc/autograd/custom_function.h>

#include <tuple>

namespace {

using at::Tensor;
using rq_torch::check;
using rq_torch::dtype_code;
using rq_torch::ptr;
using std::optional;

cudaStream_t stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

void check_rows(const Tensor& t, const char* name) {
  TORCH_CHECK(t.dim() == 2 && (t.size(1) <= 1 || t.stride(1) == 1), "rocm_qlora: ", name,
              " must be a 2-D tensor with contiguous columns");
}

// The kernels take pointers: every tensor of a call is on the first one's device.
void check_device(const Tensor& first, const Tensor& t) {
  TORCH_CHECK(t.device() == first.device(), "rocm_qlora: tensors are on different devices: ", first.device(), " and ",
              t.device());
}
void check_device(const Tensor& first, const optional<Tensor>& t) {
  if (t.has_value() && t->defined()) check_device(first, *t);
}
template <class... Rest>
void one_device(const Tensor& first, const Rest&... rest) {
  (check_device(first, rest), ...);
}

bool plan_ok(const Tensor& plan) { return plan.dim() == 1 && plan.is_contiguous() && plan.scalar_type() == at::kInt; }

void check_plan(const optional<Tensor>& plan) {
  TORCH_CHECK(!plan.has_value() || !plan->defined() || plan_ok(*plan),
              "rocm_qlora: plan must be a contiguous 1-D int32 tensor, as adapter_plan makes it");
}

// The kernels read banks and codes in 16-byte pieces: a view that starts
// between two of them is copied.
Tensor aligned(const Tensor& t) {
  return t.is_meta() || (uintptr_t)t.data_ptr() % 16 == 0 ? t : t.clone(at::MemoryFormat::Contiguous);
}

Tensor adapter_plan(const Tensor& ids, int64_t count, int64_t tile) {
  TORCH_CHECK(ids.dim() == 1 && ids.is_contiguous() && (ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt),
              "rocm_qlora: ids must be a contiguous 1-D int64 or int32 tensor");
  const int64_t words = rq_adapter_plan_words(ids.size(0), (int)count, (int)tile);
  TORCH_CHECK(words >= 0, "rocm_qlora: no plan for ", ids.size(0), " rows and ", count, " adapters");
  Tensor plan = at::empty({words}, ids.options().dtype(at::kInt));
  if (ids.is_meta()) return plan;
  const c10::cuda::CUDAGuard guard(ids.device());
  check(rq_adapter_plan(ids.data_ptr(), ids.scalar_type() == at::kLong, ids.size(0), (int)count, (int)tile,
                        plan.data_ptr<int>(), words, stream_of(ids)),
        "rq_adapter_plan");
  return plan;
}

// out (nullopt: mid only) = base + mid V^T, mid = scaling (in U)
void apply(const Tensor& in, const Tensor& U, const Tensor& V, const Tensor& scaling, const optional<Tensor>& base,
           const optional<Tensor>& plan, int64_t tile, const optional<Tensor>& mid, const optional<Tensor>& out) {
  const c10::cuda::CUDAGuard guard(in.device());
  const bool has_base = base.has_value() && base->defined(), has_plan = plan.has_value() && plan->defined();
  const Tensor u = aligned(U), v = aligned(V);
  check(rq_adapters_apply(in.data_ptr(), in.stride(0), u.data_ptr(), v.data_ptr(), scaling.data_ptr<float>(), ptr(base),
                          has_base ? base->stride(0) : 0, in.size(0), in.size(1), out ? out->size(1) : 0,
                          (int)U.size(2), (int)U.size(0), dtype_code(in.scalar_type()),
                          static_cast<const int32_t*>(ptr(plan)), has_plan ? plan->numel() : 0, (int)tile,
                          mid ? mid->data_ptr<float>() : nullptr, out ? out->data_ptr() : nullptr, out ? out->stride(0) : 0,
                          stream_of(in)),
        "rq_adapters_apply");
}

void check_bank(const Tensor& in, const Tensor& U, const Tensor& V, const Tensor& scaling,
                const optional<Tensor>& plan) {
  check_rows(in, "input");
  one_device(in, U, V, scaling, plan);
  check_plan(plan);
  TORCH_CHECK(U.dim() == 3 && V.dim() == 3 && U.is_contiguous() && V.is_contiguous() && U.size(0) == V.size(0) &&
                  U.size(2) == V.size(2) && U.size(1) == in.size(1) && U.scalar_type() == in.scalar_type() &&
                  V.scalar_type() == in.scalar_type(),
              "rocm_qlora: adapters must be contiguous [count, columns, rank] tensors of the input's dtype and size");
  TORCH_CHECK(scaling.is_contiguous() && scaling.scalar_type() == at::kFloat && scaling.numel() == U.size(0),
              "rocm_qlora: scaling must be a contiguous float32 tensor of one value an adapter");
}

void check_base(const Tensor& in, const Tensor& V, const Tensor& base) {
  one_device(in, base);
  check_rows(base, "base");
  TORCH_CHECK(base.size(0) == in.size(0) && base.size(1) == V.size(1) && base.scalar_type() == in.scalar_type(),
              "rocm_qlora: base must be [rows, ", V.size(1), "] of the input's dtype");
}

std::tuple<Tensor, Tensor> adapters_apply(const Tensor& in, const Tensor& U, const Tensor& V, const Tensor& scaling,
                                          const optional<Tensor>& base, const optional<Tensor>& plan, int64_t tile) {
  check_bank(in, U, V, scaling, plan);
  if (base.has_value() && base->defined()) check_base(in, V, *base);
  Tensor out = at::empty({in.size(0), V.size(1)}, in.options());
  Tensor mid = at::empty({in.size(0), U.size(2)}, in.options().dtype(at::kFloat));
  if (!in.is_meta()) apply(in, U, V, scaling, base, plan, tile, mid, out);
  return {out, mid};
}

Tensor adapters_apply_(Tensor out, const Tensor& in, const Tensor& U, const Tensor& V, const Tensor& scaling,
                       const Tensor& base, const optional<Tensor>& plan, int64_t tile) {
  check_bank(in, U, V, scaling, plan);
  one_device(in, out, base);
  check_rows(out, "out");
  check_rows(base, "base");
  TORCH_CHECK(out.size(0) == in.size(0) && out.size(1) == V.size(1) && out.scalar_type() == in.scalar_type() &&
                  base.sizes() == out.sizes() && base.scalar_type() == in.scalar_type(),
              "rocm_qlora: out and base must be [rows, ", V.size(1), "] of the input's dtype");
  Tensor mid = at::empty({in.size(0), U.size(2)}, in.options().dtype(at::kFloat));
  if (!in.is_meta()) apply(in, U, V, scaling, base, plan, tile, mid, out);
  return mid;
}

// Above the backends: autograd's version counter of `out` counts the write, so
// that a node which saved it refuses its backward.
Tensor adapters_apply_versioned(c10::DispatchKeySet keys, Tensor out, const Tensor& in, const Tensor& U, const Tensor& V,
                                const Tensor& scaling, const Tensor& base, const optional<Tensor>& plan, int64_t tile) {
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("rocm_qlora::adapters_apply_", "")
                             .typed<Tensor(Tensor, const Tensor&, const Tensor&, const Tensor&, const Tensor&,
                                           const Tensor&, const optional<Tensor>&, int64_t)>();
  Tensor mid;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    mid = op.redispatch(keys & c10::after_ADInplaceOrView_keyset, out, in, U, V, scaling, base, plan, tile);
  }
  torch::autograd::increment_version(out);
  return mid;
}

// The output alone, for calls without a backward.
Tensor adapters_product(const Tensor& in, const Tensor& U, const Tensor& V, const Tensor& scaling, const Tensor& base,
                        const optional<Tensor>& plan, int64_t tile) {
  check_bank(in, U, V, scaling, plan);
  check_base(in, V, base);
  Tensor out = at::empty({in.size(0), V.size(1)}, in.options());
  if (!in.is_meta()) apply(in, U, V, scaling, base, plan, tile, std::nullopt, out);
  return out;
}

Tensor adapters_mid(const Tensor& in, const Tensor& U, const Tensor& V, const Tensor& scaling,
                    const optional<Tensor>& plan, int64_t tile) {
  check_bank(in, U, V, scaling, plan);
  Tensor mid = at::empty({in.size(0), U.size(2)}, in.options().dtype(at::kFloat));
  if (!in.is_meta()) apply(in, U, V, scaling, std::nullopt, plan, tile, mid, std::nullopt);
  return mid;
}

Tensor adapters_grad(const Tensor& z, const optional<Tensor>& scales, const Tensor& mid, int64_t D, int64_t count,
                     at::ScalarType dtype, const optional<Tensor>& plan, int64_t tile) {
  check_rows(z, "rows");
  one_device(z, scales, mid, plan);
  check_plan(plan);
  const bool packed = scales.has_value() && scales->defined(), has_plan = plan.has_value() && plan->defined();
  const int64_t nb = (D + RQ_ACT8_BLOCK - 1) / RQ_ACT8_BLOCK;
  TORCH_CHECK(mid.dim() == 2 && mid.is_contiguous() && mid.size(0) == z.size(0) && mid.scalar_type() == at::kFloat,
              "rocm_qlora: mid must be a contiguous [rows, rank] float32 tensor");
  TORCH_CHECK(packed ? z.scalar_type() == at::kChar && z.size(1) == nb * RQ_ACT8_BLOCK && scales->is_contiguous() &&
                           scales->numel() == z.size(0) * nb && scales->scalar_type() == at::kFloat
                     : z.scalar_type() == dtype && z.size(1) == D,
              "rocm_qlora: rows must be [rows, ", D, "] of the adapters' dtype, or their packed form");
  Tensor grad = at::empty({count, D, mid.size(1)}, z.options().dtype(dtype));
  if (z.is_meta()) return grad;
  const c10::cuda::CUDAGuard guard(z.device());
  const Tensor rows = packed ? aligned(z) : z;
  check(rq_adapters_grad(rows.data_ptr(), rows.stride(0), static_cast<const float*>(ptr(scales)), mid.data_ptr<float>(),
                         z.size(0), D, (int)mid.size(1), (int)count, dtype_code(dtype),
                         static_cast<const int32_t*>(ptr(plan)), has_plan ? plan->numel() : 0, (int)tile,
                         grad.data_ptr(), stream_of(z)),
        "rq_adapters_grad");
  return grad;
}

int64_t blocks_of(int64_t K) { return (K + RQ_ACT8_BLOCK - 1) / RQ_ACT8_BLOCK; }

std::tuple<Tensor, Tensor> act8_pack(const Tensor& x) {
  check_rows(x, "x");
  const int64_t nb = blocks_of(x.size(1));
  Tensor codes = at::empty({x.size(0), nb * RQ_ACT8_BLOCK}, x.options().dtype(at::kChar));
  Tensor scales = at::empty({x.size(0), nb}, x.options().dtype(at::kFloat));
  if (!x.is_meta()) {
    const c10::cuda::CUDAGuard guard(x.device());
    check(rq_act8_pack(x.data_ptr(), dtype_code(x.scalar_type()), x.stride(0), x.size(0), x.size(1),
                       codes.data_ptr<int8_t>(), scales.data_ptr<float>(), stream_of(x)),
          "rq_act8_pack");
  }
  return {codes, scales};
}

void check_packed(const Tensor& codes, const Tensor& scales, int64_t K) {
  const int64_t nb = (K + RQ_ACT8_BLOCK - 1) / RQ_ACT8_BLOCK;
  one_device(codes, scales);
  TORCH_CHECK(codes.is_contiguous() && scales.is_contiguous() && codes.scalar_type() == at::kChar &&
                  scales.scalar_type() == at::kFloat && codes.dim() == scales.dim() &&
                  codes.size(-1) == nb * RQ_ACT8_BLOCK && scales.size(-1) == nb &&
                  codes.numel() == scales.numel() * RQ_ACT8_BLOCK,
              "rocm_qlora: not the packed form of rows of ", K, " values");
}

Tensor act8_unpack(const Tensor& codes, const Tensor& scales, int64_t K, at::ScalarType dtype) {
  TORCH_CHECK(codes.dim() == 2, "rocm_qlora: codes must be a 2-D tensor");
  check_packed(codes, scales, K);
  Tensor out = at::empty({codes.size(0), K}, codes.options().dtype(dtype));
  if (codes.is_meta()) return out;
  const c10::cuda::CUDAGuard guard(codes.device());
  check(rq_act8_unpack(aligned(codes).data_ptr<int8_t>(), scales.data_ptr<float>(), codes.size(0), K, out.data_ptr(),
                       dtype_code(dtype), stream_of(codes)),
        "rq_act8_unpack");
  return out;
}

std::tuple<Tensor, Tensor, Tensor> swiglu8_forward(const Tensor& gate, const Tensor& up, int64_t copies) {
  check_rows(gate, "gate");
  check_rows(up, "up");
  one_device(gate, up);
  TORCH_CHECK(gate.sizes() == up.sizes() && gate.scalar_type() == up.scalar_type(),
              "rocm_qlora: gate and up must have one shape and dtype");
  const int64_t nb = blocks_of(gate.size(1));
  Tensor codes = at::empty({copies, gate.size(0), nb * RQ_ACT8_BLOCK}, gate.options().dtype(at::kChar));
  Tensor scales = at::empty({copies, gate.size(0), nb}, gate.options().dtype(at::kFloat));
  Tensor h = at::empty({gate.size(0), gate.size(1)}, gate.options());
  if (!gate.is_meta()) {
    const c10::cuda::CUDAGuard guard(gate.device());
    check(rq_swiglu8_forward(gate.data_ptr(), gate.stride(0), up.data_ptr(), up.stride(0),
                             dtype_code(gate.scalar_type()), gate.size(0), gate.size(1), h.data_ptr(),
                             codes.data_ptr<int8_t>(), scales.data_ptr<float>(), (int)copies, stream_of(gate)),
          "rq_swiglu8_forward");
  }
  return {h, codes, scales};
}

std::tuple<Tensor, Tensor> swiglu8_backward(const Tensor& dh, const Tensor& codes, const Tensor& scales) {
  check_rows(dh, "dh");
  one_device(dh, codes);
  TORCH_CHECK(codes.dim() == 3 && codes.size(0) >= 2 && codes.size(1) == dh.size(0),
              "rocm_qlora: codes must hold the packed gate and up of dh's rows");
  check_packed(codes, scales, dh.size(1));
  Tensor dgate = at::empty({dh.size(0), dh.size(1)}, dh.options()), dup = at::empty_like(dgate);
  if (!dh.is_meta()) {
    const c10::cuda::CUDAGuard guard(dh.device());
    check(rq_swiglu8_backward(dh.data_ptr(), dh.stride(0), dtype_code(dh.scalar_type()), dh.size(0), dh.size(1),
                              codes.data_ptr<int8_t>(), scales.data_ptr<float>(), dgate.data_ptr(), dup.data_ptr(),
                              stream_of(dh)),
          "rq_swiglu8_backward");
  }
  return {dgate, dup};
}

void check_logits(const Tensor& logits, const Tensor& labels) {
  one_device(logits, labels);
  TORCH_CHECK(logits.dim() == 3 && (logits.size(2) <= 1 || logits.stride(2) == 1),
              "rocm_qlora: logits must be [batch, length, vocabulary] with a contiguous vocabulary");
  TORCH_CHECK(labels.dim() == 2 && labels.is_contiguous() && labels.scalar_type() == at::kLong &&
                  labels.size(0) == logits.size(0) && labels.size(1) == logits.size(1),
              "rocm_qlora: labels must be a contiguous [batch, length] int64 tensor");
}

void logprobs(const Tensor& logits, const Tensor& labels, int64_t ignore, const Tensor& stats, float* logps) {
  check(rq_token_logprobs(logits.data_ptr(), dtype_code(logits.scalar_type()), logits.stride(0), logits.stride(1),
                          logits.size(0), logits.size(1), logits.size(2), labels.data_ptr<int64_t>(), ignore,
                          stats.data_ptr<float>(), logps, stream_of(logits)),
        "rq_token_logprobs");
}

std::tuple<Tensor, Tensor> token_logprobs(const Tensor& logits, const Tensor& labels, int64_t ignore) {
  check_logits(logits, labels);
  const auto f32 = logits.options().dtype(at::kFloat);
  Tensor logps = at::empty({logits.size(0), logits.size(1)}, f32);
  Tensor stats = at::empty({logits.size(0), logits.size(1), 4}, f32);
  if (!logits.is_meta()) {
    const c10::cuda::CUDAGuard guard(logits.device());
    logprobs(logits, labels, ignore, stats, logps.data_ptr<float>());
  }
  return {logps, stats};
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> preference_forward(const Tensor& logits, const Tensor& labels,
                                                                      const Tensor& ref, int64_t ignore, int64_t form,
                                                                      double beta, double smooth) {
  check_logits(logits, labels);
  one_device(logits, ref);
  TORCH_CHECK(ref.sizes() == labels.sizes() && ref.is_contiguous() && ref.scalar_type() == at::kFloat,
              "rocm_qlora: ref must be a contiguous [batch, length] float32 tensor");
  const auto f32 = logits.options().dtype(at::kFloat);
  const int64_t B = logits.size(0), L = logits.size(1);
  Tensor loss = at::empty({}, f32), logps = at::empty({B}, f32), rewards = at::empty({B}, f32),
         slopes = at::empty({B}, f32), stats = at::empty({B, L, 4}, f32);
  if (!logits.is_meta()) {
    const c10::cuda::CUDAGuard guard(logits.device());
    logprobs(logits, labels, ignore, stats, nullptr);
    check(rq_preference_loss(B, L, labels.data_ptr<int64_t>(), ignore, stats.data_ptr<float>(), ref.data_ptr<float>(),
                             (int)form, (float)beta, (float)smooth, loss.data_ptr<float>(), logps.data_ptr<float>(),
                             rewards.data_ptr<float>(), slopes.data_ptr<float>(), stream_of(logits)),
          "rq_preference_loss");
  }
  return {loss, logps, rewards, slopes, stats};
}

Tensor token_logprobs_grad(const Tensor& logits, const Tensor& labels, int64_t ignore, const Tensor& stats,
                           const Tensor& slopes, const optional<Tensor>& upstream) {
  check_logits(logits, labels);
  one_device(logits, stats, slopes, upstream);
  const bool per_token = slopes.dim() == 2;
  TORCH_CHECK(slopes.is_contiguous() && slopes.scalar_type() == at::kFloat && slopes.size(0) == logits.size(0) &&
                  (!per_token || slopes.size(1) == logits.size(1)) && stats.is_contiguous() &&
                  stats.scalar_type() == at::kFloat && stats.numel() == logits.size(0) * logits.size(1) * 4,
              "rocm_qlora: slopes must be contiguous [batch] or [batch, length] float32");
  if (upstream) TORCH_CHECK(upstream->numel() == 1 && upstream->scalar_type() == at::kFloat, "rocm_qlora: upstream must be one float32");
  Tensor d = at::empty({logits.size(0), logits.size(1), logits.size(2)}, logits.options());
  if (logits.is_meta()) return d;
  const c10::cuda::CUDAGuard guard(logits.device());
  check(rq_token_logprobs_grad(logits.data_ptr(), dtype_code(logits.scalar_type()), logits.stride(0), logits.stride(1),
                               logits.size(0), logits.size(1), logits.size(2), labels.data_ptr<int64_t>(), ignore,
                               stats.data_ptr<float>(), slopes.data_ptr<float>(), per_token,
                               static_cast<const float*>(ptr(upstream)), d.data_ptr(), stream_of(logits)),
        "rq_token_logprobs_grad");
  return d;
}

// ---- the differentiable entry points: one dispatcher call forward, and a
// backward that never enters Python

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

using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

void once(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), "rocm_qlora: ", what, " is differentiable once only");
}

// t as [rows, columns]: contiguous columns, rows apart or one row for all; a
// copy where its strides are others (rows that overlap among them).
Tensor rows_of(const Tensor& t) {
  Tensor r = t.dim() == 2 ? t : t.reshape({c10::multiply_integers(t.sizes().slice(0, t.dim() - 1)), t.size(-1)});
  const bool columns = r.size(1) <= 1 || r.stride(1) == 1;
  const bool rows = r.size(0) <= 1 || r.stride(0) == 0 || r.stride(0) >= r.size(1);
  return columns && rows ? r : r.contiguous();
}

optional<Tensor> some(const Tensor& t) { return t.defined() ? optional<Tensor>(t) : std::nullopt; }

struct AdaptersAdd : Function<AdaptersAdd> {
  static Tensor forward(AutogradContext* ctx, const Tensor& base, const Tensor& x, const Tensor& A, const Tensor& B,
                        const Tensor& scaling, const optional<Tensor>& plan, int64_t tile,
                        const optional<Tensor>& codes, const optional<Tensor>& scales) {
    auto [y, mid] = RQ_VIA(adapters_apply, x, A, B, scaling, base, plan, tile);
    // x, or its packed form, is for A's gradient alone
    const bool keep = A.requires_grad(), packed = codes.has_value();
    ctx->save_for_backward({!keep ? Tensor() : packed ? *codes : x, keep && packed ? *scales : Tensor(), A, B, scaling,
                            mid, plan.value_or(Tensor())});
    ctx->saved_data["tile"] = tile;
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("adapters_add");
    const auto v = ctx->get_saved_variables();
    const Tensor &z = v[0], &A = v[2], &B = v[3], &scaling = v[4], &mid = v[5];
    const optional<Tensor> scales = some(v[1]), plan = some(v[6]);
    const int64_t tile = ctx->saved_data["tile"].toInt();
    const Tensor dy = rows_of(grads[0]);
    Tensor dx, dA, dB, gmid;
    if (ctx->needs_input_grad(1)) std::tie(dx, gmid) = RQ_VIA(adapters_apply, dy, B, A, scaling, std::nullopt, plan, tile);
    else if (ctx->needs_input_grad(2)) gmid = RQ_VIA(adapters_mid, dy, B, A, scaling, plan, tile);
    if (ctx->needs_input_grad(2)) dA = RQ_VIA(adapters_grad, z, scales, gmid, A.size(1), A.size(0), A.scalar_type(), plan, tile);
    if (ctx->needs_input_grad(3)) dB = RQ_VIA(adapters_grad, dy, std::nullopt, mid, B.size(1), B.size(0), B.scalar_type(), plan, tile);
    return {ctx->needs_input_grad(0) ? grads[0] : Tensor(), dx, dA, dB, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

void check_float(at::ScalarType t) {
  TORCH_CHECK_TYPE(t == at::kFloat || t == at::kBFloat16 || t == at::kHalf, "unsupported dtype ", t,
                   "; rocm_qlora kernels take float32, bfloat16 or float16");
}

void check_gpu(std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors) {
    TORCH_CHECK_NOT_IMPLEMENTED(!t->is_cpu(), "rocm_qlora (B200 build) computes on the GPU only: move the tensors to a CUDA device");
    TORCH_CHECK(t->device() == (*tensors.begin())->device(), "tensors are on different devices: ",
                (*tensors.begin())->device(), " and ", t->device());
  }
}

std::string sizes_of(const Tensor& t) { return c10::str(t.sizes()); }

// What a caller can get wrong, as Python's ValueError and TypeError; tensors
// off the GPU as NotImplementedError.
void check_add(const Tensor& base, const Tensor& x, const Tensor& A, const Tensor& B, const Tensor& scaling,
               const optional<Tensor>& plan, int64_t plan_rows, int64_t plan_count, const optional<Tensor>& codes,
               const optional<Tensor>& scales) {
  const auto dt = x.scalar_type();
  TORCH_CHECK_TYPE(dt == at::kBFloat16 || dt == at::kHalf, "adapters take bfloat16 or float16 activations, got ", dt);
  TORCH_CHECK_VALUE(A.dim() == 3 && B.dim() == 3 && A.size(0) == B.size(0) && A.size(2) == B.size(2),
                    "A must be [count, in, rank] and B [count, out, rank]; got ", sizes_of(A), ", ", sizes_of(B));
  TORCH_CHECK_TYPE(A.scalar_type() == dt && B.scalar_type() == dt, "adapters are ", A.scalar_type(), " and ",
                   B.scalar_type(), ", activations ", dt);
  const int64_t count = A.size(0), r = A.size(2);
  TORCH_CHECK_VALUE(r % 8 == 0 && r >= 8 && r <= 128, "rank must be a multiple of 8 up to 128, got ", r,
                    " (AdapterBank pads)");
  TORCH_CHECK_VALUE(count >= 1 && count <= RQ_ADAPTERS_MAX, "a bank holds 1 to ", RQ_ADAPTERS_MAX, " adapters, got ", count);
  TORCH_CHECK_VALUE(scaling.dim() == 1 && scaling.size(0) == count && scaling.scalar_type() == at::kFloat,
                    "scaling must be float32 [", count, "], got ", scaling.scalar_type(), " ", sizes_of(scaling));
  TORCH_CHECK_VALUE(x.dim() >= 1 && base.dim() == x.dim() && x.size(-1) == A.size(1) && base.size(-1) == B.size(1),
                    "base ", sizes_of(base), " and x ", sizes_of(x), " do not fit A ", sizes_of(A), " and B ", sizes_of(B));
  int64_t rows = 1;
  for (int64_t i = 0; i + 1 < x.dim(); ++i) {
    TORCH_CHECK_VALUE(x.size(i) == base.size(i), "base is ", sizes_of(base), ", x ", sizes_of(x));
    rows *= x.size(i);
  }
  TORCH_CHECK_TYPE(base.scalar_type() == dt, "base is ", base.scalar_type(), ", x ", dt);
  TORCH_CHECK_VALUE(plan || count == 1, "a bank of several adapters needs a plan");
  TORCH_CHECK_VALUE(!plan || plan_ok(*plan), "plan must be a contiguous 1-D int32 tensor: the data of an AdapterPlan");
  TORCH_CHECK_VALUE(!plan || (plan_rows == rows && plan_count == count), "the plan is for ", plan_rows, " rows and ",
                    plan_count, " adapters, not ", rows, " and ", count);
  if (codes) {
    const int64_t nb = (A.size(1) + RQ_ACT8_BLOCK - 1) / RQ_ACT8_BLOCK;
    TORCH_CHECK_VALUE(scales && codes->dim() == 2 && codes->size(0) == rows && codes->size(1) == nb * RQ_ACT8_BLOCK &&
                          scales->dim() == 2 && scales->size(0) == rows && scales->size(1) == nb,
                      "packed_x does not belong to x ", sizes_of(x));
    TORCH_CHECK_VALUE(codes->scalar_type() == at::kChar && scales->scalar_type() == at::kFloat &&
                          codes->is_contiguous() && scales->is_contiguous(),
                      "packed_x holds contiguous int8 codes and float32 scales, got ", codes->scalar_type(), " and ",
                      scales->scalar_type());
  }
  check_gpu({&x, &base, &A, &B, &scaling, plan ? &*plan : &x, codes ? &*codes : &x, codes ? &*scales : &x});
}

Tensor adapters_add(const Tensor& base, const Tensor& x, const Tensor& A, const Tensor& B, const Tensor& scaling,
                    const optional<Tensor>& plan, int64_t plan_rows, int64_t plan_count, int64_t tile,
                    const optional<Tensor>& codes, const optional<Tensor>& scales) {
  check_add(base, x, A, B, scaling, plan, plan_rows, plan_count, codes, scales);
  const Tensor b2 = rows_of(base), x2 = rows_of(x), a3 = A.contiguous(), b3 = B.contiguous(), s1 = scaling.contiguous();
  TORCH_CHECK_VALUE(!scaling.requires_grad(), "scaling has no gradient: fold a trainable factor into A or B");
  bool grad = at::GradMode::is_enabled() &&
              (base.requires_grad() || x.requires_grad() || A.requires_grad() || B.requires_grad());
  // a tangent of forward-mode differentiation goes to the autograd node too, which refuses it
  for (const Tensor* t : {&base, &x, &A, &B, &scaling}) grad |= t->_fw_grad(/*level=*/0).defined();
  Tensor y;
  if (grad) {
    y = AdaptersAdd::apply(b2, x2, a3, b3, s1, plan, tile, codes, scales);
  } else {  // serving: nothing is kept
    y = RQ_VIA(adapters_product, x2, a3, b3, s1, b2, plan, tile);
  }
  return base.dim() == 2 ? y : y.view(base.sizes());
}

struct Swiglu8 : Function<Swiglu8> {
  static variable_list forward(AutogradContext* ctx, const Tensor& gate, const Tensor& up, int64_t copies) {
    auto [h, codes, scales] = RQ_VIA(swiglu8_forward, rows_of(gate), rows_of(up), copies);
    ctx->save_for_backward({codes, scales});  // a third copy (of h) is in the same storage in any case
    ctx->saved_data["shape"] = gate.sizes().vec();
    ctx->mark_non_differentiable({codes, scales});
    ctx->set_materialize_grads(false);  // no zeros in the place of the codes' gradient
    return {h.view(gate.sizes()), codes, scales};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("swiglu8");
    const auto v = ctx->get_saved_variables();
    const auto shape = ctx->saved_data["shape"].toIntVector();
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor()};
    auto [dgate, dup] = RQ_VIA(swiglu8_backward, rows_of(grads[0]), v[0], v[1]);
    return {dgate.view(shape), dup.view(shape), Tensor()};
  }
};

// h and, with copies = 3, the packed form of h
std::tuple<Tensor, optional<Tensor>, optional<Tensor>> swiglu8(const Tensor& gate, const Tensor& up, int64_t copies) {
  TORCH_CHECK_VALUE(gate.sizes() == up.sizes() && gate.scalar_type() == up.scalar_type(), "gate ", gate.sizes(), " ",
                    gate.scalar_type(), " and up ", up.sizes(), " ", up.scalar_type(), " differ");
  TORCH_CHECK_VALUE(gate.dim() >= 1, "swiglu8 needs at least one dimension");
  check_float(gate.scalar_type());
  check_gpu({&gate, &up});
  auto v = Swiglu8::apply(gate, up, copies);
  if (copies < 3) return {v[0], std::nullopt, std::nullopt};
  return {v[0], v[1].select(0, 2), v[2].select(0, 2)};
}

// The public forms of pack and unpack: any shape [..., K].
std::tuple<Tensor, Tensor> pack_activation(const Tensor& x) {
  TORCH_CHECK_VALUE(x.dim() >= 1, "pack_activation needs at least one dimension");
  check_float(x.scalar_type());
  check_gpu({&x});
  return RQ_VIA(act8_pack, rows_of(x.detach()));
}

Tensor unpack_activation(const Tensor& codes, const Tensor& scales, at::IntArrayRef shape, at::ScalarType dtype) {
  check_float(dtype);
  check_gpu({&codes, &scales});
  TORCH_CHECK_VALUE(!shape.empty(), "unpack_activation needs at least one dimension");
  Tensor out = RQ_VIA(act8_unpack, codes, scales, shape.back(), dtype);
  return shape.size() == 2 ? out : out.view(shape);
}

struct Preference : Function<Preference> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& labels, const Tensor& ref,
                               int64_t ignore, int64_t form, double beta, double smooth) {
    auto [loss, logps, rewards, slopes, stats] = RQ_VIA(preference_forward, logits, labels, ref, ignore, form, beta, smooth);
    ctx->save_for_backward({logits, labels, stats, slopes});
    ctx->saved_data["ignore"] = ignore;
    ctx->mark_non_differentiable({logps, rewards});
    ctx->set_materialize_grads(false);
    return {loss, logps, rewards};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("preference_loss");
    const auto v = ctx->get_saved_variables();
    Tensor d;
    if (grads[0].defined())
      d = RQ_VIA(token_logprobs_grad, v[0], v[1], ctx->saved_data["ignore"].toInt(), v[2], v[3], grads[0]);
    return {d, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// logits with a contiguous vocabulary and contiguous labels
std::pair<Tensor, Tensor> checked_logits(const Tensor& logits, const Tensor& labels) {
  TORCH_CHECK_VALUE(logits.dim() == 3 && labels.dim() == 2 && labels.size(0) == logits.size(0) &&
                        labels.size(1) == logits.size(1),
                    "logits must be [batch, length, vocabulary] and labels [batch, length]; got ", logits.sizes(),
                    " and ", labels.sizes());
  TORCH_CHECK_TYPE(labels.scalar_type() == at::kLong, "labels must be int64, got ", labels.scalar_type());
  TORCH_CHECK_VALUE(logits.size(2) >= 1, "the vocabulary is empty");
  check_float(logits.scalar_type());
  return {logits.stride(2) == 1 || logits.size(2) == 1 ? logits : logits.contiguous(), labels.contiguous()};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> preference_loss(const Tensor& logits, const Tensor& labels,
                                                           const Tensor& ref, int64_t ignore, int64_t form,
                                                           double beta, double smooth) {
  const auto [x, y] = checked_logits(logits, labels);
  const int64_t B = x.size(0);
  TORCH_CHECK_VALUE(B >= 2 && B % 2 == 0 && x.size(1) >= 1, "a batch holds pairs (chosen, then rejected): got ", B,
                    " sequences");
  TORCH_CHECK_VALUE(ref.sizes() == y.sizes(), "ref_logps must be [batch, length] like labels, got ", ref.sizes());
  check_gpu({&logits, &labels, &ref});
  auto v = Preference::apply(x, y, ref.detach().to(at::kFloat).contiguous(), ignore, form, beta, smooth);
  return {v[0], v[1], v[2].narrow(0, 0, B / 2), v[2].narrow(0, B / 2, B / 2)};
}

struct LabelLogprobs : Function<LabelLogprobs> {
  static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& labels, int64_t ignore) {
    auto [logps, stats] = RQ_VIA(token_logprobs, logits, labels, ignore);
    ctx->save_for_backward({logits, labels, stats});
    ctx->saved_data["ignore"] = ignore;
    return logps;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("token_logprobs");
    const auto v = ctx->get_saved_variables();
    return {RQ_VIA(token_logprobs_grad, v[0], v[1], ctx->saved_data["ignore"].toInt(), v[2], grads[0].contiguous(), std::nullopt),
            Tensor(), Tensor()};
  }
};

Tensor label_logprobs(const Tensor& logits, const Tensor& labels, int64_t ignore) {
  const auto [x, y] = checked_logits(logits, labels);
  check_gpu({&logits, &labels});
  return LabelLogprobs::apply(x, y, ignore);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(rocm_qlora, m) {
  m.def("adapter_plan(Tensor ids, int count, int tile) -> Tensor");
  m.def(
      "adapters_apply(Tensor inp, Tensor u, Tensor v, Tensor scaling, Tensor? base, Tensor? plan, int tile) "
      "-> (Tensor, Tensor)");
  m.def(
      "adapters_apply_(Tensor(a!) out, Tensor inp, Tensor u, Tensor v, Tensor scaling, Tensor base, Tensor? plan, "
      "int tile) -> Tensor");
  m.def("adapters_product(Tensor inp, Tensor u, Tensor v, Tensor scaling, Tensor base, Tensor? plan, int tile) -> Tensor");
  m.def("adapters_mid(Tensor inp, Tensor u, Tensor v, Tensor scaling, Tensor? plan, int tile) -> Tensor");
  m.def(
      "adapters_grad(Tensor z, Tensor? scales, Tensor mid, int columns, int count, ScalarType dtype, Tensor? plan, "
      "int tile) -> Tensor");
  m.def("act8_pack(Tensor x) -> (Tensor, Tensor)");
  m.def("act8_unpack(Tensor codes, Tensor scales, int columns, ScalarType dtype) -> Tensor");
  m.def("swiglu8_forward(Tensor gate, Tensor up, int copies) -> (Tensor, Tensor, Tensor)");
  m.def("swiglu8_backward(Tensor dh, Tensor codes, Tensor scales) -> (Tensor, Tensor)");
  m.def("token_logprobs(Tensor logits, Tensor labels, int ignore) -> (Tensor, Tensor)");
  m.def(
      "preference_forward(Tensor logits, Tensor labels, Tensor ref, int ignore, int form, float beta, float smooth) "
      "-> (Tensor, Tensor, Tensor, Tensor, Tensor)");
  m.def(
      "token_logprobs_grad(Tensor logits, Tensor labels, int ignore, Tensor stats, Tensor slopes, Tensor? upstream) "
      "-> Tensor");
  m.def(
      "adapters_add(Tensor base, Tensor x, Tensor a, Tensor b, Tensor scaling, Tensor? plan, int plan_rows, "
      "int plan_count, int tile, Tensor? codes, Tensor? scales) -> Tensor", &adapters_add);
  m.def("swiglu8(Tensor gate, Tensor up, int copies) -> (Tensor, Tensor?, Tensor?)", &swiglu8);
  m.def("pack_activation(Tensor x) -> (Tensor, Tensor)", &pack_activation);
  m.def("unpack_activation(Tensor codes, Tensor scales, int[] shape, ScalarType dtype) -> Tensor", &unpack_activation);
  m.def(
      "preference_loss(Tensor logits, Tensor labels, Tensor ref, int ignore, int form, float beta, float smooth) "
      "-> (Tensor, Tensor, Tensor, Tensor)", &preference_loss);
  m.def("label_logprobs(Tensor logits, Tensor labels, int ignore) -> Tensor", &label_logprobs);
}

#define RQ_IMPLS(m)                                          \
  m.impl("adapter_plan", &adapter_plan);                     \
  m.impl("adapters_apply", &adapters_apply);                 \
  m.impl("adapters_apply_", &adapters_apply_);               \
  m.impl("adapters_product", &adapters_product);             \
  m.impl("adapters_mid", &adapters_mid);                     \
  m.impl("adapters_grad", &adapters_grad);                   \
  m.impl("act8_pack", &act8_pack);                           \
  m.impl("act8_unpack", &act8_unpack);                       \
  m.impl("swiglu8_forward", &swiglu8_forward);               \
  m.impl("swiglu8_backward", &swiglu8_backward);             \
  m.impl("token_logprobs", &token_logprobs);                 \
  m.impl("preference_forward", &preference_forward);         \
  m.impl("token_logprobs_grad", &token_logprobs_grad)

TORCH_LIBRARY_IMPL(rocm_qlora, CUDA, m) { RQ_IMPLS(m); }
TORCH_LIBRARY_IMPL(rocm_qlora, Meta, m) { RQ_IMPLS(m); }
TORCH_LIBRARY_IMPL(rocm_qlora, ADInplaceOrView, m) { m.impl("adapters_apply_", &adapters_apply_versioned); }

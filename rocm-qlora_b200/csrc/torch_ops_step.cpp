// torch_ops_step.cpp -- torch operators of microscaled 4-bit values and their
// products, of the gradient norm, and the AdamW step over many tensors
// (include/rq_b200.h).  As in torch_ops_train.cpp: outputs are allocated here,
// launches go to torch's current stream of the input's device, a status other
// than RQ_OK raises, and nothing is computed.
#include "torch_ops.h"

#include <torch/csrc/autograd/VariableTypeUtils.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/custom_class.h>

#include <array>
#include <tuple>
#include <vector>

namespace {

using namespace rq_torch;

// ------------------------------------------------- microscaled 4-bit values

int64_t pitch_of(int64_t K) { return (K + 127) / 128 * 128; }

void check_rows(const Tensor& t, const char* name) {
  TORCH_CHECK(t.dim() == 2 && (t.size(1) <= 1 || t.stride(1) == 1), "rocm_qlora: ", name,
              " must be a 2-D tensor with contiguous columns");
}

// What mx4_pack writes for rows of K values.
void check_packed(const Tensor& codes, const Tensor& scales, int64_t K) {
  one_device(codes, scales);
  TORCH_CHECK_VALUE(codes.dim() == 2 && scales.dim() == 3 && codes.scalar_type() == at::kByte &&
                        scales.scalar_type() == at::kByte && codes.is_contiguous() && scales.is_contiguous() &&
                        K >= 1 && codes.size(1) == pitch_of(K) / 2 && scales.size(0) == (codes.size(0) + 127) / 128 &&
                        scales.size(1) == pitch_of(K) / 128 && scales.size(2) == 512,
                    "not the packed 4-bit form of rows of ", K, " values");
}

std::tuple<Tensor, Tensor> mx4_pack(const Tensor& x) {
  check_rows(x, "x");
  const int64_t M = x.size(0), K = x.size(1), pitch = pitch_of(K);
  const auto bytes = x.options().dtype(at::kByte);
  Tensor codes = at::empty({M, pitch / 2}, bytes), scales = at::empty({(M + 127) / 128, pitch / 128, 512}, bytes);
  if (x.is_meta() || x.numel() == 0) return {codes, scales};
  const c10::cuda::CUDAGuard guard(x.device());
  check(rq_mx4_pack(x.data_ptr(), dtype_code(x.scalar_type()), x.stride(0), M, K, codes.data_ptr<uint8_t>(),
                    scales.data_ptr<uint8_t>(), stream_of(x)),
        "rq_mx4_pack");
  return {codes, scales};
}

Tensor mx4_unpack(const Tensor& codes, const Tensor& scales, int64_t K, at::ScalarType dtype) {
  check_packed(codes, scales, K);
  Tensor out = at::empty({codes.size(0), K}, codes.options().dtype(dtype));
  if (codes.is_meta()) return out;
  const c10::cuda::CUDAGuard guard(codes.device());
  const Tensor c = aligned(codes), s = aligned(scales);
  check(rq_mx4_unpack(c.data_ptr<uint8_t>(), s.data_ptr<uint8_t>(), codes.size(0), K, out.data_ptr(),
                      dtype_code(dtype), stream_of(codes)),
        "rq_mx4_unpack");
  return out;
}

Tensor mx4_product(const Tensor& a_codes, const Tensor& a_scales, const Tensor& b_codes, const Tensor& b_scales,
                   int64_t K, const optional<Tensor>& bias, at::ScalarType dtype) {
  check_packed(a_codes, a_scales, K);
  check_packed(b_codes, b_scales, K);
  one_device(a_codes, b_codes, bias);
  const int64_t M = a_codes.size(0), N = b_codes.size(0);
  Tensor out = at::empty({M, N}, a_codes.options().dtype(dtype));
  if (out.is_meta()) return out;
  const c10::cuda::CUDAGuard guard(a_codes.device());
  const Tensor ac = aligned(a_codes), as = aligned(a_scales), bc = aligned(b_codes), bs = aligned(b_scales);
  check(rq_mx4_matmul(ac.data_ptr<uint8_t>(), as.data_ptr<uint8_t>(), M, bc.data_ptr<uint8_t>(),
                      bs.data_ptr<uint8_t>(), N, K, ptr(bias), out.data_ptr(), dtype_code(dtype), stream_of(out)),
        "rq_mx4_matmul");
  return out;
}

Tensor mx4_forward(const Tensor& x, const Tensor& codes, const Tensor& scales, const optional<Tensor>& bias) {
  check_rows(x, "x");
  check_packed(codes, scales, x.size(1));
  one_device(x, codes, bias);
  const int64_t M = x.size(0), N = codes.size(0), K = x.size(1);
  Tensor out = at::empty({M, N}, x.options());
  if (out.is_meta() || out.numel() == 0) return out;
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t need = rq_mx4_linear_workspace_bytes(M, N, K);
  TORCH_CHECK(need >= 0, "rocm_qlora: no product of [", M, ", ", K, "] and [", N, ", ", K, "]");
  Tensor ws;  // one token's rows need none
  if (need > 0) ws = at::empty({need}, codes.options());
  const Tensor c = aligned(codes), s = aligned(scales);
  check(rq_mx4_linear(x.data_ptr(), dtype_code(x.scalar_type()), x.stride(0), M, c.data_ptr<uint8_t>(),
                      s.data_ptr<uint8_t>(), N, K, ptr(bias), out.data_ptr(), need > 0 ? ws.data_ptr() : nullptr, need, stream_of(x)),
        "rq_mx4_linear");
  return out;
}

Tensor mx4_dx(const Tensor& dy, const Tensor& codes, const Tensor& scales, int64_t K) {
  check_rows(dy, "dy");
  check_packed(codes, scales, K);
  one_device(dy, codes);
  TORCH_CHECK_VALUE(dy.size(1) == codes.size(0), "dy must have a column for each of the ", codes.size(0), " rows packed");
  const int64_t M = dy.size(0), N = dy.size(1);
  if (N == 0) return at::zeros({M, K}, dy.options());
  Tensor dx = at::empty({M, K}, dy.options());
  if (dx.is_meta() || M == 0) return dx;
  const c10::cuda::CUDAGuard guard(dy.device());
  Tensor d = dy;
  if (d.stride(0) % 8 || d.stride(0) < N || (uintptr_t)d.data_ptr() % 16) {  // rows as the tensor maps take them
    d = at::empty({M, (N + 7) / 8 * 8}, dy.options()).narrow(1, 0, N);
    check(rq_align_rows(dy.data_ptr(), dy.stride(0), M, N, d.data_ptr(), d.stride(0), stream_of(dy)), "rq_align_rows");
  }
  const Tensor c = aligned(codes), s = aligned(scales);
  Tensor ws;
  if (dy.scalar_type() == at::kHalf) ws = at::empty({RQ_MX4_DX_WORKSPACE}, codes.options());
  check(rq_mx4_dx(d.data_ptr(), dtype_code(d.scalar_type()), d.stride(0), M, c.data_ptr<uint8_t>(),
                  s.data_ptr<uint8_t>(), N, K, dx.data_ptr(), ws.defined() ? ws.data_ptr() : nullptr,
                  RQ_MX4_DX_WORKSPACE, stream_of(dy)),
        "rq_mx4_dx");
  return dx;
}

using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;

// The rounding of x is passed through: dx = dy . w.
struct Mx4Linear : Function<Mx4Linear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& codes, const Tensor& scales,
                        const optional<Tensor>& bias) {
    ctx->save_for_backward({codes, scales});
    ctx->saved_data["K"] = x.size(1);
    return RQ_VIA(mx4_forward, x, codes, scales, bias);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    once("mx4_linear");
    const auto v = ctx->get_saved_variables();
    return {RQ_VIA(mx4_dx, rows_of(grads[0]), v[0], v[1], ctx->saved_data["K"].toInt()), Tensor(), Tensor(), Tensor()};
  }
};

void check_half(at::ScalarType t, const char* what) {
  TORCH_CHECK_TYPE(t == at::kBFloat16 || t == at::kHalf, what, " takes bfloat16 or float16, got ", t);
}

void check_bias(const optional<Tensor>& bias, int64_t N, at::ScalarType dtype) {
  if (!bias) return;
  TORCH_CHECK_VALUE(bias->dim() == 1 && bias->size(0) == N, "bias must be [", N, "], got ", bias->sizes());
  TORCH_CHECK_TYPE(bias->scalar_type() == dtype, "bias is ", bias->scalar_type(), ", the result ", dtype);
  TORCH_CHECK_VALUE(!bias->requires_grad(), "the frozen projection's bias has no gradient");
}

// The public forms: any shape [..., K].
std::tuple<Tensor, Tensor> pack_mx4(const Tensor& x) {
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1, "pack_mx4 needs rows of at least one value, got ", x.sizes());
  check_float(x.scalar_type());
  check_gpu({&x});
  return RQ_VIA(mx4_pack, rows_of(x.detach()));
}

Tensor unpack_mx4(const Tensor& codes, const Tensor& scales, at::IntArrayRef shape, at::ScalarType dtype) {
  check_float(dtype);
  check_gpu({&codes, &scales});
  TORCH_CHECK_VALUE(!shape.empty(), "unpack_mx4 needs at least one dimension");
  TORCH_CHECK_VALUE(codes.dim() == 2 && c10::multiply_integers(shape.slice(0, shape.size() - 1)) == codes.size(0),
                    "shape ", shape, " does not have the rows of codes ", codes.sizes());
  Tensor out = RQ_VIA(mx4_unpack, codes, scales, shape.back(), dtype);
  return shape.size() == 2 ? out : out.view(shape);
}

Tensor mx4_matmul(const Tensor& a_codes, const Tensor& a_scales, const Tensor& b_codes, const Tensor& b_scales,
                  int64_t K, const optional<Tensor>& bias, at::ScalarType dtype) {
  check_half(dtype, "mx4_matmul");
  check_gpu({&a_codes, &a_scales, &b_codes, &b_scales, bias ? &*bias : &a_codes});
  check_bias(bias, b_codes.size(0), dtype);
  return RQ_VIA(mx4_product, a_codes, a_scales, b_codes, b_scales, K, bias ? optional<Tensor>(bias->contiguous()) : bias,
                dtype);
}

Tensor mx4_linear(const Tensor& x, const Tensor& codes, const Tensor& scales, int64_t K, const optional<Tensor>& bias) {
  check_half(x.scalar_type(), "mx4_linear");
  TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) == K, "x ", x.sizes(), " does not fit a weight of rows of ", K, " values");
  check_bias(bias, codes.size(0), x.scalar_type());
  check_gpu({&x, &codes, &scales, bias ? &*bias : &x});
  const Tensor x2 = rows_of(x);
  const optional<Tensor> b = bias ? optional<Tensor>(bias->contiguous()) : bias;
  // a tangent of forward-mode differentiation goes to the autograd node too, which refuses it
  const bool grad = (at::GradMode::is_enabled() && x.requires_grad()) || x._fw_grad(/*level=*/0).defined();
  const Tensor y = grad ? Mx4Linear::apply(x2, codes, scales, b) : RQ_VIA(mx4_forward, x2, codes, scales, b);
  if (x.dim() == 2) return y;
  auto shape = x.sizes().vec();
  shape.back() = codes.size(0);
  return y.view(shape);
}

// --------------------------------------------------- norm and AdamW step

// Tensors of one dtype in the kernels' form; contiguous copies stay alive
// until the launches are out.
struct Lists {
  std::array<std::vector<RqAdamTensor>, 3> by;
  std::vector<Tensor> keep;
};

template <class F>
void in_launches(const Lists& lists, F&& launch) {
  for (int dt = 0; dt < 3; ++dt) {
    const auto& v = lists.by[dt];
    for (size_t at = 0; at < v.size(); at += RQ_ADAM_TENSORS)
      launch(v.data() + at, (int)std::min<size_t>(RQ_ADAM_TENSORS, v.size() - at), dt);
  }
}

int64_t launches_of(const Lists& lists) {
  int64_t n = 0;
  in_launches(lists, [&](const RqAdamTensor*, int, int) { ++n; });
  return n;
}

Tensor norm_of(at::TensorList tensors) {
  Lists lists;
  const Tensor& first = tensors[0];
  for (const Tensor& t : tensors) {
    one_device(first, t);
    if (t.numel() == 0) continue;
    lists.keep.push_back(t.is_non_overlapping_and_dense() ? t : t.contiguous());  // any order of the values
    lists.by[dtype_code(t.scalar_type())].push_back(
        RqAdamTensor{nullptr, t.is_meta() ? nullptr : lists.keep.back().data_ptr(), t.numel(), 0, 0});
  }
  Tensor norm = at::empty({}, first.options().dtype(at::kFloat));
  if (first.is_meta()) return norm;
  const c10::cuda::CUDAGuard guard(first.device());
  const cudaStream_t st = stream_of(first);
  const int64_t n = launches_of(lists);
  Tensor partials = at::empty({n * RQ_NORM_PARTIALS}, first.options().dtype(at::kDouble));
  double* at_partials = partials.data_ptr<double>();
  in_launches(lists, [&](const RqAdamTensor* list, int count, int dt) {
    check(rq_grad_norm_partial(list, count, dt, at_partials, st), "rq_grad_norm_partial");
    at_partials += RQ_NORM_PARTIALS;
  });
  check(rq_grad_norm_end(partials.data_ptr<double>(), (int)(n * RQ_NORM_PARTIALS), norm.data_ptr<float>(), st),
        "rq_grad_norm_end");
  return norm;
}

Tensor grad_norm(at::TensorList tensors) {
  TORCH_CHECK_VALUE(!tensors.empty(), "grad_norm needs at least one tensor");
  for (const Tensor& t : tensors) {
    check_float(t.scalar_type());
    TORCH_CHECK_VALUE(t.layout() == at::kStrided, "grad_norm takes dense tensors");
    check_gpu({&tensors[0], &t});
  }
  return RQ_VIA(norm_of, tensors);
}

// The tensors of one parameter group and its arenas.
struct AdamGroup {
  std::vector<Tensor> params;
  std::vector<int64_t> blocks;  // first block of each
  Tensor m, v, scales, low, steps, ticket;
};

// Held by the optimizer, so that a step is one call whatever the number of
// parameters: their gradients are looked up here.
struct AdamW : torch::CustomClassHolder {
  std::vector<AdamGroup> groups;
  int bits;
  explicit AdamW(int64_t bits) : bits((int)bits) {
    TORCH_CHECK_VALUE(bits == 8 || bits == 32, "state_bits must be 8 or 32, got ", bits);
  }

  void add_group(std::vector<Tensor> params, Tensor m, Tensor v, optional<Tensor> scales, optional<Tensor> low,
                 Tensor steps, Tensor ticket) {
    AdamGroup g{std::move(params), {}, m, v, scales.value_or(Tensor()), low.value_or(Tensor()), steps, ticket};
    int64_t at = 0;
    for (const Tensor& p : g.params) {
      g.blocks.push_back(at);
      at += (p.numel() + RQ_ADAM_BLOCK - 1) / RQ_ADAM_BLOCK;
    }
    const auto of = bits == 8 ? at::kByte : at::kFloat;
    one_device(m, v, scales, low, steps, ticket);
    TORCH_CHECK_VALUE(m.numel() == at * RQ_ADAM_BLOCK && v.numel() == m.numel() && m.is_contiguous() &&
                          v.is_contiguous() && m.scalar_type() == of && v.scalar_type() == of &&
                          (bits == 32 || (g.scales.defined() && g.scales.is_contiguous() && g.scales.numel() == 2 * at &&
                                          g.scales.scalar_type() == at::kFloat)) &&
                          (!g.low.defined() || (g.low.is_contiguous() && g.low.numel() == m.numel() &&
                                                g.low.scalar_type() == at::kShort)) &&
                          steps.is_contiguous() && steps.scalar_type() == at::kInt &&
                          steps.numel() == (int64_t)g.params.size() && ticket.numel() == 1 &&
                          ticket.scalar_type() == at::kInt,
                      "the arenas do not fit the parameters");
    groups.push_back(std::move(g));
  }

  Lists gather(const AdamGroup& g) const {
    Lists lists;
    for (size_t i = 0; i < g.params.size(); ++i) {
      const Tensor& p = g.params[i];
      const Tensor& grad = p.grad();
      if (!grad.defined()) continue;
      TORCH_CHECK_VALUE(grad.layout() == at::kStrided, "AdamW takes dense gradients");
      TORCH_CHECK(p.device() == g.m.device() && grad.device() == g.m.device(), "a parameter or its gradient is on ",
                  p.device(), " and ", grad.device(), ", the optimizer's state on ", g.m.device());
      TORCH_CHECK_VALUE(p.is_contiguous(), "AdamW takes contiguous parameters");
      const int64_t room = (i + 1 < g.params.size() ? g.blocks[i + 1] : g.m.numel() / RQ_ADAM_BLOCK) - g.blocks[i];
      TORCH_CHECK_VALUE((p.numel() + RQ_ADAM_BLOCK - 1) / RQ_ADAM_BLOCK == room && grad.sizes() == p.sizes(),
                        "a parameter has another size than when the optimizer was made");
      check_float(p.scalar_type());
      TORCH_CHECK_TYPE(grad.scalar_type() == p.scalar_type(), "a parameter is ", p.scalar_type(), ", its gradient ",
                       grad.scalar_type());
      TORCH_CHECK_TYPE(!g.low.defined() || p.scalar_type() == at::kBFloat16,
                       "remainder keeps what bfloat16 parameters leave: a parameter is ", p.scalar_type());
      // a lazily negated view is stored with the other sign, whatever its strides
      const bool as_is = grad.is_contiguous() && !grad.is_neg();
      const Tensor flat = as_is ? grad : grad.resolve_neg().contiguous();
      if (!as_is) lists.keep.push_back(flat);
      lists.by[dtype_code(p.scalar_type())].push_back(
          RqAdamTensor{p.data_ptr(), flat.data_ptr(), p.numel(), g.blocks[i], (int32_t)i});
    }
    return lists;
  }

  // hyper: lr, beta1, beta2, eps, weight decay of each group; lrs: learning
  // rates on the device, where given; max_norm below 0: no clipping.
  void step(std::vector<double> hyper, std::vector<optional<Tensor>> lrs, double max_norm, Tensor norm) {
    TORCH_CHECK(hyper.size() == 5 * groups.size() && lrs.size() == groups.size(), "rocm_qlora: five numbers a group");
    if (groups.empty()) return;
    const Tensor& first = groups[0].m;
    std::vector<Lists> lists;
    int64_t launches = 0;
    // all is checked before the first launch: a refused step changes nothing
    for (const optional<Tensor>& lr : lrs)
      TORCH_CHECK_VALUE(!lr || (lr->numel() == 1 && lr->scalar_type() == at::kFloat && lr->device() == first.device()),
                        "a learning rate that is a tensor must be one float32 on the parameters' device");
    for (const AdamGroup& g : groups) {
      one_device(first, g.m);
      lists.push_back(gather(g));
      launches += launches_of(lists.back());
    }
    if (launches == 0) return;
    const c10::cuda::CUDAGuard guard(first.device());
    const cudaStream_t st = stream_of(first);
    const bool clip = max_norm >= 0.0;
    Tensor partials;
    int n = 0;
    if (clip) {
      TORCH_CHECK(norm.numel() == 1 && norm.scalar_type() == at::kFloat && norm.device() == first.device(),
                  "rocm_qlora: norm must be one float32 beside the state");
      partials = at::empty({launches * RQ_NORM_PARTIALS}, first.options().dtype(at::kDouble));
      for (const Lists& l : lists)
        in_launches(l, [&](const RqAdamTensor* list, int count, int dt) {
          check(rq_grad_norm_partial(list, count, dt, partials.data_ptr<double>() + n, st), "rq_grad_norm_partial");
          n += RQ_NORM_PARTIALS;
        });
    }
    for (size_t i = 0; i < groups.size(); ++i) {
      const AdamGroup& g = groups[i];
      const double* h = hyper.data() + 5 * i;
      RqAdamStep step = {};
      step.lr = h[0];
      step.beta1 = h[1];
      step.beta2 = h[2];
      step.eps = h[3];
      step.decay = h[4];
      step.lr_at = lrs[i] ? lrs[i]->data_ptr<float>() : nullptr;
      step.partials = clip ? partials.data_ptr<double>() : nullptr;
      step.n_partials = n;
      step.max_norm = (float)max_norm;
      step.norm = clip ? norm.data_ptr<float>() : nullptr;
      step.steps = g.steps.data_ptr<int32_t>();
      step.ticket = reinterpret_cast<uint32_t*>(g.ticket.data_ptr<int32_t>());
      in_launches(lists[i], [&](const RqAdamTensor* list, int count, int dt) {
        check(rq_adam_update(list, count, dt, bits, g.m.data_ptr(), g.v.data_ptr(),
                             bits == 8 ? g.scales.data_ptr<float>() : nullptr,
                             g.low.defined() ? g.low.data_ptr<int16_t>() : nullptr, &step, st),
              "rq_adam_update");
      });
    }
    for (const AdamGroup& g : groups)
      for (const Tensor& p : g.params)
        if (p.grad().defined()) torch::autograd::increment_version(p);
  }
};

std::tuple<Tensor, Tensor> adam_unpack(const Tensor& m8, const Tensor& r8, const Tensor& scales) {
  one_device(m8, r8, scales);
  TORCH_CHECK(m8.is_contiguous() && r8.is_contiguous() && scales.is_contiguous() && m8.scalar_type() == at::kByte &&
                  r8.scalar_type() == at::kByte && scales.scalar_type() == at::kFloat && m8.numel() == r8.numel() &&
                  scales.numel() * RQ_ADAM_BLOCK == 2 * m8.numel(),
              "rocm_qlora: not the 8-bit form of moments");
  Tensor m = at::empty({m8.numel()}, scales.options()), v = at::empty_like(m);
  if (m8.is_meta()) return {m, v};
  const c10::cuda::CUDAGuard guard(m8.device());
  check(rq_adam_unpack(m8.data_ptr<uint8_t>(), r8.data_ptr<uint8_t>(), scales.data_ptr<float>(),
                       m8.numel() / RQ_ADAM_BLOCK, m.data_ptr<float>(), v.data_ptr<float>(), stream_of(m8)),
        "rq_adam_unpack");
  return {m, v};
}

void adam_pack_(const Tensor& m, const Tensor& v, Tensor m8, Tensor r8, Tensor scales) {
  one_device(m, v, m8, r8, scales);
  TORCH_CHECK(m8.is_contiguous() && r8.is_contiguous() && scales.is_contiguous() && m8.scalar_type() == at::kByte &&
                  r8.scalar_type() == at::kByte && scales.scalar_type() == at::kFloat && m8.numel() == r8.numel() &&
                  scales.numel() * RQ_ADAM_BLOCK == 2 * m8.numel() && m.is_contiguous() && v.is_contiguous() &&
                  m.scalar_type() == at::kFloat && v.scalar_type() == at::kFloat && m.numel() == m8.numel() &&
                  v.numel() == m8.numel(),
              "rocm_qlora: not moments and their 8-bit form");
  if (m.is_meta()) return;
  const c10::cuda::CUDAGuard guard(m.device());
  const auto whole = [](const Tensor& t) { return (uintptr_t)t.data_ptr() % 32 ? t.clone() : t; };
  const Tensor m4 = whole(m), v4 = whole(v);
  check(rq_adam_pack(m4.data_ptr<float>(), v4.data_ptr<float>(), m8.numel() / RQ_ADAM_BLOCK, m8.data_ptr<uint8_t>(),
                     r8.data_ptr<uint8_t>(), scales.data_ptr<float>(), stream_of(m)),
        "rq_adam_pack");
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(rocm_qlora, m) {
  m.def("mx4_pack(Tensor x) -> (Tensor, Tensor)");
  m.def("mx4_unpack(Tensor codes, Tensor scales, int columns, ScalarType dtype) -> Tensor");
  m.def(
      "mx4_product(Tensor a_codes, Tensor a_scales, Tensor b_codes, Tensor b_scales, int columns, Tensor? bias, "
      "ScalarType dtype) -> Tensor");
  m.def("mx4_forward(Tensor x, Tensor codes, Tensor scales, Tensor? bias) -> Tensor");
  m.def("mx4_dx(Tensor dy, Tensor codes, Tensor scales, int columns) -> Tensor");
  m.def("norm_of(Tensor[] tensors) -> Tensor");
  m.def("grad_norm(Tensor[] tensors) -> Tensor", &grad_norm);
  m.def("adam_unpack(Tensor m, Tensor r, Tensor scales) -> (Tensor, Tensor)");
  m.def("adam_pack_(Tensor m, Tensor v, Tensor(a!) m8, Tensor(b!) r8, Tensor(c!) scales) -> ()");
  m.def("pack_mx4(Tensor x) -> (Tensor, Tensor)", &pack_mx4);
  m.def("unpack_mx4(Tensor codes, Tensor scales, int[] shape, ScalarType dtype) -> Tensor", &unpack_mx4);
  m.def(
      "mx4_matmul(Tensor a_codes, Tensor a_scales, Tensor b_codes, Tensor b_scales, int columns, Tensor? bias, "
      "ScalarType dtype) -> Tensor", &mx4_matmul);
  m.def("mx4_linear(Tensor x, Tensor codes, Tensor scales, int columns, Tensor? bias) -> Tensor", &mx4_linear);
  m.class_<AdamW>("AdamW")
      .def(torch::init<int64_t>())
      .def("add_group", &AdamW::add_group)
      .def("step", &AdamW::step);
}

#define RQ_IMPLS(m)                        \
  m.impl("mx4_pack", &mx4_pack);           \
  m.impl("mx4_unpack", &mx4_unpack);       \
  m.impl("mx4_product", &mx4_product);     \
  m.impl("mx4_forward", &mx4_forward);     \
  m.impl("mx4_dx", &mx4_dx);               \
  m.impl("norm_of", &norm_of);             \
  m.impl("adam_unpack", &adam_unpack);     \
  m.impl("adam_pack_", &adam_pack_)

TORCH_LIBRARY_IMPL(rocm_qlora, CUDA, m) { RQ_IMPLS(m); }
TORCH_LIBRARY_IMPL(rocm_qlora, Meta, m) { RQ_IMPLS(m); }

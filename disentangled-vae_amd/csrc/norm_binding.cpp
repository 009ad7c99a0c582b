// Argument checks, allocation and autograd node of the residual norm (hipvae._norm), on top of the C ABI.
//
// In C++ because the norm's smallest training calls are shorter than what a node written in Python costs: the autograd
// engine runs it in a thread of its own, which has to take the interpreter's lock and hand it back, and where idle cores
// sleep each of those turns wakes one up.  255 x 64 fp32, forward and backward: 66 us with a Python node, 47 with this; where
// idle cores sleep 126 and 78.  The same in elementary torch operations, without the engine: 91.
#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <ATen/ops/zeros.h>
#include <ATen/ops/zeros_like.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/utils/pybind.h>

#include "../../include/dvae_hip.h"

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// the library's entry points, as the Python binding has loaded them
static decltype(&dvae_add_rms_norm_fwd) norm_fwd;
static decltype(&dvae_add_rms_norm_q8) norm_q8;
static decltype(&dvae_add_rms_norm_bwd) norm_bwd;
static decltype(&dvae_add_rms_norm_bwd_ws_floats) norm_bwd_ws_floats;
static decltype(&dvae_last_error) last_error;

static void check(int rc, const char* what) {
  if (rc == 0) return;
  const char* e = last_error();
  TORCH_CHECK(false, what, " failed with code ", rc, ": ", e ? e : "");
}

static int code(const Tensor& t) { return t.scalar_type() == at::kFloat ? DVAE_DT_F32 : DVAE_DT_BF16; }
static dvae_stream_t stream_of(const Tensor& t) { return (dvae_stream_t)c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
static Tensor new_like(const Tensor& t) { return at::empty_like(t, t.options(), at::MemoryFormat::Contiguous); }

// a tensor [..., D] as rows of equal stride: copied only where its strides allow no such view
struct Rows {
  Tensor t;
  int64_t st = 0;
  Rows() {}
  Rows(const Tensor& a, int64_t D) : t(a), st(D) {
    if (!t.defined() || t.is_contiguous()) return;
    if (D > 1 && t.stride(-1) != 1) t = t.contiguous();
    else if (t.dim() != 2) t = t.reshape({-1, D});
    if (t.dim() == 2) st = t.stride(0);
  }
  const void* p() const { return t.defined() ? t.data_ptr() : nullptr; }
};

struct Args {
  Tensor x, weight;
  std::optional<Tensor> residual;
  Rows xr, rr;
  int64_t rows, D;
  int dtype, rdtype;

  Args(const char* what, const Tensor& x_, const std::optional<Tensor>& residual_, const Tensor& weight_)
      : x(x_), residual(residual_) {
    TORCH_CHECK(x.is_cuda(), what, ": input is on ", x.device(),
                "; hipvae ops need tensors on the GPU (no CPU path exists)");
    TORCH_CHECK(x.scalar_type() == at::kFloat || x.scalar_type() == at::kBFloat16, what,
                ": activations must be fp32 or bf16, got ", x.scalar_type());
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, what, ": expected [..., channels], got ", x.sizes());
    D = x.size(-1);
    rows = x.numel() / D;
    dtype = rdtype = code(x);
    if (residual) {                                    // of x's type, or fp32
      expect(what, "residual", *residual, x.sizes(), residual->scalar_type() == at::kFloat ? at::kFloat : x.scalar_type());
      rdtype = code(*residual);
      rr = Rows(*residual, D);
    }
    expect(what, "weight", weight_, {D}, at::kFloat);
    weight = weight_.contiguous();
    xr = Rows(x, D);
  }
  void expect(const char* what, const char* name, const Tensor& t, at::IntArrayRef shape, at::ScalarType type) const {
    TORCH_CHECK(t.sizes() == shape && t.scalar_type() == type && t.device() == x.device(), what, ": ", name, " is ",
                t.scalar_type(), " ", t.sizes(), " on ", t.device(), ", expected ", type, " ", shape, " on ", x.device());
  }
  Tensor new_sum() const { return residual ? new_like(*residual) : Tensor(); }
};

static std::pair<Tensor, Tensor> forward(const Args& a, double eps, const Tensor& rstd) {
  Tensor y = new_like(a.x), sum = a.new_sum();
  check(norm_fwd(a.xr.p(), a.xr.st, a.rr.p(), a.rr.st, a.weight.data_ptr<float>(), (float)eps, y.data_ptr(),
                 sum.defined() ? sum.data_ptr() : nullptr, rstd.defined() ? rstd.data_ptr<float>() : nullptr, a.rows, a.D,
                 a.dtype, a.rdtype, stream_of(a.x)),
        "add_rms_norm_fwd");
  return {y, sum};
}

struct AddRMSNorm : torch::autograd::Function<AddRMSNorm> {
  // -> {y, sum}, or {y} without a residual
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const std::optional<Tensor>& residual,
                               const Tensor& weight, double eps) {
    const Args a("add_rms_norm", x, residual, weight);
    const Tensor rstd = at::empty({a.rows}, a.weight.options());
    auto [y, sum] = ::forward(a, eps, rstd);
    ctx->save_for_backward({residual ? sum : x, a.weight, rstd});
    ctx->saved_data["bf16"] = x.scalar_type() == at::kBFloat16;
    ctx->set_materialize_grads(false);
    if (residual) return {y, sum};
    return {y};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(),
                "add_rms_norm: the gradients cannot be differentiated again (create_graph=True)");
    // (unpacking raises if one of them has been changed since; hooks may hand back other memory and strides)
    const variable_list saved = ctx->get_saved_variables();
    const bool residual = grads.size() == 2;
    Tensor dy = grads[0], dsum = residual ? grads[1] : Tensor();
    if (!dy.defined() && !dsum.defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const int64_t D = saved[0].size(-1);
    const Rows sum(saved[0], D);
    const Tensor weight = saved[1].contiguous(), rstd = saved[2].contiguous();
    const c10::DeviceGuard on(weight.device());
    const auto type = ctx->saved_data["bf16"].toBool() ? at::kBFloat16 : at::kFloat;
    if (!dy.defined()) dy = at::zeros(dsum.sizes(), dsum.options().dtype(type));
    const Rows g(dy, D), gs(dsum, D);
    const int64_t rows = dy.numel() / D;
    // Where the types are the same dx and dresidual are one tensor: autograd copies before it keeps either.
    const Tensor dres = new_like(saved[0]), dx = saved[0].scalar_type() == type ? dres : new_like(dy);
    if (rows == 0) return {dx, residual ? dres : Tensor(), at::zeros_like(weight), Tensor()};
    const Tensor dw = at::empty_like(weight), ws = at::empty({norm_bwd_ws_floats(rows, D)}, weight.options());
    check(norm_bwd(g.p(), g.st, gs.p(), gs.st, sum.p(), sum.st, weight.data_ptr<float>(), rstd.data_ptr<float>(),
                   dres.data_ptr(), dx.data_ptr(), dw.data_ptr<float>(), rows, D, type == at::kFloat ? DVAE_DT_F32 : DVAE_DT_BF16,
                   code(saved[0]), ws.data_ptr<float>(), stream_of(weight)),
          "add_rms_norm_bwd");
    return {dx, residual ? dres : Tensor(), dw, Tensor()};
  }
};

// -> y, and the sum where there is a residual
static std::tuple<Tensor, std::optional<Tensor>> add_rms_norm(const Tensor& x, const std::optional<Tensor>& residual,
                                                              const Tensor& weight, double eps) {
  const c10::DeviceGuard on(x.device());
  if (at::GradMode::is_enabled() &&
      (x.requires_grad() || weight.requires_grad() || (residual && residual->requires_grad()))) {
    const variable_list out = AddRMSNorm::apply(x, residual, weight, eps);
    return {out[0], residual ? std::optional<Tensor>(out[1]) : std::nullopt};
  }
  auto [y, sum] = forward(Args("add_rms_norm", x, residual, weight), eps, Tensor());
  return {y, residual ? std::optional<Tensor>(sum) : std::nullopt};
}

// -> q of type float8_e4m3fn, scale [...], and the sum where there is a residual
static std::tuple<Tensor, Tensor, std::optional<Tensor>> add_rms_norm_q8(const Tensor& x,
                                                                         const std::optional<Tensor>& residual,
                                                                         const Tensor& weight, double eps) {
  const c10::DeviceGuard on(x.device());
  const Args a("add_rms_norm_q8", x, residual, weight);
  const Tensor q = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn));
  const Tensor scale = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat)), sum = a.new_sum();
  check(norm_q8(a.xr.p(), a.xr.st, a.rr.p(), a.rr.st, a.weight.data_ptr<float>(), (float)eps, q.data_ptr(),
                scale.data_ptr<float>(), sum.defined() ? sum.data_ptr() : nullptr, a.rows, a.D, a.dtype, a.rdtype,
                stream_of(x)),
        "add_rms_norm_q8");
  return {q, scale, residual ? std::optional<Tensor>(sum) : std::nullopt};
}

PYBIND11_MODULE(_norm, m) {
  m.def("init", [](uintptr_t fwd, uintptr_t q8, uintptr_t bwd, uintptr_t ws_floats, uintptr_t error) {
    norm_fwd = (decltype(norm_fwd))fwd;
    norm_q8 = (decltype(norm_q8))q8;
    norm_bwd = (decltype(norm_bwd))bwd;
    norm_bwd_ws_floats = (decltype(norm_bwd_ws_floats))ws_floats;
    last_error = (decltype(last_error))error;
  });
  m.def("add_rms_norm", &add_rms_norm);
  m.def("add_rms_norm_q8", &add_rms_norm_q8);
}

// Host side of the normalisation: argument checks and the autograd node.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "host_common.h"
#include "norm.h"
#include "train_ops.h"

namespace sep {

namespace {

int type_of(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 ? kNormHalf : kNormFloat; }
bool usable(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat; }

int sms_of_current() { return at::cuda::getCurrentDeviceProperties()->multiProcessorCount; }

// `t` as rows of its last dimension, each contiguous and equally far apart; a copy where they do not lie so.
at::Tensor as_rows(const at::Tensor& t) {
  const int64_t H = t.size(-1);
  const at::Tensor m = t.dim() == 2 ? t : t.reshape({-1, H});
  return m.stride(1) == 1 || H == 1 ? m : m.contiguous();
}

struct NormCall : torch::CustomClassHolder {
  bool center;
  double eps;
};

struct NormResult { at::Tensor y, sum, stats; };

NormResult norm_forward(const NormCall& call, const at::Tensor& x, const at::Tensor& weight, const at::Tensor& bias, const at::Tensor& residual, bool keep) {
  NormResult out;
  out.y = at::empty(x.sizes(), x.options());
  if (residual.defined()) out.sum = at::empty(x.sizes(), x.options());
  const int64_t H = x.size(-1), rows = x.numel() / H;
  if (keep) out.stats = at::empty({rows, 2}, x.options().dtype(at::kFloat));
  if (rows == 0) return out;
  const at::Tensor xr = as_rows(x), w = weight.defined() ? weight.contiguous() : weight, b = bias.defined() ? bias.contiguous() : bias;
  NormParams p{};
  p.type = type_of(x); p.weight_type = w.defined() ? type_of(w) : b.defined() ? type_of(b) : kNormNone;
  p.center = call.center; p.rows = rows; p.hidden = static_cast<int>(H); p.eps = static_cast<float>(call.eps);
  p.x = xr.data_ptr(); p.x_stride = xr.stride(0);
  at::Tensor rr;
  if (residual.defined()) { rr = as_rows(residual); p.residual = rr.data_ptr(); p.residual_stride = rr.stride(0); p.sum = out.sum.data_ptr(); }
  p.weight = w.defined() ? w.data_ptr() : nullptr;
  p.bias = b.defined() ? b.data_ptr() : nullptr;
  p.y = out.y.data_ptr();
  p.stats = keep ? reinterpret_cast<float2*>(out.stats.data_ptr<float>()) : nullptr;
  SEP_CUDA_CHECK(launch_norm_forward(p, sms_of_current(), at::cuda::getCurrentCUDAStream()));
  return out;
}

class Norm : public torch::autograd::Function<Norm> {
 public:
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const std::optional<at::Tensor>& w,
                                                const std::optional<at::Tensor>& b, const std::optional<at::Tensor>& res, const c10::intrusive_ptr<NormCall>& call) {
    const at::Tensor weight = w.value_or(at::Tensor()), bias = b.value_or(at::Tensor()), residual = res.value_or(at::Tensor());
    NormResult r = norm_forward(*call, x, weight, bias, residual, true);
    ctx->save_for_backward({x, weight, r.stats, residual});
    ctx->saved_data["center"] = call->center;
    ctx->saved_data["bias"] = bias.defined() ? static_cast<int64_t>(type_of(bias)) : static_cast<int64_t>(kNormNone);
    ctx->set_materialize_grads(false);
    if (residual.defined()) return {r.y, r.sum};
    return {r.y};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    SEP_ASSERT(!at::GradMode::is_enabled(), "the normalisation has no second derivative: its backward was asked for a graph");
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &x = saved[0], &weight = saved[1], &stats = saved[2], &added = saved[3];
    const int bias_type = static_cast<int>(ctx->saved_data["bias"].toInt());
    const bool residual = added.defined();
    const at::Tensor dy = grads[0], dsum = residual ? grads[1] : at::Tensor();
    // (tensors that were left out have no edge in the graph)
    int edge = 1;
    const bool want_dw = weight.defined() && ctx->needs_input_grad(edge++), want_db = bias_type != kNormNone && ctx->needs_input_grad(edge++);
    const bool want_x = ctx->needs_input_grad(0), want_residual = residual && ctx->needs_input_grad(edge++), want_dx = want_x || want_residual;
    if (!dy.defined()) return {dsum, at::Tensor(), at::Tensor(), dsum, at::Tensor()};
    const c10::cuda::CUDAGuard guard(x.device());
    const int64_t H = x.size(-1), rows = x.numel() / H;
    at::Tensor dx, dw, db;
    if (want_dx) dx = at::empty(x.sizes(), x.options());
    const auto as_weight = x.options().dtype(bias_type == kNormHalf ? at::kBFloat16 : at::kFloat);
    if (want_dw) dw = at::empty({H}, weight.options());
    if (want_db) db = at::empty({H}, as_weight);
    if (rows == 0) {
      if (want_dw) dw.zero_();
      if (want_db) db.zero_();
    } else {
      const at::Tensor xr = as_rows(x), dyr = as_rows(dy), sr = dsum.defined() ? as_rows(dsum) : dsum, w = weight.defined() ? weight.contiguous() : weight;
      const int sms = sms_of_current();
      NormGradParams p{};
      p.type = type_of(x); p.weight_type = w.defined() ? type_of(w) : bias_type;
      p.center = ctx->saved_data["center"].toBool(); p.rows = rows; p.hidden = static_cast<int>(H);
      p.x = xr.data_ptr(); p.x_stride = xr.stride(0);
      p.dy = dyr.data_ptr(); p.dy_stride = dyr.stride(0);
      at::Tensor rr;
      if (residual) { rr = as_rows(added); p.residual = rr.data_ptr(); p.residual_stride = rr.stride(0); }
      if (sr.defined()) { p.dsum = sr.data_ptr(); p.dsum_stride = sr.stride(0); }
      p.weight = w.defined() ? w.data_ptr() : nullptr;
      p.stats = reinterpret_cast<const float2*>(stats.data_ptr<float>());
      p.dx = want_dx ? dx.data_ptr() : nullptr;
      p.dweight = want_dw ? dw.data_ptr() : nullptr;
      p.dbias = want_db ? db.data_ptr() : nullptr;
      at::Tensor parts;
      if (want_dw || want_db) {
        parts = at::empty({2 * static_cast<int64_t>(norm_parts(p, sms)) * H}, x.options().dtype(at::kFloat));
        p.parts = parts.data_ptr<float>();
      }
      SEP_CUDA_CHECK(launch_norm_backward(p, sms, at::cuda::getCurrentCUDAStream()));
    }
    return {want_x ? dx : at::Tensor(), dw, db, want_residual ? dx : at::Tensor(), at::Tensor()};
  }
};

void check_vector(const std::optional<at::Tensor>& v, const at::Tensor& x, const char* what) {
  if (!v.has_value()) return;
  SEP_ASSERT(v->dim() == 1 && v->size(0) == x.size(-1) && v->device() == x.device() && usable(*v) && v->layout() == at::kStrided,
             what << " must be a bf16 or float32 tensor of one entry for each column of x, on its device");
  SEP_ASSERT(!v->_fw_grad(0).defined(), "the normalisation has no forward-mode derivative");
}

}  // namespace

std::vector<at::Tensor> norm_rows(const at::Tensor& x, const std::optional<at::Tensor>& weight, const std::optional<at::Tensor>& bias,
                                  const std::optional<at::Tensor>& residual, bool center, double eps) {
  SEP_ASSERT(x.is_cuda() && x.layout() == at::kStrided && usable(x) && x.dim() >= 1, "x must be a [..., H] bf16 or float32 CUDA tensor");
  SEP_ASSERT(x.size(-1) >= 1 && x.size(-1) < (1ll << 30), "rows must have between 1 and 2^30 columns");
  check_vector(weight, x, "weight");
  check_vector(bias, x, "bias");
  if (weight.has_value() && bias.has_value()) SEP_ASSERT(weight->scalar_type() == bias->scalar_type(), "weight and bias must have one type");
  if (residual.has_value()) {
    SEP_ASSERT(residual->sizes() == x.sizes() && residual->scalar_type() == x.scalar_type() && residual->device() == x.device() &&
                   residual->layout() == at::kStrided, "residual must have the shape, type and device of x");
    SEP_ASSERT(!residual->_fw_grad(0).defined(), "the normalisation has no forward-mode derivative");
  }
  SEP_ASSERT(!x._fw_grad(0).defined(), "the normalisation has no forward-mode derivative");
  SEP_ASSERT(eps >= 0.0, "eps must not be negative");
  const c10::cuda::CUDAGuard guard(x.device());
  const at::Tensor w = weight.value_or(at::Tensor()), b = bias.value_or(at::Tensor()), r = residual.value_or(at::Tensor());
  auto call = c10::make_intrusive<NormCall>();
  call->center = center;
  call->eps = eps;
  auto wants = [](const at::Tensor& t) { return t.defined() && t.requires_grad(); };
  if (at::GradMode::is_enabled() && (wants(x) || wants(w) || wants(b) || wants(r))) return Norm::apply(x, weight, bias, residual, call);
  NormResult n = norm_forward(*call, x, w, b, r, false);
  if (r.defined()) return {n.y, n.sum};
  return {n.y};
}

}  // namespace sep

// Host side of the gated linear recurrence: argument checks, workspaces, the autograd node.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "host_common.h"
#include "scan.h"
#include "train_ops.h"

namespace sep {

namespace {

bool usable(const at::Tensor& t) { return t.is_cuda() && t.layout() == at::kStrided && (t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat); }

// [..., D] as rows, each contiguous and equally far apart; a copy where they do not lie so.
at::Tensor as_rows(const at::Tensor& t) {
  const at::Tensor m = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
  return m.stride(1) == 1 || m.size(1) == 1 ? m : m.contiguous();
}

struct ScanCall : torch::CustomClassHolder { ContextFn context; };

struct ScanResult { at::Tensor h, final_state; };

ScanShape shape_of(const at::Tensor& offsets, const at::Tensor& x, const at::Tensor& xr, const at::Tensor& gr, const at::Tensor& initial, const LaunchContext& ctx) {
  ScanShape p{};
  p.half = x.scalar_type() == at::kBFloat16;
  p.rows = static_cast<int>(xr.size(0)); p.channels = static_cast<int>(xr.size(1));
  if (offsets.defined()) {
    p.sequences = static_cast<int>(offsets.size(0) - 1);
    p.offsets = offsets.data_ptr();
    p.offsets_wide = offsets.scalar_type() == at::kLong;
  } else {
    p.sequences = static_cast<int>(x.size(0));
    p.length = static_cast<int>(x.size(1));
  }
  p.x = xr.data_ptr(); p.x_stride = xr.stride(0);
  p.gate = gr.data_ptr(); p.gate_stride = gr.stride(0);
  p.initial = initial.defined() ? initial.data_ptr<float>() : nullptr;
  p.status = ctx.status; p.rank = ctx.rank;
  return p;
}

at::Tensor workspace(const ScanSplit& split, int channels, const at::Tensor& like) {
  const int64_t bytes = scan_space(split, channels);
  return bytes > 0 ? at::empty({bytes}, like.options().dtype(at::kByte)) : at::Tensor();
}
void* pointer(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

ScanResult scan_forward(const ScanCall& call, const at::Tensor& x, const at::Tensor& gate, const at::Tensor& initial, const at::Tensor& offsets,
                        bool want_state) {
  ScanResult out;
  out.h = at::empty(x.sizes(), x.options());
  const LaunchContext ctx = call.context(0);
  const at::Tensor xr = as_rows(x), gr = as_rows(gate), start = initial.defined() ? initial.contiguous() : initial;
  ScanParams p{};
  static_cast<ScanShape&>(p) = shape_of(offsets, x, xr, gr, start, ctx);
  if (want_state) out.final_state = at::empty({p.sequences, p.channels}, x.options().dtype(at::kFloat));
  if (p.sequences == 0) { out.h.zero_(); return out; }
  p.h = out.h.data_ptr();
  p.final_state = want_state ? out.final_state.data_ptr<float>() : nullptr;
  const ScanSplit split = scan_split(p, ctx.sms);
  const at::Tensor space = workspace(split, p.channels, x);
  SEP_CUDA_CHECK(launch_scan_forward(p, split, pointer(space), call.context(split.within ? 1 : 2).stream));
  return out;
}

class Scan : public torch::autograd::Function<Scan> {
 public:
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& gate,
                                                const std::optional<at::Tensor>& first, const std::optional<at::Tensor>& cuts,
                                                const c10::intrusive_ptr<ScanCall>& call, bool want_state) {
    const at::Tensor initial = first.value_or(at::Tensor()), offsets = cuts.value_or(at::Tensor());
    ScanResult r = scan_forward(*call, x, gate, initial, offsets, want_state);
    ctx->save_for_backward({x, gate, initial, r.h, offsets});
    ctx->saved_data["call"] = c10::IValue::make_capsule(call);
    ctx->set_materialize_grads(false);
    if (want_state) return {r.h, r.final_state};
    return {r.h};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    SEP_ASSERT(!at::GradMode::is_enabled(), "gated_scan has no second derivative: its backward was asked for a graph");
    auto call = c10::static_intrusive_pointer_cast<ScanCall>(ctx->saved_data["call"].toCapsule());
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &x = saved[0], &gate = saved[1], &initial = saved[2], &h = saved[3], &offsets = saved[4];
    const at::Tensor dh = grads[0], dfinal = grads.size() > 1 ? grads[1] : at::Tensor();
    if (!dh.defined() && !dfinal.defined()) return {at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
    const bool want_dx = ctx->needs_input_grad(0), want_dgate = ctx->needs_input_grad(1), want_dinitial = initial.defined() && ctx->needs_input_grad(2);
    const c10::cuda::CUDAGuard guard(x.device());
    const LaunchContext context = call->context(0);
    const at::Tensor xr = as_rows(x), gr = as_rows(gate), start = initial.defined() ? initial.contiguous() : initial, hr = as_rows(h);
    const at::Tensor dhr = dh.defined() ? as_rows(dh) : dh, dfr = dfinal.defined() ? dfinal.contiguous() : dfinal;
    ScanGradParams p{};
    static_cast<ScanShape&>(p) = shape_of(offsets, x, xr, gr, start, context);
    at::Tensor dx, dgate, dinitial;
    if (want_dx) dx = at::empty(x.sizes(), x.options());
    if (want_dgate) dgate = at::empty(x.sizes(), x.options());
    if (want_dinitial) dinitial = at::empty(initial.sizes(), initial.options());
    if (p.sequences == 0) {
      if (want_dx) dx.zero_();
      if (want_dgate) dgate.zero_();
    } else {
      p.h = hr.data_ptr();
      if (dhr.defined()) { p.dh = dhr.data_ptr(); p.dh_stride = dhr.stride(0); }
      p.dfinal = dfr.defined() ? dfr.data_ptr<float>() : nullptr;
      p.dx = want_dx ? dx.data_ptr() : nullptr;
      p.dgate = want_dgate ? dgate.data_ptr() : nullptr;
      p.dinitial = want_dinitial ? dinitial.data_ptr<float>() : nullptr;
      const ScanSplit split = scan_split(p, context.sms);
      const at::Tensor space = workspace(split, p.channels, x);
      SEP_CUDA_CHECK(launch_scan_backward(p, split, pointer(space), call->context(split.within ? 1 : 2).stream));
    }
    return {dx, dgate, dinitial, at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

}  // namespace

std::vector<at::Tensor> gated_scan(const ContextFn& context, const at::Tensor& x, const at::Tensor& gate, const std::optional<at::Tensor>& initial,
                                   const std::optional<at::Tensor>& offsets, bool want_state) {
  SEP_ASSERT(usable(x) && x.dim() == (offsets.has_value() ? 2 : 3), "x must be a bf16 or float32 CUDA tensor, [B, T, D], or [N, D] with offsets");
  SEP_ASSERT(gate.sizes() == x.sizes() && gate.scalar_type() == x.scalar_type() && gate.device() == x.device() && gate.layout() == at::kStrided,
             "gate must have the shape, type and device of x");
  SEP_ASSERT(x.size(-1) >= 1 && x.size(-1) < (1ll << 30) && x.numel() / x.size(-1) < (1ll << 30), "x must have at least one channel, and less than 2^30 rows and channels");
  if (offsets.has_value())
    SEP_ASSERT(offsets->dim() == 1 && offsets->size(0) >= 1 && offsets->size(0) < (1ll << 30) && offsets->device() == x.device() &&
                   (offsets->scalar_type() == at::kInt || offsets->scalar_type() == at::kLong),
               "offsets must be a list of int32 or int64 numbers on the device of x, one more than there are sequences");
  else
    SEP_ASSERT(x.size(0) < (1ll << 30), "x has too many sequences");
  const int64_t sequences = offsets.has_value() ? offsets->size(0) - 1 : x.size(0);
  if (initial.has_value())
    SEP_ASSERT(initial->dim() == 2 && initial->size(0) == sequences && initial->size(1) == x.size(-1) && initial->scalar_type() == at::kFloat &&
                   initial->device() == x.device() && initial->layout() == at::kStrided,
               "initial_state must be float32, one row of all channels for each sequence, on the device of x");
  SEP_ASSERT(!x._fw_grad(0).defined() && !gate._fw_grad(0).defined() && !(initial.has_value() && initial->_fw_grad(0).defined()),
             "gated_scan has no forward-mode derivative");
  const c10::cuda::CUDAGuard guard(x.device());
  auto call = c10::make_intrusive<ScanCall>();
  call->context = context;
  std::optional<at::Tensor> cuts;
  if (offsets.has_value()) cuts = offsets->contiguous();
  SEP_ASSERT(context(0).device == x.get_device(), "x is not on the device of the buffer that this call reports into");
  if (at::GradMode::is_enabled() && (x.requires_grad() || gate.requires_grad() || (initial.has_value() && initial->requires_grad())))
    return Scan::apply(x, gate, initial, cuts, call, want_state);
  ScanResult r = scan_forward(*call, x, gate, initial.value_or(at::Tensor()), cuts.value_or(at::Tensor()), want_state);
  if (want_state) return {r.h, r.final_state};
  return {r.h};
}

at::Tensor gated_scan_step(const at::Tensor& state, const at::Tensor& x, const at::Tensor& gate) {
  SEP_ASSERT(usable(x) && x.dim() == 2 && x.size(1) >= 1 && x.size(1) < (1ll << 30) && x.size(0) < (1ll << 30), "x must be a [S, D] bf16 or float32 CUDA tensor");
  SEP_ASSERT(gate.sizes() == x.sizes() && gate.scalar_type() == x.scalar_type() && gate.device() == x.device() && gate.layout() == at::kStrided,
             "gate must have the shape, type and device of x");
  SEP_ASSERT(state.sizes() == x.sizes() && state.scalar_type() == at::kFloat && state.device() == x.device() && state.layout() == at::kStrided,
             "state must be float32 and have the shape and device of x");
  SEP_ASSERT((state.size(1) == 1 || state.stride(1) == 1) && (state.size(0) <= 1 || state.stride(0) >= state.size(1)),
             "state is changed in place: its rows must be contiguous and must not overlap");
  SEP_ASSERT(!state.is_alias_of(x) && !state.is_alias_of(gate), "state is changed in place: it must not share memory with x or gate");
  SEP_ASSERT(!(at::GradMode::is_enabled() && (x.requires_grad() || gate.requires_grad() || state.requires_grad())),
             "gated_scan_step_ has no gradient: call it under torch.no_grad(), or gated_scan");
  SEP_ASSERT(!x._fw_grad(0).defined() && !gate._fw_grad(0).defined() && !state._fw_grad(0).defined(), "gated_scan_step_ has no forward-mode derivative");
  const c10::cuda::CUDAGuard guard(x.device());
  const at::Tensor h = at::empty(x.sizes(), x.options());
  if (x.numel() == 0) return h;
  const at::Tensor xr = as_rows(x), gr = as_rows(gate);
  ScanStepParams p{};
  p.half = x.scalar_type() == at::kBFloat16;
  p.rows = static_cast<int>(x.size(0)); p.channels = static_cast<int>(x.size(1));
  p.x = xr.data_ptr(); p.x_stride = xr.stride(0);
  p.gate = gr.data_ptr(); p.gate_stride = gr.stride(0);
  p.state = state.data_ptr<float>(); p.state_stride = state.stride(0);
  p.h = h.data_ptr();
  SEP_CUDA_CHECK(launch_scan_step(p, at::cuda::getCurrentCUDAStream()));
  if (!state.is_inference()) state.unsafeGetTensorImpl()->bump_version();
  return h;
}

}  // namespace sep

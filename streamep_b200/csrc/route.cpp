// Host side of routing that is trained: argument checks, the router's launch with what its losses need, the autograd node.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "api.h"
#include "host_common.h"
#include "route.h"
#include "train_ops.h"

namespace sep {

namespace {

// bf16 rows as the tensor maps read them; a copy where they do not lie so.
at::Tensor readable(const at::Tensor& t) { return aligned_rows(t.contiguous()); }

struct RouteCall : torch::CustomClassHolder {
  ContextFn context;
  int top_k, num_ranks;
  bool renormalize;
};

// `kept`, for the backward: probabilities [T, E], logsumexp [T], load [E] and 1 / n; behind them what the blocks leave to be added up.
struct Route { at::Tensor idx, weights, in_rank, balance, z, counts, kept; };
struct Kept {
  float *probs, *lse, *load;
  float2 *other_parts, *parts;
  int64_t floats;
  Kept(float* base, int64_t T, int64_t E, int64_t blocks) {
    const int64_t at_lse = T * E, at_load = at_lse + T, at_other = (at_load + E + 1 + 1) / 2 * 2, at_parts = at_other + 2 * blocks;
    floats = at_parts + 2 * blocks * E;
    probs = base; lse = base + at_lse; load = base + at_load;
    other_parts = reinterpret_cast<float2*>(base + at_other); parts = reinterpret_cast<float2*>(base + at_parts);
  }
};

const unsigned char* mask_of(const at::Tensor& mask) { return mask.defined() ? reinterpret_cast<const unsigned char*>(mask.data_ptr<bool>()) : nullptr; }

Route route_forward(const RouteCall& call, const at::Tensor& x, const at::Tensor& w, const at::Tensor& mask) {
  const int64_t T = x.size(0), H = x.size(1), E = w.size(0), K = call.top_k;
  const auto f32 = x.options().dtype(at::kFloat);
  Route r;
  r.idx = at::empty({T, K}, x.options().dtype(at::kLong));
  r.weights = at::empty({T, K}, f32);
  r.in_rank = at::empty({T, call.num_ranks}, x.options().dtype(at::kBool));
  r.balance = at::empty({}, f32);
  r.z = at::empty({}, f32);
  r.counts = at::empty({E}, x.options().dtype(at::kLong));
  const LaunchContext ctx = call.context(T > 0 ? 2 : 1);
  RouterParams p{};
  p.x = x.data_ptr(); p.w_gate = w.data_ptr();
  p.num_tokens = static_cast<int>(T); p.hidden = static_cast<int>(H); p.num_experts = static_cast<int>(E); p.num_topk = call.top_k;
  p.num_ranks = call.num_ranks; p.renormalize = call.renormalize ? 1 : 0;
  p.topk_idx = reinterpret_cast<long long*>(r.idx.data_ptr<int64_t>());
  p.topk_weights = r.weights.data_ptr<float>();
  p.is_token_in_rank = reinterpret_cast<unsigned char*>(r.in_rank.data_ptr<bool>());
  RouteStatsParams s{};
  s.experts = static_cast<int>(E); s.top_k = call.top_k;
  s.mask = mask_of(mask);
  const RouteTile tile = route_tile(p, ctx.sms);
  s.blocks = tile.grid;
  r.kept = at::empty({Kept(nullptr, T, E, s.blocks).floats}, f32);
  const Kept kept(r.kept.data_ptr<float>(), T, E, s.blocks);
  p.probs = kept.probs; p.lse = kept.lse;
  s.other_parts = kept.other_parts; s.parts = kept.parts; s.load = kept.load;
  s.balance = r.balance.data_ptr<float>(); s.z = r.z.data_ptr<float>();
  s.counts = reinterpret_cast<long long*>(r.counts.data_ptr<int64_t>());
  CUtensorMap mw{}, mx{};
  if (T > 0) {
    mw = make_tmap(w.data_ptr(), H, E, 1, H, E * H, 64, 128);
    mx = make_tmap(x.data_ptr(), H, T, 1, H, T * H, 64, tile.tile_tokens);
  }
  SEP_CUDA_CHECK(launch_route_forward(p, s, &mw, &mx, ctx.sms, ctx.status, ctx.wait_budget_ns, ctx.stream));
  return r;
}

class BalancedRoute : public torch::autograd::Function<BalancedRoute> {
 public:
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w_gate,
                                                const std::optional<at::Tensor>& counted, const c10::intrusive_ptr<RouteCall>& call) {
    const at::Tensor mask = counted.value_or(at::Tensor());
    Route r = route_forward(*call, readable(x), readable(w_gate), mask);
    ctx->save_for_backward({x, w_gate, mask, r.kept, r.idx, r.weights});
    ctx->saved_data["call"] = c10::IValue::make_capsule(call);
    ctx->set_materialize_grads(false);
    ctx->mark_non_differentiable({r.idx, r.in_rank, r.counts});
    return {r.idx, r.weights, r.in_rank, r.balance, r.z, r.counts};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    SEP_ASSERT(!at::GradMode::is_enabled(), "balanced_router has no second derivative: its backward was asked for a graph");
    auto call = c10::static_intrusive_pointer_cast<RouteCall>(ctx->saved_data["call"].toCapsule());
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &x = saved[0], &w_gate = saved[1], &mask = saved[2], &idx = saved[4], &weights = saved[5];
    if (!grads[1].defined() && !grads[3].defined() && !grads[4].defined()) return {at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
    const bool want_dx = ctx->needs_input_grad(0), want_dw = ctx->needs_input_grad(1);
    const int64_t T = x.size(0), H = x.size(1), E = w_gate.size(0);
    const Kept kept(saved[3].data_ptr<float>(), T, E, 0);
    const c10::cuda::CUDAGuard guard(x.device());
    // A thread of the autograd engine may not have made a call of the CUDA runtime yet, and the driver encodes tensor maps only
    // with a context bound to the thread.
    SEP_CUDA_CHECK(cudaSetDevice(x.get_device()));
    at::Tensor dx, dw;
    if (want_dx) dx = at::empty({T, H}, x.options());
    if (want_dw) dw = T > 0 ? at::empty({E, H}, w_gate.options()) : at::zeros({E, H}, w_gate.options());
    if (T > 0) {
      const LaunchContext context = call->context(0);
      const at::Tensor xr = readable(x), wr = readable(w_gate);
      const RouteGradPlan plan = route_grad_plan(static_cast<int>(T), static_cast<int>(H), static_cast<int>(E), context.sms);
      call->context(want_dw ? plan.dw_splits > 1 ? 3 : 2 : 1);
      at::Tensor up[3];
      for (int i = 0; i < 3; ++i) {
        const at::Tensor& g = grads[i == 0 ? 1 : i + 2];
        if (g.defined()) up[i] = g.scalar_type() == at::kFloat && g.is_contiguous() ? g : g.to(at::kFloat).contiguous();
      }
      RouteGradParams p{};
      p.tokens = static_cast<int>(T); p.experts = static_cast<int>(E); p.top_k = call->top_k; p.hidden = static_cast<int>(H); p.renormalize = call->renormalize;
      p.probs = kept.probs; p.lse = kept.lse; p.load = kept.load;
      p.idx = reinterpret_cast<const long long*>(idx.data_ptr<int64_t>());
      p.weights = weights.data_ptr<float>();
      p.mask = mask_of(mask);
      p.dweights = up[0].defined() ? up[0].data_ptr<float>() : nullptr;
      p.dbalance = up[1].defined() ? up[1].data_ptr<float>() : nullptr;
      p.dz_loss = up[2].defined() ? up[2].data_ptr<float>() : nullptr;
      p.dx = want_dx ? dx.data_ptr() : nullptr;
      p.dw = want_dw ? dw.data_ptr() : nullptr;
      p.status = context.status; p.rank = context.rank; p.wait_budget_ns = context.wait_budget_ns;
      at::Tensor space;                          // dz, and the parts of dw
      const int64_t dz_bytes = (plan.layers * T * plan.padded * 2 + 255) / 256 * 256, parts = plan.dw_splits > 1 ? plan.dw_splits : 0;
      if (want_dw) {
        space = at::empty({dz_bytes + parts * E * H * 4}, x.options().dtype(at::kByte));
        p.dz = space.data_ptr();
      }
      CUtensorMap map_w{}, map_dx{};
      if (want_dx) {
        map_w = make_tmap(wr.data_ptr(), H, E, 1, H, E * H, 64, 64);
        map_dx = make_tmap(p.dx, H, T, 1, H, T * H, 64, 32);
      }
      SEP_CUDA_CHECK(launch_route_dx(p, plan, &map_w, &map_dx, context.stream));
      if (want_dw) {
        float* sums = reinterpret_cast<float*>(static_cast<char*>(space.data_ptr()) + dz_bytes);
        const CUtensorMap map_dz = make_tmap(p.dz, plan.padded, T, plan.layers, plan.padded, T * plan.padded, 64, 64), map_x = make_tmap(xr.data_ptr(), H, T, 1, H, T * H, 64, 64),
                          map_out = parts > 0 ? make_tmap(sums, H, E, parts, H, E * H, 32, 32, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_DATA_TYPE_FLOAT32)
                                              : make_tmap(p.dw, H, E, 1, H, E * H, 64, 32);
        SEP_CUDA_CHECK(launch_route_dw(p, plan, &map_dz, &map_x, &map_out, sums, context.stream));
      }
    }
    return {dx, dw, at::Tensor(), at::Tensor()};
  }
};

}  // namespace

std::vector<at::Tensor> balanced_router(const ContextFn& context, const at::Tensor& x, const at::Tensor& w_gate, int64_t top_k, int64_t num_ranks,
                                        bool renormalize, const std::optional<at::Tensor>& mask) {
  auto rows = [](const at::Tensor& t) { return t.is_cuda() && t.layout() == at::kStrided && t.dim() == 2 && t.scalar_type() == at::kBFloat16; };
  SEP_ASSERT(rows(x), "x must be a [T, H] bf16 CUDA tensor");
  SEP_ASSERT(rows(w_gate) && w_gate.device() == x.device() && w_gate.size(1) == x.size(1), "w_gate must be an [E, H] bf16 tensor on the device of x");
  SEP_ASSERT(x.size(1) > 0 && x.size(1) % 8 == 0 && x.size(1) < (1ll << 30), "hidden must be a positive multiple of 8");
  SEP_ASSERT(x.size(0) < (1ll << 26), "too many tokens for one call");
  const int64_t E = w_gate.size(0);
  SEP_ASSERT(E >= 1 && E <= 512, "the router takes 1 to 512 experts");
  SEP_ASSERT(top_k >= 1 && top_k <= 32 && top_k <= E, "top_k must be between 1 and 32, and no more than there are experts");
  SEP_ASSERT(num_ranks >= 1 && num_ranks <= 32 && E % num_ranks == 0, "the experts must divide evenly over 1 to 32 ranks");
  if (mask.has_value())
    SEP_ASSERT(mask->dim() == 1 && mask->size(0) == x.size(0) && mask->scalar_type() == at::kBool && mask->device() == x.device() && mask->layout() == at::kStrided,
               "mask must hold one truth value for each token, on the device of x");
  SEP_ASSERT(!x._fw_grad(0).defined() && !w_gate._fw_grad(0).defined(), "balanced_router has no forward-mode derivative");
  const c10::cuda::CUDAGuard guard(x.device());
  auto call = c10::make_intrusive<RouteCall>();
  call->context = context;
  call->top_k = static_cast<int>(top_k); call->num_ranks = static_cast<int>(num_ranks);
  call->renormalize = renormalize;
  SEP_ASSERT(context(0).device == x.get_device(), "x is not on the device of the buffer that this call reports into");
  std::optional<at::Tensor> counted;
  if (mask.has_value()) counted = mask->contiguous();
  if (at::GradMode::is_enabled() && (x.requires_grad() || w_gate.requires_grad())) return BalancedRoute::apply(x, w_gate, counted, call);
  const Route r = route_forward(*call, readable(x), readable(w_gate), counted.value_or(at::Tensor()));
  return {r.idx, r.weights, r.in_rank, r.balance, r.z, r.counts};
}

}  // namespace sep

// Host side of the output projection with softmax cross entropy: argument checks, the plan of the backward (pieces of the
// vocabulary, splits), workspaces, and the autograd node.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>

#include "host_common.h"
#include "linear_loss.h"
#include "train_ops.h"

namespace sep {

namespace {

int64_t ceil_of(int64_t a, int64_t b) { return (a + b - 1) / b; }

// One dz buffer holds at most about this much, of which there are two.  Larger pieces mean fewer additions to the fp32 sums of dx: with 48, 128,
// 256 and 512 MB 8192 x 2048 x 65536 (tokens, hidden, vocabulary) took 7530, 7026, 6978 and 6946 us, 16384 x 1024 x 50000 7388, 6050, 5909 and 5855.
constexpr int64_t kPieceBytes = 256ll << 20;
constexpr int64_t kSplitTokens = 64;             // calls whose dz is kept as a sum of two bf16 numbers: one k-block of tokens
constexpr int64_t kDirectBlocks = 32;            // k-blocks of dx that are not worth splitting
constexpr int64_t kNarrowTokens = 576;           // three token tiles of 192, three quarters of 256
constexpr int64_t kBandBytes = 48ll << 20;       // rows of x that a band of units shares in L2

// Tokens as columns (the narrow form) where that multiplies at least a quarter less; always where dz is split.  Hidden 2048, V 100003, with rows
// and with columns, forward alone: 96 tokens 103 and 90 us, 160 107 and 102, 192 109 and 107, 224 111 and 113, 300 175 and 166, 384 178 and
// 177, 448 183 and 188; with gradients 418 and 382, 467 and 440, 474 and 460, 492 and 494, 702 and 669, 739 and 725, 779 and 777.
// 513 243 and 238, with gradients 994 and 968, 576 246 and 240, 1016 and 978.  576 tokens, hidden 4096, V 32000: 167 and 165, with gradients 661 and
// 643.  Short reductions lose, forward alone: hidden 512 and 300 tokens 31 and 35, 576 (V 50257) 44.1 and 46.4, with gradients 181 and 186.
// 1 token, hidden 4096, V 128000, forward: 248 and 172.
void plan_tiles(LossParams& p, bool backward) {
  const int64_t T = p.T, units = ceil_of(T, kLossUnit), tokens = ceil_of(ceil_of(T, units), 32) * 32;
  p.narrow = T <= kSplitTokens || (T <= kNarrowTokens && tokens * 4 <= 3 * kLossUnit);
  p.tile_tokens = p.narrow ? static_cast<int>(tokens) : kLossUnit;
  p.row_units = static_cast<int>(units);
  // The tensor cores take bf16, so dz is rounded to it before its products (8 bits: 2^-8 at most, of each term and not of a sum that may cancel), as
  // bf16 training code rounds the gradient of its logits.  That does not average out: a target's row of dW is mostly one token's (p - 1) x.
  // The gradients' 2-norm error against 64 bits goes from 1.7e-3, the result's own rounding, to 2.0e-3 - 2.3e-3.  Up to 64 tokens dz is kept
  // to 16 bits instead, as a sum of two bf16 numbers, since twice the products of dx and dW cost little beside the reads of the projection: with
  // gradients 1 x 4096 x 128000 (tokens, hidden, vocabulary) 709 -> 728 us, 16 and 64 x 2048 x 100003 315 -> 323 and 351 -> 376, 64 x 512 x 32000
  // 98 -> 97.  Of longer calls the products take most of the time, and there would be 5 for every 3.
  p.split2 = T <= kSplitTokens ? 1 : 0;
  // Up to 32 tokens dw takes 32 at a time, so that a stage of the ring need not hold more than 128 rows of the projection and those tokens, and more
  // of the projection is on its way: 1 token, hidden 4096, V 128000 581 -> 547 us, 16 tokens, hidden 2048, V 100003 255 -> 241.  (40
  // tokens in two such blocks: 259 -> 287.)
  p.dw_rows = T <= 32 ? 32 : 64;
  loss_narrow_ring(p, backward);
}
void plan_backward(LossParams& p, int sms, int64_t piece_bytes) {
  const int64_t T = p.T, H = p.H, V = p.V, pairs = sms / 2;
  p.h_units = static_cast<int>(ceil_of(H, kLossUnit));
  const int64_t row_bytes = T * 2 * (p.split2 ? 2 : 1);
  const int64_t want = ceil_of(V * row_bytes, piece_bytes);
  p.piece = static_cast<int>(ceil_of(ceil_of(V, want), kLossUnit) * kLossUnit);
  p.pieces = static_cast<int>(ceil_of(V, p.piece));
  p.last_cols = static_cast<int>(V - static_cast<int64_t>(p.pieces - 1) * p.piece);
  p.ahead = std::min(1, p.pieces);
  p.buffers = std::min(p.ahead + 1, p.pieces);
  const int64_t v_blocks = ceil_of(V, 64), t_blocks = ceil_of(T, p.dw_rows) * (p.split2 ? 2 : 1), tiles = ceil_of(V, kLossUnit);
  // k-blocks of all the work, for each pair
  const int64_t all = (p.row_units * tiles * ceil_of(H, 64) + (p.want_dx ? p.row_units * p.h_units * v_blocks : 0) +
                       (p.want_dw ? tiles * p.h_units * t_blocks : 0)) / pairs + 1;
  // dx units of one place follow each other piece by piece: a chain of v_blocks / splits k-blocks, which is to stay within half of the
  // time that the whole takes; and a unit within an eighth of it, so that pairs end together.  But no more splits than keep the
  // traffic of the partial sums (4 bytes, written and read) within an eighth of reading the projection.  Where the dx units of a piece
  // are few rounds of all pairs, the number whose rounds are fullest is taken.
  const int64_t piece_blocks = ceil_of(std::min<int64_t>(V, p.piece), 64), places = static_cast<int64_t>(p.row_units) * p.h_units;
  const int64_t chain = ceil_of(2 * v_blocks, all), even = std::min(ceil_of(8 * piece_blocks, all), V / (32 * T));
  const int64_t most = std::max<int64_t>(1, std::min({std::max(chain, even), piece_blocks / 4, static_cast<int64_t>(64)}));
  int64_t best = most, best_time = -1;
  for (int64_t s = std::max<int64_t>(1, std::max(chain, most / 2)); s <= most; ++s) {
    const int64_t time = ceil_of(places * s, pairs) * ceil_of(piece_blocks, s);
    if (best_time < 0 || time < best_time) { best = s; best_time = time; }
  }
  p.splits = static_cast<int>(best);
  p.split_blocks = static_cast<int>(ceil_of(piece_blocks, p.splits));
  p.splits = static_cast<int>(ceil_of(piece_blocks, p.split_blocks));
  // Small vocabularies are not split: such calls are bound by the host, to whom the kernel that joins the splits costs a launch (64 tokens,
  // hidden 256, V 1000: 87 -> 81 us a training pass).
  if (v_blocks <= kDirectBlocks) { p.splits = 1; p.split_blocks = static_cast<int>(piece_blocks); }
  p.dx_direct = p.splits == 1 && p.pieces == 1;
  // dw units of few k-blocks take several column tiles, as long as there are a few units for every pair: claiming one and asking
  // whether its dz is there takes longer than its products.
  const int64_t per_pair = tiles * p.h_units / pairs;
  p.dw_group = static_cast<int>(std::max<int64_t>(1, std::min({static_cast<int64_t>(p.h_units), 24 / t_blocks, per_pair / 4})));
  // A single piece has nothing but its own dz ahead of its products.  Some dw units, which can begin on the first finished column
  // tiles of dz, bridge the wait for the last ones; the others come after the longer dx units.
  p.dw_lead = p.pieces == 1 ? static_cast<int>(pairs) : 0;
}
// Units of few k-blocks are claimed further ahead: a claim takes about as long as the operands of four k-blocks.
int claim_lead(const LossParams& p, bool backward) {
  const int64_t shortest = std::min<int64_t>(ceil_of(p.H, 64), backward ? ceil_of(p.T, 64) : 1 << 20);
  return shortest <= 8 ? 2 : 0;
}
void plan_band(LossParams& p) {
  const int64_t rows = std::max<int64_t>(kBandBytes / (2 * static_cast<int64_t>(p.H)), kLossUnit);
  // bands of equal height
  const int64_t bands = ceil_of(p.row_units, std::max<int64_t>(rows / p.tile_tokens, 1));
  p.band = static_cast<int>(ceil_of(p.row_units, bands));
}

// [rows, cols] bf16 with rows 16 bytes apart at least, as TMA reads them; a copy where they are not.
at::Tensor readable(const at::Tensor& t) {
  const bool fits = t.stride(1) == 1 && is_aligned(t) && (t.size(0) <= 1 || (t.stride(0) % 8 == 0 && t.stride(0) >= t.size(1)));
  if (fits) return t;
  return aligned_rows(t.contiguous());
}
int64_t pitch(const at::Tensor& t) { return t.size(0) <= 1 ? t.size(1) : t.stride(0); }

// Places in one workspace, 256 bytes apart.
struct Carver {
  int64_t bytes = 0;
  int64_t take(int64_t n) { const int64_t at = bytes; bytes += ceil_of(std::max<int64_t>(n, 1), 256) * 256; return at; }
};

struct LossCall : torch::CustomClassHolder {
  ContextFn context;
  int64_t ignore_index;
  int reduction;
  int64_t piece_bytes;
  bool want_dx = false, want_dw = false;
  // The forward's kernel clears the backward's counters, for one backward after it.  A backward clears them itself when another has run
  // (retain_graph), and when the two are not of one captured graph (or of none): one may be replayed without the other.
  bool counters_used = false;
  unsigned long long capture = 0;
};

// The capture that the stream takes part in, 0: none.
unsigned long long capture_of(cudaStream_t stream) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  SEP_CUDA_CHECK(cudaStreamGetCaptureInfo(stream, &status, &id));
  return status == cudaStreamCaptureStatusActive ? id : 0;
}

// The loss; and what the backward needs: [3][T] softmax statistics, 1 / counted tokens, and from `counters_at` on the counters of its kernel,
// which the forward's kernel clears.
struct Forward { at::Tensor loss, stats; };

LossParams plan(int64_t T, int64_t H, int64_t V, bool want_dx, bool want_dw, int sms, int64_t piece_bytes) {
  LossParams p{};
  p.T = static_cast<int>(T); p.H = static_cast<int>(H); p.V = static_cast<int>(V);
  p.want_dx = want_dx; p.want_dw = want_dw;
  plan_tiles(p, true);
  plan_backward(p, sms, piece_bytes);
  plan_band(p);
  p.claim_lead = claim_lead(p, true);
  return p;
}
int64_t counters_at(int64_t T) { return ceil_of(3 * T + 1, 64) * 64; }
int64_t counter_ints(const LossParams& p) { return 4 + (3 + p.piece / kLossUnit) * static_cast<int64_t>(p.pieces); }

Forward loss_forward(LossCall& call, const at::Tensor& x, const at::Tensor& w, const at::Tensor& targets) {
  const int64_t T = x.size(0), H = x.size(1), V = w.size(0);
  const auto f32 = x.options().dtype(at::kFloat);
  const bool reduced = call.reduction != kLossNone;
  Forward out;
  if (T == 0) {
    out.stats = at::empty({1}, f32);
    out.loss = reduced ? at::full({}, call.reduction == kLossMean ? std::numeric_limits<float>::quiet_NaN() : 0.0, f32) : at::empty({0}, f32);
    return out;
  }
  out.loss = reduced ? at::empty({}, f32) : at::empty({T}, f32);
  const LaunchContext ctx = call.context(2);
  LossParams p{};
  p.T = static_cast<int>(T); p.H = static_cast<int>(H); p.V = static_cast<int>(V);
  plan_tiles(p, false);
  plan_band(p);
  p.claim_lead = claim_lead(p, false);
  const int64_t parts = loss_forward_parts(p, ctx.sms);
  Carver c;
  const int64_t counters = c.take(64), part_at = c.take(parts * T * 8), logit_at = c.take(T * 4), each_at = reduced ? c.take(T * 4) : 0;
  const at::Tensor space = at::empty({c.bytes}, x.options().dtype(at::kByte));
  char* base = static_cast<char*>(space.data_ptr());
  p.parts = reinterpret_cast<float2*>(base + part_at);
  p.target_logit = reinterpret_cast<float*>(base + logit_at);
  p.targets = reinterpret_cast<const long long*>(targets.data_ptr<int64_t>());
  p.ignore_index = call.ignore_index;
  int* ticket = reinterpret_cast<int*>(base + counters) + 1;
  p.zero = ticket; p.zero_ints = 1;
  if (call.want_dx || call.want_dw) {
    // the ticket stands behind the backward's counters, to be cleared with them
    const int64_t ints = counter_ints(plan(T, H, V, call.want_dx, call.want_dw, ctx.sms, call.piece_bytes));
    out.stats = at::empty({counters_at(T) + ints + 1}, f32);
    call.capture = capture_of(ctx.stream);
    p.zero = reinterpret_cast<int*>(out.stats.data_ptr<float>() + counters_at(T));
    p.zero_ints = static_cast<int>(ints + 1);
    ticket = p.zero + ints;
  } else {
    out.stats = at::empty({3 * T + 1}, f32);
  }
  p.status = ctx.status; p.rank = ctx.rank; p.wait_budget_ns = ctx.wait_budget_ns;
  LossMaps m{};
  m.x_k = make_tmap(x.data_ptr(), H, T, 1, pitch(x), pitch(x) * T, 64, p.tile_tokens / 2);
  m.w_k = make_tmap(w.data_ptr(), H, V, 1, pitch(w), pitch(w) * V, 64, 128);
  // Units of the narrow form are dealt out in turn, since each warp keeps one statistic of all that it gets: claimed by whoever is free
  // first, a repeated call would add in another order and not give the same bits.  (Of the others each unit has its own part; and with
  // a unit a pair there is nothing to claim.)
  if (!p.narrow && static_cast<int64_t>(p.row_units) * ceil_of(V, kLossUnit) > ctx.sms / 2) {
    p.claim = reinterpret_cast<int*>(base + counters);
    SEP_CUDA_CHECK(cudaMemsetAsync(p.claim, 0, sizeof(int), ctx.stream));
  }
  SEP_CUDA_CHECK(launch_loss_forward(p, m, ctx.sms, ctx.stream));

  LossFinalParams f{};
  f.T = p.T; f.V = p.V; f.num_parts = static_cast<int>(parts);
  f.parts = p.parts; f.target_logit = p.target_logit; f.targets = p.targets; f.ignore_index = p.ignore_index;
  f.mean = call.reduction == kLossMean; f.sum = call.reduction == kLossSum;
  f.each = reduced ? reinterpret_cast<float*>(base + each_at) : out.loss.data_ptr<float>();
  f.top = out.stats.data_ptr<float>();
  f.loss = reduced ? out.loss.data_ptr<float>() : nullptr;
  f.inv_count = f.top + 3 * T;
  f.ticket = ticket;
  f.status = ctx.status; f.rank = ctx.rank;
  SEP_CUDA_CHECK(launch_loss_final(f, ctx.stream));
  return out;
}

std::pair<at::Tensor, at::Tensor> loss_backward(LossCall& call, const at::Tensor& x, const at::Tensor& w, const at::Tensor& targets,
                                                const at::Tensor& stats, const at::Tensor& upstream, bool want_dx, bool want_dw) {
  const int64_t T = x.size(0), H = x.size(1), V = w.size(0);
  at::Tensor dx, dw;
  if (T == 0) {
    if (want_dx) dx = at::empty({0, H}, x.options());
    if (want_dw) dw = at::zeros({V, H}, w.options());
    return {dx, dw};
  }
  if (want_dx) dx = at::empty({T, H}, x.options());
  if (want_dw) dw = at::empty({V, H}, w.options());
  const LaunchContext ctx = call.context(1);
  const at::Tensor up = upstream.to(at::kFloat).contiguous();

  LossParams p = plan(T, H, V, want_dx, want_dw, ctx.sms, call.piece_bytes);
  SEP_ASSERT(loss_backward_units(p) < (1ll << 30), "this loss has too many tiles for one call: split the tokens");
  const int64_t z_layers = p.split2 ? 2 : 1, slots = p.splits;
  Carver c;
  const int64_t z_at = c.take(p.buffers * z_layers * T * p.piece * 2), dx_at = want_dx && !p.dx_direct ? c.take(slots * T * H * 4) : 0;
  const at::Tensor space = at::empty({c.bytes}, x.options().dtype(at::kByte));
  char* base = static_cast<char*>(space.data_ptr());
  p.targets = reinterpret_cast<const long long*>(targets.data_ptr<int64_t>());
  p.ignore_index = call.ignore_index;
  p.top = stats.data_ptr<float>();
  if (call.reduction == kLossNone) p.row_scale = up.data_ptr<float>();
  else p.scale = up.data_ptr<float>();
  if (call.reduction == kLossMean) p.scale2 = p.top + 3 * T;
  p.claim = reinterpret_cast<int*>(stats.data_ptr<float>() + counters_at(T));
  p.done = p.claim + 4;
  p.status = ctx.status; p.rank = ctx.rank; p.wait_budget_ns = ctx.wait_budget_ns;

  LossMaps m{};
  m.x_k = make_tmap(x.data_ptr(), H, T, 1, pitch(x), pitch(x) * T, 64, p.tile_tokens / 2);
  m.w_k = make_tmap(w.data_ptr(), H, V, 1, pitch(w), pitch(w) * V, 64, 128);
  if (want_dw) m.x_mn = make_tmap(x.data_ptr(), H, T, 1, pitch(x), pitch(x) * T, 64, p.dw_rows);
  if (want_dx) m.w_mn = make_tmap(w.data_ptr(), H, V, 1, pitch(w), pitch(w) * V, 64, 64);
  const int64_t panels = p.buffers * z_layers * (p.piece / 64);
  auto z_map = [&](int cols, int rows, CUtensorMapSwizzle swizzle) { return make_tmap(base + z_at, 64, T, panels, 64, T * 64, cols, rows, swizzle); };
  if (want_dx) m.z_k = z_map(64, p.split2 ? p.tile_tokens : p.tile_tokens / 2, CU_TENSOR_MAP_SWIZZLE_128B);
  if (want_dw) m.z_mn = z_map(64, p.dw_rows, CU_TENSOR_MAP_SWIZZLE_128B);
  m.z_out = p.narrow ? z_map(32, 32, CU_TENSOR_MAP_SWIZZLE_64B) : z_map(64, 32, CU_TENSOR_MAP_SWIZZLE_128B);
  if (want_dw) m.dw = make_tmap(dw.data_ptr(), H, V, 1, H, H * V, 64, 32);
  p.dx_parts = reinterpret_cast<float*>(base + dx_at);
  p.dx = want_dx ? dx.data_ptr() : nullptr;
  if (want_dx && p.dx_direct) m.dx = make_tmap(dx.data_ptr(), H, T, 1, H, T * H, 64, 32);
  else if (want_dx && !p.narrow) m.dx = make_tmap(base + dx_at, H, T, slots, H, T * H, 32, 32, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_DATA_TYPE_FLOAT32);
  if (call.counters_used || call.capture != capture_of(ctx.stream)) SEP_CUDA_CHECK(cudaMemsetAsync(p.claim, 0, counter_ints(p) * sizeof(int), ctx.stream));
  call.counters_used = true;
  SEP_CUDA_CHECK(launch_loss_backward(p, m, ctx.sms, ctx.stream));
  if (want_dx && !p.dx_direct) {
    LossDxParams d{};
    d.T = p.T; d.H = p.H; d.slots = static_cast<int>(slots);
    d.parts = reinterpret_cast<const float*>(base + dx_at);
    d.scale = p.scale; d.scale2 = p.scale2;
    d.dx = dx.data_ptr();
    SEP_CUDA_CHECK(launch_loss_dx(d, call.context(1).stream));
  }
  return {dx, dw};
}

class LinearLoss : public torch::autograd::Function<LinearLoss> {
 public:
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const at::Tensor& weight, const at::Tensor& targets,
                            const c10::intrusive_ptr<LossCall>& call) {
    const at::Tensor xr = readable(x), wr = readable(weight), y = targets.contiguous();
    Forward f = loss_forward(*call, xr, wr, y);
    ctx->save_for_backward({x, weight, targets, f.stats});
    ctx->saved_data["call"] = c10::IValue::make_capsule(call);
    return f.loss;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    SEP_ASSERT(!at::GradMode::is_enabled(), "linear_cross_entropy has no second derivative: its backward was asked for a graph");
    auto call = c10::static_intrusive_pointer_cast<LossCall>(ctx->saved_data["call"].toCapsule());
    const auto saved = ctx->get_saved_variables();
    if (!grads[0].defined()) return {at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
    const c10::cuda::CUDAGuard guard(saved[0].device());
    // A thread of the autograd engine may not have made a call of the CUDA runtime yet, and the driver encodes tensor maps only
    // with a context bound to the thread.
    SEP_CUDA_CHECK(cudaSetDevice(saved[0].get_device()));
    auto g = loss_backward(*call, readable(saved[0]), readable(saved[1]), saved[2].contiguous(), saved[3], grads[0],
                           call->want_dx && ctx->needs_input_grad(0), call->want_dw && ctx->needs_input_grad(1));
    return {g.first, g.second, at::Tensor(), at::Tensor()};
  }
};

}  // namespace

at::Tensor linear_loss(const ContextFn& context, const at::Tensor& x, const at::Tensor& weight, const at::Tensor& targets,
                       int64_t ignore_index, int reduction, int64_t piece_bytes) {
  SEP_ASSERT(x.is_cuda() && x.dim() == 2 && x.scalar_type() == at::kBFloat16, "x must be a [..., H] bf16 CUDA tensor");
  SEP_ASSERT(weight.dim() == 2 && weight.scalar_type() == at::kBFloat16 && weight.device() == x.device() && weight.size(1) == x.size(1),
             "weight must be a [V, H] bf16 tensor on the device of x");
  SEP_ASSERT(targets.dim() == 1 && targets.scalar_type() == at::kLong && targets.device() == x.device() && targets.size(0) == x.size(0),
             "targets must be int64, one for each row of x, on its device");
  SEP_ASSERT(x.size(1) > 0 && x.size(1) % 8 == 0, "hidden must be a positive multiple of 8");
  SEP_ASSERT(weight.size(0) >= 1, "the vocabulary is empty");
  SEP_ASSERT(x.size(0) < (1ll << 30) && weight.size(0) < (1ll << 30) && x.size(1) < (1ll << 30) &&
                 ceil_of(x.size(0), kLossUnit) * ceil_of(weight.size(0), kLossUnit) < (1ll << 30),
             "this loss has too many tiles for one call: split the tokens");
  SEP_ASSERT(reduction >= kLossNone && reduction <= kLossSum, "unknown reduction");
  SEP_ASSERT(piece_bytes >= 0, "piece_bytes must not be negative");
  SEP_ASSERT(!x._fw_grad(0).defined() && !weight._fw_grad(0).defined(), "linear_cross_entropy has no forward-mode derivative");
  const c10::cuda::CUDAGuard guard(x.device());
  auto call = c10::make_intrusive<LossCall>();
  call->context = context;
  call->ignore_index = ignore_index;
  call->reduction = reduction;
  call->piece_bytes = piece_bytes > 0 ? piece_bytes : kPieceBytes;
  SEP_ASSERT(context(0).device == x.get_device(), "x is not on the device of the buffer that this call reports into");
  if (!(at::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad())))
    return loss_forward(*call, readable(x), readable(weight), targets.contiguous()).loss;
  call->want_dx = x.requires_grad();
  call->want_dw = weight.requires_grad();
  return LinearLoss::apply(x, weight, targets, call);
}

std::vector<std::vector<int>> linear_loss_schedule(int64_t tokens, int64_t hidden, int64_t vocab, int sms, bool want_dx, bool want_dw, int64_t piece_bytes) {
  const LossParams p = plan(tokens, hidden, vocab, want_dx, want_dw, sms, piece_bytes > 0 ? piece_bytes : kPieceBytes);
  std::vector<std::vector<int>> out = {{p.pieces, p.piece, p.splits, p.ahead, p.buffers, p.row_units, p.split2, p.dw_group}};
  const long long units = loss_backward_units(p);
  for (long long i = 0; i < units; ++i) {
    int v[7];
    loss_backward_unit(p, static_cast<int>(i), v);
    out.emplace_back(v, v + 7);
  }
  return out;
}

}  // namespace sep

// Host side of the operators over lists of tensors: checks, the lists as kernel arguments, launches.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>
#include <deque>

#include "host_common.h"
#include "list_kernels.h"
#include "train_ops.h"

namespace sep {

namespace {

bool is_half(const at::Tensor& t) { return t.scalar_type() == at::kBFloat16; }

constexpr char kListMessage[] = "the tensors of a list must be dense tensors on one CUDA device, bf16 or float32";

bool usable(const at::Tensor& t, const at::Device& device) {
  return t.defined() && t.layout() == at::kStrided && t.device() == device && (t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat);
}

// What is written in place must not lie in two entries: its owner would be undefined.
struct Ranges {
  using List = std::vector<std::pair<uintptr_t, uintptr_t>>;
  List all;                      // sorted so far
  static bool less(const List::value_type& a, const List::value_type& b) { return a.first < b.first; }
  static List::value_type of(const at::Tensor& t) {
    const auto p = reinterpret_cast<uintptr_t>(t.data_ptr());
    return {p, p + t.numel() * t.element_size()};
  }
  // (lists are mostly in the order of their addresses, and one behind the other: nothing to sort or merge)
  void add(List&& more) {
    if (!std::is_sorted(more.begin(), more.end(), less)) std::sort(more.begin(), more.end(), less);
    if (all.empty()) { all = std::move(more); return; }
    if (more.empty()) return;
    if (less(more.back(), all.front())) all.swap(more);
    const size_t n = all.size();
    const bool behind = !less(more.front(), all.back());
    all.insert(all.end(), more.begin(), more.end());
    if (!behind) std::inplace_merge(all.begin(), all.begin() + n, all.end(), less);
  }
  void check() const {
    for (size_t i = 1; i < all.size(); ++i)
      SEP_ASSERT(all[i].first >= all[i - 1].second, "two tensors that are written in place share memory");
  }
};

int num_sms() { return at::cuda::getCurrentDeviceProperties()->multiProcessorCount; }

// Elements of a chunk: about eight chunks a block, so that blocks end together, and no less than two elements a thread.
int chunk_of(int64_t elements, int64_t blocks) {
  int64_t chunk = 1024;
  while (chunk < 16384 && chunk * blocks * 8 < elements) chunk *= 2;
  return static_cast<int>(chunk);
}

// Cuts `tensors` (none of them empty) into lists of at most kNormEntries.
template <class Launch>
void for_norm_lists(const TensorList& tensors, Launch launch) {
  int64_t elements = 0;
  for (const at::Tensor* t : tensors) elements += t->numel();
  NormList list;
  const int most = num_sms() * kNormBlocksPerSm;
  list.chunk = chunk_of(elements, most);
  for (size_t at = 0; at < tensors.size(); at += kNormEntries) {
    list.count = static_cast<int>(std::min<size_t>(kNormEntries, tensors.size() - at));
    int64_t chunks = 0;
    for (int i = 0; i < list.count; ++i) {
      const at::Tensor& t = *tensors[at + i];
      list.data[i] = t.data_ptr();
      list.length[i] = static_cast<unsigned long long>(t.numel()) | (static_cast<unsigned long long>(is_half(t) ? kListHalf : 0) << kListTypeShift);
      list.first[i] = static_cast<int>(chunks);
      chunks += (t.numel() + list.chunk - 1) / list.chunk;
      SEP_ASSERT(chunks < (1ll << 31), "the list is too large");
    }
    list.first[list.count] = list.chunks = static_cast<int>(chunks);
    launch(list, static_cast<int>(std::min<int64_t>(most, chunks)));
  }
}

// The tensors to read for a norm: dense ones as they lie (the order of elements does not matter), others as contiguous copies.
struct Readable {
  TensorList list;
  std::deque<at::Tensor> copies;
  Readable(const TensorList& tensors, const at::Device& device) {
    list.reserve(tensors.size());
    for (const at::Tensor* t : tensors) {
      SEP_ASSERT(usable(*t, device), kListMessage);
      if (t->numel() == 0) continue;
      if (t->is_non_overlapping_and_dense()) { list.push_back(t); continue; }
      copies.push_back(t->detach().contiguous());
      list.push_back(&copies.back());
    }
  }
};

// The partial sums of squares of a list, one double per block of every launch.
at::Tensor squares(const TensorList& tensors, cudaStream_t stream, int& count) {
  const int64_t lists = (static_cast<int64_t>(tensors.size()) + kNormEntries - 1) / kNormEntries;
  const at::Tensor sums = at::empty({lists * num_sms() * kNormBlocksPerSm}, tensors[0]->options().dtype(at::kDouble));
  count = 0;
  for_norm_lists(tensors, [&](const NormList& list, int blocks) {
    SEP_CUDA_CHECK(launch_list_squares(list, sums.data_ptr<double>() + count, blocks, stream));
    count += blocks;
  });
  return sums;
}

void scale_lists(const TensorList& tensors, const double* sums, int count, float* norm, double max_norm, cudaStream_t stream) {
  for_norm_lists(tensors, [&](const NormList& list, int blocks) {
    SEP_CUDA_CHECK(launch_list_scale(list, sums, count, norm, static_cast<float>(max_norm), blocks, stream));
  });
}

void changed(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// Tensors that will be scaled in place: dense ones themselves; others through contiguous copies that go back afterwards.
struct InPlace {
  TensorList work;
  std::deque<at::Tensor> copies;
  std::vector<const at::Tensor*> back;             // whose copies they are
  InPlace(const TensorList& tensors, const at::Device& device) {
    Ranges::List ranges;
    work.reserve(tensors.size());
    ranges.reserve(tensors.size());
    for (const at::Tensor* t : tensors) {
      SEP_ASSERT(usable(*t, device), kListMessage);
      if (t->numel() == 0) continue;
      if (t->is_non_overlapping_and_dense()) {
        ranges.push_back(Ranges::of(*t));
        work.push_back(t);
      } else {
        for (int64_t d = 0; d < t->dim(); ++d)
          SEP_ASSERT(t->size(d) <= 1 || t->stride(d) != 0, "an expanded tensor cannot be changed in place");
        copies.push_back(t->detach().contiguous());
        back.push_back(t);
        work.push_back(&copies.back());
      }
    }
    Ranges r;
    r.add(std::move(ranges));
    r.check();
  }
  void finish(const TensorList& tensors) {
    for (size_t i = 0; i < back.size(); ++i) back[i]->detach().copy_(copies[i]);
    for (const at::Tensor* t : tensors) changed(*t);
  }
};

// The device of a list; the current one for an empty list.
at::Device device_of(const TensorList& tensors) {
  if (tensors.empty()) return at::Device(at::kCUDA, c10::cuda::current_device());
  SEP_ASSERT(tensors[0]->defined() && tensors[0]->is_cuda(), kListMessage);
  return tensors[0]->device();
}

void check_max_norm(double max_norm) { SEP_ASSERT(max_norm >= 0.0, "max_norm must not be negative"); }

}  // namespace

std::pair<at::Tensor, at::Tensor> list_norm(const TensorList& tensors) {
  const at::Device device = device_of(tensors);
  const auto options = at::TensorOptions().device(device);
  const c10::cuda::CUDAGuard guard(device);
  const Readable r(tensors, device);
  if (r.list.empty()) return {at::zeros({}, options.dtype(at::kFloat)), at::zeros({}, options.dtype(at::kDouble))};
  const auto stream = at::cuda::getCurrentCUDAStream();
  const at::Tensor norm = at::empty({}, options.dtype(at::kFloat)), total = at::empty({}, options.dtype(at::kDouble));
  int count = 0;
  const at::Tensor sums = squares(r.list, stream, count);
  SEP_CUDA_CHECK(launch_list_norm(sums.data_ptr<double>(), count, norm.data_ptr<float>(), total.data_ptr<double>(), stream));
  return {norm, total};
}

at::Tensor list_clip(const TensorList& tensors, double max_norm) {
  check_max_norm(max_norm);
  const at::Device device = device_of(tensors);
  const auto options = at::TensorOptions().device(device).dtype(at::kFloat);
  const c10::cuda::CUDAGuard guard(device);
  InPlace list(tensors, device);
  if (list.work.empty()) return at::zeros({}, options);
  const auto stream = at::cuda::getCurrentCUDAStream();
  const at::Tensor norm = at::empty({}, options);
  int count = 0;
  const at::Tensor sums = squares(list.work, stream, count);
  scale_lists(list.work, sums.data_ptr<double>(), count, norm.data_ptr<float>(), max_norm, stream);
  list.finish(tensors);
  return norm;
}

void list_scale(const TensorList& tensors, const at::Tensor& norm, double max_norm) {
  check_max_norm(max_norm);
  if (tensors.empty()) return;
  const at::Device device = device_of(tensors);
  SEP_ASSERT(norm.device() == device && norm.scalar_type() == at::kFloat && norm.numel() == 1, "norm must be one float32 number on the tensors' device");
  const c10::cuda::CUDAGuard guard(device);
  InPlace list(tensors, device);
  if (list.work.empty()) return;
  scale_lists(list.work, nullptr, 0, norm.data_ptr<float>(), max_norm, at::cuda::getCurrentCUDAStream());
  list.finish(tensors);
}

void list_adamw(const TensorList& params, const TensorList& grads, const TensorList& exp_avgs, const TensorList& exp_avg_sqs,
                const TensorList& masters, const std::optional<at::Tensor>& norm, const AdamOptions& o) {
  const size_t n = params.size();
  SEP_ASSERT(grads.size() == n && exp_avgs.size() == n && exp_avg_sqs.size() == n && (masters.empty() || masters.size() == n),
             "params, grads, exp_avgs, exp_avg_sqs and masters must be lists of one length");
  SEP_ASSERT(o.device_step.has_value() || o.step >= 1, "step counts from 1");
  SEP_ASSERT(o.lr >= 0.0 && o.eps >= 0.0 && o.weight_decay >= 0.0 && o.beta1 >= 0.0 && o.beta1 < 1.0 && o.beta2 >= 0.0 && o.beta2 < 1.0,
             "lr, eps and weight_decay must not be negative, betas within [0, 1)");
  if (n == 0) return;
  const at::Device device = device_of(params);
  if (norm.has_value())
    SEP_ASSERT(norm->device() == device && norm->scalar_type() == at::kFloat && norm->numel() == 1, "norm must be one float32 number on the parameters' device");
  if (o.device_step.has_value())
    SEP_ASSERT(o.device_step->device() == device && o.device_step->scalar_type() == at::kLong && o.device_step->numel() == 1,
               "a step that is a tensor must be one int64 number on the parameters' device");
  const c10::cuda::CUDAGuard guard(device);
  const bool have_masters = !masters.empty();
  std::deque<at::Tensor> held;                       // gradients that had to be laid out like their parameters
  TensorList grad_at = grads;
  Ranges::List ranges[4];
  for (Ranges::List& r : ranges) r.reserve(n);
  int64_t elements = 0;
  for (size_t i = 0; i < n; ++i) {
    const at::Tensor &p = *params[i], &g = *grads[i];
    SEP_ASSERT(usable(p, device) && usable(g, device), kListMessage);
    SEP_ASSERT(g.sizes() == p.sizes(), "a gradient does not have its parameter's shape");
    SEP_ASSERT(p.is_non_overlapping_and_dense(), "a parameter with gaps or repeats in memory cannot be updated in place");
    const bool plain = p.is_contiguous();
    auto same_layout = [&](const at::Tensor& t) { return plain ? t.is_contiguous() : t.strides() == p.strides(); };
    auto state = [&](const at::Tensor& t, const char* what, Ranges::List& r) {
      SEP_ASSERT(usable(t, device) && t.scalar_type() == at::kFloat && t.sizes() == p.sizes() && same_layout(t),
                 what << " must be float32 and laid out like their parameters");
      if (t.numel() > 0) r.push_back(Ranges::of(t));
    };
    state(*exp_avgs[i], "exp_avgs", ranges[1]);
    state(*exp_avg_sqs[i], "exp_avg_sqs", ranges[2]);
    if (have_masters) state(*masters[i], "masters", ranges[3]);
    if (!same_layout(g)) {
      held.push_back(at::empty_strided(p.sizes(), p.strides(), g.options()));
      held.back().copy_(g.detach());
      grad_at[i] = &held.back();
    }
    elements += p.numel();
    if (p.numel() > 0) ranges[0].push_back(Ranges::of(p));
  }
  Ranges written;
  for (Ranges::List& r : ranges) written.add(std::move(r));
  written.check();
  AdamParams a{};
  if (o.device_step.has_value()) {
    a.step = reinterpret_cast<const long long*>(o.device_step->data_ptr<int64_t>());
    a.lr = static_cast<float>(o.lr);
    a.log_beta1 = std::log(o.beta1); a.log_beta2 = std::log(o.beta2);
  } else {
    const double c1 = 1.0 - std::pow(o.beta1, static_cast<double>(o.step)), c2 = 1.0 - std::pow(o.beta2, static_cast<double>(o.step));
    a.step_size = static_cast<float>(o.lr / c1);
    a.inv_sqrt_correction = static_cast<float>(1.0 / std::sqrt(c2));
  }
  a.beta1 = static_cast<float>(o.beta1); a.one_minus_beta1 = static_cast<float>(1.0 - o.beta1);
  a.beta2 = static_cast<float>(o.beta2); a.one_minus_beta2 = static_cast<float>(1.0 - o.beta2);
  a.eps = static_cast<float>(o.eps); a.keep = static_cast<float>(1.0 - o.lr * o.weight_decay);
  a.norm = norm.has_value() ? norm->data_ptr<float>() : nullptr;
  a.max_norm = static_cast<float>(o.max_norm); a.skip_nonfinite = o.skip_nonfinite ? 1 : 0;
  const auto stream = at::cuda::getCurrentCUDAStream();
  const int most = num_sms() * kAdamBlocksPerSm;
  AdamList list;
  // Long lists with master copies: chunks of one vector a thread, dealt out in turn, so that the blocks that run together read and write one
  // window of each of the seven arrays and not 296: 411 M elements 1948 -> 1841 us, 20 M in 400 tensors 108 -> 100 (any larger
  // chunk or window 1926 to 1948).  Not without masters, where the arrays are of one width and such windows meet in the same DRAM banks (203 M
  // elements fp32 1033 -> 1137 us, bf16 812 -> 977).  Short lists: a run of chunks for every block, one search for each: 250 tensors of 5 M
  // elements in all, 101 -> 90.
  const bool in_turn = have_masters && elements >= 8'000'000;
  list.chunk = in_turn ? 4 * kListThreads : chunk_of(elements, most);
  list.count = 0;
  int64_t chunks = 0;
  auto flush = [&] {
    if (list.count == 0) return;
    list.first[list.count] = list.chunks = static_cast<int>(chunks);
    list.window = in_turn ? 1 : static_cast<int>((chunks + most - 1) / most);
    SEP_CUDA_CHECK(launch_list_adamw(list, a, static_cast<int>(std::min<int64_t>(most, chunks)), stream));
    list.count = 0; chunks = 0;
  };
  for (size_t i = 0; i < n; ++i) {
    const at::Tensor &p = *params[i], &g = *grad_at[i];
    if (p.numel() == 0) continue;
    if (list.count == kAdamEntries) flush();
    const int at = list.count++;
    list.param[at] = p.data_ptr();
    list.grad[at] = g.data_ptr();
    list.exp_avg[at] = static_cast<float*>(exp_avgs[i]->data_ptr());
    list.exp_avg_sq[at] = static_cast<float*>(exp_avg_sqs[i]->data_ptr());
    list.master[at] = have_masters ? static_cast<float*>(masters[i]->data_ptr()) : nullptr;
    // the first element at which all of them stand on a boundary of four elements
    auto place = [](const void* q, int width) { return static_cast<int>(reinterpret_cast<uintptr_t>(q) / width % 4); };
    const int off = place(list.exp_avg[at], 4);
    const bool together = place(list.param[at], is_half(p) ? 2 : 4) == off && place(list.grad[at], is_half(g) ? 2 : 4) == off &&
                          place(list.exp_avg_sq[at], 4) == off && (!have_masters || place(list.master[at], 4) == off);
    const int lead = together ? (4 - off) % 4 : 0;
    const unsigned long long flags = (is_half(p) ? kListHalf : 0) | (is_half(g) ? kListGradHalf : 0) | (together ? 0 : kListScalar) |
                                     (static_cast<unsigned long long>(lead) << kListHeadShift);
    list.length[at] = static_cast<unsigned long long>(p.numel()) | (flags << kListTypeShift);
    list.first[at] = static_cast<int>(chunks);
    chunks += std::max<int64_t>(1, (p.numel() - lead + list.chunk - 1) / list.chunk);
    SEP_ASSERT(chunks < (1ll << 31), "the list is too large");
  }
  flush();
  for (const TensorList* l : {&params, &exp_avgs, &exp_avg_sqs, &masters})
    for (const at::Tensor* t : *l) changed(*t);
}

}  // namespace sep

// Operators of a training step around the MoE layer, host side: the loss over the vocabulary (linear_loss.cpp), and lists
// of tensors (list_ops.cpp): gradients' norm and clipping, AdamW.
#pragma once

#include <functional>
#include <optional>
#include <string>
#include <utility>
#include <vector>

#include <cuda_runtime.h>
#include <torch/types.h>

#include "status.h"

namespace sep {

// What an operator takes from the Runtime it reports into.
struct LaunchContext {
  StatusBlock* status;
  unsigned long long wait_budget_ns;
  int rank, sms, device;
  cudaStream_t stream;           // the current one
};
using ContextFn = std::function<LaunchContext(int launches)>;   // `launches`: how many kernels the caller is about to launch

enum LossReduction : int { kLossNone = 0, kLossMean = 1, kLossSum = 2 };
// x [T, H], weight [V, H] bf16, targets [T] int64; differentiable in x and weight.  `piece_bytes`: what a piece of the backward may take (0: the
// plan's own limit; tests give less, so that small calls have many pieces)
at::Tensor linear_loss(const ContextFn& context, const at::Tensor& x, const at::Tensor& weight, const at::Tensor& targets,
                       int64_t ignore_index, int reduction, int64_t piece_bytes);
// The backward's units in order, for the schedule's test: each {kind, piece, unit row, unit column, split, first k-block, k-blocks};
// first of all {pieces, columns of a piece, splits, ahead, buffers, row units, split2, column tiles of a dw unit}.
std::vector<std::vector<int>> linear_loss_schedule(int64_t tokens, int64_t hidden, int64_t vocab, int sms, bool want_dx, bool want_dw,
                                                   int64_t piece_bytes);

// Tensors that the caller (a Python list) keeps alive during the call.
using TensorList = std::vector<const at::Tensor*>;
// {norm (fp32), sum of squares (fp64)}, 0-dim
std::pair<at::Tensor, at::Tensor> list_norm(const TensorList& tensors);
at::Tensor list_clip(const TensorList& tensors, double max_norm);
void list_scale(const TensorList& tensors, const at::Tensor& norm, double max_norm);
struct AdamOptions {
  int64_t step;
  std::optional<at::Tensor> device_step;           // instead of `step`: one int64 on the device
  double lr, beta1, beta2, eps, weight_decay;
  double max_norm;               // < 0: no clipping
  bool skip_nonfinite;
};
void list_adamw(const TensorList& params, const TensorList& grads, const TensorList& exp_avgs, const TensorList& exp_avg_sqs,
                const TensorList& masters, const std::optional<at::Tensor>& norm, const AdamOptions& o);

}  // namespace sep

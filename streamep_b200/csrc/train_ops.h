// Operators of a training step around the MoE layer, host side: the loss over the vocabulary (linear_loss.cpp).
#pragma once

#include <functional>
#include <string>
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
// x [T, H], weight [V, H] bf16, targets [T] int64; differentiable in x and weight
at::Tensor linear_loss(const ContextFn& context, const at::Tensor& x, const at::Tensor& weight, const at::Tensor& targets,
                       int64_t ignore_index, int reduction);
// The backward's units in order, for the schedule's test: each {kind, piece, unit row, unit column, split, first k-block, k-blocks};
// first of all {pieces, columns of a piece, splits, ahead, buffers, row units, split2}.
std::vector<std::vector<int>> linear_loss_schedule(int64_t tokens, int64_t hidden, int64_t vocab, int sms, bool want_dx, bool want_dw);

}  // namespace sep

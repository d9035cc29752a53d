// Normalisation of rows: launches of norm_kernels.cu.
#pragma once

#include <cuda_runtime.h>

namespace sep {

enum NormType : int { kNormNone = 0, kNormHalf = 1, kNormFloat = 2 };   // an array that is not there, bf16, fp32

struct NormParams {
  int type;                      // of rows: x, residual, y, sum and their gradients
  int weight_type;               // of weight and bias (kNormNone: neither)
  int center;                    // 1: subtract the mean (layer norm), 0: root mean square only
  long long rows;
  int hidden;
  float eps;
  const void* x;                 // [rows, hidden], rows `x_stride` elements apart
  const void* residual;          // the same, or null
  long long x_stride, residual_stride;
  const void* weight;            // [hidden] or null
  const void* bias;              // [hidden] or null
  void* y;                       // [rows, hidden] contiguous
  void* sum;                     // [rows, hidden] contiguous: x + residual (null without one)
  float2* stats;                 // [rows] (mean, 1 / deviation) or null
};
cudaError_t launch_norm_forward(const NormParams& p, int sms, cudaStream_t stream);

struct NormGradParams {
  int type, weight_type, center;
  long long rows;
  int hidden;
  const void* x;
  const void* residual;          // or null
  const void* dy;
  const void* dsum;              // the sum's own gradient, or null
  long long x_stride, residual_stride, dy_stride, dsum_stride;
  const void* weight;
  const float2* stats;
  void* dx;                      // [rows, hidden] contiguous
  void* dweight;                 // [hidden] or null
  void* dbias;                   // [hidden] or null
  float* parts;                  // [2][norm_parts][hidden] sums of the blocks' rows
};
// How many blocks leave sums of their own for the gradients of weight and bias.
int norm_parts(const NormGradParams& p, int sms);
cudaError_t launch_norm_backward(const NormGradParams& p, int sms, cudaStream_t stream);

}  // namespace sep

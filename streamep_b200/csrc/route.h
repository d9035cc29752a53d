// Routing that is trained: statistics of the router's probabilities, and its gradients (route_kernels.cu).
#pragma once

#include <cuda_runtime.h>

namespace sep {

struct RouteStatsParams {
  int tokens, experts, top_k;
  const float* probs;            // [tokens, experts]
  const float* lse;              // [tokens]
  const long long* idx;          // [tokens, top_k]
  const unsigned char* mask;     // [tokens] or null: tokens that count
  int blocks;                    // route_stats_blocks()
  float* prob_parts;             // [blocks][experts] sums over a block's tokens
  int* count_parts;              // [blocks][experts]
  float2* other_parts;           // [blocks] (sum of lse^2, bits of the number of tokens that count)
  float* balance;                // one number each
  float* z;
  long long* counts;             // [experts]
  float* load;                   // [experts + 1]: experts * counts / (top_k * n); behind them 1 / n (0 without any that count)
};
int route_stats_blocks(int tokens, int sms);
cudaError_t launch_route_stats(const RouteStatsParams& p, cudaStream_t stream);

struct RouteGradParams {
  int tokens, experts, top_k, hidden, renormalize;
  const float* probs;
  const float* lse;
  const long long* idx;
  const float* weights;          // [tokens, top_k]
  const unsigned char* mask;
  const float* load;
  const float* dweights;         // [tokens, top_k] or null
  const float* dbalance;         // one number or null
  const float* dz_loss;          // one number or null
  float* dlogits;                // [tokens, experts]
  const void* x;                 // [tokens, hidden] bf16
  const void* w_gate;            // [experts, hidden] bf16
  void* dx;                      // or null
  void* dw;                      // or null
};
cudaError_t launch_route_backward(const RouteGradParams& p, cudaStream_t stream);

}  // namespace sep

// Routing that is trained: statistics of the router's probabilities, and its gradients (route_kernels.cu, route_grad_kernels.cu).
#pragma once

#include <cuda_runtime.h>

#include "api.h"
#include "status.h"

namespace sep {

struct RouteStatsParams {
  int experts, top_k;
  const unsigned char* mask;     // [tokens] or null: tokens that count
  int blocks;                    // RouteTile::grid (0 without tokens)
  float2* parts;                 // [blocks][experts] (sum of probabilities, bits of the count)
  float2* other_parts;           // [blocks] (sum of lse^2, bits of the number of tokens that count)
  float* balance;                // one number each
  float* z;
  long long* counts;             // [experts]
  float* load;                   // [experts + 1]: experts * counts / (top_k * n); behind them 1 / n (0 without any that count)
};
struct RouteTile : RouterTile {
  int pairs;                     // 1: blocks multiply in pairs
  int grid;
};
RouteTile route_tile(const RouterParams& p, int sms);
// Maps as for the router (api.h); all outputs of `p`, probs and lse too.
cudaError_t launch_route_forward(const RouterParams& p, const RouteStatsParams& s, const void* map_w, const void* map_x, int sms, StatusBlock* status, unsigned long long wait_budget_ns,
                                 cudaStream_t stream);

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
  void* dz;                      // [layers, tokens, padded] bf16: the logits' gradients, or null (no dw)
  void* dx;                      // [tokens, hidden] bf16, or null
  void* dw;                      // [experts, hidden] bf16, or null
  StatusBlock* status;
  int rank;
  unsigned long long wait_budget_ns;
};
// How the products are cut up: `padded` experts (a multiple of 64), in `layers` matrices; blocks that share the columns of 128 tokens' dx; experts (in blocks of 128) and parts of
// the tokens of a unit of dW.
struct RouteGradPlan {
  int padded, layers;            // of dz: bf16 numbers that add up to it
  int dx_pairs, dx_splits, dx_stages, dx_staging, dx_smem;
  int dw_pairs, dw_blocks, dw_splits, dw_units, dw_stages, dw_smem;             // (units: as blocks of the grid)
};
RouteGradPlan route_grad_plan(int tokens, int hidden, int experts, int sms);
// Maps: `map_w` [E, H] boxes of 64 x 64, `map_dx` [T, H] boxes of 32 rows x 64; `map_dz` [layers, T, padded] and `map_x` [T, H] boxes of 64 x 64; `map_out` dW boxes of
// 32 x 64 (bf16), or with several parts [splits, E, H] fp32 boxes of 32 x 32 over `parts`.  All with 128-byte swizzle.
cudaError_t launch_route_dx(const RouteGradParams& p, const RouteGradPlan& g, const void* map_w, const void* map_dx, cudaStream_t stream);
cudaError_t launch_route_dw(const RouteGradParams& p, const RouteGradPlan& g, const void* map_dz, const void* map_x, const void* map_out, float* parts, cudaStream_t stream);

}  // namespace sep

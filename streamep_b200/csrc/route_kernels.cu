// Routing that is trained: from the router's probabilities p = softmax(z), z = x W^T, and its choice of top_k experts a token
//
//   counts_e = tokens (that count: n) that chose e,   load_e = E counts_e / (top_k n)
//   balance = sum_e load_e mean_t p_te,   z_loss = mean_t logsumexp(z_t)^2
//
// and the gradients of both and of the weights w:
//
//   dz_t = [counts] (db p_t (load - <p_t, load>) + 2 dz_loss lse_t p_t) / n
//          + w (dw - <w, dw>) at the chosen experts where w is the softmax over them, or p (dp - <p, dp>) with dp = dw there
//   dx = dz W,   dW = dz^T x
#include "route.h"

#include "ptx.cuh"

namespace sep {

namespace {

constexpr int kStatThreads = 512;                // one expert a thread
constexpr int kMaxExperts = 512;

__global__ void __launch_bounds__(kStatThreads) route_stats_kernel(const RouteStatsParams p) {
  __shared__ int hist[kMaxExperts];
  const int e = threadIdx.x;
  hist[e] = 0;
  __syncthreads();
  const int begin = static_cast<int>(static_cast<long long>(p.tokens) * blockIdx.x / p.blocks), end = static_cast<int>(static_cast<long long>(p.tokens) * (blockIdx.x + 1) / p.blocks);
  float sum = 0.f, squares = 0.f;
  int live = 0;
  for (int t = begin; t < end; ++t) {
    if (p.mask != nullptr && p.mask[t] == 0) continue;
    if (e < p.experts) sum += p.probs[static_cast<long long>(t) * p.experts + e];
    if (e < p.top_k) atomicAdd(&hist[p.idx[static_cast<long long>(t) * p.top_k + e]], 1);
    const float lse = p.lse[t];
    squares = fmaf(lse, lse, squares);
    ++live;
  }
  __syncthreads();
  if (e < p.experts) {
    p.prob_parts[blockIdx.x * p.experts + e] = sum;
    p.count_parts[blockIdx.x * p.experts + e] = hist[e];
  }
  if (e == 0) p.other_parts[blockIdx.x] = make_float2(squares, __int_as_float(live));
}

__global__ void __launch_bounds__(kStatThreads) route_join_kernel(const RouteStatsParams p) {
  __shared__ float scratch[kStatThreads / 32];
  const int e = threadIdx.x;
  float squares = 0.f;
  int n = 0;
  for (int b = 0; b < p.blocks; ++b) { const float2 o = p.other_parts[b]; squares += o.x; n += __float_as_int(o.y); }
  const float share = n > 0 ? 1.f / static_cast<float>(n) : 0.f;
  float term = 0.f;
  if (e < p.experts) {
    float sum = 0.f;
    long long count = 0;
    for (int b = 0; b < p.blocks; ++b) { sum += p.prob_parts[b * p.experts + e]; count += p.count_parts[b * p.experts + e]; }
    const float load = static_cast<float>(static_cast<double>(count) * p.experts / p.top_k) * share;
    p.counts[e] = count;
    p.load[e] = load;
    term = load * (sum * share);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) term += __shfl_xor_sync(0xffffffffu, term, o);
  if ((e & 31) == 0) scratch[e >> 5] = term;
  __syncthreads();
  if (e != 0) return;
  float balance = 0.f;
  for (int w = 0; w < kStatThreads / 32; ++w) balance += scratch[w];
  *p.balance = balance;
  *p.z = squares * share;
  p.load[p.experts] = share;
}

}  // namespace

int route_stats_blocks(int tokens, int sms) {
  const int most = (tokens + 15) / 16;
  return most < sms ? most : sms;
}

cudaError_t launch_route_stats(const RouteStatsParams& p, cudaStream_t stream) {
  if (p.blocks > 0) route_stats_kernel<<<p.blocks, kStatThreads, 0, stream>>>(p);
  route_join_kernel<<<1, kStatThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace sep

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

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// One warp a token.
__global__ void __launch_bounds__(256) route_dlogits_kernel(const RouteGradParams p) {
  const int t = (blockIdx.x * 256 + threadIdx.x) >> 5, lane = threadIdx.x & 31;
  if (t >= p.tokens) return;
  const float* probs = p.probs + static_cast<long long>(t) * p.experts;
  float* out = p.dlogits + static_cast<long long>(t) * p.experts;
  const bool counts = p.mask == nullptr || p.mask[t] != 0;
  const float share = p.load[p.experts];
  const float cb = counts && p.dbalance != nullptr ? *p.dbalance * share : 0.f;
  const float cz = counts && p.dz_loss != nullptr ? 2.f * *p.dz_loss * share * p.lse[t] : 0.f;
  int e_mine = -1;
  float up = 0.f, w = 0.f;
  if (lane < p.top_k) {
    e_mine = static_cast<int>(p.idx[static_cast<long long>(t) * p.top_k + lane]);
    w = p.weights[static_cast<long long>(t) * p.top_k + lane];
    up = p.dweights != nullptr ? p.dweights[static_cast<long long>(t) * p.top_k + lane] : 0.f;
  }
  float mean_load = 0.f;
  if (cb != 0.f) for (int e = lane; e < p.experts; e += 32) mean_load = fmaf(probs[e], p.load[e], mean_load);
  mean_load = warp_sum(mean_load);
  const float mean_up = warp_sum(lane < p.top_k ? w * up : 0.f);        // (w is p at the chosen experts where it is not normalised again)
  const float at_chosen = p.renormalize ? w * (up - mean_up) : w * up;
  for (int e0 = 0; e0 < p.experts; e0 += 32) {
    const int e = e0 + lane;
    float v = 0.f;
    if (e < p.experts) {
      const float prob = probs[e];
      if (cb != 0.f) v = cb * prob * (p.load[e] - mean_load);
      if (cz != 0.f) v = fmaf(cz, prob, v);
      if (!p.renormalize && p.dweights != nullptr) v = fmaf(-prob, mean_up, v);
    }
    for (int k = 0; k < p.top_k; ++k) {
      const int chosen = __shfl_sync(0xffffffffu, e_mine, k);
      const float add = __shfl_sync(0xffffffffu, at_chosen, k);
      if (chosen == e && p.dweights != nullptr) v += add;
    }
    if (e < p.experts) out[e] = v;
  }
}

// c[m, n] = sum_k a(m, k) b[k, n], 64 x 64 a block, 16 results a thread, a(m, k) = a[k * lda + m] (kTransposed) or a[m * lda + k].
template <bool kTransposed>
__global__ void __launch_bounds__(256) route_product_kernel(const float* a, int lda, const __nv_bfloat16* b, int ldb, __nv_bfloat16* c, int ldc, int M, int N, int K) {
  __shared__ float sa[16][65], sb[16][65];
  const int m0 = blockIdx.y * 64, n0 = blockIdx.x * 64, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < K; k0 += 16) {
    for (int i = threadIdx.x; i < 1024; i += 256) {
      const int kk = kTransposed ? i >> 6 : i & 15, mm = kTransposed ? i & 63 : i >> 4;
      const long long at = kTransposed ? static_cast<long long>(k0 + kk) * lda + m0 + mm : static_cast<long long>(m0 + mm) * lda + k0 + kk;
      sa[kk][mm] = k0 + kk < K && m0 + mm < M ? a[at] : 0.f;
      const int kb = i >> 6, nn = i & 63;
      sb[kb][nn] = k0 + kb < K && n0 + nn < N ? __bfloat162float(b[static_cast<long long>(k0 + kb) * ldb + n0 + nn]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sa[k][ty + i * 16], sb[k][tx + j * 16], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int m = m0 + ty + i * 16, n = n0 + tx + j * 16;
      if (m < M && n < N) c[static_cast<long long>(m) * ldc + n] = __float2bfloat16_rn(acc[i][j]);
    }
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

cudaError_t launch_route_backward(const RouteGradParams& p, cudaStream_t stream) {
  route_dlogits_kernel<<<(p.tokens + 7) / 8, 256, 0, stream>>>(p);
  const int columns = (p.hidden + 63) / 64;
  if (p.dx != nullptr)
    route_product_kernel<false><<<dim3(columns, (p.tokens + 63) / 64), 256, 0, stream>>>(
        p.dlogits, p.experts, static_cast<const __nv_bfloat16*>(p.w_gate), p.hidden, static_cast<__nv_bfloat16*>(p.dx), p.hidden, p.tokens, p.hidden, p.experts);
  if (p.dw != nullptr)
    route_product_kernel<true><<<dim3(columns, (p.experts + 63) / 64), 256, 0, stream>>>(
        p.dlogits, p.experts, static_cast<const __nv_bfloat16*>(p.x), p.hidden, static_cast<__nv_bfloat16*>(p.dw), p.hidden, p.experts, p.hidden, p.tokens);
  return cudaGetLastError();
}

}  // namespace sep

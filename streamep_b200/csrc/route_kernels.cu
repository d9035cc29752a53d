// Routing that is trained: the router's product and choice with what its losses need.
//
//   z = x W^T,  p = softmax(z),  the top_k experts of each token and their weights
//   counts_e = tokens (that count: n) that chose e,   load_e = E counts_e / (top_k n)
//   balance = sum_e load_e mean_t p_te,   z_loss = mean_t logsumexp(z_t)^2
//
// One kernel multiplies, chooses, leaves p and the logsumexp for the backward and adds up its tokens' probabilities, counts and squares; a small one adds
// up the blocks' sums, in one order (a repeated call gives the same bits).
//
// What bounds it: reading x once (HBM), for many experts what the SMs read from L2, and the choice (16384 tokens of 256 experts: 1.1 us for each one chosen).
#include <algorithm>
#include <atomic>
#include <cuda.h>
#include <type_traits>

#include "api.h"
#include "ptx.cuh"
#include "route.h"

namespace sep {

namespace {

constexpr int kThreads = 512;
constexpr int kBK = 64;
// The tensor cores cut off what an accumulator cannot hold instead of rounding, so it starts anew every 256 elements of the reduction and the
// segments are added up in registers: with one accumulator over 7168 elements the z loss came out 6e-6 too small, with segments 2e-7 off.
constexpr int kSegment = 4;                      // k-blocks
constexpr int kDrainFirst = 4, kDrainers = 12;   // warps that take the segments' sums: three for each quarter of the accumulator's lanes
constexpr int kMostChunks = 6;                   // of 16 columns, of up to 256, for one of the three
constexpr int kMaxStages = 8, kMaxSplits = 8, kMostExperts = 512;
__host__ __device__ constexpr int e_pad_of(int experts) { return (experts + 127) / 128 * 128 + 1; }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// What a warp adds up over its tokens.
template <int EPL> struct Sums { float probs[EPL], squares; int live; };

// One warp finishes N tokens side by side (t[i]; those that `there` are) from their fp32 logits: softmax, the top_k by repeated arg-max (ties: lowest expert), weights,
// ranks, sums.
template <int EPL, int N, class Row>
__device__ __forceinline__ void finish_tokens(const RouterParams& p, const RouteStatsParams& s, Row row, const int (&t)[N], const bool (&there)[N], int lane, int* hist, Sums<EPL>& sums) {
  const int E = p.num_experts, K = p.num_topk;
  float v[N][EPL], top[N], sum[N], inv[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    top[i] = -INFINITY;
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      const int e = j * 32 + lane;
      v[i][j] = e < E ? (there[i] ? row(i, e) : 0.f) : -INFINITY;
      top[i] = fmaxf(top[i], v[i][j]);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
#pragma unroll
  for (int i = 0; i < N; ++i) {
    sum[i] = 0.f;
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      v[i][j] = j * 32 + lane < E ? expf(v[i][j] - top[i]) : 0.f;
      sum[i] += v[i][j];
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], o);
  bool counts[N];
  unsigned key[N][EPL];          // probability bits + 1, which order like the values (0: taken, or no such expert)
#pragma unroll
  for (int i = 0; i < N; ++i) {
    inv[i] = 1.f / sum[i];
    const float lse = top[i] + logf(sum[i]);
    counts[i] = there[i] && (s.mask == nullptr || s.mask[t[i]] != 0);
#pragma unroll
    for (int j = 0; j < EPL; ++j) {
      const int e = j * 32 + lane;
      const float prob = v[i][j] * inv[i];
      if (e < E && there[i]) p.probs[static_cast<size_t>(t[i]) * E + e] = prob;
      if (counts[i]) sums.probs[j] += prob;
      key[i][j] = e < E ? __float_as_uint(prob) + 1u : 0u;
    }
    if (counts[i]) { sums.squares = fmaf(lse, lse, sums.squares); ++sums.live; }
    if (lane == 0 && there[i]) p.lse[t[i]] = lse;
  }
  float wsum[N], my_w[N];
  int my_e[N];
#pragma unroll
  for (int i = 0; i < N; ++i) { wsum[i] = my_w[i] = 0.f; my_e[i] = 0; }
  for (int k = 0; k < K; ++k) {
    unsigned most[N];
    int e[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      unsigned best = 0;
#pragma unroll
      for (int j = 0; j < EPL; ++j) best = max(best, key[i][j]);
      most[i] = __reduce_max_sync(0xffffffffu, best);
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      unsigned mine = 0x7fffffffu;
#pragma unroll
      for (int j = EPL - 1; j >= 0; --j)
        if (key[i][j] == most[i]) mine = j * 32 + lane;
      e[i] = static_cast<int>(__reduce_min_sync(0xffffffffu, mine));
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
      for (int j = 0; j < EPL; ++j)
        if (j * 32 + lane == e[i]) key[i][j] = 0;
      const float w = __uint_as_float(most[i] - 1u);
      if (lane == k) { my_w[i] = w; my_e[i] = e[i]; }
      wsum[i] += w;
    }
  }
  const int e_local = E / p.num_ranks;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const unsigned ranks = __reduce_or_sync(0xffffffffu, lane < K ? 1u << my_e[i] / e_local : 0u);
    if (!there[i]) continue;
    if (lane < K) {
      p.topk_idx[static_cast<size_t>(t[i]) * K + lane] = my_e[i];
      p.topk_weights[static_cast<size_t>(t[i]) * K + lane] = p.renormalize ? my_w[i] / wsum[i] : my_w[i];
      if (counts[i]) atomicAdd(&hist[my_e[i]], 1);             // (whole numbers: the order does not matter)
    }
    if (lane < p.num_ranks) p.is_token_in_rank[static_cast<size_t>(t[i]) * p.num_ranks + lane] = (ranks >> lane) & 1u;
  }
}

// A unit of `g.tile_tokens` tokens belongs to a cluster of `splits` blocks; each multiplies its share of the hidden dimension, W (experts, 128 per
// accumulator) times the tokens (16 to 128 columns), and leaves its partial logits in shared memory; then every block of the cluster finishes its
// share of the tokens, adding the partial sums over distributed shared memory.
// CG = 2: no splits; the blocks of a pair multiply their 2 x 128 tokens with 256 experts together, each with half of W in its shared memory, and each then has the logits of half
// of the experts for the tokens of both, of which it hands the other's over.  What the SMs
// read from L2 bounds long rows: x once and W for every 128 tokens, or 256 (16384 tokens, hidden 7168, 256 experts: 92.4 -> 78.5 us).
template <int EPL, int CG>
__global__ void __launch_bounds__(kThreads, 1) route_forward_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const RouterParams p,
                                                                    const RouteStatsParams s, const RouteTile g, StatusBlock* status, unsigned long long budget) {
  extern __shared__ unsigned char smem_dyn[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full_bar[kMaxStages], empty_bar[kMaxStages], tmem_full[2], tmem_empty[2];
  __shared__ uint32_t s_tmem;
  __shared__ int hist[kMostExperts];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = static_cast<int>(blockIdx.x) % g.splits, tile = static_cast<int>(blockIdx.x) / g.splits;
  const int rank = CG == 2 ? static_cast<int>(cluster_ctarank()) : 0;
  const bool leader = rank == 0;
  const int n = g.tile_tokens, nb = g.blocks, set = nb * n;    // (of a pair: one block of experts and twice the tokens)
  const int own_blocks = nb / CG;                // of experts, in this block's shared memory
  const int k_blocks = (p.hidden + kBK - 1) / kBK;
  const int kb0 = k_blocks * split / g.splits, kb1 = k_blocks * (split + 1) / g.splits;
  const int segments = (kb1 - kb0 + kSegment - 1) / kSegment;
  const int stage_bytes = own_blocks * 128 * 128 + n * 128;
  int tmem_cols = 32;
  while (tmem_cols < 2 * set) tmem_cols *= 2;
  grid_release();
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&map_w);
    tma_prefetch_desc(&map_x);
    for (int i = 0; i < g.stages; ++i) { mbar_init(&full_bar[i], 1); mbar_init(&empty_bar[i], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&tmem_full[i], 1); mbar_init(&tmem_empty[i], kDrainers * CG); }
    mbar_fence_init();
  }
  if (warp == 1) { tmem_alloc<CG>(&s_tmem, tmem_cols); tmem_relinquish<CG>(); }
  hist[threadIdx.x] = 0;
  tc_fence_before_sync();
  if constexpr (CG == 2) cluster_sync(); else __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = s_tmem;
  bool ok = true;
  float acc[kMostChunks][16];
#pragma unroll
  for (int i = 0; i < kMostChunks; ++i)
#pragma unroll
    for (int c = 0; c < 16; ++c) acc[i][c] = 0.f;
  const int quarter = warp & 3, third = (warp - kDrainFirst) >> 2, chunks = set / 16;
  if (warp == 0) {
    if (lane == 0) {
      int stage = 0; uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&empty_bar[stage], phase ^ 1, budget, status)) { ok = false; break; }
        unsigned char* at = smem + stage * stage_bytes;
        if constexpr (CG == 2) {                 // (the bytes of both are counted on the first one's barrier)
          if (leader) mbar_arrive_expect_tx(&full_bar[stage], 2 * stage_bytes);
          const uint32_t bar = cluster_map(&full_bar[stage], 0);
          tma_load_3d_pair(at, &map_w, bar, kb * kBK, rank * 128, 0);
          tma_load_3d_pair(at + 128 * 128, &map_x, bar, kb * kBK, tile * n, 0);
        } else {
          mbar_arrive_expect_tx(&full_bar[stage], stage_bytes);
          for (int b = 0; b < nb; ++b) tma_load_3d(at + b * 128 * 128, &map_w, &full_bar[stage], kb * kBK, b * 128, 0);
          tma_load_3d(at + nb * 128 * 128, &map_x, &full_bar[stage], kb * kBK, tile * n, 0);
        }
        if (++stage == g.stages) { stage = 0; phase ^= 1; }
      }
      if (!ok) {
        report_failure(status, kStatusTimeoutPipeline, kKernelRoute, 6, 0, tile, split, 0);
        const unsigned long long t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 2000000ull) {}          // copies in flight land before the block leaves (bounded)
      }
    }
  } else if (warp == 1 && leader) {
    const uint32_t idesc = umma_idesc_bf16(128 * CG, 0, 0, 0) | (static_cast<uint32_t>(n * CG >> 3) << 17);
    int stage = 0; uint32_t phase = 0;
    for (int q = 0; q < segments && ok; ++q) {
      const int first = kb0 + q * kSegment, last = min(first + kSegment, kb1);
      if (!__all_sync(0xffffffffu, mbar_wait<CG == 2>(&tmem_empty[q & 1], ((q >> 1) & 1) ^ 1, budget, status))) { ok = false; break; }
      tc_fence_after_sync();
      for (int kb = first; kb < last; ++kb) {
        if (!__all_sync(0xffffffffu, mbar_wait<CG == 2>(&full_bar[stage], phase, budget, status))) { ok = false; break; }
        tc_fence_after_sync();
        if (elect_one()) {
          const uint32_t a = smem_u32(smem + stage * stage_bytes), b = a + own_blocks * 128 * 128;
          for (int m = 0; m < own_blocks; ++m)
#pragma unroll
            for (int j = 0; j < kBK / 16; ++j)
              umma_bf16_ss<CG>(tmem + (q & 1) * set + m * n, umma_smem_desc(a + m * 128 * 128 + j * 32, 16, 1024), umma_smem_desc(b + j * 32, 16, 1024), idesc,
                              (kb > first || j > 0) ? 1u : 0u);
          umma_commit<CG>(&empty_bar[stage]);
          if (kb == last - 1) umma_commit<CG>(&tmem_full[q & 1]);
        }
        __syncwarp();
        if (++stage == g.stages) { stage = 0; phase ^= 1; }
      }
    }
    if (!ok && lane == 0) report_failure(status, kStatusTimeoutPipeline, kKernelRoute, 7, 0, tile, split, 0);
  } else if (warp >= kDrainFirst) {
    // accumulator lane = expert within its block of 128, column = token (of a pair: of 256)
    for (int q = 0; q < segments; ++q) {
      if (!__all_sync(0xffffffffu, mbar_wait(&tmem_full[q & 1], (q >> 1) & 1, budget, status))) { ok = false; break; }
      tc_fence_after_sync();
#pragma unroll
      for (int i = 0; i < kMostChunks; ++i) {
        const int c = third + i * 3;
        if (c >= chunks) break;
        uint32_t r[16];
        tmem_ld_32x16(tmem + (static_cast<uint32_t>(quarter * 32) << 16) + (q & 1) * set + c * 16, r);
        tmem_ld_wait();
#pragma unroll
        for (int k = 0; k < 16; ++k) acc[i][k] += __uint_as_float(r[k]);
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        if constexpr (CG == 2) mbar_arrive_cluster(cluster_map(&tmem_empty[q & 1], 0)); else mbar_arrive(&tmem_empty[q & 1]);
      }
    }
    if (!ok && lane == 0) report_failure(status, kStatusTimeoutPipeline, kKernelRoute, 8, 0, tile, split, 0);
  }
  __syncwarp();
  const int e_pad = e_pad_of(p.num_experts);
  float* logits = reinterpret_cast<float*>(smem);              // the operand ring is free once the products are done
  ok = __syncthreads_and(ok ? 1 : 0) != 0;
  if (ok && warp >= kDrainFirst) {
#pragma unroll
    for (int i = 0; i < kMostChunks; ++i) {
      const int c = third + i * 3;
      if (c >= chunks) break;
      const int block = c * 16 / n, token = c * 16 - block * n;
      if constexpr (CG == 2) {                   // (the products, and with them the other's ring, are done: so said the last accumulator)
        const uint32_t at = cluster_map(&logits[token * e_pad + rank * 128 + quarter * 32 + lane], block);
#pragma unroll
        for (int k = 0; k < 16; ++k) st_cluster(at + k * e_pad * 4, __float_as_int(acc[i][k]));
      } else {
#pragma unroll
        for (int k = 0; k < 16; ++k) logits[(token + k) * e_pad + block * 128 + quarter * 32 + lane] = acc[i][k];
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (CG == 2 || g.splits > 1) cluster_sync();
  if (warp == 1) { tc_fence_after_sync(); tmem_dealloc<CG>(tmem, tmem_cols); }
  Sums<EPL> sums;
#pragma unroll
  for (int j = 0; j < EPL; ++j) sums.probs[j] = 0.f;
  sums.squares = 0.f; sums.live = 0;
  if (ok) {
    constexpr int kWarps = kThreads / 32;
    auto finish = [&](auto at_once) {
      constexpr int kAtOnce = decltype(at_once)::value;
      for (int tt = split + warp * g.splits; tt < n && tile * n + tt < p.num_tokens; tt += g.splits * kWarps * kAtOnce) {
        int at[kAtOnce], t[kAtOnce];
        bool there[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
          at[i] = tt + i * g.splits * kWarps;
          t[i] = tile * n + at[i];
          there[i] = at[i] < n && t[i] < p.num_tokens;
        }
        if (g.splits == 1) {
          finish_tokens<EPL, kAtOnce>(p, s, [&](int i, int e) { return logits[at[i] * e_pad + e]; }, t, there, lane, hist, sums);
        } else {
          finish_tokens<EPL, kAtOnce>(p, s, [&](int i, int e) {
            float v[kMaxSplits];
#pragma unroll
            for (int q = 0; q < kMaxSplits; ++q) v[q] = q < g.splits ? ld_cluster_f32(cluster_map(&logits[at[i] * e_pad + e], q)) : 0.f;
            float sum = 0.f;
#pragma unroll
            for (int q = 0; q < kMaxSplits; ++q) sum += v[q];
            return sum;
          }, t, there, lane, hist, sums);
        }
      }
    };
    // Two tokens at once hide each other's latency (16384 tokens, hidden 7168, 256 experts, top-8: 87.4 -> 82.4 us; four no less); a warp with one works for nobody (64 tokens, hidden
    // 4096, 256 experts: 14.5 -> 15.7).
    if (n > kWarps * g.splits) finish(std::integral_constant<int, 2>{}); else finish(std::integral_constant<int, 1>{});
  }
  if (g.splits > 1) cluster_sync();              // the peers have read this block's logits
  __syncthreads();
  // the warps' sums, in place of the logits
  float* all = logits;                           // [16 warps][experts]
  __shared__ float2 others[kThreads / 32];
#pragma unroll
  for (int j = 0; j < EPL; ++j)
    if (j * 32 + lane < p.num_experts) all[warp * p.num_experts + j * 32 + lane] = sums.probs[j];
  if (lane == 0) others[warp] = make_float2(sums.squares, __int_as_float(sums.live));
  __syncthreads();
  const int e = threadIdx.x;
  if (e < p.num_experts) {
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) sum += all[w * p.num_experts + e];
    s.parts[static_cast<size_t>(blockIdx.x) * p.num_experts + e] = make_float2(sum, __int_as_float(hist[e]));
  }
  if (e == 0) {
    float squares = 0.f;
    int live = 0;
    for (int w = 0; w < kThreads / 32; ++w) { squares += others[w].x; live += __float_as_int(others[w].y); }
    s.other_parts[blockIdx.x] = make_float2(squares, __int_as_float(live));
  }
}

// A sum of numbers of one sign with what its roundings lose beside it: of tens of thousands of blocks that are alike (the same token over and over) a plain one came
// out 2e-4 off.
struct LongSum {
  float sum = 0.f, lost = 0.f;
  __device__ __forceinline__ void add(float v) {
    const float s = __fadd_rn(sum, v);
    lost = __fadd_rn(lost, __fsub_rn(v, __fsub_rn(s, sum)));
    sum = s;
  }
  __device__ __forceinline__ float get() const { return sum + lost; }
};

// One block adds up the blocks' sums: `rows` threads for each expert.
constexpr int kJoinThreads = 1024;
__global__ void __launch_bounds__(kJoinThreads) route_join_kernel(const RouteStatsParams p) {
  __shared__ float sums[kJoinThreads];
  __shared__ int counts[kJoinThreads];
  __shared__ float other[32];
  __shared__ int live[32];
  const int E = p.experts, rows = kJoinThreads / E, e = threadIdx.x % E, row = threadIdx.x / E, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_wait();
  LongSum probs, lse2;
  int count = 0, n = 0;
  if (row < rows) {
#pragma unroll 8
    for (int b = row; b < p.blocks; b += rows) {
      const float2 v = p.parts[static_cast<size_t>(b) * E + e];
      probs.add(v.x); count += __float_as_int(v.y);
    }
  }
  for (int b = threadIdx.x; b < p.blocks; b += kJoinThreads) { const float2 v = p.other_parts[b]; lse2.add(v.x); n += __float_as_int(v.y); }
  float squares = warp_sum(lse2.get());
  n = __reduce_add_sync(0xffffffffu, n);
  sums[threadIdx.x] = probs.get();
  counts[threadIdx.x] = count;
  if (lane == 0) { other[warp] = squares; live[warp] = n; }
  __syncthreads();
  squares = warp_sum(other[lane]);
  n = __reduce_add_sync(0xffffffffu, live[lane]);
  const float share = n > 0 ? 1.f / static_cast<float>(n) : 0.f;
  float term = 0.f;
  if (threadIdx.x < E) {
    long long total = 0;
    LongSum all;
    for (int r = 0; r < rows; ++r) { all.add(sums[r * E + e]); total += counts[r * E + e]; }
    const float load = static_cast<float>(static_cast<double>(total) * E / p.top_k) * share;
    p.counts[e] = total;
    p.load[e] = load;
    term = load * (all.get() * share);
  }
  __syncthreads();
  term = warp_sum(term);
  if (lane == 0) other[warp] = term;
  __syncthreads();
  if (warp != 0) return;
  term = warp_sum(other[lane]);
  if (lane != 0) return;
  *p.balance = term;
  *p.z = squares * share;
  p.load[E] = share;
}

template <int EPL, int CG>
cudaError_t launch_width(const RouterParams& p, const RouteStatsParams& s, const RouteTile& g, const CUtensorMap& map_w, const CUtensorMap& map_x, StatusBlock* status,
                         unsigned long long budget, cudaStream_t stream) {
  auto kernel = route_forward_kernel<EPL, CG>;
  static std::atomic<bool> configured[64];       // the shared-memory limit is an attribute of the function on a device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 224 * 1024);
    if (e != cudaSuccess) return e;
    configured[dev].store(true, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(s.blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = g.smem_bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = g.splits * CG; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, map_w, map_x, p, s, g, status, budget);
}

}  // namespace

RouteTile route_tile(const RouterParams& p, int sms) {
  RouteTile g{router_tile(p, sms), 0};
  const int tiles = (p.num_tokens + g.tile_tokens - 1) / g.tile_tokens;
  // (16384 tokens, 256 experts, without and with pairs: hidden 512 29.8 and 31.2 us, 2048 44.5 and 42.4, 4096 64.2 and 57.5)
  g.pairs = g.blocks == 2 && g.splits == 1 && g.tile_tokens == 128 && p.hidden > 1024 ? 1 : 0;
  if (g.pairs) {
    const int stage = 2 * 128 * 128, logits = 128 * e_pad_of(p.num_experts) * 4;
    g.stages = kMaxStages - 2;
    g.smem_bytes = std::max(g.stages * stage, logits) + 1024;
  }
  g.grid = g.pairs ? (tiles + 1) / 2 * 2 : tiles * g.splits;
  return g;
}

cudaError_t launch_route_forward(const RouterParams& p, const RouteStatsParams& s, const void* map_w, const void* map_x, int sms, StatusBlock* status, unsigned long long wait_budget_ns,
                                 cudaStream_t stream) {
  cudaError_t e = cudaSuccess;
  if (s.blocks > 0) {
    const RouteTile g = route_tile(p, sms);
    const CUtensorMap &mw = *static_cast<const CUtensorMap*>(map_w), &mx = *static_cast<const CUtensorMap*>(map_x);
    if (g.pairs) e = launch_width<8, 2>(p, s, g, mw, mx, status, wait_budget_ns, stream);
    else if (p.num_experts <= 32) e = launch_width<1, 1>(p, s, g, mw, mx, status, wait_budget_ns, stream);
    else if (p.num_experts <= 64) e = launch_width<2, 1>(p, s, g, mw, mx, status, wait_budget_ns, stream);
    else if (p.num_experts <= 128) e = launch_width<4, 1>(p, s, g, mw, mx, status, wait_budget_ns, stream);
    else if (p.num_experts <= 256) e = launch_width<8, 1>(p, s, g, mw, mx, status, wait_budget_ns, stream);
    else e = launch_width<16, 1>(p, s, g, mw, mx, status, wait_budget_ns, stream);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(1);
  cfg.blockDim = dim3(kJoinThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = s.blocks > 0 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, route_join_kernel, s);
}

}  // namespace sep

// Gradients of routing on the tensor cores: from the gradients of weights, balance and z loss that of the logits, dz [T, E], and from it
//
//   dx = dz W  [T, H]      a block takes 128 tokens: their dz is formed in shared memory, where it stays as the left operand, and W's columns go by
//   dW = dz^T x  [E, H]    a block takes up to 256 experts, 256 columns and a part of the tokens; the parts are added up by a small kernel
//
// For both products dz is rounded to bf16, 2^-8 of each term at most, as bf16 training code rounds the gradient of its logits: against 64 bits dx and dW are
// 2.3e-3 off in 2-norm, where their own rounding is 1.7e-3.  Up to 128 experts, where twice the products cost nothing beside the reads of x and the writes of
// dx, dz is kept to 16 bits as the sum of two bf16 numbers, and they are 1.7e-3 off.  All sums are fp32; of dx over up to 512 experts in one accumulator, of dW over up to 4096 tokens.
// What bounds them: x is read and dx written once (HBM), for many experts what the SMs read from L2; and for short calls the forming of dz.  All operands lie in memory as TMA brings them in, dz as
// [layers, T, experts rounded up to 64]; nothing is transposed.  Parts and sums have a fixed order: a repeated call gives the same bits.
#include <algorithm>
#include <atomic>
#include <cuda.h>
#include <type_traits>

#include "ptx.cuh"
#include "route.h"

namespace sep {

namespace {

constexpr int kThreads = 320;                    // TMA, MMA, 8 warps of epilogue
constexpr int kEpiWarps = 8;
constexpr int kTokens = 128, kCols = 256, kBK = 64;
constexpr int kChunk = 64 * 128;                 // a box of 64 x 64 bf16
constexpr int kStaging = 4096;
constexpr int kMostSmem = 226 * 1024;
constexpr int kMostStages = 8;
// Tokens of a part of dW.  The tensor cores cut off what an accumulator cannot hold instead of rounding, at every 16 tokens and each layer of dz: 17 numbers of which
// each may lose 2^-23 of the largest, so that at most 512 steps make 17 2^-15 = 5e-4 of the sum, an eighth of the result's own rounding.  Measured: 2e-5; parts of 65536
// tokens came out 3.6e-4 too small, of 2^20 6e-3.
constexpr int kMostPart = 4096;

__device__ __forceinline__ void mbar_arrive_release_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" :: "r"(cluster_addr) : "memory");
}

// The gradients of N tokens' logits, by one warp: lane l has experts 2 l, 2 l + 1, 64 + 2 l, ... in P pairs.  All loads first: a warp has 16 tokens to form before the first
// product.  What the chosen experts get beside the others is handed to their lanes through `chosen` (shared memory of the warp's own, N rows
// of 64 P numbers, zeros before and after): looking for each choice in all lanes took 0.8 us a choice
// (top-8, dx of 16384 tokens, hidden 7168, 256 experts 82 -> 71 us, of 8192 tokens, hidden 2048, 64 experts 19.4 -> 15.9).
template <int P, int N>
__device__ __forceinline__ void token_gradients(const RouteGradParams& p, int t0, int step, int lane, float share, float db, float dzl, const float2 (&load)[P], float* chosen,
                                                float2 (&v)[N][P]) {
  float2 prob[N][P];
  float up[N], w[N], lse[N];
  int mine[N];
  bool counts[N];
  const bool even = p.experts % 2 == 0;          // (pairs then lie on their boundaries)
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int t = t0 + i * step;
    const bool there = t < p.tokens;
    const float* row = p.probs + static_cast<long long>(t) * p.experts;
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const int e = j * 64 + lane * 2;
      prob[i][j] = make_float2(0.f, 0.f);
      if (there && e < p.experts) {
        if (even) {
          prob[i][j] = *reinterpret_cast<const float2*>(row + e);
        } else {
          prob[i][j].x = row[e];
          if (e + 1 < p.experts) prob[i][j].y = row[e + 1];
        }
      }
    }
    mine[i] = -1; up[i] = w[i] = 0.f;
    if (there && lane < p.top_k && p.dweights != nullptr) {
      const long long at = static_cast<long long>(t) * p.top_k + lane;
      mine[i] = static_cast<int>(p.idx[at]);
      w[i] = p.weights[at];
      up[i] = p.dweights[at];
    }
    counts[i] = there && (p.mask == nullptr || p.mask[t] != 0);
    lse[i] = there && dzl != 0.f ? p.lse[t] : 0.f;
  }
  float mean_load[N], mean_up[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    mean_load[i] = 0.f;
#pragma unroll
    for (int j = 0; j < P; ++j) mean_load[i] = fmaf(prob[i][j].x, load[j].x, fmaf(prob[i][j].y, load[j].y, mean_load[i]));
    // (where the weights are not normalised again, w is the probability itself)
    mean_up[i] = w[i] * up[i];
  }
  if (db != 0.f) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
      for (int i = 0; i < N; ++i) mean_load[i] += __shfl_xor_sync(0xffffffffu, mean_load[i], o);
  }
  if (p.dweights != nullptr) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
      for (int i = 0; i < N; ++i) mean_up[i] += __shfl_xor_sync(0xffffffffu, mean_up[i], o);
    __syncwarp();                // (the zeros are back)
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (static_cast<unsigned>(mine[i]) < static_cast<unsigned>(p.experts)) chosen[i * P * 64 + mine[i]] = p.renormalize ? w[i] * (up[i] - mean_up[i]) : w[i] * up[i];
    __syncwarp();
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float cb = counts[i] ? db * share : 0.f, cz = counts[i] ? 2.f * dzl * share * lse[i] : 0.f, all = p.renormalize ? 0.f : mean_up[i];
#pragma unroll
    for (int j = 0; j < P; ++j) {
      // (a token that does not count is not multiplied with: it may hold anything)
      v[i][j].x = counts[i] ? fmaf(cz, prob[i][j].x, cb * prob[i][j].x * (load[j].x - mean_load[i])) : 0.f;
      v[i][j].y = counts[i] ? fmaf(cz, prob[i][j].y, cb * prob[i][j].y * (load[j].y - mean_load[i])) : 0.f;
      if (p.dweights != nullptr) {
        const float2 add = *reinterpret_cast<const float2*>(chosen + (i * P + j) * 64 + lane * 2);
        v[i][j].x = fmaf(-all, prob[i][j].x, v[i][j].x) + add.x;
        v[i][j].y = fmaf(-all, prob[i][j].y, v[i][j].y) + add.y;
      }
    }
  }
  if (p.dweights != nullptr) {
    __syncwarp();
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (static_cast<unsigned>(mine[i]) < static_cast<unsigned>(p.experts)) chosen[i * P * 64 + mine[i]] = 0.f;
  }
}

// A failed wait: the copies that this thread may have in flight land before the block leaves (bounded).
__device__ __forceinline__ void give_up(StatusBlock* status, int role, int rank, int where) {
  report_failure(status, kStatusTimeoutPipeline, kKernelRoute, role, rank, where, 0, 0);
  const unsigned long long t0 = globaltimer_ns();
  while (globaltimer_ns() - t0 < 2000000ull) {}
}

// 32 rows and 64 columns of an accumulator leave as bf16.
__device__ __forceinline__ void store_half_tile(uint32_t taddr, unsigned char* tile, const CUtensorMap* map, int x, int y, int lane) {
  uint32_t a[32], b[32];
  tmem_ld_32x32(taddr, a);
  tmem_ld_32x32(taddr + 32, b);
  tmem_ld_wait();
  const uint32_t stg = smem_u32(tile);
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    uint32_t o[4];
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const int i = (q & 3) * 8 + h * 2;
      o[h] = pack_bf16x2(__uint_as_float(q < 4 ? a[i] : b[i]), __uint_as_float(q < 4 ? a[i + 1] : b[i + 1]));
    }
    st_shared_v4(stg + stage_off<128>(lane, q), o[0], o[1], o[2], o[3]);
  }
  fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) { tma_store_3d(map, tile, x, y, 0); bulk_commit(); }
}

// CG = 2: the blocks of a pair multiply their 256 tokens together, each with half of W's columns in its shared memory.  The kernels of
// 16384 tokens, hidden 7168 and 256 experts are bound by what the SMs read from L2 (8 TB/s): with the whole of W for every 128 tokens this one took 82 us, for every 256 67.
template <int EPL, int CG>
__global__ void __launch_bounds__(kThreads, 1) route_dx_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_dx, const RouteGradParams p,
                                                               const RouteGradPlan g) {
  constexpr int kLayers = EPL <= 4 ? 2 : 1;      // g.layers
  extern __shared__ unsigned char smem_dyn[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
  constexpr int kHalf = 4 / CG;                  // chunks of W in a stage
  __shared__ uint64_t full_bar[kMostStages], empty_bar[kMostStages], tmem_full[2], tmem_empty[2], dz_bar;
  __shared__ uint32_t s_tmem;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = CG == 2 ? static_cast<int>(cluster_ctarank()) : 0, unit = static_cast<int>(blockIdx.x) / CG;
  const int tile = unit / g.dx_splits * CG + rank, split = unit % g.dx_splits;
  const bool leader = rank == 0;
  const int k_blocks = g.padded / kBK, n_tiles = p.dx != nullptr ? (p.hidden + kCols - 1) / kCols : 0;
  const int n0 = n_tiles * split / g.dx_splits, n1 = n_tiles * (split + 1) / g.dx_splits;
  unsigned char* dz = smem;                      // [layers][k_blocks][128 rows][128 bytes]
  const int layer_bytes = k_blocks * kTokens * 128;
  unsigned char* stages = dz + kLayers * layer_bytes;
  unsigned char* staging = stages + g.dx_stages * kHalf * kChunk;
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&map_w);
    for (int s = 0; s < g.dx_stages; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
    for (int b = 0; b < 2; ++b) { mbar_init(&tmem_full[b], 1); mbar_init(&tmem_empty[b], kEpiWarps * CG); }
    mbar_init(&dz_bar, kEpiWarps * CG);
    mbar_fence_init();
  }
  if (warp == 1) { tmem_alloc<CG>(&s_tmem, 512); tmem_relinquish<CG>(); }
  tc_fence_before_sync();
  if constexpr (CG == 2) cluster_sync(); else __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = s_tmem;
  if (warp == 0) {
    if (lane == 0) {
      int stage = 0; uint32_t phase = 0; bool ok = true;
      for (int n = n0; n < n1 && ok; ++n) {
        // (of a pair, each has half of the columns that are multiplied)
        const int half = CG == 2 ? min(kCols, (p.hidden - n * kCols + 31) / 32 * 32) / 2 : min(kCols, p.hidden - n * kCols), chunks = (half + 63) / 64;
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1, p.wait_budget_ns, p.status)) { ok = false; break; }
          // (both blocks' bytes are counted on the first one's barrier, which that one arms for the sum)
          if (leader) mbar_arrive_expect_tx(&full_bar[stage], CG * chunks * kChunk);
          for (int c = 0; c < chunks; ++c) {
            unsigned char* to = stages + (stage * kHalf + c) * kChunk;
            if constexpr (CG == 2) tma_load_3d_pair(to, &map_w, cluster_map(&full_bar[stage], 0), n * kCols + rank * half + c * 64, kb * kBK, 0);
            else tma_load_3d(to, &map_w, &full_bar[stage], n * kCols + c * 64, kb * kBK, 0);
          }
          if (++stage == g.dx_stages) { stage = 0; phase ^= 1; }
        }
      }
      if (!ok) give_up(p.status, 0, p.rank, tile);
    }
  } else if (warp == 1) {
    if (leader) {
    bool ok = __all_sync(0xffffffffu, mbar_wait<CG == 2>(&dz_bar, 0, p.wait_budget_ns, p.status));
    int stage = 0, acc = 0; uint32_t phase = 0, acc_phase = 0;
    for (int n = n0; n < n1 && ok; ++n) {
      const int cols = min(kCols, (p.hidden - n * kCols + 31) / 32 * 32);
      const uint32_t idesc = umma_idesc_bf16(kTokens * CG, 0, 0, 1) | (static_cast<uint32_t>(cols >> 3) << 17);
      if (!__all_sync(0xffffffffu, mbar_wait<CG == 2>(&tmem_empty[acc], acc_phase ^ 1, p.wait_budget_ns, p.status))) { ok = false; break; }
      tc_fence_after_sync();
      for (int kb = 0; kb < k_blocks; ++kb) {
        if (!__all_sync(0xffffffffu, mbar_wait<CG == 2>(&full_bar[stage], phase, p.wait_budget_ns, p.status))) { ok = false; break; }
        tc_fence_after_sync();
        if (elect_one()) {
          const uint32_t a = smem_u32(dz + kb * kTokens * 128), b = smem_u32(stages + stage * kHalf * kChunk);
#pragma unroll
          for (int l = 0; l < kLayers; ++l)
#pragma unroll
            for (int j = 0; j < kBK / 16; ++j)
              umma_bf16_ss<CG>(tmem + acc * kCols, umma_smem_desc(a + l * layer_bytes + j * 32, 16, 1024), umma_smem_desc(b + j * 16 * 128, kChunk, 1024), idesc,
                              (kb > 0 || l > 0 || j > 0) ? 1u : 0u);
          umma_commit<CG>(&empty_bar[stage]);
          if (kb == k_blocks - 1) umma_commit<CG>(&tmem_full[acc]);
        }
        __syncwarp();
        if (++stage == g.dx_stages) { stage = 0; phase ^= 1; }
      }
      acc ^= 1; if (acc == 0) acc_phase ^= 1;
    }
    if (!ok && lane == 0) report_failure(p.status, kStatusTimeoutPipeline, kKernelRoute, 1, p.rank, tile, 0, 0);
    }
  } else {
    const int w = warp - 2, quarter = warp & 3, side = w >> 2;
    const float share = p.load[p.experts], db = p.dbalance != nullptr ? *p.dbalance : 0.f, dzl = p.dz_loss != nullptr ? *p.dz_loss : 0.f;
    constexpr int P = EPL / 2, kAtOnce = EPL <= 4 ? 8 : EPL <= 8 ? 4 : 2;
    static_assert(kAtOnce * P * 64 * 4 <= kStaging, "the place of the results serves for what the choices hand over");
    float* const chosen = reinterpret_cast<float*>(staging + w * g.dx_staging * kStaging);
#pragma unroll
    for (int i = lane; i < kAtOnce * P * 16; i += 32) reinterpret_cast<float4*>(chosen)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    float2 load[P];
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const int e = j * 64 + lane * 2;
      load[j] = db != 0.f ? make_float2(e < p.experts ? p.load[e] : 0.f, e + 1 < p.experts ? p.load[e + 1] : 0.f) : make_float2(0.f, 0.f);
    }
    for (int r0 = w; r0 < kTokens; r0 += kEpiWarps * kAtOnce) {
      float2 v[kAtOnce][P];
      token_gradients<P, kAtOnce>(p, tile * kTokens + r0, kEpiWarps, lane, share, db, dzl, load, chosen, v);
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int r = r0 + i * kEpiWarps, t = tile * kTokens + r;
#pragma unroll
        for (int j = 0; j < P; ++j) {
          const int e = j * 64 + lane * 2;
          if (j * 64 >= g.padded) continue;
          float2 left = v[i][j];                 // (zeros where there is no such token or expert)
#pragma unroll
          for (int l = 0; l < kLayers; ++l) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(left.x, left.y);
            left.x -= __bfloat162float(b.x); left.y -= __bfloat162float(b.y);
            *reinterpret_cast<__nv_bfloat162*>(dz + l * layer_bytes + j * kTokens * 128 + stage_off<128>(r, lane / 4) + lane % 4 * 4) = b;
            if (split == 0 && t < p.tokens && p.dz != nullptr)
              *reinterpret_cast<__nv_bfloat162*>(static_cast<__nv_bfloat16*>(p.dz) + (static_cast<long long>(l) * p.tokens + t) * g.padded + e) = b;
          }
        }
      }
    }
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) {             // (the first block's tensor cores read this block's dz: a release that reaches it)
      if constexpr (CG == 2) mbar_arrive_release_cluster(cluster_map(&dz_bar, 0)); else mbar_arrive(&dz_bar);
    }
    int acc = 0, flip = 0; uint32_t acc_phase = 0;
    unsigned char* const mine = staging + w * g.dx_staging * kStaging;
    const int row0 = tile * kTokens + quarter * 32;
    for (int n = n0; n < n1; ++n) {
      if (!__all_sync(0xffffffffu, mbar_wait(&tmem_full[acc], acc_phase, p.wait_budget_ns, p.status))) {
        if (lane == 0) report_failure(p.status, kStatusTimeoutPipeline, kKernelRoute, 2, p.rank, tile, n, 0);
        break;
      }
      tc_fence_after_sync();
#pragma unroll 1
      for (int c = 0; c < 128; c += 64) {
        const int col = side * 128 + c;
        if (n * kCols + col >= p.hidden || row0 >= p.tokens) continue;
        if (lane == 0) { if (g.dx_staging == 2) bulk_wait_read_but_one(); else bulk_wait_read(); }
        __syncwarp();
        store_half_tile(tmem + (static_cast<uint32_t>(quarter * 32) << 16) + acc * kCols + col, mine + flip * kStaging, &map_dx, n * kCols + col, row0, lane);
        if (g.dx_staging == 2) flip ^= 1;
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        if constexpr (CG == 2) mbar_arrive_cluster(cluster_map(&tmem_empty[acc], 0)); else mbar_arrive(&tmem_empty[acc]);
      }
      acc ^= 1; if (acc == 0) acc_phase ^= 1;
    }
    if (lane == 0) bulk_wait_all();
  }
  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();         // (the pair's operands, accumulators and barriers are no longer in use)
  if (warp == 1) { tc_fence_after_sync(); tmem_dealloc<CG>(tmem, 512); }
}

// A unit: `g.dw_blocks` blocks of 128 experts, 256 columns, a part of the tokens.  CG = 2: a pair of blocks, each with 128 experts, and 512 columns, of which each has half in its
// shared memory; dz is then read half as often (16384 tokens, hidden 7168, 256 experts 61.4 -> 56.7 us).
template <int CG>
__global__ void __launch_bounds__(kThreads, 1) route_dw_kernel(const __grid_constant__ CUtensorMap map_dz, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_out,
                                                               const RouteGradParams p, const RouteGradPlan g) {
  extern __shared__ unsigned char smem_dyn[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full_bar[4], empty_bar[4], done_bar;
  __shared__ uint32_t s_tmem;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kUnit = kCols * CG;
  const int rank = CG == 2 ? static_cast<int>(cluster_ctarank()) : 0, unit = static_cast<int>(blockIdx.x) / CG;
  const bool leader = rank == 0;
  const int n_tiles = (p.hidden + kUnit - 1) / kUnit;
  const int n = unit % n_tiles, rest = unit / n_tiles, split = rest % g.dw_splits, group = rest / g.dw_splits;
  // this block's experts: m0, ... in blocks of 128
  const int all_blocks = (p.experts + 127) / 128, m0 = group * g.dw_blocks + rank, blocks = CG == 2 ? 1 : min(g.dw_blocks, all_blocks - m0);
  const int k_blocks = (p.tokens + kBK - 1) / kBK, kb0 = static_cast<int>(static_cast<long long>(k_blocks) * split / g.dw_splits),
            kb1 = static_cast<int>(static_cast<long long>(k_blocks) * (split + 1) / g.dw_splits);
  // of the h-th 256 columns: those that are multiplied, and the 64-wide pieces of them in this block's shared memory
  auto cols_of = [&](int h) { return max(0, min(kCols, (p.hidden - n * kUnit - h * kCols + 31) / 32 * 32)); };
  auto chunks_of = [&](int h) { return CG == 2 ? (cols_of(h) / 2 + 63) / 64 : (min(kCols, p.hidden - n * kUnit) + 63) / 64; };
  auto experts_of = [&](int block) { return max(0, min((CG == 2 ? 1 : blocks) * 2, g.padded / 64 - block * 2)); };      // (chunks)
  const int layer_chunks = g.dw_blocks * 2 / CG, stage_bytes = (g.layers * layer_chunks + 4) * kChunk, tmem_cols = g.dw_blocks * kCols;
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&map_dz);
    tma_prefetch_desc(&map_x);
    for (int s = 0; s < g.dw_stages; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
    mbar_init(&done_bar, 1);
    mbar_fence_init();
  }
  if (warp == 1) { tmem_alloc<CG>(&s_tmem, tmem_cols); tmem_relinquish<CG>(); }
  tc_fence_before_sync();
  if constexpr (CG == 2) cluster_sync(); else __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = s_tmem;
  if (warp == 0) {
    if (lane == 0) {
      int stage = 0; uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(&empty_bar[stage], phase ^ 1, p.wait_budget_ns, p.status)) { give_up(p.status, 3, p.rank, static_cast<int>(blockIdx.x)); break; }
        unsigned char* s = smem + stage * stage_bytes;
        // (experts beyond the padded ones: chunks outside are not fetched, and their rows of the result not stored)
        const int left = experts_of(m0);
        if constexpr (CG == 2) {                 // (the bytes of both are counted on the first one's barrier)
          if (leader) mbar_arrive_expect_tx(&full_bar[stage], (left + experts_of(m0 + 1) + 2 * (chunks_of(0) + chunks_of(1))) * kChunk);
          const uint32_t bar = cluster_map(&full_bar[stage], 0);
          for (int c = 0; c < left; ++c) tma_load_3d_pair(s + c * kChunk, &map_dz, bar, (m0 * 2 + c) * 64, kb * kBK, 0);
          for (int h = 0; h < 2; ++h)
            for (int c = 0; c < chunks_of(h); ++c)
              tma_load_3d_pair(s + (2 + h * 2 + c) * kChunk, &map_x, bar, n * kUnit + h * kCols + rank * (cols_of(h) / 2) + c * 64, kb * kBK, 0);
        } else {
          const int chunks = chunks_of(0);
          mbar_arrive_expect_tx(&full_bar[stage], (g.layers * left + chunks) * kChunk);
          for (int l = 0; l < g.layers; ++l)
            for (int c = 0; c < left; ++c) tma_load_3d(s + (l * layer_chunks + c) * kChunk, &map_dz, &full_bar[stage], (m0 * 2 + c) * 64, kb * kBK, l);
          for (int c = 0; c < chunks; ++c) tma_load_3d(s + (g.layers * layer_chunks + c) * kChunk, &map_x, &full_bar[stage], n * kCols + c * 64, kb * kBK, 0);
        }
        if (++stage == g.dw_stages) { stage = 0; phase ^= 1; }
      }
    }
  } else if (warp == 1) {
    if (leader) {
    const uint32_t idesc = umma_idesc_bf16(128 * CG, 0, 1, 1);
    int stage = 0; uint32_t phase = 0; bool ok = true;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!__all_sync(0xffffffffu, mbar_wait<CG == 2>(&full_bar[stage], phase, p.wait_budget_ns, p.status))) { ok = false; break; }
      tc_fence_after_sync();
      if (elect_one()) {
        const uint32_t a = smem_u32(smem + stage * stage_bytes), b = a + g.layers * layer_chunks * kChunk;
        for (int l = 0; l < g.layers; ++l)
          for (int m = 0; m < (CG == 2 ? 2 : blocks); ++m) {           // accumulators: of experts, or of a pair's columns
            const int cols = cols_of(CG == 2 ? m : 0);
            if (cols == 0) break;
            const uint32_t am = a + (l * layer_chunks + (CG == 2 ? 0 : m * 2)) * kChunk, bm = b + (CG == 2 ? m * 2 : 0) * kChunk;
#pragma unroll
            for (int j = 0; j < kBK / 16; ++j)
              umma_bf16_ss<CG>(tmem + m * kCols, umma_smem_desc(am + j * 16 * 128, kChunk, 1024), umma_smem_desc(bm + j * 16 * 128, kChunk, 1024),
                               idesc | (static_cast<uint32_t>(cols >> 3) << 17), (kb > kb0 || l > 0 || j > 0) ? 1u : 0u);
          }
        umma_commit<CG>(&empty_bar[stage]);
        if (kb == kb1 - 1) umma_commit<CG>(&done_bar);
      }
      __syncwarp();
      if (++stage == g.dw_stages) { stage = 0; phase ^= 1; }
    }
    if (!ok && lane == 0) report_failure(p.status, kStatusTimeoutPipeline, kKernelRoute, 4, p.rank, static_cast<int>(blockIdx.x), 0, 0);
    }
  } else {
    // (the operands' place is free once the products are done)
    const bool have = kb1 > kb0;
    const bool ok = !have || __all_sync(0xffffffffu, mbar_wait(&done_bar, 0, p.wait_budget_ns, p.status));
    if (!ok && lane == 0) report_failure(p.status, kStatusTimeoutPipeline, kKernelRoute, 5, p.rank, static_cast<int>(blockIdx.x), 0, 0);
    if (ok) {
      tc_fence_after_sync();
      const int w = warp - 2, quarter = warp & 3, side = w >> 2;
      unsigned char* const mine = smem + w * 2 * kStaging;
      int flip = 0;
      for (int m = 0; m < (CG == 2 ? 2 : blocks); ++m) {
        const int row0 = (CG == 2 ? m0 : m0 + m) * 128 + quarter * 32, col0 = n * kUnit + (CG == 2 ? m * kCols : 0);
        if (row0 >= p.experts) continue;
        const uint32_t taddr = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + m * kCols;
        for (int c = side * 128; c < side * 128 + 128; c += g.dw_splits > 1 ? 32 : 64) {
          if (col0 + c >= p.hidden) break;
          if (lane == 0) bulk_wait_read_but_one();
          __syncwarp();
          unsigned char* tile = mine + flip * kStaging;
          flip ^= 1;
          if (g.dw_splits == 1) {
            store_half_tile(taddr + c, tile, &map_out, col0 + c, row0, lane);
            continue;
          }
          uint32_t r[32];
          tmem_ld_32x32(taddr + c, r);
          tmem_ld_wait();
          const uint32_t stg = smem_u32(tile);
#pragma unroll
          for (int q = 0; q < 8; ++q) st_shared_v4(stg + stage_off<128>(lane, q), r[q * 4], r[q * 4 + 1], r[q * 4 + 2], r[q * 4 + 3]);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) { tma_store_3d(&map_out, tile, col0 + c, row0, split); bulk_commit(); }
        }
      }
      if (lane == 0) bulk_wait_all();
    }
  }
  __syncwarp();
  tc_fence_before_sync();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();         // (the pair's operands, accumulators and barriers are no longer in use)
  if (warp == 1) { tc_fence_after_sync(); tmem_dealloc<CG>(tmem, tmem_cols); }
}

// The sum of the parts of dW, 8 elements a thread.
__global__ void __launch_bounds__(256) route_dw_join_kernel(const float* parts, void* dw, long long elements, int splits) {
  grid_wait();
  const long long i = (static_cast<long long>(blockIdx.x) * 256 + threadIdx.x) * 8;
  if (i >= elements) return;
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    const float4* at = reinterpret_cast<const float4*>(parts + s * elements + i);
    const float4 u = at[0], v = at[1];
    a.x += u.x; a.y += u.y; a.z += u.z; a.w += u.w;
    b.x += v.x; b.y += v.y; b.z += v.z; b.w += v.w;
  }
  *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(dw) + i) = make_uint4(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w), pack_bf16x2(b.x, b.y), pack_bf16x2(b.z, b.w));
}

template <auto kKernel, class... Args>
cudaError_t launch(unsigned grid, int cluster, int smem, cudaStream_t stream, const Args&... args) {
  static std::atomic<bool> configured[64];       // the shared-memory limit is an attribute of the function on a device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[dev].load(std::memory_order_acquire)) {
    if ((e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem)) != cudaSuccess) return e;
    configured[dev].store(true, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kKernel, args...);
}

}  // namespace

RouteGradPlan route_grad_plan(int tokens, int hidden, int experts, int sms) {
  RouteGradPlan g{};
  g.padded = (experts + 63) / 64 * 64;
  g.layers = experts <= 128 ? 2 : 1;
  const int tiles = (tokens + kTokens - 1) / kTokens, n_tiles = (hidden + kCols - 1) / kCols;
  // dx: a block forms the gradient of its tokens' logits, so several for the same tokens only where there are few
  // (blocks in pairs cost 1.4 us and halve what is read of W: even at 48 MB of it, without and with pairs 15.0 and 16.0 us for 2048 tokens,
  // hidden 4096 and 128 experts, 27.5 and 26.0 for 8192, 43.8 and 38.8 for 16384; at 64 experts the writes hide it: 1 us lost up to 32768 tokens, hidden 2048)
  g.dx_pairs = g.padded > 64 && static_cast<long long>(tiles) * g.padded * hidden * 2 >= 48ll << 20 ? 1 : 0;
  const int group = g.dx_pairs ? 2 : 1, groups = (tiles + group - 1) / group;
  g.dx_splits = groups > 0 ? sms / group / groups : 1;
  if (g.dx_splits > n_tiles) g.dx_splits = n_tiles;
  if (g.dx_splits < 1) g.dx_splits = 1;
  // (a fourth stage of W is worth more than a second tile of results a warp)
  g.dx_staging = g.padded <= 128 ? 2 : 1;
  const int fixed = 1024 + g.layers * g.padded * kTokens * 2 + kEpiWarps * g.dx_staging * kStaging, stage = 4 / group * kChunk;
  g.dx_stages = (kMostSmem - fixed) / stage;
  if (g.dx_stages > kMostStages) g.dx_stages = kMostStages;
  g.dx_smem = fixed + g.dx_stages * stage;
  // dW: tokens are split to fill the GPU, into no shorter parts than 4 blocks of 64, and rather into whole rounds of all SMs
  const int blocks = (experts + 127) / 128;
  g.dw_blocks = blocks > 1 ? 2 : 1;
  const int groups_of_experts = (blocks + g.dw_blocks - 1) / g.dw_blocks;
  // (256 experts, without and with pairs: 1000 tokens of hidden 7168 12.2 and 12.8 us, 4096 23.5 and 22.3, 32768 of hidden 1000 27.8 and 29.4, of 2048 41.4 and 40.1)
  g.dw_pairs = g.dw_blocks == 2 && hidden >= 2048 && static_cast<long long>(tokens) * hidden * groups_of_experts >= 1 << 24 ? 1 : 0;
  const int of = g.dw_pairs ? 2 : 1, unit_cols = kCols * of;
  const int units = groups_of_experts * ((hidden + unit_cols - 1) / unit_cols), most = (tokens + 4 * kBK - 1) / (4 * kBK);
  const int least = (tokens + kMostPart - 1) / kMostPart;
  int best = least;
  double best_time = 0.0;
  for (int s = least; s <= most && s <= std::max(64, least + 32); ++s) {
    const int rounds = (units * s + sms / of - 1) / (sms / of);
    // a round's blocks of tokens, and what an output tile costs: about as much as 6 blocks
    const double time = rounds * (static_cast<double>((tokens + kBK - 1) / kBK) / s + 6.0);
    if (s == least || time < best_time) { best = s; best_time = time; }
  }
  g.dw_splits = best;
  // stages of 64 KB: two blocks, or two layers of one; of a pair of 48
  g.dw_stages = g.dw_pairs ? 4 : 3;
  g.dw_smem = 1024 + g.dw_stages * (g.layers * g.dw_blocks * 2 / of + 4) * kChunk;
  g.dw_units = units * best * of;
  return g;
}

cudaError_t launch_route_dx(const RouteGradParams& p, const RouteGradPlan& g, const void* map_w, const void* map_dx, cudaStream_t stream) {
  const CUtensorMap &mw = *static_cast<const CUtensorMap*>(map_w), &mdx = *static_cast<const CUtensorMap*>(map_dx);
  RouteGradPlan q = g;
  if (p.dx == nullptr) q.dx_splits = 1;
  const int group = g.dx_pairs ? 2 : 1, tiles = (p.tokens + kTokens - 1) / kTokens;
  const unsigned grid = static_cast<unsigned>((tiles + group - 1) / group * group * q.dx_splits);
  auto with = [&](auto experts) {
    constexpr int EPL = decltype(experts)::value;
    if constexpr (EPL >= 4) if (g.dx_pairs) return launch<route_dx_kernel<EPL, 2>>(grid, 2, g.dx_smem, stream, mw, mdx, p, q);
    return launch<route_dx_kernel<EPL, 1>>(grid, 1, g.dx_smem, stream, mw, mdx, p, q);
  };
  if (p.experts <= 64) return with(std::integral_constant<int, 2>{});
  if (p.experts <= 128) return with(std::integral_constant<int, 4>{});
  if (p.experts <= 256) return with(std::integral_constant<int, 8>{});
  return with(std::integral_constant<int, 16>{});
}

cudaError_t launch_route_dw(const RouteGradParams& p, const RouteGradPlan& g, const void* map_dz, const void* map_x, const void* map_out, float* parts, cudaStream_t stream) {
  const CUtensorMap &mz = *static_cast<const CUtensorMap*>(map_dz), &mx = *static_cast<const CUtensorMap*>(map_x), &mo = *static_cast<const CUtensorMap*>(map_out);
  const cudaError_t e = g.dw_pairs ? launch<route_dw_kernel<2>>(static_cast<unsigned>(g.dw_units), 2, g.dw_smem, stream, mz, mx, mo, p, g)
                                   : launch<route_dw_kernel<1>>(static_cast<unsigned>(g.dw_units), 1, g.dw_smem, stream, mz, mx, mo, p, g);
  if (e != cudaSuccess || g.dw_splits == 1) return e;
  const long long elements = static_cast<long long>(p.experts) * p.hidden;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>((elements / 8 + 255) / 256));
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, route_dw_join_kernel, static_cast<const float*>(parts), p.dw, elements, g.dw_splits);
}

}  // namespace sep

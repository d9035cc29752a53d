// Output projection with softmax cross entropy, without logits in memory: z = x W^T, and for each token t with target y
//   loss_t = log sum_v exp(z_tv) - z_ty,   dz_tv = c_t (exp(z_tv - lse_t) - [v = y]),   dx = dz W,   dW = dz^T x.
//
// All four products run in one kernel template over units of 256 x 256 (tcgen05 on CTA pairs, fp32 accumulators in tensor memory,
// operands by TMA).  Forward: the epilogue reduces each row's 128 columns to a maximum m and the sum of exp(z - m) and drops the
// tile; a second kernel joins the parts in a fixed order.  Backward: ONE launch walks the vocabulary in pieces.  The logits of a piece are
// computed again and leave as dz (bf16, a buffer of a fixed size, not of T x V); dx and dW units of a piece follow when its
// dz is complete, while the dz units of the next piece keep the tensor cores busy in between.
//
// What bounds it: the tensor cores, 2THV operations forward and 6THV backward (one of the three products is the recomputation, the price
// of not keeping the logits); below a few hundred tokens the reads of W and the writes of dW.
//
// Order and progress.  Units are claimed one after another from a counter, by CTAs that run, so a unit that waits for others
// only waits for units that are already being worked on: the kernel needs no number of co-resident CTAs.
#include <atomic>

#include "linear_loss.h"
#include "ptx.cuh"

namespace sep {

namespace {

constexpr int kBK = 64;                          // bf16 elements of a k-block: one 128-byte swizzle row
constexpr int kStages = 6;
constexpr int kOperandBytes = 128 * kBK * 2;     // A or B of one CTA: 128 rows of a k-block
constexpr int kStageBytes = 2 * kOperandBytes;
constexpr int kEpiWarps = 8;
constexpr int kThreads = (2 + kEpiWarps + 1) * 32;   // 0 TMA producer, 1 MMA, 2..9 epilogue, 10 scheduler
constexpr int kStagingBytes = 4096;              // per epilogue warp: 32 rows of 128 bytes
constexpr int kQueue = 4;
constexpr int kSmemBytes = kStages * kStageBytes + kEpiWarps * kStagingBytes + 1024;
constexpr int kTmemCols = 512;
constexpr int kDoneWarps = 2 * kEpiWarps;        // reports per unit
// The scheduler claims the next unit when the producer has this many k-blocks of the one before left: a claimed unit is work that
// no idle pair can take any more.
constexpr int kClaimAhead = 10;
constexpr float kLog2e = 1.4426950408889634f;
// The tensor cores cut off what an fp32 accumulator cannot hold instead of rounding it, so every 16 elements of K a logit loses half a unit
// of its last place on average, always towards zero: at H 7168 the mean loss came out 6e-6 too small (relative).  The forward
// therefore starts its accumulators anew after this many k-blocks and adds them up in registers, rounded to nearest.
constexpr int kSegmentBlocks = 8;

__host__ __device__ __forceinline__ int lesser(int a, int b) { return a < b ? a : b; }
__host__ __device__ __forceinline__ int greater(int a, int b) { return a > b ? a : b; }

struct Unit {
  int kind, piece, m, n;         // unit row and column in its product
  int k0, k_blocks;              // first k-block (dx: of the piece) and how many
  int split;
  bool last;                     // of the last, possibly narrower, piece
};

__host__ __device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }

// Row units of a band are walked first, then the next column: pairs that work at the same time share a band's rows of A (kept in
// L2 by the choice of `band`) and few columns of B.
__host__ __device__ __forceinline__ void band_decode(int band, int lin, int num_m, int num_n, int& m, int& n) {
  const int b = lin / (band * num_n);
  const int rem = lin - b * (band * num_n);
  const int m0 = b * band, height = band < num_m - m0 ? band : num_m - m0;
  n = rem / height;
  m = m0 + (rem - n * height);
}

struct Counts {                  // units of a full piece and of the last
  int dz, dz_last, dx, dw, dw_last;
};
__host__ __device__ inline Counts loss_counts(const LossParams& p) {
  Counts c;
  c.dz = p.row_units * (p.piece / kLossUnit);
  c.dz_last = p.row_units * ((p.last_cols + kLossUnit - 1) / kLossUnit);
  c.dx = p.want_dx ? p.row_units * p.h_units * p.splits : 0;
  c.dw = p.want_dw ? (p.piece / kLossUnit) * p.h_units : 0;
  c.dw_last = p.want_dw ? ((p.last_cols + kLossUnit - 1) / kLossUnit) * p.h_units : 0;
  return c;
}

// Backward order: dz of the first `ahead` pieces; then for each piece j: dz of piece j + ahead, dx and dW of piece j.
__host__ __device__ __forceinline__ Unit unit_of(const LossParams& p, int lin) {
  const Counts c = loss_counts(p);
  Unit u;
  u.split = 0; u.k0 = 0;
  const int last = p.pieces - 1;
  int kind = kLossDz, piece = 0, rem = lin;
  const int lead = lesser(p.ahead, p.pieces);                   // pieces of the lead-in
  const int lead_units = lead < p.pieces ? lead * c.dz : last * c.dz + c.dz_last;
  if (rem < lead_units) {
    piece = lesser(rem / c.dz, last);
    rem -= piece * c.dz;
  } else {
    rem -= lead_units;
    const int full = c.dz + c.dx + c.dw;
    int j = lesser(rem / full, greater(last - p.ahead, 0));         // steps whose dz piece is a full one
    rem -= j * full;
    if (j + p.ahead == last && j < last) {                   // ... then the one with the last piece
      const int size = c.dz_last + c.dx + c.dw;
      if (rem >= size) { rem -= size; ++j; }
    }
    if (j + p.ahead > last) {                                // ... then steps without any
      const int k = lesser(rem / (c.dx + c.dw > 0 ? c.dx + c.dw : 1), last - j);
      rem -= k * (c.dx + c.dw);
      j += k;
    }
    piece = j;
    const int here = j + p.ahead < last ? c.dz : j + p.ahead == last ? c.dz_last : 0;
    if (rem < here) {
      piece = j + p.ahead;
    } else {
      rem -= here;
      if (rem < c.dx) kind = kLossDx;
      else { rem -= c.dx; kind = kLossDw; }
    }
  }
  u.kind = kind; u.piece = piece; u.last = piece == last;
  const int cols = u.last ? p.last_cols : p.piece;
  if (kind == kLossDz) {
    band_decode(p.band, rem, p.row_units, ceil_div(cols, kLossUnit), u.m, u.n);
    u.k_blocks = ceil_div(p.H, kBK);
  } else if (kind == kLossDx) {
    const int per = p.row_units * p.h_units;
    u.split = rem / per;
    band_decode(8, rem - u.split * per, p.row_units, p.h_units, u.m, u.n);
    u.k0 = u.split * p.split_blocks;
    u.k_blocks = greater(lesser(p.split_blocks, ceil_div(cols, kBK) - u.k0), 0);
  } else {
    band_decode(8, rem, ceil_div(cols, kLossUnit), p.h_units, u.m, u.n);
    u.k_blocks = ceil_div(p.T, kBK) * (p.split2 ? 2 : 1);
  }
  return u;
}

// Columns of a tile that are multiplied (a multiple of 32, at most 256).
__device__ __forceinline__ int tile_cols(int n, int n0) { return min(kLossUnit, (n - n0 + 31) / 32 * 32); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mbar_arrive_release_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" :: "r"(cluster_addr) : "memory");
}
// Adds a tile to global memory in fp32 (clipped at the tensor's bounds), tracked by bulk async-groups.
__device__ __forceinline__ void tma_reduce_add_3d(const void* tmap, const void* smem_src, int x, int y, int z) {
  asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3, %4}], [%1];"
               :: "l"(tmap), "r"(smem_u32(smem_src)), "r"(x), "r"(y), "r"(z) : "memory");
}

template <bool FWD>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
linear_loss_kernel(const __grid_constant__ LossParams p, const __grid_constant__ LossMaps maps) {
  extern __shared__ unsigned char smem_dyn[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
  unsigned char* stage_base = smem;
  unsigned char* staging = smem + kStages * kStageBytes;
  __shared__ uint64_t full_bar[kStages], empty_bar[kStages], tmem_full[2], tmem_empty[2], queue_full[kQueue], queue_empty[kQueue];
  __shared__ int s_queue[kQueue];
  __shared__ int s_progress;           // units whose operands the producer has nearly all requested
  __shared__ uint32_t s_tmem;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int half = static_cast<int>(cluster_ctarank());
  const bool leader = half == 0;
  const unsigned long long budget = p.wait_budget_ns;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) { mbar_init(&full_bar[s], 1); mbar_init(&empty_bar[s], 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(&tmem_full[a], 1); mbar_init(&tmem_empty[a], kEpiWarps * 2); }
    // readers of a queue entry: both producers, the MMA warp, both CTAs' epilogue warps
    for (int q = 0; q < kQueue; ++q) { mbar_init(&queue_full[q], 1); mbar_init(&queue_empty[q], 2 + 1 + 2 * kEpiWarps); }
    mbar_fence_init();
    s_progress = 0;
  }
  if (warp == 1) {
    tmem_alloc<2>(&s_tmem, kTmemCols);
    tmem_relinquish<2>();
  }
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync();
  tc_fence_after_sync();
  const uint32_t tmem_base = s_tmem;

  int total;
  if (FWD) {
    total = p.row_units * ceil_div(p.V, kLossUnit);
  } else {
    const Counts c = loss_counts(p);
    total = (p.pieces - 1) * (c.dz + c.dw) + c.dz_last + c.dw_last + p.pieces * c.dx;
  }
  auto decode = [&](int lin) {
    if constexpr (FWD) {
      Unit u;
      u.kind = kLossStats; u.piece = 0; u.split = 0; u.k0 = 0; u.last = true;
      band_decode(p.band, lin, p.row_units, ceil_div(p.V, kLossUnit), u.m, u.n);
      u.k_blocks = ceil_div(p.H, kBK);
      return u;
    } else {
      return unit_of(p, lin);
    }
  };
  // The next queue entry (warp-uniform for whole warps); false: a wait gave up.
  auto next_unit = [&](int it, int& lin) {
    const int q = it % kQueue;
    const bool got = leader ? mbar_wait<false>(&queue_full[q], (it / kQueue) & 1, budget, p.status)
                            : mbar_wait<true>(&queue_full[q], (it / kQueue) & 1, budget, p.status);
    if (!got) return false;
    lin = *reinterpret_cast<volatile int*>(&s_queue[q]);
    return true;
  };
  auto release_entry = [&](int it) {
    uint64_t* bar = &queue_empty[it % kQueue];
    if (leader) mbar_arrive(bar); else mbar_arrive_cluster(cluster_map(bar, 0));
  };

  if (warp == 10) {
    // ------------------------------------------------------------------ scheduler (first CTA of a pair)
    if (leader && lane == 0) {
      for (int it = 0;; ++it) {
        const int q = it % kQueue;
        if (!mbar_wait<true>(&queue_empty[q], ((it / kQueue) & 1) ^ 1, budget, p.status)) break;
        if (!spin_until([&] { return *reinterpret_cast<volatile int*>(&s_progress) >= it; }, budget, p.status)) break;
        const int lin = atomicAdd(p.claim, 1);
        s_queue[q] = lin;
        st_cluster(cluster_map(&s_queue[q], 1), lin);
        mbar_arrive(&queue_full[q]);
        mbar_arrive_release_cluster(cluster_map(&queue_full[q], 1));
        if (lin >= total) break;
      }
    }
  } else if (warp == 0) {
    // ------------------------------------------------------------------ TMA producer
    if (lane == 0) {
      int stage = 0; uint32_t phase = 0; int issued = 0; bool ok = true;
      for (int it = 0; ok; ++it) {
        int lin;
        if (!next_unit(it, lin)) { ok = false; break; }
        release_entry(it);
        if (lin >= total) break;
        const Unit u = decode(lin);
        if (!FWD) {
          // what this unit reads, or overwrites, of other units' results (all of lower numbers)
          const Counts c = loss_counts(p);
          auto reached = [&](int list, int piece, int units) {
            const int* d = p.done + list * p.pieces + piece;
            if (spin_until([&] { return ld_acquire_gpu(d) >= units * kDoneWarps; }, budget, p.status)) return true;
            report_failure(p.status, kStatusTimeoutTileGate, kKernelLoss, list, p.rank, piece, units * kDoneWarps, ld_acquire_gpu(d));
            return false;
          };
          if (u.kind == kLossDz) {
            if (u.piece >= p.buffers)      // the buffer's piece before was never the last one
              ok = reached(1, u.piece - p.buffers, c.dx) && reached(2, u.piece - p.buffers, c.dw);
          } else {
            ok = reached(0, u.piece, u.last ? c.dz_last : c.dz);
            // sums of pieces are added in the order of the pieces, so that a repeated call gives the same bits
            if (ok && u.kind == kLossDx && u.piece > 0) ok = reached(1, u.piece - 1, c.dx);
          }
          if (!ok) break;
          fence_proxy_async();
        }
        const int n_cols = (u.kind <= kLossDz) ? (FWD ? p.V : (u.last ? p.last_cols : p.piece)) : p.H;
        const int n0 = u.n * kLossUnit;
        const int b0 = n0 + half * (tile_cols(n_cols, n0) / 2);
        const int a0 = u.m * kLossUnit + half * 128;
        const int v0 = u.piece * (FWD ? 0 : p.piece);
        const int zbuf = FWD ? 0 : (u.piece % p.buffers) * (p.split2 ? 2 : 1);
        const int t_blocks = ceil_div(p.T, kBK);
        const int warn = max(u.k_blocks - kClaimAhead, 0);
        if (u.k_blocks == 0 && leader) st_volatile_shared(&s_progress, it + 1);
        for (int kb = 0; kb < u.k_blocks; ++kb) {
          if (leader && kb == warn) st_volatile_shared(&s_progress, it + 1);
          if (!mbar_wait(&empty_bar[stage], phase ^ 1, budget, p.status)) {
            report_failure(p.status, kStatusTimeoutPipeline, kKernelLoss, 0, p.rank, lin, kb, stage);
            ok = false; break;
          }
          unsigned char* sa = stage_base + stage * kStageBytes;
          unsigned char* sb = sa + kOperandBytes;
          // Both CTAs' bytes are counted on the first CTA's barrier, which that CTA arms for the sum.
          if (leader) mbar_arrive_expect_tx(&full_bar[stage], 2 * kStageBytes);
          const uint32_t bar = cluster_map(&full_bar[stage], 0);
          const int k = (u.k0 + kb) * kBK;
          if (FWD || u.kind == kLossDz) {
            tma_load_3d_pair(sa, &maps.x_k, bar, k, a0, 0);
            tma_load_3d_pair(sb, &maps.w_k, bar, k, v0 + b0, 0);
          } else if (u.kind == kLossDx) {
            // split2: the first CTA multiplies the leading halves of dz, the second the remainders
            if (p.split2) tma_load_3d_pair(sa, &maps.z_k[u.last], bar, k, 0, zbuf + half);
            else tma_load_3d_pair(sa, &maps.z_k[u.last], bar, k, a0, zbuf);
            tma_load_3d_pair(sb, &maps.w_mn, bar, b0, v0 + k, 0);
            tma_load_3d_pair(sb + kOperandBytes / 2, &maps.w_mn, bar, b0 + 64, v0 + k, 0);
          } else {
            const int rest = kb >= t_blocks ? 1 : 0;         // split2: all leading halves, then all remainders
            const int t = (kb - rest * t_blocks) * kBK;
            tma_load_3d_pair(sa, &maps.z_mn[u.last], bar, a0, t, zbuf + rest);
            tma_load_3d_pair(sa + kOperandBytes / 2, &maps.z_mn[u.last], bar, a0 + 64, t, zbuf + rest);
            tma_load_3d_pair(sb, &maps.x_mn, bar, b0, t, 0);
            tma_load_3d_pair(sb + kOperandBytes / 2, &maps.x_mn, bar, b0 + 64, t, 0);
          }
          ++issued;
          if (++stage == kStages) { stage = 0; phase ^= 1; }
        }
      }
      if (!ok && issued > 0) {       // let the copies in flight land before the CTA may exit (bounded)
        const unsigned long long t0 = globaltimer_ns();
        while (globaltimer_ns() - t0 < 2000000ull) {}
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------ MMA issuer (first CTA of a pair)
    if (leader) {
      constexpr uint32_t idesc_kk = umma_idesc_bf16(256, 0, 0, 0), idesc_km = umma_idesc_bf16(256, 0, 0, 1), idesc_mm = umma_idesc_bf16(256, 0, 1, 1);
      int stage = 0; uint32_t phase = 0; int acc = 0; uint32_t acc_phase = 0; bool ok = true;
      for (int it = 0; ok; ++it) {
        int lin = 0;
        if (!__all_sync(0xffffffffu, next_unit(it, lin))) { ok = false; break; }
        __syncwarp();
        if (lane == 0) release_entry(it);
        if (lin >= total) break;
        const Unit u = decode(lin);
        if (u.k_blocks == 0) continue;
        const bool a_mn = !FWD && u.kind == kLossDw, b_mn = !FWD && u.kind >= kLossDx;
        const int n_cols = (u.kind <= kLossDz) ? (FWD ? p.V : (u.last ? p.last_cols : p.piece)) : p.H;
        const uint32_t idesc = (a_mn ? idesc_mm : b_mn ? idesc_km : idesc_kk) | (static_cast<uint32_t>(tile_cols(n_cols, u.n * kLossUnit) >> 3) << 17);
        // per 16 elements of K: 32 bytes along a K-major row, 16 rows of 128 bytes of an MN-major box
        const uint32_t step_a = a_mn ? 16 * 128 : 32, step_b = b_mn ? 16 * 128 : 32;
        const uint32_t lbo_a = a_mn ? kBK * 128 : 16, lbo_b = b_mn ? kBK * 128 : 16;
        const int segment = FWD ? kSegmentBlocks : u.k_blocks;
        for (int first = 0; first < u.k_blocks && ok; first += segment) {
        if (!__all_sync(0xffffffffu, mbar_wait<true>(&tmem_empty[acc], acc_phase ^ 1, budget, p.status))) { ok = false; break; }
        tc_fence_after_sync();
        const uint32_t tmem_d = tmem_base + acc * kLossUnit;
        const int end = min(first + segment, u.k_blocks);
        for (int kb = first; kb < end; ++kb) {
          if (!__all_sync(0xffffffffu, mbar_wait<true>(&full_bar[stage], phase, budget, p.status))) { ok = false; break; }
          tc_fence_after_sync();
          if (elect_one()) {
            const uint32_t a_addr = smem_u32(stage_base + stage * kStageBytes), b_addr = a_addr + kOperandBytes;
#pragma unroll
            for (int j = 0; j < kBK / 16; ++j)
              umma_bf16_ss<2>(tmem_d, umma_smem_desc(a_addr + j * step_a, lbo_a, 1024), umma_smem_desc(b_addr + j * step_b, lbo_b, 1024),
                              idesc, (kb > first || j > 0) ? 1u : 0u);
            umma_commit<2>(&empty_bar[stage]);
            if (kb == end - 1) umma_commit<2>(&tmem_full[acc]);
          }
          __syncwarp();
          if (++stage == kStages) { stage = 0; phase ^= 1; }
        }
        acc ^= 1; if (acc == 0) acc_phase ^= 1;
        }
      }
      if (!ok && lane == 0) report_failure(p.status, kStatusTimeoutPipeline, kKernelLoss, 1, p.rank, 0, 0, 0);
    }
  } else {
    // ------------------------------------------------------------------ epilogue: a warp reads the 32 accumulator lanes of its quarter,
    // warps 2..5 the left 128 columns of the tile and warps 6..9 the right ones.  Warps do not wait for one another.
    const int quarter = warp & 3, side = (warp - 2) >> 2;
    unsigned char* stage_tile = staging + (warp - 2) * kStagingBytes;
    const uint32_t stg = smem_u32(stage_tile);
    int acc = 0; uint32_t acc_phase = 0;
    for (int it = 0;; ++it) {
      int lin = 0;
      if (!__all_sync(0xffffffffu, next_unit(it, lin))) break;
      __syncwarp();
      if (lane == 0) release_entry(it);
      if (lin >= total) break;
      const Unit u = decode(lin);
      const int n_cols = (u.kind <= kLossDz) ? (FWD ? p.V : (u.last ? p.last_cols : p.piece)) : p.H;
      const int n0 = u.n * kLossUnit + side * 128;                 // first column of this warp
      const int chunks = min(4, max(0, (n_cols - n0 + 31) / 32));
      const int row0 = u.m * kLossUnit + half * 128 + quarter * 32;  // first row of this warp
      const int row = row0 + lane;
      const bool empty = u.k_blocks == 0;
      // fetched while the tensor cores still work on the tile
      int col = -1; float lse2 = 0.f, c_t = 0.f;
      bool dead = true;              // an ignored token (or no token): zeros whatever its logits are
      float scale = 1.f;
      if (u.kind <= kLossDz) {
        if (row < p.T) {
          const long long y = p.targets[row];
          const long long rel = y - (FWD ? 0 : static_cast<long long>(u.piece) * p.piece) - n0;
          if (rel >= 0 && rel < 128 && y < p.V) col = static_cast<int>(rel);
          if (!FWD && y != p.ignore_index) {
            dead = false;
            c_t = p.row_scale != nullptr ? p.row_scale[row] : 1.f;
            lse2 = p.lse[row] * kLog2e;
          }
        }
      } else if (u.kind == kLossDw) {
        if (p.scale != nullptr) scale = *p.scale;
        if (p.scale2 != nullptr) scale *= *p.scale2;
      }
      auto accumulated = [&] {
        if (!__all_sync(0xffffffffu, mbar_wait(&tmem_full[acc], acc_phase, budget, p.status))) {
          if (lane == 0) report_failure(p.status, kStatusTimeoutPipeline, kKernelLoss, 2, p.rank, lin, acc, 0);
          return false;
        }
        tc_fence_after_sync();
        return true;
      };
      if (!FWD && !empty && !accumulated()) break;
      const uint32_t lanes = tmem_base + side * 128 + (static_cast<uint32_t>(quarter * 32) << 16);
      const uint32_t taddr = lanes + acc * kLossUnit;
      auto give_back = [&] {
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(cluster_map(&tmem_empty[acc], 0));
      };
      uint32_t r[32];
      auto fetch = [&](int c) {
        if (empty) {
#pragma unroll
          for (int i = 0; i < 32; ++i) r[i] = 0;
        } else {
          tmem_ld_32x32(taddr + c * 32, r); tmem_ld_wait();
        }
      };
      if (FWD) {
        float z[128];
#pragma unroll
        for (int i = 0; i < 128; ++i) z[i] = 0.f;
        bool ok = true;
        for (int first = 0; first < u.k_blocks; first += kSegmentBlocks) {
          if (!(ok = accumulated())) break;
#pragma unroll
          for (int c = 0; c < 8; ++c) {       // (16 columns at a time: 32 spill)
            uint32_t part[16];
            tmem_ld_32x16(lanes + acc * kLossUnit + c * 16, part); tmem_ld_wait();
            if (c == 7) give_back();
#pragma unroll
            for (int i = 0; i < 16; ++i) z[c * 16 + i] += __uint_as_float(part[i]);
          }
          acc ^= 1; if (acc == 0) acc_phase ^= 1;
        }
        if (!ok) break;
        const int left = n_cols - n0;        // (columns that were not multiplied hold anything)
        if (left <= 0) continue;
        const float ninf = __int_as_float(0xff800000);
        if (left < 128) {
#pragma unroll
          for (int i = 0; i < 128; ++i) if (i >= left) z[i] = ninf;
        }
        if (__any_sync(0xffffffffu, col >= 0)) {
          float zt = 0.f;
#pragma unroll
          for (int i = 0; i < 128; ++i) if (col == i) zt = z[i];
          if (col >= 0) p.target_logit[row] = zt;
        }
        float top[4] = {ninf, ninf, ninf, ninf};
#pragma unroll
        for (int i = 0; i < 128; ++i) top[i & 3] = fmaxf(top[i & 3], z[i]);
        const float m = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        // (a row of -inf: subtract 0, every term is exp(-inf) = 0)
        const float ref = m == ninf ? 0.f : m * kLog2e;
        float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 128; ++i) s[i & 3] += ex2(fmaf(z[i], kLog2e, -ref));
        if (row < p.T) p.parts[static_cast<size_t>(u.n * 2 + side) * p.T + row] = make_float2(m, (s[0] + s[1]) + (s[2] + s[3]));
      } else if (u.kind == kLossDz) {
        const CUtensorMap* out = &maps.z_out[u.last];
        const int zbuf = (u.piece % p.buffers) * (p.split2 ? 2 : 1);
        const int passes = p.split2 ? 2 : 1;
        const bool rows = row0 < p.T;
#pragma unroll 1
        for (int part = 0; part < passes; ++part) {
#pragma unroll 1
          for (int c = 0; c < chunks; ++c) {
            fetch(c);
            if (c == chunks - 1 && part == passes - 1) give_back();
            if (!rows) continue;
            const int left = n_cols - n0 - c * 32;
            const bool target_here = __any_sync(0xffffffffu, (col >> 5) == c);
            if ((c & 1) == 0) {
              if (lane == 0) bulk_wait_read();
              __syncwarp();
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              uint32_t o[4];
#pragma unroll
              for (int h = 0; h < 4; ++h) {
                float d[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const int i = q * 8 + h * 2 + e;
                  float v = ex2(fmaf(__uint_as_float(r[i]), kLog2e, -lse2));
                  if (target_here && col == c * 32 + i) v -= 1.f;
                  v *= c_t;
                  if (dead || i >= left) v = 0.f;
                  d[e] = v;
                }
                o[h] = pack_bf16x2(d[0], d[1]);
                if (part == 1) {
                  const float2 lead = unpack_bf16x2(o[h]);
                  o[h] = pack_bf16x2(d[0] - lead.x, d[1] - lead.y);
                }
              }
              st_shared_v4(stg + stage_off<128>(lane, (c & 1) * 4 + q), o[0], o[1], o[2], o[3]);
            }
            if ((c & 1) == 1 || c == chunks - 1) {
              fence_proxy_async_smem();
              __syncwarp();
              if (lane == 0) { tma_store_3d(out, stage_tile, n0 + (c & ~1) * 32, row0, zbuf + part); bulk_commit(); }
            }
          }
        }
        if (chunks == 0) give_back();
        __syncwarp();
        if (lane == 0) { bulk_wait_all(); fence_proxy_async(); red_release_gpu_add(p.done + u.piece, 1); }
      } else if (u.kind == kLossDx) {
        const int z = p.split2 ? u.split * 2 + half : u.split;
        const int y = p.split2 ? quarter * 32 : row0;
#pragma unroll 1
        for (int c = 0; c < chunks; ++c) {
          fetch(c);
          if (c == chunks - 1 && !empty) give_back();
          if (y >= p.T) continue;
          if (lane == 0) bulk_wait_read();
          __syncwarp();
#pragma unroll
          for (int q = 0; q < 8; ++q) st_shared_v4(stg + stage_off<128>(lane, q), r[q * 4], r[q * 4 + 1], r[q * 4 + 2], r[q * 4 + 3]);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (u.piece == 0) tma_store_3d(&maps.dx, stage_tile, n0 + c * 32, y, z);
            else tma_reduce_add_3d(&maps.dx, stage_tile, n0 + c * 32, y, z);
            bulk_commit();
          }
        }
        if (chunks == 0 && !empty) give_back();
        __syncwarp();
        if (lane == 0) { bulk_wait_all(); red_release_gpu_add(p.done + p.pieces + u.piece, 1); }
      } else {
        const int v = u.piece * p.piece + row0;
#pragma unroll 1
        for (int c = 0; c < chunks; ++c) {
          fetch(c);
          if (c == chunks - 1) {
            give_back();
            if (lane == 0) red_release_gpu_add(p.done + 2 * p.pieces + u.piece, 1);   // the operands have been read
          }
          if (v >= p.V) continue;
          if ((c & 1) == 0) {
            if (lane == 0) bulk_wait_read();
            __syncwarp();
          }
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t o[4];
#pragma unroll
            for (int h = 0; h < 4; ++h)
              o[h] = pack_bf16x2(scale * __uint_as_float(r[q * 8 + h * 2]), scale * __uint_as_float(r[q * 8 + h * 2 + 1]));
            st_shared_v4(stg + stage_off<128>(lane, (c & 1) * 4 + q), o[0], o[1], o[2], o[3]);
          }
          if ((c & 1) == 1 || c == chunks - 1) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) { tma_store_3d(&maps.dw, stage_tile, n0 + (c & ~1) * 32, v, 0); bulk_commit(); }
          }
        }
        if (chunks == 0) {
          give_back();
          if (lane == 0) red_release_gpu_add(p.done + 2 * p.pieces + u.piece, 1);
        }
      }
      if (!FWD && !empty) { acc ^= 1; if (acc == 0) acc_phase ^= 1; }
    }
    if (lane == 0) bulk_wait_all();
  }

  // ---------------------------------------------------------------------- teardown
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc<2>(tmem_base, kTmemCols);
  }
}

template <bool FWD>
cudaError_t launch_pairs(const LossParams& p, const LossMaps& m, long long units, int sms, cudaStream_t stream) {
  auto kernel = linear_loss_kernel<FWD>;
  static std::atomic<bool> configured[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[dev].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes);
    if (e != cudaSuccess) return e;
    configured[dev].store(true, std::memory_order_release);
  }
  const long long pairs = units < sms / 2 ? units : sms / 2;
  kernel<<<static_cast<unsigned>(pairs * 2), kThreads, kSmemBytes, stream>>>(p, m);
  return cudaGetLastError();
}

// ---------------------------------------------------------------------------------------------
// Joins the parts of each row, and the rows' losses.  A block takes 32 rows: lanes are rows, warps take parts in turn.
// ---------------------------------------------------------------------------------------------
constexpr int kFinalWarps = 16;

__global__ void __launch_bounds__(kFinalWarps * 32) loss_final_kernel(const LossFinalParams p) {
  __shared__ float2 joined[kFinalWarps][32];
  __shared__ double sums[kFinalWarps];
  __shared__ int counts[kFinalWarps];
  __shared__ bool last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long row = static_cast<long long>(blockIdx.x) * 32 + lane;
  const float ninf = __int_as_float(0xff800000);
  auto join = [&](float2 a, float2 b) {
    const float m = fmaxf(a.x, b.x);
    if (m == ninf) return make_float2(m, a.y + b.y);
    return make_float2(m, a.y * exp2f((a.x - m) * kLog2e) + b.y * exp2f((b.x - m) * kLog2e));
  };
  float2 v = make_float2(ninf, 0.f);
  if (row < p.T) {
#pragma unroll 4
    for (int i = warp; i < p.num_parts; i += kFinalWarps) v = join(v, p.parts[static_cast<size_t>(i) * p.T + row]);
  }
  joined[warp][lane] = v;
  __syncthreads();
  if (warp == 0 && row < p.T) {
    for (int w = 1; w < kFinalWarps; ++w) v = join(v, joined[w][lane]);
    float lse = v.x + logf(v.y);
    const long long y = p.targets[row];
    float loss = 0.f;
    if (y != p.ignore_index) {
      if (y < 0 || y >= p.V) {       // the loss and every gradient become NaN, and the caller can ask why
        report_note(p.status, kStatusBadTarget, kKernelLoss, 0, p.rank, static_cast<int>(row), p.V, static_cast<int>(y));
        lse = loss = __int_as_float(0x7fc00000);
      } else {
        loss = lse - p.target_logit[row];
      }
    }
    p.lse[row] = lse;
    p.each[row] = loss;
  }
  if (!p.mean && !p.sum) return;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(p.ticket, 1) == static_cast<int>(gridDim.x) - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  double sum = 0.0; int count = 0;
  for (int t = threadIdx.x; t < p.T; t += blockDim.x) {
    sum += static_cast<double>(__ldcg(p.each + t));
    count += p.targets[t] != p.ignore_index ? 1 : 0;
  }
  for (int d = 16; d > 0; d >>= 1) {
    sum += __shfl_down_sync(0xffffffffu, sum, d);
    count += __shfl_down_sync(0xffffffffu, count, d);
  }
  if (lane == 0) { sums[warp] = sum; counts[warp] = count; }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kFinalWarps; ++w) { sum += sums[w]; count += counts[w]; }
    // without a counted token the mean is 0 / 0, and its gradients are zeros
    *p.loss = static_cast<float>(p.mean ? sum / static_cast<double>(count) : sum);
    if (p.mean) *p.inv_count = count > 0 ? static_cast<float>(1.0 / count) : 0.f;
  }
}

// dx = scale * sum of its slots, rounded once.
__global__ void __launch_bounds__(256) loss_dx_kernel(const LossDxParams p) {
  const size_t n = static_cast<size_t>(p.T) * p.H;
  float scale = p.scale != nullptr ? *p.scale : 1.f;
  if (p.scale2 != nullptr) scale *= *p.scale2;
  for (size_t i = (static_cast<size_t>(blockIdx.x) * blockDim.x + threadIdx.x) * 8; i < n; i += static_cast<size_t>(gridDim.x) * blockDim.x * 8) {
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
    for (int s = 0; s < p.slots; ++s) {
      const float4* q = reinterpret_cast<const float4*>(p.parts + s * n + i);
      const float4 u = __ldcs(q), w = __ldcs(q + 1);
      a.x += u.x; a.y += u.y; a.z += u.z; a.w += u.w;
      b.x += w.x; b.y += w.y; b.z += w.z; b.w += w.w;
    }
    *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.dx) + i) =
        make_uint4(pack_bf16x2(scale * a.x, scale * a.y), pack_bf16x2(scale * a.z, scale * a.w),
                   pack_bf16x2(scale * b.x, scale * b.y), pack_bf16x2(scale * b.z, scale * b.w));
  }
}

}  // namespace

void loss_backward_unit(const LossParams& p, int lin, int (&out)[7]) {
  const Unit u = unit_of(p, lin);
  const int v[7] = {u.kind, u.piece, u.m, u.n, u.split, u.k0, u.k_blocks};
  for (int i = 0; i < 7; ++i) out[i] = v[i];
}
long long loss_backward_units(const LossParams& p) {
  const Counts c = loss_counts(p);
  return static_cast<long long>(p.pieces - 1) * (c.dz + c.dw) + c.dz_last + c.dw_last + static_cast<long long>(p.pieces) * c.dx;
}

cudaError_t launch_loss_forward(const LossParams& p, const LossMaps& m, int sms, cudaStream_t stream) {
  return launch_pairs<true>(p, m, static_cast<long long>(p.row_units) * ((p.V + kLossUnit - 1) / kLossUnit), sms, stream);
}
cudaError_t launch_loss_backward(const LossParams& p, const LossMaps& m, int sms, cudaStream_t stream) {
  return launch_pairs<false>(p, m, loss_backward_units(p), sms, stream);
}
cudaError_t launch_loss_final(const LossFinalParams& p, cudaStream_t stream) {
  loss_final_kernel<<<static_cast<unsigned>((p.T + 31) / 32), kFinalWarps * 32, 0, stream>>>(p);
  return cudaGetLastError();
}
cudaError_t launch_loss_dx(const LossDxParams& p, cudaStream_t stream) {
  const long long vectors = static_cast<long long>(p.T) * p.H / 8;
  const long long blocks = (vectors + 255) / 256;
  loss_dx_kernel<<<static_cast<unsigned>(blocks < 148 * 8 ? blocks : 148 * 8), 256, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace sep

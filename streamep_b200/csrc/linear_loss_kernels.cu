// Output projection with softmax cross entropy, without logits in memory: z = x W^T, and for each token t with target y
//   loss_t = log sum_v exp(z_tv) - z_ty,   dz_tv = c_t (exp(z_tv) / sum_v exp(z_tv) - [v = y]),   dx = dz W,   dW = dz^T x.
// Differences with the row's maximum are formed first, (z - max) log2 e and not z log2 e - max log2 e: logits masked with the type's lowest
// value would overflow in the second form.
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
// Two forms.  The tensor cores multiply 256 rows at a time however few of them exist, so with the tokens as rows a call of 300 pays for 512
// and one of 1 for 256.  The narrow form makes the vocabulary (for dx: the hidden dimension) the rows, and 32 to 192 tokens the columns of
// a unit, which cost what they are; its epilogues turn 32 x 32 pieces around in shared memory, so that a thread has a token again.
//
// Order and progress.  Units are claimed one after another from a counter, by CTAs that run, so a unit that waits for others
// only waits for units that are already being worked on: the kernel needs no number of co-resident CTAs.
#include <atomic>

#include "linear_loss.h"
#include "ptx.cuh"

namespace sep {

namespace {

constexpr int kBK = 64;                          // bf16 elements of a k-block: one 128-byte swizzle row
constexpr int kOperandBytes = 128 * kBK * 2;     // A or B of one CTA: 128 rows of a k-block
constexpr int kStageBytes = 2 * kOperandBytes;
constexpr int kEpiWarps = 8;
constexpr int kThreads = (2 + kEpiWarps + 1) * 32;   // 0 TMA producer, 1 MMA, 2..9 epilogue, 10 scheduler
constexpr int kTileBytes = 4096;                 // 32 rows of 128 bytes
constexpr int kStagingBytes = 2 * kTileBytes;    // per epilogue warp of the backward: two of them
// Of the two tiles that begin at `own` the one that is not at `tile`, wherever shared memory places them.
__host__ __device__ constexpr uint32_t other_tile(uint32_t own, uint32_t tile) { return own + kTileBytes - (tile - own); }
constexpr bool tiles_take_turns() {
  for (uint32_t own = 0; own < 4 * kStagingBytes; own += 1024)
    if (other_tile(own, own) != own + kTileBytes || other_tile(own, own + kTileBytes) != own) return false;
  return true;
}
static_assert(tiles_take_turns(), "a warp's two staging tiles take turns at every alignment of shared memory");
constexpr int kQueue = 4;
// The forward's epilogue stores nothing but statistics, so all shared memory is its operand ring's.
// The narrow forward needs one tile a warp, keeps each warp's statistics of all its units beside it (a part for every 32 columns made the
// joining kernel longer than the product: 100 tokens, V 100003 92 -> 108 us), and has as many stages as its few tokens leave room for.
constexpr int kNarrowStages = 9, kNarrowRing = 5 * kStageBytes;
constexpr int kNarrowUnits = 3, kNarrowTiles = 3;   // units of tokens of the narrow form, and a warp's 32-token pieces of one, at most
constexpr int kNarrowStats = kNarrowUnits * kNarrowTiles * 32 * 8;   // bytes a warp: [unit][its 32-token pieces][lane] (maximum, sum)
constexpr int stages_of(bool fwd, bool narrow) { return narrow ? kNarrowStages : fwd ? 7 : 5; }
constexpr int ring_bytes(bool fwd, bool narrow) { return narrow ? kNarrowRing : stages_of(fwd, narrow) * kStageBytes; }
constexpr int smem_bytes(bool fwd, bool narrow) { return ring_bytes(fwd, narrow) + (fwd ? (narrow ? kEpiWarps * (4096 + kNarrowStats) : 0) : kEpiWarps * kStagingBytes) + 1024; }
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
  int tiles;                     // column tiles, one after another (dw)
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
  const int groups = (p.h_units + p.dw_group - 1) / p.dw_group;
  c.dw = p.want_dw ? (p.piece / kLossUnit) * groups : 0;
  c.dw_last = p.want_dw ? ((p.last_cols + kLossUnit - 1) / kLossUnit) * groups : 0;
  return c;
}

// Backward order: dz of the first `ahead` pieces; then for each piece j: dz of piece j + ahead, dx and dW of piece j (`dw_lead` dw units of
// it before the dx units).
__host__ __device__ __forceinline__ Unit unit_of(const LossParams& p, int lin) {
  const Counts c = loss_counts(p);
  Unit u;
  u.split = 0; u.k0 = 0; u.tiles = 1;
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
      const int lead_dw = lesser(p.dw_lead, j == last ? c.dw_last : c.dw);
      kind = rem >= lead_dw && rem < lead_dw + c.dx ? kLossDx : kLossDw;
      if (kind == kLossDx) rem -= lead_dw;
      else if (rem >= lead_dw) rem -= c.dx;
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
    band_decode(8, rem, ceil_div(cols, kLossUnit), ceil_div(p.h_units, p.dw_group), u.m, u.n);
    u.n *= p.dw_group;
    u.tiles = lesser(p.dw_group, p.h_units - u.n);
    u.k_blocks = ceil_div(p.T, p.dw_rows) * (p.split2 ? 2 : 1);
  }
  return u;
}

// dz lies in panels of 64 columns, [panel][T][64]: what a load or a store moves is one contiguous block (with rows of a whole piece,
// 128 bytes here and the next 200 KB away, calls of 1 to 800 tokens took 2 to 4 % longer).  The first panel of a piece, of its leading halves or (split2) remainders:
__device__ __forceinline__ int panel_of(const LossParams& p, int piece, int rest) {
  return ((piece % p.buffers) * (p.split2 ? 2 : 1) + rest) * (p.piece / 64);
}

// Columns of a tile that are multiplied (a multiple of 32, at most 256).
__device__ __forceinline__ int tile_cols(int n, int n0) { return min(kLossUnit, (n - n0 + 31) / 32 * 32); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Two fp32 operations in one instruction, for the epilogues of the wide form: 4001 tokens, hidden 2048, V 100003 forward 1225 -> 1175 us,
// 8192 x 512 x 32000 with gradients 1135 -> 1113.  (The narrow form, turned around in between, gained nothing by them.)
struct Pair { unsigned long long v; };
__device__ __forceinline__ Pair pair_of(float a, float b) { Pair p; asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(a), "f"(b)); return p; }
__device__ __forceinline__ void parts_of(Pair p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p.v)); }
__device__ __forceinline__ Pair operator+(Pair a, Pair b) { Pair d; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v)); return d; }
__device__ __forceinline__ Pair operator*(Pair a, Pair b) { Pair d; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v)); return d; }
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) { Pair d; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v)); return d; }
__device__ __forceinline__ Pair ex2(Pair p) { float a, b; parts_of(p, a, b); return pair_of(ex2(a), ex2(b)); }
__device__ __forceinline__ void mbar_arrive_release_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" :: "r"(cluster_addr) : "memory");
}
// Adds a tile to global memory in fp32 (clipped at the tensor's bounds), tracked by bulk async-groups.
__device__ __forceinline__ void tma_reduce_add_3d(const void* tmap, const void* smem_src, int x, int y, int z) {
  asm volatile("cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.tile.bulk_group [%0, {%2, %3, %4}], [%1];"
               :: "l"(tmap), "r"(smem_u32(smem_src)), "r"(x), "r"(y), "r"(z) : "memory");
}

__device__ __forceinline__ void st_shared_b16(uint32_t addr, uint32_t low_half) {
  asm volatile("{\n\t.reg .b16 h;\n\tcvt.u16.u32 h, %1;\n\tst.shared.b16 [%0], h;\n\t}" :: "r"(addr), "r"(low_half) : "memory");
}
// p - 1 of the target, from the forward's own logit: the one computed again lacks what kSegmentBlocks is for, 1e-4 of a logit of 12 at H 7168,
// which is more than 1 - p of a token that the model is sure of.
__device__ __forceinline__ float target_gradient(float target_z, float top, float log2_sum) {
  return expm1f(fmaf(-0.693147181f, log2_sum, target_z - top));
}
// Lane l has element i of 32 in v[i]; afterwards lane l has in v[j] what lane j had in v[l].  `tile`: 4 KB of the warp's own.
__device__ __forceinline__ void st_shared_f32(uint32_t addr, float v) { asm volatile("st.shared.f32 [%0], %1;" :: "r"(addr), "f"(v) : "memory"); }
__device__ __forceinline__ float ld_shared_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void turn_write(uint32_t tile, int lane, int i, float v) { st_shared_f32(tile + (i * 32 + (lane ^ i)) * 4, v); }
__device__ __forceinline__ float turn_read(uint32_t tile, int lane, int j) { return ld_shared_f32(tile + (lane * 32 + (j ^ lane)) * 4); }

template <bool FWD, bool NARROW>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
linear_loss_kernel(const __grid_constant__ LossParams p, const __grid_constant__ LossMaps maps) {
  constexpr int kStages = stages_of(FWD, NARROW);
  const int stages = NARROW ? p.stages : kStages;
  const int stage_bytes = NARROW ? p.stage_bytes : kStageBytes;
  const int dw_rows = NARROW ? p.dw_rows : kBK;
  extern __shared__ unsigned char smem_dyn[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
  unsigned char* stage_base = smem;
  unsigned char* staging = smem + ring_bytes(FWD, NARROW);
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
  grid_release();
  if (FWD && blockIdx.x == 0)
    for (int i = threadIdx.x; i < p.zero_ints; i += kThreads) p.zero[i] = 0;

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
      u.kind = kLossStats; u.piece = 0; u.split = 0; u.k0 = 0; u.tiles = 1; u.last = true;
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
        if (!spin_until([&] { return *reinterpret_cast<volatile int*>(&s_progress) >= it - p.claim_lead; }, budget, p.status)) break;
        const int lin = FWD && p.claim == nullptr ? static_cast<int>(blockIdx.x / 2 + it * (gridDim.x / 2)) : atomicAdd(p.claim, 1);
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
      int seen_dz = -1, seen_free = -1, seen_sum = -1;      // pieces whose counters were found complete: not asked for again
      for (int it = 0; ok; ++it) {
        int lin;
        if (!next_unit(it, lin)) { ok = false; break; }
        release_entry(it);
        if (lin >= total) break;
        Unit u = decode(lin);
        if (!FWD) {
          // what this unit reads, or overwrites, of other units' results (all of lower numbers)
          const Counts c = loss_counts(p);
          auto reached = [&](int list, int piece, int units) {
            const int* d = p.done + list * p.pieces + piece;       // (list 3: by column tile)
            if (spin_until([&] { return ld_acquire_gpu(d) >= units * kDoneWarps; }, budget, p.status)) return true;
            report_failure(p.status, kStatusTimeoutTileGate, kKernelLoss, list, p.rank, piece, units * kDoneWarps, ld_acquire_gpu(d));
            return false;
          };
          bool asked = false;
          auto once = [&](int& seen, int piece, auto ask) {
            if (piece <= seen) return true;
            if (!ask()) return false;
            seen = piece; asked = true;
            return true;
          };
          if (u.kind == kLossDz) {
            if (u.piece >= p.buffers)      // (the piece that was in this buffer was not the last one)
              ok = once(seen_free, u.piece - p.buffers, [&] { return reached(1, u.piece - p.buffers, c.dx) && reached(2, u.piece - p.buffers, c.dw); });
          } else if (u.kind == kLossDx) {
            ok = once(seen_dz, u.piece, [&] { return reached(0, u.piece, u.last ? c.dz_last : c.dz); });
            // sums of pieces are added in the order of the pieces, so that a repeated call gives the same bits
            if (ok && u.piece > 0) ok = once(seen_sum, u.piece - 1, [&] { return reached(1, u.piece - 1, c.dx); });
          } else if (u.piece > seen_dz) {
            asked = true;
            if (ld_acquire_gpu(p.done + u.piece) >= (u.last ? c.dz_last : c.dz) * kDoneWarps) seen_dz = u.piece;
            else ok = reached(3, u.piece * (p.piece / kLossUnit) + u.m, p.row_units);      // one column tile of dz is enough
          }
          if (!ok) break;
          if (asked) fence_proxy_async();
        }
        const int n_cols = (u.kind <= kLossDz) ? (FWD ? p.V : (u.last ? p.last_cols : p.piece)) : p.H;
        const int a0 = u.m * kLossUnit + half * 128;
        const int v0 = u.piece * (FWD ? 0 : p.piece);
        const int z0 = FWD ? 0 : panel_of(p, u.piece, 0);
        const int t_blocks = ceil_div(p.T, dw_rows);
        // narrow: rows of x / dz that this CTA loads, and which (split2: the leading halves of dz by the first CTA, the remainders by the second)
        const bool both = NARROW && !FWD && u.kind == kLossDx && p.split2;
        const int my_tokens = NARROW ? (both ? p.tile_tokens : p.tile_tokens / 2) : 0;
        const int t0 = NARROW ? u.m * p.tile_tokens + (both ? 0 : half * my_tokens) : 0;
        const uint32_t pair_bytes = NARROW ? 2 * (FWD || u.kind != kLossDw ? kOperandBytes + my_tokens * 128 : 4 * dw_rows * 128) : 2 * kStageBytes;
        const int warn = max(u.k_blocks - kClaimAhead, 0);
        if (u.k_blocks == 0 && leader) st_volatile_shared(&s_progress, it + 1);
        for (int tile = 0; tile < u.tiles && ok; ++tile, ++u.n) {
        const int n0 = u.n * kLossUnit;
        const int b0 = n0 + half * (NARROW && (FWD || u.kind != kLossDw) ? 128 : tile_cols(n_cols, n0) / 2);
        for (int kb = 0; kb < u.k_blocks; ++kb) {
          if (leader && kb == warn && tile == u.tiles - 1) st_volatile_shared(&s_progress, it + 1);
          if (!mbar_wait(&empty_bar[stage], phase ^ 1, budget, p.status)) {
            report_failure(p.status, kStatusTimeoutPipeline, kKernelLoss, 0, p.rank, lin, kb, stage);
            ok = false; break;
          }
          unsigned char* sa = stage_base + stage * stage_bytes;
          unsigned char* sb = sa + kOperandBytes;
          // Both CTAs' bytes are counted on the first CTA's barrier, which that CTA arms for the sum.
          if (leader) mbar_arrive_expect_tx(&full_bar[stage], pair_bytes);
          const uint32_t bar = cluster_map(&full_bar[stage], 0);
          const int k = (u.k0 + kb) * kBK;
          if (FWD || u.kind == kLossDz) {
            tma_load_3d_pair(sa, NARROW ? &maps.w_k : &maps.x_k, bar, k, NARROW ? v0 + b0 : a0, 0);
            tma_load_3d_pair(sb, NARROW ? &maps.x_k : &maps.w_k, bar, k, NARROW ? t0 : v0 + b0, 0);
          } else if (u.kind == kLossDx) {
            unsigned char* sw = NARROW ? sa : sb;
            tma_load_3d_pair(NARROW ? sb : sa, &maps.z_k, bar, 0, NARROW ? t0 : a0, (both && half ? panel_of(p, u.piece, 1) : z0) + u.k0 + kb);
            tma_load_3d_pair(sw, &maps.w_mn, bar, b0, v0 + k, 0);
            tma_load_3d_pair(sw + kOperandBytes / 2, &maps.w_mn, bar, b0 + 64, v0 + k, 0);
          } else {
            const int rest = kb >= t_blocks ? 1 : 0;         // split2: all leading halves, then all remainders
            const int t = (kb - rest * t_blocks) * dw_rows, box = dw_rows * 128;
            unsigned char* const sx = sa + 2 * box;
            const int panel = (rest ? panel_of(p, u.piece, 1) : z0) + a0 / 64;
            tma_load_3d_pair(sa, &maps.z_mn, bar, 0, t, panel);
            tma_load_3d_pair(sa + box, &maps.z_mn, bar, 0, t, panel + 1);
            tma_load_3d_pair(sx, &maps.x_mn, bar, b0, t, 0);
            tma_load_3d_pair(sx + box, &maps.x_mn, bar, b0 + 64, t, 0);
          }
          ++issued;
          if (++stage == stages) { stage = 0; phase ^= 1; }
        }
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
      int stage = 0; uint32_t phase = 0; int acc = 0; uint32_t acc_phase = 0; bool ok = true;
      for (int it = 0; ok; ++it) {
        int lin = 0;
        if (!__all_sync(0xffffffffu, next_unit(it, lin))) { ok = false; break; }
        __syncwarp();
        if (lane == 0) release_entry(it);
        if (lin >= total) break;
        Unit u = decode(lin);
        if (u.k_blocks == 0) continue;
        const bool a_mn = !FWD && (u.kind == kLossDw || (NARROW && u.kind == kLossDx)), b_mn = !FWD && (u.kind == kLossDw || (!NARROW && u.kind == kLossDx));
        const bool tokens = NARROW && (FWD || u.kind != kLossDw);      // columns are tokens
        const int n_cols = (u.kind <= kLossDz) ? (FWD ? p.V : (u.last ? p.last_cols : p.piece)) : p.H;
        for (int tile = 0; tile < u.tiles && ok; ++tile, ++u.n) {
        const int cols = tokens ? (!FWD && u.kind == kLossDx && p.split2 ? 2 : 1) * p.tile_tokens : tile_cols(n_cols, u.n * kLossUnit);
        const uint32_t idesc = umma_idesc_bf16(256, 0, 0, 0) | (a_mn ? 1u << 15 : 0) | (b_mn ? 1u << 16 : 0) | (static_cast<uint32_t>(cols >> 3) << 17);
        // per 16 elements of K: 32 bytes along a K-major row, 16 rows of 128 bytes of an MN-major box
        const uint32_t step_a = a_mn ? 16 * 128 : 32, step_b = b_mn ? 16 * 128 : 32;
        const bool half_blocks = NARROW && !FWD && u.kind == kLossDw && dw_rows != kBK;
        const uint32_t rows = half_blocks ? kBK / 2 : kBK;           // of K in a stage
        const uint32_t lbo_a = a_mn ? rows * 128 : 16, lbo_b = b_mn ? rows * 128 : 16;
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
            const uint32_t a_addr = smem_u32(stage_base + stage * stage_bytes), b_addr = a_addr + kOperandBytes / kBK * rows;
#pragma unroll
            for (int j = 0; j < kBK / 16; ++j)
              if (!NARROW || j < 2 || !half_blocks) umma_bf16_ss<2>(tmem_d, umma_smem_desc(a_addr + j * step_a, lbo_a, 1024), umma_smem_desc(b_addr + j * step_b, lbo_b, 1024),
                              idesc, (kb > first || j > 0) ? 1u : 0u);
            umma_commit<2>(&empty_bar[stage]);
            if (kb == end - 1) umma_commit<2>(&tmem_full[acc]);
          }
          __syncwarp();
          if (++stage == stages) { stage = 0; phase ^= 1; }
        }
        acc ^= 1; if (acc == 0) acc_phase ^= 1;
        }
        }
      }
      if (!ok && lane == 0) report_failure(p.status, kStatusTimeoutPipeline, kKernelLoss, 1, p.rank, 0, 0, 0);
    }
  } else {
    // ------------------------------------------------------------------ epilogue: a warp reads the 32 accumulator lanes of its quarter,
    // warps 2..5 the left 128 columns of the tile and warps 6..9 the right ones.  Warps do not wait for one another.
    const int quarter = warp & 3, side = (warp - 2) >> 2;
    // A tile of results is written to shared memory and leaves by a bulk store, while the warp fills the other one.
    const uint32_t own_tiles = (warp - 2) * (FWD ? kTileBytes : kStagingBytes);          // from `staging` on
    unsigned char* stage_tile = staging + own_tiles;
    auto next_tile = [&] {               // whole warp: the tile that the store before the last one has read
      stage_tile = staging + other_tile(own_tiles, static_cast<uint32_t>(stage_tile - staging));
      if (lane == 0) bulk_wait_read_but_one();
      __syncwarp();
      return smem_u32(stage_tile);
    };
    uint32_t stg = 0;
    // narrow: this warp's 32-token pieces of a unit
    const int pieces32 = NARROW ? p.tile_tokens / 32 : 0;
    const int first32 = side == 0 ? 0 : (pieces32 + 1) / 2, count32 = side == 0 ? (pieces32 + 1) / 2 : pieces32 / 2;
    const uint32_t turn = smem_u32(stage_tile);                    // narrow: where pieces are turned around ...
    unsigned char* const narrow_out = stage_tile + 4096;           // ... and where dz waits for its stores
    int flip = 0;
    float2* const stats = reinterpret_cast<float2*>(staging + kEpiWarps * 4096 + (warp - 2) * kNarrowStats) + lane;    // (forward) [unit row * kNarrowTiles + piece] * 32
    if (FWD && NARROW)
      for (int i = 0; i < kNarrowUnits * kNarrowTiles; ++i) stats[i * 32] = make_float2(__int_as_float(0xff800000), 0.f);
    float scale = 1.f;                   // of dw
    if (!FWD && p.scale != nullptr) scale = *p.scale;
    if (!FWD && p.scale2 != nullptr) scale *= *p.scale2;
    int acc = 0; uint32_t acc_phase = 0;
    bool ok = true;
    for (int it = 0; ok; ++it) {
      int lin = 0;
      if (!__all_sync(0xffffffffu, next_unit(it, lin))) break;
      __syncwarp();
      if (lane == 0) release_entry(it);
      if (lin >= total) break;
      Unit u = decode(lin);
      const int n_cols = (u.kind <= kLossDz) ? (FWD ? p.V : (u.last ? p.last_cols : p.piece)) : p.H;
      for (int tile = 0; tile < u.tiles; ++tile, ++u.n) {
      const int n0 = u.n * kLossUnit + side * 128;                 // first column of this warp
      const int chunks = min(4, max(0, (n_cols - n0 + 31) / 32));
      const int row0 = u.m * kLossUnit + half * 128 + quarter * 32;  // first row of this warp
      const int row = row0 + lane;
      const bool empty = u.k_blocks == 0;
      // fetched while the tensor cores still work on the tile
      int col = -1; float top = 0.f, log2_sum = 0.f, target_z = 0.f, c_t = 0.f;
      bool dead = true;              // an ignored token (or no token): zeros whatever its logits are
      if (!NARROW && u.kind <= kLossDz) {
        if (row < p.T) {
          const long long y = p.targets[row];
          const long long rel = y - (FWD ? 0 : static_cast<long long>(u.piece) * p.piece) - n0;
          if (rel >= 0 && rel < 128 && y < p.V) col = static_cast<int>(rel);
          if (!FWD && y != p.ignore_index) {
            dead = false;
            c_t = p.row_scale != nullptr ? p.row_scale[row] : 1.f;
            top = p.top[row]; log2_sum = p.top[p.T + row]; target_z = p.top[2 * static_cast<size_t>(p.T) + row];
          }
        }
      }
      auto accumulated = [&] {
        if (!__all_sync(0xffffffffu, mbar_wait(&tmem_full[acc], acc_phase, budget, p.status))) {
          if (lane == 0) report_failure(p.status, kStatusTimeoutPipeline, kKernelLoss, 2, p.rank, lin, acc, 0);
          return false;
        }
        tc_fence_after_sync();
        return true;
      };
      if (!FWD && !empty && !(ok = accumulated())) break;
      const bool tokens = NARROW && (FWD || u.kind != kLossDw);      // columns are tokens
      const uint32_t lanes = tmem_base + (tokens ? first32 * 32 : side * 128) + (static_cast<uint32_t>(quarter * 32) << 16);
      const int v_first = u.n * kLossUnit + half * 128 + quarter * 32;   // (tokens) first row of this warp: in the vocabulary's piece, or of H
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
      if (FWD && NARROW) {
        float z[kNarrowTiles * 32];
#pragma unroll
        for (int i = 0; i < kNarrowTiles * 32; ++i) z[i] = 0.f;
        for (int first = 0; first < u.k_blocks; first += kSegmentBlocks) {
          if (!(ok = accumulated())) break;
          if (count32 == 0) give_back();
#pragma unroll
          for (int c = 0; c < 2 * kNarrowTiles; ++c) {
            if (c < 2 * count32) {
              uint32_t part[16];
              tmem_ld_32x16(lanes + acc * kLossUnit + c * 16, part); tmem_ld_wait();
              if (c == 2 * count32 - 1) give_back();
#pragma unroll
              for (int i = 0; i < 16; ++i) z[c * 16 + i] += __uint_as_float(part[i]);
            }
          }
          acc ^= 1; if (acc == 0) acc_phase ^= 1;
        }
        if (!ok) break;
        if (v_first >= p.V) continue;
        const float ninf = __int_as_float(0xff800000);
        const bool exists = v_first + lane < p.V;
#pragma unroll
        for (int c = 0; c < kNarrowTiles; ++c) {
          if (c < count32) {
            const int t = u.m * p.tile_tokens + (first32 + c) * 32 + lane;
            const long long y = t < p.T ? p.targets[t] : -1;
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 32; ++i) turn_write(turn, lane, i, exists ? z[c * 32 + i] : ninf);
            __syncwarp();
            float2& so_far = stats[(u.m * kNarrowTiles + c) * 32];
            const float2 before = so_far;
            float v[32], most[4] = {before.x, ninf, ninf, ninf}, s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < 32; ++j) { v[j] = turn_read(turn, lane, j); most[j & 3] = fmaxf(most[j & 3], v[j]); }
            const float m = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
            const float ref = m == ninf ? 0.f : m;         // (a row of -inf: subtract 0, every term is exp(-inf) = 0)
#pragma unroll
            for (int j = 0; j < 32; ++j) s[j & 3] += ex2((v[j] - ref) * kLog2e);
            so_far = make_float2(m, before.y * ex2((before.x - ref) * kLog2e) + ((s[0] + s[1]) + (s[2] + s[3])));
            if (t < p.T) {
              if (y >= v_first && y < v_first + 32 && y < p.V) p.target_logit[t] = turn_read(turn, lane, static_cast<int>(y) - v_first);
            }
          }
        }
      } else if (NARROW && u.kind == kLossDz) {
        if (count32 == 0) give_back();
        if (lane == 0) bulk_wait_read();       // (stores of a dw unit before still read both tiles)
        __syncwarp();
#pragma unroll 1
        for (int c = 0; c < count32; ++c) {
          const int t_first = u.m * p.tile_tokens + (first32 + c) * 32, t = t_first + lane;
          float top = 0.f, log2_sum = 0.f, target_z = 0.f, c_t = 0.f;
          int target = -1;               // among this warp's rows
          bool dead = true;
          if (t < p.T) {
            const long long y = p.targets[t];
            if (y != p.ignore_index) {
              dead = false;
              c_t = p.row_scale != nullptr ? p.row_scale[t] : 1.f;
              top = p.top[t]; log2_sum = p.top[p.T + t]; target_z = p.top[2 * static_cast<size_t>(p.T) + t];
              const long long rel = y - static_cast<long long>(u.piece) * p.piece - v_first;
              if (rel >= 0 && rel < 32) target = static_cast<int>(rel);
            }
          }
          fetch(c);
          if (c == count32 - 1) give_back();
          if (v_first >= (n_cols + 63) / 64 * 64 || t_first >= p.T) continue;     // (the last panel is filled up with zeros)
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 32; ++i) turn_write(turn, lane, i, __uint_as_float(r[i]));
          // the stores before must have read where this piece will stand (split2: both halves, else the one before the last)
          if (lane == 0) { if (p.split2) bulk_wait_read(); else bulk_wait_read_but_one(); }
          __syncwarp();
          unsigned char* const lead_tile = narrow_out + (p.split2 ? 0 : flip * 2048);
          flip ^= 1;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t o[4], rest[4];
#pragma unroll
            for (int h = 0; h < 4; ++h) {
              const int j = q * 8 + h * 2;
              float a = ex2(fmaf(turn_read(turn, lane, j) - top, kLog2e, -log2_sum)) * c_t, b = ex2(fmaf(turn_read(turn, lane, j + 1) - top, kLog2e, -log2_sum)) * c_t;
              if (dead || v_first + j >= n_cols) a = 0.f;
              if (dead || v_first + j + 1 >= n_cols) b = 0.f;
              o[h] = pack_bf16x2(a, b);
              const float2 lead = unpack_bf16x2(o[h]);
              rest[h] = pack_bf16x2(a - lead.x, b - lead.y);
            }
            st_shared_v4(smem_u32(lead_tile) + stage_off<64>(lane, q), o[0], o[1], o[2], o[3]);
            if (p.split2) st_shared_v4(smem_u32(lead_tile) + 2048 + stage_off<64>(lane, q), rest[0], rest[1], rest[2], rest[3]);
          }
          if (target >= 0) {                 // (a lane writes over what it wrote itself)
            const float d = target_gradient(target_z, top, log2_sum) * c_t;
            const uint32_t at = smem_u32(lead_tile) + stage_off<64>(lane, target / 8) + (target & 7) * 2, lead = pack_bf16x2(d, 0.f);
            st_shared_b16(at, lead);
            if (p.split2) st_shared_b16(at + 2048, pack_bf16x2(d - unpack_bf16x2(lead).x, 0.f));
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_3d(&maps.z_out, lead_tile, v_first % 64, t_first, panel_of(p, u.piece, 0) + v_first / 64);
            if (p.split2) tma_store_3d(&maps.z_out, lead_tile + 2048, v_first % 64, t_first, panel_of(p, u.piece, 1) + v_first / 64);
            bulk_commit();
          }
        }
        __syncwarp();
        if (lane == 0) {
          bulk_wait_all();
          fence_proxy_async();
          red_release_gpu_add(p.done + u.piece, 1);
          red_release_gpu_add(p.done + 3 * p.pieces + u.piece * (p.piece / kLossUnit) + u.n, 1);
        }
      } else if (NARROW && u.kind == kLossDx) {
        if (count32 == 0 && !empty) give_back();
        const int h = v_first + lane;
#pragma unroll 1
        for (int c = 0; c < count32; ++c) {
          fetch(c);
          if (p.split2 && !empty) {          // the products of the remainders
            uint32_t r2[32];
            tmem_ld_32x32(taddr + p.tile_tokens + c * 32, r2); tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) + __uint_as_float(r2[i]));
          }
          if (c == count32 - 1 && !empty) give_back();
          const int t_first = u.m * p.tile_tokens + (first32 + c) * 32;
          float* out = p.dx_parts + (static_cast<size_t>(u.split) * p.T + t_first) * p.H + h;
          if (h < p.H) {                     // 32 lanes write 128 contiguous bytes of each token (64 of the finished bf16)
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              if (t_first + i < p.T) {
                if (p.dx_direct) static_cast<__nv_bfloat16*>(p.dx)[static_cast<size_t>(t_first + i) * p.H + h] = __float2bfloat16_rn(scale * __uint_as_float(r[i]));
                else if (u.piece == 0) out[static_cast<size_t>(i) * p.H] = __uint_as_float(r[i]);
                else red_add_f32(out + static_cast<size_t>(i) * p.H, __uint_as_float(r[i]));
              }
            }
          }
        }
        __syncwarp();
        if (lane == 0 && p.pieces > 1) red_release_gpu_add(p.done + p.pieces + u.piece, 1);
      } else if (FWD) {
        Pair z[64];
        for (int first = 0; first < u.k_blocks; first += kSegmentBlocks) {
          if (!(ok = accumulated())) break;
          if (row0 < p.T) {
#pragma unroll
            for (int c = 0; c < 8; ++c) {       // (16 columns at a time: 32 spill)
              uint32_t part[16];
              tmem_ld_32x16(lanes + acc * kLossUnit + c * 16, part); tmem_ld_wait();
              if (c == 7) give_back();
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const Pair add = pair_of(__uint_as_float(part[2 * i]), __uint_as_float(part[2 * i + 1]));
                z[c * 8 + i] = first == 0 ? add : z[c * 8 + i] + add;
              }
            }
          } else {
            give_back();
          }
          acc ^= 1; if (acc == 0) acc_phase ^= 1;
        }
        if (!ok) break;
        const int left = n_cols - n0;        // (columns that were not multiplied hold anything)
        if (left <= 0 || row0 >= p.T) continue;
        const float ninf = __int_as_float(0xff800000);
        if (left < 128) {
#pragma unroll
          for (int i = 0; i < 64; ++i) {
            float a, b;
            parts_of(z[i], a, b);
            z[i] = pair_of(2 * i < left ? a : ninf, 2 * i + 1 < left ? b : ninf);
          }
        }
        if (__any_sync(0xffffffffu, col >= 0)) {
          float zt = 0.f;
#pragma unroll
          for (int i = 0; i < 64; ++i) {
            float a, b;
            parts_of(z[i], a, b);
            if (col == 2 * i) zt = a;
            if (col == 2 * i + 1) zt = b;
          }
          if (col >= 0) p.target_logit[row] = zt;
        }
        float most[4] = {ninf, ninf, ninf, ninf};
#pragma unroll
        for (int i = 0; i < 64; ++i) {
          float a, b;
          parts_of(z[i], a, b);
          most[i & 3] = fmaxf(most[i & 3], fmaxf(a, b));
        }
        const float m = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
        // (a row of -inf: subtract 0, every term is exp(-inf) = 0)
        const float ref = m == ninf ? 0.f : m;
        const Pair minus = pair_of(-ref, -ref), log2e = pair_of(kLog2e, kLog2e);
        Pair s[2] = {pair_of(0.f, 0.f), pair_of(0.f, 0.f)};
#pragma unroll
        for (int i = 0; i < 64; ++i) s[i & 1] = s[i & 1] + ex2((z[i] + minus) * log2e);
        float s0, s1;
        parts_of(s[0] + s[1], s0, s1);
        if (row < p.T) p.parts[static_cast<size_t>(u.n * 2 + side) * p.T + row] = make_float2(m, s0 + s1);
      } else if (u.kind == kLossDz) {
        const int z_chunks = (chunks + 1) / 2 * 2;       // (the last panel is filled up with zeros)
        const Pair minus_top = pair_of(-top, -top), minus_sum = pair_of(-log2_sum, -log2_sum), log2e = pair_of(kLog2e, kLog2e), scale_t = pair_of(c_t, c_t);
        const uint32_t target_dz = pack_bf16x2(target_gradient(target_z, top, log2_sum) * c_t, 0.f);
        const bool rows = row0 < p.T;
        if (!rows) give_back();
#pragma unroll 1
        for (int c = 0; c < z_chunks && rows; ++c) {
          fetch(c);
          if (c == z_chunks - 1) give_back();
          const int left = n_cols - n0 - c * 32;
          const bool target_here = __any_sync(0xffffffffu, (col >> 5) == c);
          if ((c & 1) == 0) stg = next_tile();
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t o[4];
#pragma unroll
            for (int h = 0; h < 4; ++h) {
              const int i = q * 8 + h * 2;
              float a, b;
              parts_of(ex2(fma2(pair_of(__uint_as_float(r[i]), __uint_as_float(r[i + 1])) + minus_top, log2e, minus_sum)) * scale_t, a, b);
              o[h] = dead ? 0u : pack_bf16x2(a, b);
              if (left < 32) {                 // (uniform: the piece ends here)
                if (i >= left) o[h] = 0u;
                else if (i + 1 >= left) o[h] &= 0xffffu;
              }
            }
            st_shared_v4(stg + stage_off<128>(lane, (c & 1) * 4 + q), o[0], o[1], o[2], o[3]);
          }
          if (target_here) {                 // (a lane writes over what it wrote itself)
            if ((col >> 5) == c) st_shared_b16(stg + stage_off<128>(lane, (c & 1) * 4 + (col & 31) / 8) + (col & 7) * 2, target_dz);
          }
          if ((c & 1) == 1) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) { tma_store_3d(&maps.z_out, stage_tile, 0, row0, panel_of(p, u.piece, 0) + (n0 + c * 32) / 64); bulk_commit(); }
          }
        }
        if (chunks == 0 && rows) give_back();
        __syncwarp();
        if (lane == 0) {
          bulk_wait_all();
          fence_proxy_async();
          red_release_gpu_add(p.done + u.piece, 1);
          red_release_gpu_add(p.done + 3 * p.pieces + u.piece * (p.piece / kLossUnit) + u.n, 1);
        }
      } else if (u.kind == kLossDx && !p.dx_direct) {
        const bool rows = row0 < p.T;
        if (!rows && !empty) give_back();
#pragma unroll 1
        for (int c = 0; c < chunks && rows; ++c) {
          fetch(c);
          if (c == chunks - 1 && !empty) give_back();
          stg = next_tile();
#pragma unroll
          for (int q = 0; q < 8; ++q) st_shared_v4(stg + stage_off<128>(lane, q), r[q * 4], r[q * 4 + 1], r[q * 4 + 2], r[q * 4 + 3]);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (u.piece == 0) tma_store_3d(&maps.dx, stage_tile, n0 + c * 32, row0, u.split);
            else tma_reduce_add_3d(&maps.dx, stage_tile, n0 + c * 32, row0, u.split);
            bulk_commit();
          }
        }
        if (chunks == 0 && rows && !empty) give_back();
        __syncwarp();
        if (lane == 0 && p.pieces > 1) { bulk_wait_all(); red_release_gpu_add(p.done + p.pieces + u.piece, 1); }
      } else {
        // finished rows of dW, or (the only unit of its place, a single piece) of dx
        const bool is_dw = u.kind == kLossDw;
        const int y = is_dw ? u.piece * p.piece + row0 : row0, y_end = is_dw ? p.V : p.T;
        const bool report = is_dw && p.pieces > 1 && tile == u.tiles - 1;      // the operands have been read
#pragma unroll 1
        for (int c = 0; c < chunks; c += 2) {
          uint32_t r2[32];             // two chunks on their way at once (columns past the last were not multiplied and are not stored)
          tmem_ld_32x32(taddr + c * 32, r);
          tmem_ld_32x32(taddr + c * 32 + 32, r2);
          tmem_ld_wait();
          if (c + 2 >= chunks) {
            give_back();
            if (lane == 0 && report) red_release_gpu_add(p.done + 2 * p.pieces + u.piece, 1);
          }
          if (y >= y_end) continue;
          stg = next_tile();
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            uint32_t o[4];
#pragma unroll
            for (int h = 0; h < 4; ++h) {
              const int i = (q & 3) * 8 + h * 2;
              o[h] = pack_bf16x2(scale * __uint_as_float(q < 4 ? r[i] : r2[i]), scale * __uint_as_float(q < 4 ? r[i + 1] : r2[i + 1]));
            }
            st_shared_v4(stg + stage_off<128>(lane, q), o[0], o[1], o[2], o[3]);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) { tma_store_3d(is_dw ? &maps.dw : &maps.dx, stage_tile, n0 + c * 32, y, 0); bulk_commit(); }
        }
        if (chunks == 0) {
          give_back();
          if (lane == 0 && report) red_release_gpu_add(p.done + 2 * p.pieces + u.piece, 1);
        }
      }
      if (!FWD && !empty) { acc ^= 1; if (acc == 0) acc_phase ^= 1; }
      }
    }
    if (FWD && NARROW) {
      for (int m = 0; m < p.row_units; ++m)
        for (int c = 0; c < count32; ++c) {
          const int t = m * p.tile_tokens + (first32 + c) * 32 + lane;
          if (t < p.T) p.parts[static_cast<size_t>(blockIdx.x * 4 + quarter) * p.T + t] = stats[(m * kNarrowTiles + c) * 32];
        }
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

template <bool FWD, bool NARROW>
cudaError_t launch_pairs(const LossParams& p, const LossMaps& m, long long units, int sms, cudaStream_t stream) {
  auto kernel = linear_loss_kernel<FWD, NARROW>;
  static std::atomic<bool> configured[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[dev].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes(FWD, NARROW));
    if (e != cudaSuccess) return e;
    configured[dev].store(true, std::memory_order_release);
  }
  const long long pairs = units < sms / 2 ? units : sms / 2;
  kernel<<<static_cast<unsigned>(pairs * 2), kThreads, smem_bytes(FWD, NARROW), stream>>>(p, m);
  return cudaGetLastError();
}

// ---------------------------------------------------------------------------------------------
// Joins the parts of each row, and the rows' losses.  A block takes 8 rows (64 contiguous bytes of every part) and 64 threads for
// each: with 32 rows and 16 threads a call of one token waited for 49 loads in a row (V 100003: 16.6 us).
// ---------------------------------------------------------------------------------------------
constexpr int kFinalRows = 8, kFinalThreads = 512, kFinalLanes = kFinalThreads / kFinalRows;

__global__ void __launch_bounds__(kFinalThreads) loss_final_kernel(const LossFinalParams p) {
  __shared__ float2 joined[kFinalLanes][kFinalRows];
  __shared__ double sums[kFinalThreads / 32];
  __shared__ int counts[kFinalThreads / 32];
  __shared__ bool last;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int r = threadIdx.x % kFinalRows, part = threadIdx.x / kFinalRows;
  const long long row = static_cast<long long>(blockIdx.x) * kFinalRows + r;
  const float ninf = __int_as_float(0xff800000);
  auto join = [&](float2 a, float2 b) {
    const float m = fmaxf(a.x, b.x);
    const float ref = m == ninf ? 0.f : m;
    return make_float2(m, a.y * ex2((a.x - ref) * kLog2e) + b.y * ex2((b.x - ref) * kLog2e));
  };
  grid_wait();
  float2 v = make_float2(ninf, 0.f);
  if (row < p.T) {
    const float2* q = p.parts + row;
    int i = part;
    for (; i + 3 * kFinalLanes < p.num_parts; i += 4 * kFinalLanes) {
      float2 u[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) u[j] = q[static_cast<size_t>(i + j * kFinalLanes) * p.T];
      v = join(v, join(join(u[0], u[1]), join(u[2], u[3])));
    }
    for (; i < p.num_parts; i += kFinalLanes) v = join(v, q[static_cast<size_t>(i) * p.T]);
  }
  joined[part][r] = v;
  __syncthreads();
  if (warp == 0) {
    // four lanes for each row
    v = joined[part][r];
    for (int w = part + 4; w < kFinalLanes; w += 4) v = join(v, joined[w][r]);
    for (int d = 8; d < 32; d *= 2) v = join(v, make_float2(__shfl_xor_sync(0xffffffffu, v.x, d), __shfl_xor_sync(0xffffffffu, v.y, d)));
    if (lane < kFinalRows && row < p.T) {
      // The maximum and the logarithm of the sum stay apart: next to a maximum of the type's lowest value, or a loss near zero, their sum
      // would have lost the logarithm.
      const long long y = p.targets[row];
      float loss = 0.f;
      if (y != p.ignore_index) {
        if (y < 0 || y >= p.V) {       // the loss and every gradient become NaN, and the caller can ask why
          report_note(p.status, kStatusBadTarget, kKernelLoss, 0, p.rank, static_cast<int>(row), p.V, static_cast<int>(y));
          v.x = loss = __int_as_float(0x7fc00000);
        } else {
          loss = (v.x - p.target_logit[row]) + logf(v.y);
        }
      }
      p.top[row] = v.x;
      p.top[p.T + row] = log2f(v.y);
      p.top[2 * static_cast<size_t>(p.T) + row] = p.target_logit[row];
      p.each[row] = loss;
    }
  }
  if (!p.mean && !p.sum) return;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(p.ticket, 1) == static_cast<int>(gridDim.x) - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  double sum = 0.0; int count = 0;
  for (int t = threadIdx.x; t < p.T; t += kFinalThreads) {
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
    for (int w = 1; w < kFinalThreads / 32; ++w) { sum += sums[w]; count += counts[w]; }
    // without a counted token the mean is 0 / 0, and its gradients are zeros
    *p.loss = static_cast<float>(p.mean ? sum / static_cast<double>(count) : sum);
    if (p.mean) *p.inv_count = count > 0 ? static_cast<float>(1.0 / count) : 0.f;
  }
}

// dx = scale * sum of its slots, rounded once.  Calls of few elements and many slots share the slots of four elements among several
// threads (16 tokens, hidden 2048, 60 slots: one thread after another waited for 60 loads in a row, 40 us).
constexpr int kDxThreads = 256;

__global__ void __launch_bounds__(kDxThreads) loss_dx_kernel(const LossDxParams p) {
  __shared__ float4 shared[kDxThreads];
  const size_t n = static_cast<size_t>(p.T) * p.H / 4;            // vectors (H is a multiple of 8)
  const int per_block = kDxThreads / p.lanes, lane = threadIdx.x / per_block, v = threadIdx.x % per_block;
  grid_wait();
  float scale = p.scale != nullptr ? *p.scale : 1.f;
  if (p.scale2 != nullptr) scale *= *p.scale2;
  auto add = [](float4 a, float4 b) { return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w); };
  for (size_t first = static_cast<size_t>(blockIdx.x) * per_block; first < n; first += static_cast<size_t>(gridDim.x) * per_block) {
    const size_t i = first + v;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    if (i < n) {
      const float4* q = reinterpret_cast<const float4*>(p.parts) + i;
      int s = lane;
      for (; s + 3 * p.lanes < p.slots; s += 4 * p.lanes) {
        float4 u[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) u[j] = __ldcs(q + (s + j * p.lanes) * n);
        a = add(a, add(add(u[0], u[1]), add(u[2], u[3])));
      }
      for (; s < p.slots; s += p.lanes) a = add(a, __ldcs(q + s * n));
    }
    if (p.lanes > 1) {
      shared[threadIdx.x] = a;
      __syncthreads();
      if (lane == 0)
        for (int l = 1; l < p.lanes; ++l) a = add(a, shared[l * per_block + v]);
      __syncthreads();
    }
    if (lane == 0 && i < n)
      *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.dx) + i * 4) = make_uint2(pack_bf16x2(scale * a.x, scale * a.y), pack_bf16x2(scale * a.z, scale * a.w));
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

void loss_narrow_ring(LossParams& p, bool backward) {
  const int tokens = backward && p.split2 ? p.tile_tokens : p.tile_tokens / 2;      // that a CTA loads
  p.stage_bytes = kOperandBytes + (tokens * 128 + 1023) / 1024 * 1024;              // (operands stand on 1024-byte boundaries)
  if (backward) p.stage_bytes = greater(p.stage_bytes, 4 * p.dw_rows * 128);
  p.stages = lesser(kNarrowStages, kNarrowRing / p.stage_bytes);
}
static long long forward_units(const LossParams& p) { return static_cast<long long>(p.row_units) * ((p.V + kLossUnit - 1) / kLossUnit); }
long long loss_forward_parts(const LossParams& p, int sms) {
  if (!p.narrow) return (static_cast<long long>(p.V) + kLossPart - 1) / kLossPart;
  const long long units = forward_units(p);
  return (units < sms / 2 ? units : sms / 2) * 2 * 4;           // one for each warp quarter of every CTA
}
cudaError_t launch_loss_forward(const LossParams& p, const LossMaps& m, int sms, cudaStream_t stream) {
  const long long units = forward_units(p);
  return p.narrow ? launch_pairs<true, true>(p, m, units, sms, stream) : launch_pairs<true, false>(p, m, units, sms, stream);
}
cudaError_t launch_loss_backward(const LossParams& p, const LossMaps& m, int sms, cudaStream_t stream) {
  return p.narrow ? launch_pairs<false, true>(p, m, loss_backward_units(p), sms, stream) : launch_pairs<false, false>(p, m, loss_backward_units(p), sms, stream);
}
// Both follow the kernel whose results they read, and may be launched while it drains.
template <class Params>
static cudaError_t launch_after(void (*kernel)(const Params), const Params& p, long long blocks, int threads, cudaStream_t stream) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr; cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}
cudaError_t launch_loss_final(const LossFinalParams& p, cudaStream_t stream) {
  return launch_after(loss_final_kernel, p, (p.T + kFinalRows - 1) / kFinalRows, kFinalThreads, stream);
}
cudaError_t launch_loss_dx(const LossDxParams& p_in, cudaStream_t stream) {
  LossDxParams p = p_in;
  const long long vectors = static_cast<long long>(p.T) * p.H / 4;
  p.lanes = 1;
  while (p.lanes < 16 && p.lanes * 4 <= p.slots && vectors * p.lanes < 148 * 1024) p.lanes *= 2;
  const long long per_block = kDxThreads / p.lanes, blocks = (vectors + per_block - 1) / per_block;
  return launch_after(loss_dx_kernel, p, blocks < 148 * 8 ? blocks : 148 * 8, kDxThreads, stream);
}

}  // namespace sep

// Gated linear recurrence along sequences, and its gradients.
//
//   keep_t = sigmoid(gate_t), take_t = 1 - keep_t:   h_t = keep_t h_{t-1} + take_t x_t
//   g_t = dh_t + keep_{t+1} g_{t+1}:   dx_t = take_t g_t,   dgate_t = g_t keep_t take_t (h_{t-1} - x_t),   dh_{-1} = keep_0 g_0
//
// The state, and everything that is added up along a sequence, is fp32.
#include "scan.h"
#include "ptx.cuh"

namespace sep {

namespace {

constexpr int kThreads = 128;                    // of the form for one more token
constexpr int kScanThreads = 256;
constexpr int kScanGroup = 32;                   // chunks between two states that are handed on

// What the blocks of a call hand on to one another.
struct ScanChain {
  int chunks, tiles;
  int* ticket;                   // null: one chunk, nothing is handed on
  int* flags;                    // [chunks + groups][tiles]: the run, the group's state is there
  float2* runs;                  // [chunks][channels]
  float* states;                 // [groups][channels] behind each group
};

template <class T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// sigmoid(gate) and sigmoid(-gate), each to its own last digits: the smaller one is computed and kept, with the sign of the gate; the other is
// its difference to 1.  For bf16 gates the exponent is rounded once (|gate| 2^-24 of the result), for fp32 ones it is not.
template <class T> __device__ __forceinline__ float smaller(float g);
template <> __device__ __forceinline__ float smaller<__nv_bfloat16>(float g) {
  float e, m;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fabsf(g) * 1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(m) : "f"(1.f + e));
  return copysignf(m, g);
}
template <> __device__ __forceinline__ float smaller<float>(float g) { return copysignf(__frcp_rn(1.f + expf(fabsf(g))), g); }
struct Gate { float keep, take; };
__device__ __forceinline__ Gate gate_of(float s) {
  const float m = fabsf(s), o = 1.f - m;
  return signbit(s) ? Gate{m, o} : Gate{o, m};
}

// What a run of rows does to the state in front of it: h -> a h + b, or h -> b where a sequence starts within (a is then -0, and stays negative
// in products: a state of the sequence before, infinite or NaN as it may be, is not multiplied with).
struct Run { float a, b; };
__device__ __forceinline__ float apply(Run r, float h) { return signbit(r.a) ? r.b : fmaf(r.a, h, r.b); }
__device__ __forceinline__ Run join(Run first, Run then) {
  return signbit(then.a) ? then : Run{then.a * first.a, fmaf(then.a, first.b, then.b)};
}
__device__ __forceinline__ Run nothing() { return {1.f, 0.f}; }

__device__ __forceinline__ long long offset_of(const ScanShape& p, int i) {
  return p.offsets_wide ? static_cast<const long long*>(p.offsets)[i] : static_cast<const int*>(p.offsets)[i];
}
// The sequence that row `t` belongs to, -1 for none.  Whatever the offsets are, it is one that exists.
__device__ __forceinline__ int sequence_of(const ScanShape& p, int t) {
  if (t < 0 || t >= p.rows) return -1;
  if (p.offsets == nullptr) return t / p.length;
  int lo = -1, hi = p.sequences + 1;             // offsets[lo] <= t < offsets[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (offset_of(p, mid) <= t) lo = mid; else hi = mid;
  }
  return lo < p.sequences ? lo : -1;
}
__device__ __forceinline__ long long first_row(const ScanShape& p, int s) { return p.offsets == nullptr ? static_cast<long long>(s) * p.length : offset_of(p, s); }

template <class T, int VEC> struct Raw;
template <> struct Raw<__nv_bfloat16, 8> {
  uint4 v;
  __device__ __forceinline__ void load(const void* base, long long at) { v = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(base) + at); }
  __device__ __forceinline__ void clear() { v = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ float get(int i) const {
    const uint32_t u = i < 2 ? v.x : i < 4 ? v.y : i < 6 ? v.z : v.w;
    return __uint_as_float(i & 1 ? u & 0xffff0000u : u << 16);
  }
};
template <> struct Raw<float, 4> {
  float4 v;
  __device__ __forceinline__ void load(const void* base, long long at) { v = *reinterpret_cast<const float4*>(static_cast<const float*>(base) + at); }
  __device__ __forceinline__ void clear() { v = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ float get(int i) const { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
};
template <class T> struct Raw<T, 1> {
  T v;
  __device__ __forceinline__ void load(const void* base, long long at) { v = static_cast<const T*>(base)[at]; }
  __device__ __forceinline__ void clear() { v = from_float<T>(0.f); }
  __device__ __forceinline__ float get(int) const { return to_float(v); }
};
template <class T, int VEC>
__device__ __forceinline__ void store_row(void* base, long long at, const float (&f)[VEC]) {
  if constexpr (VEC == 8) {
    *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(base) + at) =
        make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  } else if constexpr (VEC == 4) {
    *reinterpret_cast<float4*>(static_cast<float*>(base) + at) = make_float4(f[0], f[1], f[2], f[3]);
  } else {
    static_cast<T*>(base)[at] = from_float<T>(f[0]);
  }
}
template <int VEC>
__device__ __forceinline__ void load_state(const float* base, long long at, float (&f)[VEC]) {
  if (base == nullptr) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = 0.f;
  } else if constexpr (VEC >= 4) {
#pragma unroll
    for (int i = 0; i < VEC; i += 4) {
      const float4 v = *reinterpret_cast<const float4*>(base + at + i);
      f[i] = v.x; f[i + 1] = v.y; f[i + 2] = v.z; f[i + 3] = v.w;
    }
  } else {
    f[0] = base[at];
  }
}
template <int VEC>
__device__ __forceinline__ void store_state(float* base, long long at, const float (&f)[VEC]) {
  if constexpr (VEC >= 4) {
#pragma unroll
    for (int i = 0; i < VEC; i += 4) *reinterpret_cast<float4*>(base + at + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
  } else {
    base[at] = f[0];
  }
}

// A unit of work: a chunk of rows and a tile of channels.  A thread holds R rows of VEC channels in registers, LANES threads lie side by side
// across the channels, and the others above one another along time.
template <class T, int V> struct Tile {
  static constexpr int VEC = V;
  static constexpr int LANES = V > 1 ? 8 : 32;
  static constexpr int R = V == 8 ? 4 : V == 4 ? 8 : 16;
  static constexpr int PILES = kScanThreads / LANES;           // of R rows
  static constexpr int ROWS = PILES * R;
  static constexpr int COLS = LANES * V;
  static constexpr int PARTS = kScanThreads / COLS;            // threads that share the joining of one channel
};

// Chunks are dealt out in the order in which they depend on one another, by a ticket: a chunk waits only for chunks that were dealt out before it
// and are running or done, however many blocks are resident.  `order` counts chunks from where the recurrence starts (the first row, or the last
// one for the backward).  Each leaves what it does to the state (Run) as soon as it knows it; the state in front of a chunk is that of its group of
// 32 chunks, and the runs of the chunks between, joined in one order: no rounding depends on who was first.  Only the
// groups' states follow one another.
template <class Tl>
struct Chain {
  const ScanChain& c;
  const ScanShape& p;
  int order, tile, col0;

  __device__ __forceinline__ float2* runs_at(int k) const { return c.runs + static_cast<long long>(k) * p.channels + col0; }
  __device__ __forceinline__ float* state_at(int g) const { return c.states + static_cast<long long>(g) * p.channels + col0; }
  __device__ __forceinline__ int* flag_at(int k) const { return c.flags + static_cast<long long>(k) * c.tiles + tile; }
  __device__ __forceinline__ int* group_flag_at(int g) const { return c.flags + static_cast<long long>(c.chunks + g) * c.tiles + tile; }

  // Thread i < COLS has the chunk's run for its channel; all threads call.
  __device__ __forceinline__ void publish(Run run) const {
    if (threadIdx.x < Tl::COLS && col0 + static_cast<int>(threadIdx.x) < p.channels) __stcg(runs_at(order) + threadIdx.x, make_float2(run.a, run.b));
    __syncthreads();
    if (threadIdx.x == 0) { __threadfence(); red_release_gpu_add(flag_at(order), 1); }
  }
  __device__ __forceinline__ void publish_state(float state) const {
    if (threadIdx.x < Tl::COLS && col0 + static_cast<int>(threadIdx.x) < p.channels) __stcg(state_at(order / kScanGroup) + threadIdx.x, state);
    __syncthreads();
    if (threadIdx.x == 0) { __threadfence(); red_release_gpu_add(group_flag_at(order / kScanGroup), 1); }
  }
  // The state in front of this chunk for threads i < COLS, of a sequence that starts in chunk `from` (in this order).  All threads call; `scratch`
  // holds PARTS x COLS runs.
  __device__ __forceinline__ float state_before(int from, Run* scratch) const {
    const int group = order / kScanGroup, group_start = group * kScanGroup;
    const bool whole = from < group_start;
    const int begin = whole ? group_start : from, n = order - begin;
    bool ok = true;
    if (threadIdx.x < 64) {
      const int i = threadIdx.x;
      int* flag = i < n ? flag_at(begin + i) : i == 63 && whole ? group_flag_at(group - 1) : nullptr;
      if (flag != nullptr) {
        ok = spin_until([&] { return ld_acquire_gpu(flag) != 0; }, p.wait_budget_ns, p.status);
        if (!ok) report_failure(p.status, kStatusTimeoutPipeline, kKernelScan, 0, p.rank, order, begin + i, tile);
      }
    }
    ok = __syncthreads_and(ok) != 0;
    const int ch = threadIdx.x % Tl::COLS, part = threadIdx.x / Tl::COLS;
    const bool mine = col0 + ch < p.channels;
    float state = 0.f;
    if (whole && mine && part == 0) state = __ldcg(state_at(group - 1) + ch);
    Run run = nothing();
    if (mine) {
      const int last = begin + n * (part + 1) / Tl::PARTS;
#pragma unroll 4
      for (int k = begin + n * part / Tl::PARTS; k < last; ++k) {
        const float2 v = __ldcg(runs_at(k) + ch);
        run = join(run, Run{v.x, v.y});
      }
    }
    scratch[threadIdx.x] = run;
    __syncthreads();
    if (part == 0) {
#pragma unroll
      for (int i = 0; i < Tl::PARTS; ++i) state = apply(scratch[i * Tl::COLS + ch], state);
    }
    return ok ? state : __int_as_float(0x7fc00000);
  }
};

// Which chunk this block takes; the same for all of its threads.
__device__ __forceinline__ int claim_unit(const ScanChain& c, int* slot) {
  if (c.ticket == nullptr) return blockIdx.x;
  if (threadIdx.x == 0) *slot = atomicAdd(c.ticket, 1);
  __syncthreads();
  return *slot;
}

// Runs of the threads of a block that lie above one another, `mine` in the order of threads: what all threads before this one do, and
// for threads i < COLS what the whole block does to channel i.
template <class Tl>
__device__ __forceinline__ void block_runs(Run (&mine)[Tl::VEC], Run (&before)[Tl::VEC], Run& whole, Run (*scratch)[Tl::COLS]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, side = threadIdx.x % Tl::LANES;
  // within the warp
#pragma unroll
  for (int d = Tl::LANES; d < 32; d *= 2) {
#pragma unroll
    for (int i = 0; i < Tl::VEC; ++i) {
      const Run prev = {__shfl_up_sync(0xffffffffu, mine[i].a, d), __shfl_up_sync(0xffffffffu, mine[i].b, d)};
      if (lane >= d) mine[i] = join(prev, mine[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < Tl::VEC; ++i) {
    if (lane >= 32 - Tl::LANES) scratch[warp][side * Tl::VEC + i] = mine[i];
    if constexpr (Tl::LANES < 32) {
      const Run prev = {__shfl_up_sync(0xffffffffu, mine[i].a, Tl::LANES), __shfl_up_sync(0xffffffffu, mine[i].b, Tl::LANES)};
      before[i] = lane >= Tl::LANES ? prev : nothing();
    } else {
      before[i] = nothing();
    }
  }
  __syncthreads();
  whole = nothing();
  if (threadIdx.x < Tl::COLS) {
#pragma unroll
    for (int w = 0; w < kScanThreads / 32; ++w) {
      const Run r = scratch[w][threadIdx.x];
      scratch[w][threadIdx.x] = whole;
      whole = join(whole, r);
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < Tl::VEC; ++i) before[i] = join(scratch[warp][side * Tl::VEC + i], before[i]);
}

// Sequences without rows hand their state on (`from` to `to`); offsets that are none are reported.  A block looks at its share of the sequences.
template <class Tl>
__device__ __forceinline__ void empty_sequences(const ScanShape& p, const ScanChain& c, int chunk, int tile, const float* from, float* to, bool report) {
  if (p.offsets == nullptr && p.length > 0) return;
  const int begin = static_cast<int>(static_cast<long long>(p.sequences) * chunk / c.chunks), end = static_cast<int>(static_cast<long long>(p.sequences) * (chunk + 1) / c.chunks);
  for (int s = begin + threadIdx.x; s < end; s += kScanThreads) {
    const long long a = first_row(p, s), b = first_row(p, s + 1);
    if (a < 0 || b < a || b > p.rows) {
      if (report && tile == 0)
        report_note(p.status, kStatusBadOffsets, kKernelScan, 0, p.rank, s, static_cast<int>(min(max(a, -1ll << 31), (1ll << 31) - 1)),
                    static_cast<int>(min(max(b, -1ll << 31), (1ll << 31) - 1)));
      continue;
    }
    if (a != b || to == nullptr) continue;
    for (int i = tile * Tl::COLS; i < min((tile + 1) * Tl::COLS, p.channels); ++i)
      to[static_cast<long long>(s) * p.channels + i] = from != nullptr ? from[static_cast<long long>(s) * p.channels + i] : 0.f;
  }
}

template <class T, int V>
__global__ void __launch_bounds__(kScanThreads, 2) scan_forward_kernel(const ScanParams p, const ScanChain c) {
  using Tl = Tile<T, V>;
  __shared__ int seq[Tl::ROWS + 2];              // of the rows from the one before the chunk to the one behind it
  __shared__ Run warps[kScanThreads / 32][Tl::COLS];
  __shared__ Run parts[kScanThreads];
  __shared__ float carry[Tl::COLS];
  __shared__ int slot;
  const int unit = claim_unit(c, &slot), chunk = unit / c.tiles, tile = unit - chunk * c.tiles;
  const int row0 = chunk * Tl::ROWS, col0 = tile * Tl::COLS;
  const int side = threadIdx.x % Tl::LANES, pile = threadIdx.x / Tl::LANES;
  const int col = col0 + side * V, first = row0 + pile * Tl::R;
  const bool in = col < p.channels;
  Raw<T, V> x[Tl::R], gate[Tl::R];
#pragma unroll
  for (int r = 0; r < Tl::R; ++r) {
    if (in && first + r < p.rows) {
      gate[r].load(p.gate, (first + r) * p.gate_stride + col);
      x[r].load(p.x, (first + r) * p.x_stride + col);
    } else {
      gate[r].clear(); x[r].clear();
    }
  }
  for (int i = threadIdx.x; i < Tl::ROWS + 2; i += kScanThreads) seq[i] = sequence_of(p, row0 - 1 + i);
  empty_sequences<Tl>(p, c, chunk, tile, p.initial, p.final_state, true);
  __syncthreads();

  float small[Tl::R][V];
  Run mine[V], before[V], whole;
#pragma unroll
  for (int i = 0; i < V; ++i) mine[i] = nothing();
#pragma unroll
  for (int r = 0; r < Tl::R; ++r) {
    const int at = pile * Tl::R + r + 1, s = seq[at];
    if (s != seq[at - 1] || s < 0) {
      float start[V];
      load_state<V>(s >= 0 && in ? p.initial : nullptr, static_cast<long long>(s) * p.channels + col, start);
#pragma unroll
      for (int i = 0; i < V; ++i) mine[i] = {-0.f, start[i]};
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      small[r][i] = smaller<T>(gate[r].get(i));
      if (s >= 0) {
        const Gate g = gate_of(small[r][i]);
        mine[i] = {mine[i].a * g.keep, fmaf(g.keep, mine[i].b, g.take * x[r].get(i))};
      }
    }
  }
  block_runs<Tl>(mine, before, whole, warps);

  const Chain<Tl> chain{c, p, chunk, tile, col0};
  if (c.ticket != nullptr) chain.publish(whole);
  const bool continues = seq[1] >= 0 && seq[1] == seq[0];
  float state = 0.f;
  if (continues) state = chain.state_before(static_cast<int>(max(first_row(p, seq[1]), 0ll) / Tl::ROWS), parts);
  if (threadIdx.x < Tl::COLS) carry[threadIdx.x] = state;
  if (c.ticket != nullptr && chunk % kScanGroup == kScanGroup - 1) chain.publish_state(apply(whole, state));
  __syncthreads();
  if (!in) return;

  float h[V];
#pragma unroll
  for (int i = 0; i < V; ++i) h[i] = apply(before[i], carry[side * V + i]);
#pragma unroll
  for (int r = 0; r < Tl::R; ++r) {
    if (first + r >= p.rows) break;
    const int at = pile * Tl::R + r + 1, s = seq[at];
    if (s != seq[at - 1] || s < 0) load_state<V>(s >= 0 ? p.initial : nullptr, static_cast<long long>(s) * p.channels + col, h);
    if (s >= 0) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const Gate g = gate_of(small[r][i]);
        h[i] = fmaf(g.keep, h[i], g.take * x[r].get(i));
      }
      if (p.final_state != nullptr && seq[at + 1] != s) store_state<V>(p.final_state, static_cast<long long>(s) * p.channels + col, h);
    }
    store_row<T, V>(p.h, static_cast<long long>(first + r) * p.channels + col, h);
  }
}

// As the forward, from the last row to the first: what runs along is keep_t g_t.
template <class T, int V>
__global__ void __launch_bounds__(kScanThreads, 2) scan_backward_kernel(const ScanGradParams p, const ScanChain c) {
  using Tl = Tile<T, V>;
  __shared__ int seq[Tl::ROWS + 2];
  __shared__ Run warps[kScanThreads / 32][Tl::COLS];
  __shared__ Run parts[kScanThreads];
  __shared__ float carry[Tl::COLS];
  __shared__ int slot;
  const int unit = claim_unit(c, &slot), order = unit / c.tiles, tile = unit - order * c.tiles;
  const int chunk = c.chunks - 1 - order, row0 = chunk * Tl::ROWS, col0 = tile * Tl::COLS;
  const int side = threadIdx.x % Tl::LANES, pile = Tl::PILES - 1 - static_cast<int>(threadIdx.x) / Tl::LANES;
  const int col = col0 + side * V, first = row0 + pile * Tl::R;
  const bool in = col < p.channels;
  Raw<T, V> x[Tl::R], gate[Tl::R], dh[Tl::R], before_row[Tl::R];
#pragma unroll
  for (int r = 0; r < Tl::R; ++r) {
    const int t = first + r;
    const bool there = in && t < p.rows;
    if (there) gate[r].load(p.gate, t * p.gate_stride + col); else gate[r].clear();
    if (there && p.dh != nullptr) dh[r].load(p.dh, t * p.dh_stride + col); else dh[r].clear();
    if (there && p.dgate != nullptr) x[r].load(p.x, t * p.x_stride + col); else x[r].clear();
    if (there && p.dgate != nullptr && t > 0) before_row[r].load(p.h, static_cast<long long>(t - 1) * p.channels + col); else before_row[r].clear();
  }
  for (int i = threadIdx.x; i < Tl::ROWS + 2; i += kScanThreads) seq[i] = sequence_of(p, row0 - 1 + i);
  empty_sequences<Tl>(p, c, order, tile, p.dfinal, p.dinitial, false);
  __syncthreads();

  float small[Tl::R][V];
  Run mine[V], before[V], whole;
#pragma unroll
  for (int i = 0; i < V; ++i) mine[i] = nothing();
#pragma unroll
  for (int r = Tl::R - 1; r >= 0; --r) {
    const int at = pile * Tl::R + r + 1, s = seq[at];
    if (s != seq[at + 1] || s < 0) {
      float end[V];
      load_state<V>(s >= 0 && in ? p.dfinal : nullptr, static_cast<long long>(s) * p.channels + col, end);
#pragma unroll
      for (int i = 0; i < V; ++i) mine[i] = {-0.f, end[i]};
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      small[r][i] = smaller<T>(gate[r].get(i));
      if (s >= 0) {
        const float keep = gate_of(small[r][i]).keep;
        mine[i] = {mine[i].a * keep, __fmul_rn(keep, __fadd_rn(mine[i].b, dh[r].get(i)))};
      }
    }
  }
  block_runs<Tl>(mine, before, whole, warps);

  const Chain<Tl> chain{c, p, order, tile, col0};
  if (c.ticket != nullptr) chain.publish(whole);
  const int last = seq[Tl::ROWS];
  float state = 0.f;
  if (last >= 0 && last == seq[Tl::ROWS + 1]) {
    const long long end = min(max(first_row(p, last + 1), 1ll), static_cast<long long>(p.rows)) - 1;      // the sequence's last row
    state = chain.state_before(max(c.chunks - 1 - static_cast<int>(end / Tl::ROWS), 0), parts);
  }
  if (threadIdx.x < Tl::COLS) carry[threadIdx.x] = state;
  if (c.ticket != nullptr && order % kScanGroup == kScanGroup - 1) chain.publish_state(apply(whole, state));
  __syncthreads();
  if (!in) return;

  float back[V];                                 // keep_{t+1} g_{t+1}
#pragma unroll
  for (int i = 0; i < V; ++i) back[i] = apply(before[i], carry[side * V + i]);
#pragma unroll
  for (int r = Tl::R - 1; r >= 0; --r) {
    const int t = first + r;
    if (t >= p.rows) continue;
    const int at = pile * Tl::R + r + 1, s = seq[at];
    float dx[V], dgate[V];
    if (s >= 0) {
      const long long state_at = static_cast<long long>(s) * p.channels + col;
      if (s != seq[at + 1]) load_state<V>(p.dfinal, state_at, back);
      const bool start = s != seq[at - 1];
      float h[V];
      if (start) {
        load_state<V>(p.initial, state_at, h);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) h[i] = before_row[r].get(i);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const Gate k = gate_of(small[r][i]);
        const float g = __fadd_rn(back[i], dh[r].get(i));
        dx[i] = k.take * g;
        dgate[i] = g * (k.keep * k.take) * (h[i] - x[r].get(i));
        back[i] = __fmul_rn(k.keep, g);
      }
      if (start && p.dinitial != nullptr) store_state<V>(p.dinitial, state_at, back);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) dx[i] = dgate[i] = 0.f;
    }
    const long long out = static_cast<long long>(t) * p.channels + col;
    if (p.dx != nullptr) store_row<T, V>(p.dx, out, dx);
    if (p.dgate != nullptr) store_row<T, V>(p.dgate, out, dgate);
  }
}

template <class T>
__global__ void __launch_bounds__(kThreads) scan_step_kernel(const ScanStepParams p) {
  const int d = blockIdx.x * kThreads + threadIdx.x;
  if (d >= p.channels) return;
  for (long long s = blockIdx.y; s < p.rows; s += gridDim.y) {
    float* state = p.state + s * p.state_stride + d;
    const Gate g = gate_of(smaller<T>(to_float(static_cast<const T*>(p.gate)[s * p.gate_stride + d])));
    const float h = fmaf(g.keep, *state, g.take * to_float(static_cast<const T*>(p.x)[s * p.x_stride + d]));
    *state = h;
    static_cast<T*>(p.h)[s * p.channels + d] = from_float<T>(h);
  }
}

dim3 step_grid(int channels, int rows) { return dim3((channels + kThreads - 1) / kThreads, rows < 65535 ? rows : 65535); }

bool whole_vectors(const ScanShape& p) {
  const int vec = p.half ? 8 : 4;
  auto fits = [&](const void* base, long long stride) { return reinterpret_cast<uintptr_t>(base) % 16 == 0 && stride % vec == 0; };
  return p.channels % vec == 0 && fits(p.x, p.x_stride) && fits(p.gate, p.gate_stride) && fits(p.initial, 0);
}
bool whole_vectors(const ScanGradParams& p) {
  return whole_vectors(static_cast<const ScanShape&>(p)) && reinterpret_cast<uintptr_t>(p.dh) % 16 == 0 && p.dh_stride % (p.half ? 8 : 4) == 0 &&
         reinterpret_cast<uintptr_t>(p.dfinal) % 16 == 0;
}

template <class Tl>
ScanPlan plan(const ScanShape& p) {
  ScanPlan s{};
  s.tiles = (p.channels + Tl::COLS - 1) / Tl::COLS;
  s.chunks = p.rows > Tl::ROWS ? (p.rows + Tl::ROWS - 1) / Tl::ROWS : 1;
  return s;
}
template <class F>
auto by_tile(bool half, bool vectors, F f) {
  if (half) return vectors ? f(Tile<__nv_bfloat16, 8>{}, __nv_bfloat16{}) : f(Tile<__nv_bfloat16, 1>{}, __nv_bfloat16{});
  return vectors ? f(Tile<float, 4>{}, float{}) : f(Tile<float, 1>{}, float{});
}

// Where the parts of the workspace lie.
cudaError_t lay_out(ScanChain& c, const ScanPlan& s, int channels, void* space, cudaStream_t stream) {
  c.chunks = s.chunks; c.tiles = s.tiles;
  if (s.chunks == 1) return cudaSuccess;
  const int groups = (s.chunks + kScanGroup - 1) / kScanGroup;
  c.ticket = static_cast<int*>(space);
  c.flags = c.ticket + 4;
  const size_t ints = 4 + static_cast<size_t>(s.chunks + groups) * s.tiles;
  c.runs = reinterpret_cast<float2*>(c.ticket + (ints + 3) / 4 * 4);
  c.states = reinterpret_cast<float*>(c.runs + static_cast<size_t>(s.chunks) * channels);
  return cudaMemsetAsync(space, 0, ints * sizeof(int), stream);
}

}  // namespace

ScanPlan scan_plan(const ScanParams& p) { return by_tile(p.half, whole_vectors(p), [&](auto tile, auto) { return plan<decltype(tile)>(p); }); }
ScanPlan scan_plan(const ScanGradParams& p) { return by_tile(p.half, whole_vectors(p), [&](auto tile, auto) { return plan<decltype(tile)>(p); }); }
long long scan_space(const ScanPlan& s, int channels) {
  if (s.chunks == 1) return 0;
  const long long groups = (s.chunks + kScanGroup - 1) / kScanGroup;
  return 32 + 4 * (s.chunks + groups) * s.tiles + 8ll * s.chunks * channels + 4ll * groups * channels;
}

cudaError_t launch_scan_forward(const ScanParams& p, void* space, cudaStream_t stream) {
  return by_tile(p.half, whole_vectors(p), [&](auto tile, auto type) {
    const ScanPlan s = plan<decltype(tile)>(p);
    ScanChain c{};
    const cudaError_t e = lay_out(c, s, p.channels, space, stream);
    if (e != cudaSuccess) return e;
    scan_forward_kernel<decltype(type), decltype(tile)::VEC><<<static_cast<unsigned>(s.chunks) * s.tiles, kScanThreads, 0, stream>>>(p, c);
    return cudaGetLastError();
  });
}

cudaError_t launch_scan_backward(const ScanGradParams& p, void* space, cudaStream_t stream) {
  return by_tile(p.half, whole_vectors(p), [&](auto tile, auto type) {
    const ScanPlan s = plan<decltype(tile)>(p);
    ScanChain c{};
    const cudaError_t e = lay_out(c, s, p.channels, space, stream);
    if (e != cudaSuccess) return e;
    scan_backward_kernel<decltype(type), decltype(tile)::VEC><<<static_cast<unsigned>(s.chunks) * s.tiles, kScanThreads, 0, stream>>>(p, c);
    return cudaGetLastError();
  });
}

cudaError_t launch_scan_step(const ScanStepParams& p, int sms, cudaStream_t stream) {
  (void)sms;
  if (p.half) scan_step_kernel<__nv_bfloat16><<<step_grid(p.channels, p.rows), kThreads, 0, stream>>>(p);
  else scan_step_kernel<float><<<step_grid(p.channels, p.rows), kThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace sep

// Gated linear recurrence along sequences, and its gradients.
//
//   keep_t = sigmoid(gate_t), take_t = 1 - keep_t:   h_t = keep_t h_{t-1} + take_t x_t
//   g_t = dh_t + keep_{t+1} g_{t+1}:   dx_t = take_t g_t,   dgate_t = g_t keep_t take_t (h_{t-1} - x_t),   dh_{-1} = keep_0 g_0
//
// The state, and everything that is added up along a sequence, is fp32.
#include <atomic>

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
  float2* runs;                  // [chunks][channels]
  float* states;                 // [groups][channels] behind each group
};

template <class T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Two fp32 numbers that one instruction works on.
struct Pair { unsigned long long v; };
__device__ __forceinline__ Pair pair_of(float a, float b) { Pair p; asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(a), "f"(b)); return p; }
__device__ __forceinline__ void parts_of(Pair p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p.v)); }
__device__ __forceinline__ Pair operator+(Pair a, Pair b) { Pair d; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v)); return d; }
__device__ __forceinline__ Pair operator*(Pair a, Pair b) { Pair d; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v)); return d; }
__device__ __forceinline__ Pair fused(Pair a, Pair b, Pair c) { Pair d; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v)); return d; }
// V numbers of a thread, of one row.  (Sums and products are written out, so that the bits do not depend on what else a call computes.)
template <int V> struct Row {
  Pair p[V / 2];
  __device__ __forceinline__ static Row all(float f) { Row r; for (int i = 0; i < V / 2; ++i) r.p[i] = pair_of(f, f); return r; }
  __device__ __forceinline__ void put(int i, float a, float b) { p[i] = pair_of(a, b); }
  __device__ __forceinline__ void get(float (&f)[V]) const { _Pragma("unroll") for (int i = 0; i < V / 2; ++i) parts_of(p[i], f[2 * i], f[2 * i + 1]); }
  __device__ __forceinline__ static Row of(const float (&f)[V]) { Row r; _Pragma("unroll") for (int i = 0; i < V / 2; ++i) r.p[i] = pair_of(f[2 * i], f[2 * i + 1]); return r; }
};
template <> struct Row<1> {
  float f;
  __device__ __forceinline__ static Row all(float f) { return Row{f}; }
  __device__ __forceinline__ void get(float (&o)[1]) const { o[0] = f; }
  __device__ __forceinline__ static Row of(const float (&o)[1]) { return Row{o[0]}; }
};
template <int V> __device__ __forceinline__ Row<V> operator+(Row<V> a, const Row<V>& b) {
  if constexpr (V == 1) a.f = __fadd_rn(a.f, b.f);
  else { _Pragma("unroll") for (int i = 0; i < V / 2; ++i) a.p[i] = a.p[i] + b.p[i]; }
  return a;
}
template <int V> __device__ __forceinline__ Row<V> operator*(Row<V> a, const Row<V>& b) {
  if constexpr (V == 1) a.f = __fmul_rn(a.f, b.f);
  else { _Pragma("unroll") for (int i = 0; i < V / 2; ++i) a.p[i] = a.p[i] * b.p[i]; }
  return a;
}
template <int V> __device__ __forceinline__ Row<V> fused(const Row<V>& a, const Row<V>& b, Row<V> c) {
  if constexpr (V == 1) c.f = fmaf(a.f, b.f, c.f);
  else { _Pragma("unroll") for (int i = 0; i < V / 2; ++i) c.p[i] = fused(a.p[i], b.p[i], c.p[i]); }
  return c;
}

// sigmoid(gate) and sigmoid(-gate), each to its own last digits: 1 / (1 + e) and e / (1 + e) of e = exp(gate), which is held at 2^126 (a gate of
// 87; NaN stays).  For bf16 gates the exponent is rounded once (|gate| 2^-24 of the result), for fp32 ones it is not.
__device__ __forceinline__ float at_most(float v, float top) { float r; asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(top)); return r; }
__device__ __forceinline__ float ex2(float v) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; }
__device__ __forceinline__ float reciprocal(float v) { float r; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; }
template <class T, int V>
__device__ __forceinline__ void gates_of(const Row<V>& gate, Row<V>& keep, Row<V>& take) {
  float e[V];
  if constexpr (sizeof(T) == 2) {
    const Row<V> scaled = gate * Row<V>::all(1.4426950408889634f);
    scaled.get(e);
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = ex2(at_most(e[i], 126.f));
  } else {
    gate.get(e);
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = expf(at_most(e[i], 87.f));
  }
  const Row<V> power = Row<V>::of(e), sum = power + Row<V>::all(1.f);
  sum.get(e);
#pragma unroll
  for (int i = 0; i < V; ++i) e[i] = sizeof(T) == 2 ? reciprocal(e[i]) : __frcp_rn(e[i]);
  take = Row<V>::of(e);
  keep = power * take;
}
__device__ __forceinline__ void gate_of(float gate, float& keep, float& take, bool half) {
  Row<1> k, t;
  if (half) gates_of<__nv_bfloat16, 1>(Row<1>{gate}, k, t); else gates_of<float, 1>(Row<1>{gate}, k, t);
  keep = k.f; take = t.f;
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

template <class T, int V>
__device__ __forceinline__ void store_row(void* base, long long at, const Row<V>& row) {
  float f[V];
  row.get(f);
  if constexpr (V == 8) {
    *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(base) + at) =
        make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  } else if constexpr (V == 4) {
    *reinterpret_cast<float4*>(static_cast<float*>(base) + at) = make_float4(f[0], f[1], f[2], f[3]);
  } else {
    static_cast<T*>(base)[at] = from_float<T>(f[0]);
  }
}
template <int V>
__device__ __forceinline__ Row<V> load_state(const float* base, long long at) {
  if (base == nullptr) return Row<V>::all(0.f);
  float f[V];
  if constexpr (V >= 4) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const float4 v = *reinterpret_cast<const float4*>(base + at + i);
      f[i] = v.x; f[i + 1] = v.y; f[i + 2] = v.z; f[i + 3] = v.w;
    }
  } else {
    f[0] = base[at];
  }
  return Row<V>::of(f);
}
template <int V>
__device__ __forceinline__ void store_state(float* base, long long at, const Row<V>& row) {
  float f[V];
  row.get(f);
  if constexpr (V >= 4) {
#pragma unroll
    for (int i = 0; i < V; i += 4) *reinterpret_cast<float4*>(base + at + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
  } else {
    base[at] = f[0];
  }
}

// A unit of work: a chunk of rows and a tile of channels.  A thread has R rows of V channels; LANES threads lie side by side across the
// channels, and the piles of R rows above one another along time.
template <class Type, int Vec> struct Tile {
  using T = Type;
  static constexpr int V = Vec;
  static constexpr int LANES = V > 1 ? 8 : 32;
  static constexpr int R = V > 1 ? 4 : 16;
  static constexpr int PILES = kScanThreads / LANES;
  static constexpr int ROWS = PILES * R;
  static constexpr int COLS = LANES * V;
  static constexpr int PARTS = kScanThreads / COLS;            // threads that share a channel where runs are joined
  static constexpr int PART_PILES = PILES / PARTS;
  static constexpr int WARP_COLS = COLS / (kScanThreads / 32); // there, a warp has these channels of all parts
  // Each thread copies its rows into places of its own in shared memory (nobody has to wait for anybody else's copies): row r of thread i lies at
  // r * PITCH + slot(i).  When the gates have been read, the run of a pile and channel takes the place of two of them; the pitch, and 16 bytes between
  // the threads of two parts, keep what half a warp reads together in different banks.
  static constexpr int SLOT = V > 1 ? 16 : 4;
  static constexpr int PITCH = kScanThreads * SLOT + (V == 8 ? 160 : V == 4 ? 192 : 0);
  __device__ __forceinline__ static int slot(int thread) { return thread * SLOT + (V > 1 ? thread / (PART_PILES * LANES) * 16 : 0); }
  static constexpr int ARRAY = R * PITCH;
  static constexpr int RUNS = V > 1 ? 0 : PILES * COLS * 8;     // (with one channel a thread the runs lie by themselves)
  __device__ __forceinline__ static unsigned char* run_at(unsigned char* gates, unsigned char* runs, int pile_order, int ch) {
    if constexpr (V > 1) return gates + (ch % V) / 2 * PITCH + slot(pile_order * LANES + ch / V) + (ch & 1) * 8;
    else return runs + (pile_order * COLS + ch) * 8;
  }
};
template <class Tl>
__device__ __forceinline__ void fetch(unsigned char* place, const void* base, long long at, bool there) {
  using T = typename Tl::T;
  if constexpr (Tl::V > 1) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" :: "r"(smem_u32(place)), "l"(static_cast<const T*>(base) + (there ? at : 0)), "r"(there ? 16 : 0) : "memory");
  } else if constexpr (sizeof(T) == 4) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" :: "r"(smem_u32(place)), "l"(static_cast<const T*>(base) + (there ? at : 0)), "r"(there ? 4 : 0) : "memory");
  } else {
    *reinterpret_cast<float*>(place) = there ? to_float(static_cast<const T*>(base)[at]) : 0.f;
  }
}
template <class Tl>
__device__ __forceinline__ Row<Tl::V> fetched(const unsigned char* place) {
  if constexpr (Tl::V == 8) {
    const uint4 v = *reinterpret_cast<const uint4*>(place);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    Row<8> r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r.put(i, __uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    return r;
  } else if constexpr (Tl::V == 4) {
    const float4 v = *reinterpret_cast<const float4*>(place);
    Row<4> r;
    r.put(0, v.x, v.y); r.put(1, v.z, v.w);
    return r;
  } else {
    return Row<1>{*reinterpret_cast<const float*>(place)};
  }
}
__device__ __forceinline__ void fetch_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft> __device__ __forceinline__ void fetch_wait() { asm volatile("cp.async.wait_group %0;" :: "n"(kLeft) : "memory"); }

// The rows of a unit and what is handed on within its block.
template <class Tl>
struct ScanShared {
  int seq[2][Tl::ROWS + 2];      // sequences of the rows from the one before the chunk to the one behind it, of two units
  float carry[Tl::PARTS][Tl::COLS];
  int next;                      // the unit after this one
};

// Chunks are dealt out in the order in which they depend on one another, by a ticket: a chunk waits only for chunks that were dealt out before it, and
// every block works on its chunks in that order, so the first unfinished one never waits, however many blocks are resident.
// `order` counts chunks from where the recurrence starts (the first row, or the last one for the backward).  Each leaves what it does to the state
// (its run) as soon as it knows it; the state in front of a chunk is that behind the group of 32 chunks before it, and the runs of the chunks
// between, joined in one order: no rounding depends on who was first.  Only the groups' states follow one another.
//
// A number says by itself that it is there: the workspace is filled with ones, which no number that is left has (NaN is left as 0x7fffffff), a run is
// written and read as one 8-byte word, and nothing else is handed on with it that would have to be in order.  (With a flag beside it, its
// writer waits for the numbers to arrive before the flag, its reader for the flag before the numbers: 8192 rows of 2048 channels 46.7 us, in
// four barriers a unit instead of two.)
constexpr uint32_t kAbsent = 0xffffffffu;
__device__ __forceinline__ uint32_t present(float f) { const uint32_t u = __float_as_uint(f); return u == kAbsent ? 0x7fffffffu : u; }
__device__ __forceinline__ void leave(float2* at, Run r) {
  const unsigned long long v = static_cast<unsigned long long>(present(r.b)) << 32 | present(r.a);
  asm volatile("st.relaxed.gpu.global.b64 [%0], %1;" :: "l"(at), "l"(v) : "memory");
}
__device__ __forceinline__ void leave(float* at, float f) { asm volatile("st.relaxed.gpu.global.b32 [%0], %1;" :: "l"(at), "r"(present(f)) : "memory"); }
__device__ __forceinline__ uint2 look(const float2* at) {
  unsigned long long v;
  asm volatile("ld.relaxed.gpu.global.b64 %0, [%1];" : "=l"(v) : "l"(at) : "memory");
  return make_uint2(static_cast<uint32_t>(v), static_cast<uint32_t>(v >> 32));
}
__device__ __forceinline__ uint32_t look(const float* at) { uint32_t v; asm volatile("ld.relaxed.gpu.global.b32 %0, [%1];" : "=r"(v) : "l"(at) : "memory"); return v; }

template <class Tl>
struct Chain {
  const ScanChain& c;
  const ScanShape& p;
  ScanShared<Tl>& sh;
  int order, tile;
  // this thread works on channel `ch` of the tile, for part `part` of what is joined; the other parts belong to lanes of its warp
  int ch, part, col;
  Run before, whole;             // of this chunk: of the parts before, of all

  __device__ __forceinline__ Chain(const ScanChain& c, const ScanShape& p, ScanShared<Tl>& sh, int order, int tile) : c(c), p(p), sh(sh), order(order), tile(tile) {
    const int lane = threadIdx.x & 31;
    ch = (threadIdx.x >> 5) * Tl::WARP_COLS + lane % Tl::WARP_COLS;
    part = lane / Tl::WARP_COLS;
    col = tile * Tl::COLS + ch;
  }
  __device__ __forceinline__ float2* run_at(int k) const { return c.runs + static_cast<long long>(k) * p.channels + col; }
  __device__ __forceinline__ float* state_at(int g) const { return c.states + static_cast<long long>(g) * p.channels + col; }

  // `run` of each part becomes that of all parts up to it.
  __device__ __forceinline__ Run join_parts(Run run) const {
#pragma unroll
    for (int d = Tl::WARP_COLS; d < 32; d *= 2) {
      const Run prev = {__shfl_up_sync(0xffffffffu, run.a, d), __shfl_up_sync(0xffffffffu, run.b, d)};
      if (static_cast<int>(threadIdx.x & 31) >= d) run = join(prev, run);
    }
    return run;
  }
  __device__ __forceinline__ static Run of_last_part(Run run) {
    const int from = 32 - Tl::WARP_COLS + static_cast<int>(threadIdx.x & 31) % Tl::WARP_COLS;
    return {__shfl_sync(0xffffffffu, run.a, from), __shfl_sync(0xffffffffu, run.b, from)};
  }

  // From the runs of the piles in shared memory (in order): each becomes the run of the piles before it in its part.  Leaves the whole chunk's run
  // to the chunks behind.
  template <class RunAt>
  __device__ __forceinline__ void join_piles(RunAt run_in_smem) {
    Run run = nothing();
#pragma unroll
    for (int i = 0; i < Tl::PART_PILES; ++i) {
      float2* at = reinterpret_cast<float2*>(run_in_smem(part * Tl::PART_PILES + i, ch));
      const float2 v = *at;
      *at = make_float2(run.a, run.b);
      run = join(run, Run{v.x, v.y});
    }
    run = join_parts(run);
    before = {__shfl_up_sync(0xffffffffu, run.a, Tl::WARP_COLS), __shfl_up_sync(0xffffffffu, run.b, Tl::WARP_COLS)};
    if (part == 0) before = nothing();
    whole = of_last_part(run);
    if (part == 0 && col < p.channels && c.ticket != nullptr) leave(run_at(order), whole);
  }

  // The state in front of this chunk, of a sequence that starts in chunk `from` (in this order).
  __device__ __forceinline__ float state_before(int from) {
    const int group = order / kScanGroup, group_start = group * kScanGroup;
    const bool handed = from < group_start;
    const int start = handed ? group_start : from, n = max(order - start, 0);
    const int begin = start + n * part / Tl::PARTS, count = start + n * (part + 1) / Tl::PARTS - begin;
    constexpr int kMost = kScanGroup / Tl::PARTS;              // (n is less than kScanGroup)
    uint2 got[kMost];
    uint32_t state = 0;
    bool ok = true;
    if (col < p.channels) {
      ok = spin_until([&] {
        bool all = true;
        if (handed) { state = look(state_at(group - 1)); all = state != kAbsent; }
#pragma unroll
        for (int i = 0; i < kMost; ++i) if (i < count) got[i] = look(run_at(begin + i));
#pragma unroll
        for (int i = 0; i < kMost; ++i) if (i < count) all = all && got[i].x != kAbsent;
        return all;
      }, p.wait_budget_ns, p.status);
      if (!ok) report_failure(p.status, kStatusTimeoutPipeline, kKernelScan, 0, p.rank, order, begin, tile);
    }
    Run run = nothing();
    if (col < p.channels) {
#pragma unroll
      for (int i = 0; i < kMost; ++i) if (i < count) run = join(run, Run{__uint_as_float(got[i].x), __uint_as_float(got[i].y)});
    }
    if (!ok) run = {-0.f, __int_as_float(0x7fc00000)};
    return apply(of_last_part(join_parts(run)), __uint_as_float(state));
  }
  // The state behind the chunk goes to the group behind; the state in front of each part to the block's threads.
  __device__ __forceinline__ void spread(float state) {
    if (part == 0 && col < p.channels && c.ticket != nullptr && order % kScanGroup == kScanGroup - 1) leave(state_at(order / kScanGroup), apply(whole, state));
    sh.carry[part][ch] = apply(before, state);
    __syncthreads();
  }
  // The state in front of this thread's pile.
  template <class RunAt>
  __device__ __forceinline__ Row<Tl::V> state_of_pile(RunAt run_in_smem, int pile_order, int side) const {
    float f[Tl::V];
#pragma unroll
    for (int i = 0; i < Tl::V; ++i) {
      const float2 r = *reinterpret_cast<const float2*>(run_in_smem(pile_order, side * Tl::V + i));
      f[i] = apply(Run{r.x, r.y}, sh.carry[pile_order / Tl::PART_PILES][side * Tl::V + i]);
    }
    return Row<Tl::V>::of(f);
  }
};

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

// The first unit of a block; thread 0 has the next one in hand, and claims the one after it when it gives that out.  (No block has a second
// unit where there is one for each.)
__device__ __forceinline__ int claim(const ScanChain& c, int units) {
  return c.ticket != nullptr && units > static_cast<int>(gridDim.x) ? atomicAdd(c.ticket, 1) + 1 : units;
}
__device__ __forceinline__ int first_unit(const ScanChain& c, int* next) {
  if (c.ticket == nullptr) return blockIdx.x;
  if (threadIdx.x == 0) *next = atomicAdd(c.ticket, 1) + 1;
  __syncthreads();
  const int unit = *next;
  __syncthreads();
  return unit;
}

// Rows of the unit after this one are on their way while this one's are worked on.
template <class Tl>
__global__ void __launch_bounds__(kScanThreads, 2) scan_forward_kernel(const ScanParams p, const ScanChain c) {
  using T = typename Tl::T;
  constexpr int V = Tl::V, R = Tl::R;
  extern __shared__ __align__(16) unsigned char space[];       // [2 units][gate, x], runs
  __shared__ ScanShared<Tl> sh;
  const int side = threadIdx.x % Tl::LANES, pile = threadIdx.x / Tl::LANES, units = c.chunks * c.tiles;
  auto array = [&](int buffer, int which) { return space + (buffer * 2 + which) * Tl::ARRAY; };
  auto place = [&](int buffer, int which, int r) { return array(buffer, which) + r * Tl::PITCH + Tl::slot(threadIdx.x); };
  auto issue = [&](int unit, int buffer) {
    if (unit < units) {
      const int chunk = unit / c.tiles, tile = unit - chunk * c.tiles, row0 = chunk * Tl::ROWS, col = tile * Tl::COLS + side * V;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int t = row0 + pile * R + r;
        const bool there = col < p.channels && t < p.rows;
        fetch<Tl>(place(buffer, 0, r), p.gate, t * p.gate_stride + col, there);
        fetch<Tl>(place(buffer, 1, r), p.x, t * p.x_stride + col, there);
      }
      for (int i = threadIdx.x; i < Tl::ROWS + 2; i += kScanThreads) sh.seq[buffer][i] = sequence_of(p, row0 - 1 + i);
    }
    fetch_commit();
  };
  int claimed = units, buffer = 0, unit = first_unit(c, &sh.next);
  issue(unit, 0);
  if (threadIdx.x == 0) claimed = claim(c, units);
  __syncthreads();
  for (; unit < units; buffer ^= 1) {
    const int chunk = unit / c.tiles, tile = unit - chunk * c.tiles;
    const int first = chunk * Tl::ROWS + pile * R, col = tile * Tl::COLS + side * V;
    const bool in = col < p.channels;
    const int* seq = sh.seq[buffer];
    auto run_at = [&](int pile_order, int ch) { return Tl::run_at(array(buffer, 0), space + 4 * Tl::ARRAY, pile_order, ch); };
    empty_sequences<Tl>(p, c, chunk, tile, p.initial, p.final_state, true);
    if (threadIdx.x == 0) sh.next = claimed;
    fetch_wait<0>();

    Row<V> keep[R], add[R];                      // h -> keep h + add
    Row<V> a = Row<V>::all(1.f), b = Row<V>::all(0.f);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int at = pile * R + r + 1, s = seq[at];
      gates_of<T, V>(fetched<Tl>(place(buffer, 0, r)), keep[r], add[r]);
      add[r] = add[r] * fetched<Tl>(place(buffer, 1, r));
      if (s != seq[at - 1] || s < 0) {
        a = Row<V>::all(-0.f);
        b = load_state<V>(s >= 0 && in ? p.initial : nullptr, static_cast<long long>(s) * p.channels + col);
      }
      if (s >= 0) {
        a = a * keep[r];
        b = fused(keep[r], b, add[r]);
      }
    }
    {
      float fa[V], fb[V];
      a.get(fa); b.get(fb);
#pragma unroll
      for (int i = 0; i < V; ++i) *reinterpret_cast<float2*>(run_at(pile, side * V + i)) = make_float2(fa[i], fb[i]);
    }
    Chain<Tl> chain(c, p, sh, chunk, tile);
    __syncthreads();
    const int next = sh.next;
    if (threadIdx.x == 0 && next < units) claimed = claim(c, units);
    chain.join_piles(run_at);
    issue(next, buffer ^ 1);
    float state = 0.f;
    if (seq[1] >= 0 && seq[1] == seq[0]) state = chain.state_before(static_cast<int>(max(first_row(p, seq[1]), 0ll) / Tl::ROWS));
    chain.spread(state);

    Row<V> h = chain.state_of_pile(run_at, pile, side);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (!in || first + r >= p.rows) break;
      const int at = pile * R + r + 1, s = seq[at];
      if (s != seq[at - 1] || s < 0) h = load_state<V>(s >= 0 ? p.initial : nullptr, static_cast<long long>(s) * p.channels + col);
      if (s >= 0) {
        h = fused(keep[r], h, add[r]);
        if (p.final_state != nullptr && seq[at + 1] != s) store_state<V>(p.final_state, static_cast<long long>(s) * p.channels + col, h);
      }
      store_row<T, V>(p.h, static_cast<long long>(first + r) * p.channels + col, h);
    }
    unit = next;
  }
}

// As the forward, from the last row to the first: what runs along is keep_t g_t.
template <class Tl>
__global__ void __launch_bounds__(kScanThreads, 2) scan_backward_kernel(const ScanGradParams p, const ScanChain c) {
  using T = typename Tl::T;
  constexpr int V = Tl::V, R = Tl::R;
  extern __shared__ __align__(16) unsigned char space[];       // [2 units][gate, dh], x, h of the row before, runs
  __shared__ ScanShared<Tl> sh;
  const int side = threadIdx.x % Tl::LANES, pile_order = threadIdx.x / Tl::LANES, pile = Tl::PILES - 1 - pile_order, units = c.chunks * c.tiles;
  auto array = [&](int buffer, int which) { return space + (buffer * 2 + which) * Tl::ARRAY; };
  auto place = [&](int buffer, int which, int r) { return array(buffer, which) + r * Tl::PITCH + Tl::slot(threadIdx.x); };
  auto issue = [&](int unit, int buffer) {
    if (unit < units) {
      const int order = unit / c.tiles, tile = unit - order * c.tiles, row0 = (c.chunks - 1 - order) * Tl::ROWS, col = tile * Tl::COLS + side * V;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int t = row0 + pile * R + r;
        const bool there = col < p.channels && t < p.rows;
        fetch<Tl>(place(buffer, 0, r), p.gate, t * p.gate_stride + col, there);
        fetch<Tl>(place(buffer, 1, r), p.dh, t * p.dh_stride + col, there && p.dh != nullptr);
      }
      for (int i = threadIdx.x; i < Tl::ROWS + 2; i += kScanThreads) sh.seq[buffer][i] = sequence_of(p, row0 - 1 + i);
    }
    fetch_commit();
  };
  // what only the gate's gradient needs, later than the rest
  auto issue_late = [&](int unit) {
    if (unit < units && p.dgate != nullptr) {
      const int order = unit / c.tiles, tile = unit - order * c.tiles, row0 = (c.chunks - 1 - order) * Tl::ROWS, col = tile * Tl::COLS + side * V;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const int t = row0 + pile * R + r;
        const bool there = col < p.channels && t < p.rows;
        fetch<Tl>(place(2, 0, r), p.x, t * p.x_stride + col, there);
        fetch<Tl>(place(2, 1, r), p.h, static_cast<long long>(t - 1) * p.channels + col, there && t > 0);
      }
    }
    fetch_commit();
  };
  int claimed = units, buffer = 0, unit = first_unit(c, &sh.next);
  issue(unit, 0);
  issue_late(unit);
  if (threadIdx.x == 0) claimed = claim(c, units);
  __syncthreads();
  for (; unit < units; buffer ^= 1) {
    const int order = unit / c.tiles, tile = unit - order * c.tiles, chunk = c.chunks - 1 - order;
    const int first = chunk * Tl::ROWS + pile * R, col = tile * Tl::COLS + side * V;
    const bool in = col < p.channels;
    const int* seq = sh.seq[buffer];
    auto run_at = [&](int order_of_pile, int ch) { return Tl::run_at(array(buffer, 0), space + 6 * Tl::ARRAY, order_of_pile, ch); };
    empty_sequences<Tl>(p, c, order, tile, p.dfinal, p.dinitial, false);
    if (threadIdx.x == 0) sh.next = claimed;
    fetch_wait<1>();

    Row<V> keep[R], take[R];
    Row<V> a = Row<V>::all(1.f), b = Row<V>::all(0.f);
#pragma unroll
    for (int r = R - 1; r >= 0; --r) {
      const int at = pile * R + r + 1, s = seq[at];
      gates_of<T, V>(fetched<Tl>(place(buffer, 0, r)), keep[r], take[r]);
      if (s != seq[at + 1] || s < 0) {
        a = Row<V>::all(-0.f);
        b = load_state<V>(s >= 0 && in ? p.dfinal : nullptr, static_cast<long long>(s) * p.channels + col);
      }
      if (s >= 0) {
        a = a * keep[r];
        b = keep[r] * (b + fetched<Tl>(place(buffer, 1, r)));
      }
    }
    {
      float fa[V], fb[V];
      a.get(fa); b.get(fb);
#pragma unroll
      for (int i = 0; i < V; ++i) *reinterpret_cast<float2*>(run_at(pile_order, side * V + i)) = make_float2(fa[i], fb[i]);
    }
    Chain<Tl> chain(c, p, sh, order, tile);
    __syncthreads();
    const int next = sh.next;
    if (threadIdx.x == 0 && next < units) claimed = claim(c, units);
    chain.join_piles(run_at);
    issue(next, buffer ^ 1);
    const int last = seq[Tl::ROWS];
    float state = 0.f;
    if (last >= 0 && last == seq[Tl::ROWS + 1]) {
      const long long end = min(max(first_row(p, last + 1), 1ll), static_cast<long long>(p.rows)) - 1;      // the sequence's last row
      state = chain.state_before(max(c.chunks - 1 - static_cast<int>(end / Tl::ROWS), 0));
    }
    chain.spread(state);

    Row<V> back = chain.state_of_pile(run_at, pile_order, side);                   // keep_{t+1} g_{t+1}
    fetch_wait<1>();
#pragma unroll
    for (int r = R - 1; r >= 0; --r) {
      const int t = first + r;
      if (!in || t >= p.rows) continue;
      const int at = pile * R + r + 1, s = seq[at];
      Row<V> dx = Row<V>::all(0.f), dgate = dx;
      if (s >= 0) {
        const long long state_at = static_cast<long long>(s) * p.channels + col;
        if (s != seq[at + 1]) back = load_state<V>(p.dfinal, state_at);
        const bool start = s != seq[at - 1];
        const Row<V> g = back + fetched<Tl>(place(buffer, 1, r));
        dx = take[r] * g;
        if (p.dgate != nullptr) {
          const Row<V> h = start ? load_state<V>(p.initial, state_at) : fetched<Tl>(place(2, 1, r));
          dgate = g * (keep[r] * take[r]) * fused(Row<V>::all(-1.f), fetched<Tl>(place(2, 0, r)), h);
        }
        back = keep[r] * g;
        if (start && p.dinitial != nullptr) store_state<V>(p.dinitial, state_at, back);
      }
      const long long out = static_cast<long long>(t) * p.channels + col;
      if (p.dx != nullptr) store_row<T, V>(p.dx, out, dx);
      if (p.dgate != nullptr) store_row<T, V>(p.dgate, out, dgate);
    }
    issue_late(next);
    unit = next;
  }
}

template <class T>
__global__ void __launch_bounds__(kThreads) scan_step_kernel(const ScanStepParams p) {
  const int d = blockIdx.x * kThreads + threadIdx.x;
  if (d >= p.channels) return;
  for (long long s = blockIdx.y; s < p.rows; s += gridDim.y) {
    float* state = p.state + s * p.state_stride + d;
    float keep, take;
    gate_of(to_float(static_cast<const T*>(p.gate)[s * p.gate_stride + d]), keep, take, sizeof(T) == 2);
    const float h = fmaf(keep, *state, __fmul_rn(take, to_float(static_cast<const T*>(p.x)[s * p.x_stride + d])));
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
  if (half) return vectors ? f(Tile<__nv_bfloat16, 8>{}) : f(Tile<__nv_bfloat16, 1>{});
  return vectors ? f(Tile<float, 4>{}) : f(Tile<float, 1>{});
}

// Where the parts of the workspace lie.  The ticket counts up from -1, as all of it is filled.
cudaError_t lay_out(ScanChain& c, const ScanPlan& s, int channels, void* space, cudaStream_t stream) {
  c.chunks = s.chunks; c.tiles = s.tiles;
  if (s.chunks == 1) return cudaSuccess;
  c.ticket = static_cast<int*>(space);
  c.runs = reinterpret_cast<float2*>(c.ticket + 4);
  c.states = reinterpret_cast<float*>(c.runs + static_cast<size_t>(s.chunks) * channels);
  return cudaMemsetAsync(space, 0xff, static_cast<size_t>(scan_space(s, channels)), stream);
}

}  // namespace

ScanPlan scan_plan(const ScanParams& p) { return by_tile(p.half, whole_vectors(p), [&](auto tile) { return plan<decltype(tile)>(p); }); }
ScanPlan scan_plan(const ScanGradParams& p) { return by_tile(p.half, whole_vectors(p), [&](auto tile) { return plan<decltype(tile)>(p); }); }
long long scan_space(const ScanPlan& s, int channels) {
  if (s.chunks == 1) return 0;
  const long long groups = (s.chunks + kScanGroup - 1) / kScanGroup;
  return 16 + 8ll * s.chunks * channels + 4ll * groups * channels;
}

namespace {

template <class Tl, class Params>
cudaError_t launch_scan(void (*kernel)(const Params, const ScanChain), const Params& p, int arrays, int sms, void* space, cudaStream_t stream) {
  const ScanPlan s = plan<Tl>(p);
  ScanChain c{};
  cudaError_t e = lay_out(c, s, p.channels, space, stream);
  if (e != cudaSuccess) return e;
  const int smem = arrays * Tl::ARRAY + Tl::RUNS;
  static std::atomic<bool> configured[64];       // the shared-memory limit is an attribute of the function on a device
  int dev = 0;
  if ((e = cudaGetDevice(&dev)) != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[dev].load(std::memory_order_acquire)) {
    if ((e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) != cudaSuccess) return e;
    configured[dev].store(true, std::memory_order_release);
  }
  const long long units = static_cast<long long>(s.chunks) * s.tiles;
  const unsigned grid = static_cast<unsigned>(s.chunks == 1 || units < 2 * sms ? units : 2 * sms);
  kernel<<<grid, kScanThreads, smem, stream>>>(p, c);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_scan_forward(const ScanParams& p, int sms, void* space, cudaStream_t stream) {
  return by_tile(p.half, whole_vectors(p), [&](auto tile) { return launch_scan<decltype(tile)>(scan_forward_kernel<decltype(tile)>, p, 4, sms, space, stream); });
}
cudaError_t launch_scan_backward(const ScanGradParams& p, int sms, void* space, cudaStream_t stream) {
  return by_tile(p.half, whole_vectors(p), [&](auto tile) { return launch_scan<decltype(tile)>(scan_backward_kernel<decltype(tile)>, p, 6, sms, space, stream); });
}

cudaError_t launch_scan_step(const ScanStepParams& p, int sms, cudaStream_t stream) {
  (void)sms;
  if (p.half) scan_step_kernel<__nv_bfloat16><<<step_grid(p.channels, p.rows), kThreads, 0, stream>>>(p);
  else scan_step_kernel<float><<<step_grid(p.channels, p.rows), kThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace sep

// Gated linear recurrence along sequences, and its gradients.
//
//   keep_t = sigmoid(gate_t), take_t = 1 - keep_t:   h_t = keep_t h_{t-1} + take_t x_t = h_{t-1} + take_t (x_t - h_{t-1})
//   g_t = dh_t + keep_{t+1} g_{t+1}:   dx_t = take_t g_t,   dgate_t = g_t keep_t take_t (h_{t-1} - x_t),   dh_{-1} = keep_0 g_0
//
// The state, and everything that is added up along a sequence, is fp32.
//
// What bounds it: memory (two arrays read and one written, four and two in the backward), and two special-function results an element.  A thread
// walks one vector of channels through a segment of rows.  Where sequences and channels alone are threads enough, a segment is a whole
// sequence, and that is all.  Else time is split: what each segment does to the state in front of it (its run, h -> a h + b) is formed first, the
// runs of a block's segments are joined, and a second walk begins from each segment's state.  Where the segments of a sequence lie in one block, one
// kernel does both; else a first kernel leaves the runs, and the second one's blocks join those of the blocks before.  The second reading comes
// from L2 as far as that reaches.  No block waits for another, and all is added in one order: a repeated call gives the same bits.
#include <algorithm>
#include <atomic>
#include <initializer_list>
#include <type_traits>
#include <utility>

#include "scan.h"
#include "ptx.cuh"
#include "rows.cuh"

namespace sep {

namespace {

constexpr int kScanThreads = 128;               // (256: 8192 rows of 2048 channels forward 40.8 -> 48 us, backward 58.6 -> 61)
// Blocks an SM: 72 registers a thread.  With 80 and 6 blocks 8192 rows of 2048 bf16 channels forward took 42.9 us instead of 37.5, 7488 of 1001 61.6 instead of 45.5.
constexpr int kScanBlocks = 7;

// e = exp(gate), held at 2^126 (a gate of 87; NaN stays), and sigmoid(-gate) = 1 / (1 + e), what a row takes; it keeps e / (1 + e), to that one's own last
// digits too.  For bf16 gates the exponent is rounded once (|gate| 2^-24 of the result), for fp32 ones it is not.
__device__ __forceinline__ float at_most(float v, float top) { float r; asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(top)); return r; }
__device__ __forceinline__ float ex2(float v) { float r; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; }
__device__ __forceinline__ float reciprocal(float v) { float r; asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v)); return r; }
template <class T, int V>
__device__ __forceinline__ void gates_of(const Row<V>& gate, Row<V>& power, Row<V>& take) {
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
  power = Row<V>::of(e);
  const Row<V> sum = power + Row<V>::all(1.f);
  sum.get(e);
#pragma unroll
  for (int i = 0; i < V; ++i) e[i] = reciprocal(e[i]);
  take = Row<V>::of(e);
}
// keep h + take x, and keep h alone.  Where less than half is taken, as h + take (x - h) and h - take h: 32 bits cannot hold a `keep` near 1 and 1 - keep
// alike, and what `keep` is off by, at every row to one side, makes a state that lasts e^gate rows drift away from its inputs (300000 rows whose inputs
// equal the state, gates of 12 to 18: by up to 0.9 %; in these forms by 2e-6).  Else as x - keep (x - h).  Written with predicates, which leave the selections that a
// compiler makes of it out (131072 rows of 1024 bf16 channels forward 250 -> 242 us).
// kAny: also where the state, or the difference, is infinite; else that makes a NaN, which stays in the state and is seen at its end.
__device__ __forceinline__ bool finite(float v) { return fabsf(v) < INFINITY; }
template <bool kAny> __device__ __forceinline__ float follow(float h, float x, float power, float take) {
  const float d = x - h, keep = power * take;
  if (kAny && !finite(d)) return fmaf(keep, h, take * x);
  float r;
  asm("{\n .reg .pred near;\n setp.gt.f32 near, %1, 0f3F800000;\n @near fma.rn.f32 %0, %2, %4, %5;\n @!near fma.rn.f32 %0, %3, %4, %6;\n}"
      : "=f"(r) : "f"(power), "f"(take), "f"(-keep), "f"(d), "f"(h), "f"(x));
  return r;
}
template <bool kAny> __device__ __forceinline__ float fade(float g, float power, float take) {
  const float keep = power * take;
  if (kAny && !finite(g)) return keep * g;
  float r;
  asm("{\n .reg .pred near;\n setp.gt.f32 near, %1, 0f3F800000;\n @near fma.rn.f32 %0, %2, %4, %4;\n @!near mul.rn.f32 %0, %3, %4;\n}"
      : "=f"(r) : "f"(power), "f"(-take), "f"(keep), "f"(g));
  return r;
}
template <bool kAny, int V> __device__ __forceinline__ Row<V> follow(const Row<V>& h, const Row<V>& x, const Row<V>& power, const Row<V>& take) {
  Row<V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.f[i] = follow<kAny>(h.f[i], x.f[i], power.f[i], take.f[i]);
  return r;
}
template <bool kAny, int V> __device__ __forceinline__ Row<V> fade(const Row<V>& g, const Row<V>& power, const Row<V>& take) {
  Row<V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.f[i] = fade<kAny>(g.f[i], power.f[i], take.f[i]);
  return r;
}
// of the first `count` channels (the ring holds anything for those that are not there)
template <int V> __device__ __forceinline__ bool finite(const Row<V>& r, int count) {
  bool all = true;
#pragma unroll
  for (int i = 0; i < V; ++i) all = all && (i >= count || finite(r.f[i]));
  return all;
}
// What a run of rows does to the state in front of it: h -> a h + b, or h -> b where a sequence starts within (a is then -0: a state of the sequence
// before, infinite or NaN as it may be, is not multiplied with).  For the same reason as above it knows 1 - a too, and for an a of a half or more goes by that.
struct Run { float a, lost, b; };                // lost: 1 - a
__device__ __forceinline__ float apply(Run r, float h) {
  if (signbit(r.a)) h = 0.f;
  const bool near = r.lost <= 0.5f && finite(h);
  return fmaf(near ? -r.lost : r.a, h, r.b) + (near ? h : 0.f);
}
__device__ __forceinline__ Run join(Run first, Run then) {
  return {signbit(then.a) ? then.a : then.a * first.a, fmaf(then.lost, 1.f - first.lost, first.lost), apply(then, first.b)};
}
__device__ __forceinline__ Run nothing() { return {1.f, 0.f, 0.f}; }
// a and 1 - a in one number: a start, -(1 - a), or a
constexpr float kStarts = 2.f;
__device__ __forceinline__ float factor_of(Run r) { return signbit(r.a) ? kStarts : r.lost <= 0.5f ? -r.lost : r.a; }
__device__ __forceinline__ Run run_of(float factor, float b) {
  if (factor == kStarts) return {-0.f, 1.f, b};
  return signbit(factor) ? Run{1.f + factor, -factor, b} : Run{factor, 1.f - factor, b};
}

__device__ __forceinline__ long long offset_of(const ScanShape& p, int i) {
  if (p.offsets == nullptr) return static_cast<long long>(i) * p.length;
  return p.offsets_wide ? static_cast<const long long*>(p.offsets)[i] : static_cast<const int*>(p.offsets)[i];
}
// The sequences of neighbouring rows; -1 where a row belongs to none.  Whatever the offsets are, it is one that exists.
struct SequenceWalk {
  int i;                         // offsets[i] <= row < offsets[i + 1]
  long long first, behind;
  __device__ __forceinline__ void bounds(const ScanShape& p) {
    first = i < 0 ? -(1ll << 60) : offset_of(p, i);
    behind = i >= p.sequences ? 1ll << 60 : offset_of(p, i + 1);
  }
  __device__ __forceinline__ SequenceWalk(const ScanShape& p, int t) {
    int lo = -1, hi = p.sequences + 1;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (offset_of(p, mid) <= t) lo = mid; else hi = mid;
    }
    i = lo;
    bounds(p);
  }
  __device__ __forceinline__ int at(const ScanShape& p, int t) {
    while (t >= behind && i < p.sequences) { ++i; bounds(p); }
    while (t < first && i >= 0) { --i; bounds(p); }
    return t >= 0 && t < p.rows && i >= 0 && i < p.sequences ? i : -1;
  }
  // Whether rows [t, end) and the one before them, where the walk stands, are of one sequence.
  __device__ __forceinline__ bool all_within(const ScanShape& p, int end) const { return i >= 0 && i < p.sequences && end <= behind && end <= p.rows; }
};
// Of a packed batch: whether all rows from `before` to `end` are of one sequence.  Then nothing starts or ends among them, which saves the rows' own
// looks (7488 rows of 1001 fp32 channels in 9 sequences, forward and backward, 252 -> 131 us).
__device__ __forceinline__ bool within_one(const ScanShape& p, int before, int end) {
  if (before < 0) return false;
  SequenceWalk walk(p, before);
  return walk.at(p, before) >= 0 && walk.all_within(p, end);
}

// The same for all segments of a warp: one that looks at each row makes the others wait for it, so that then all do (7488 rows of 1000 fp32 channels in 9
// sequences, forward and backward, 129 -> 103 us of kernels).
template <class Seg> __device__ __forceinline__ bool all_plain(const ScanShape& p, const Seg& seg, int before, int end) {
  return p.offsets == nullptr || __all_sync(0xffffffffu, !seg.there || within_one(p, before, end));
}

// A block's threads: LANES side by side across the channels, V channels each, and SEGS segments above one another.  Where runs are joined, PARTS
// threads share a channel.  A thread's channels are one vector; or with kApart, where rows do not begin on boundaries of vectors, every 32nd: a warp then
// reads and writes neighbouring numbers, and still has V of them for each row that it counts off (7488 rows of 1001 fp32 channels with gradients 131 us
// one by one, 115 so).
template <int Vec, bool kApart> struct Tile {
  static constexpr int V = Vec;
  static constexpr bool kStrided = kApart;
  static constexpr int LANES = !kApart && V >= 4 ? 8 : 32;
  static constexpr int COLS = LANES * V;
  static constexpr int SEGS = kScanThreads / LANES;
  static constexpr int PARTS = kScanThreads / COLS;
  static_assert(SEGS % PARTS == 0, "parts of equal length");
  // of channel i of the thread `side`: its place in the tile, and its distance to the thread's first one
  __device__ __forceinline__ static constexpr int place(int side, int i) { return kApart ? side + i * 32 : side * V + i; }
  __device__ __forceinline__ static constexpr int apart(int i) { return kApart ? i * 32 : i; }
  // V numbers from a thread's first one on, of which `count` are there
  __device__ __forceinline__ static Row<V> load(const float* at, int count) {
    if constexpr (!kApart) {
      return load_state<V>(at);
    } else {
      Row<V> r;
#pragma unroll
      for (int i = 0; i < V; ++i) r.f[i] = i < count ? at[apart(i)] : 0.f;
      return r;
    }
  }
  __device__ __forceinline__ static void store(float* at, const Row<V>& r, int count) {
    if constexpr (!kApart) {
      store_state<V>(at, r);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) if (i < count) at[apart(i)] = r.f[i];
    }
  }
  template <class T> __device__ __forceinline__ static void store_rounded(T* at, const Row<V>& r, int count) {
    if constexpr (!kApart) {
      store_row<T, V>(at, r);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) if (i < count) at[apart(i)] = from_float<T>(r.f[i]);
    }
  }
};

// What a thread works on: V channels from `col` on, and rows [first, last) of a segment.  `order` counts segments from where the recurrence starts:
// the first one, or with kBack the last one.
template <class Tl, bool kBack>
struct Segment {
  int order, index, sequence, part, col, count, first, last;
  bool there;
  __device__ __forceinline__ Segment(const ScanShape& p, const ScanSplit& s, int block, int tile) {
    order = block * Tl::SEGS + static_cast<int>(threadIdx.x) / Tl::LANES;
    col = tile * Tl::COLS + Tl::place(static_cast<int>(threadIdx.x) % Tl::LANES, 0);
    count = Tl::kStrided ? min(Tl::V, (p.channels - col + 31) / 32) : Tl::V;     // of the V channels, those that there are
    there = order < s.segments && col < p.channels;
    index = kBack ? s.segments - 1 - order : order;
    sequence = index / s.parts;
    part = index - sequence * s.parts;
    if (order >= s.segments) { first = last = 0; return; }
    const int base = p.offsets == nullptr ? sequence * p.length : 0, end = p.offsets == nullptr ? base + p.length : p.rows;
    first = min(base + part * s.rows, end);
    last = min(first + s.rows, end);
  }
};

// Rows that are on their way while one is worked on: in places of the thread's own in shared memory, filled by asynchronous copies (nobody waits for
// anybody else's).  Five of two arrays, three of four: more rows leave fewer blocks (8 and 5: 40.8 -> 45 us, 58.6 -> 64 for 8192 rows of 2048
// channels).  bf16 channels taken one by one, 2 bytes, come through registers.
template <class T, class Tl> constexpr bool by_copies() { return Tl::kStrided ? sizeof(T) == 4 : Tl::V * sizeof(T) >= 4; }
template <class T, class Tl, int kArrays> constexpr int rows_ahead() {
  return !by_copies<T, Tl>() ? 8 / kArrays : Tl::V * sizeof(T) == 16 ? (kArrays == 2 ? 5 : 3) : 8;
}
template <class T, class Tl, int kArrays> constexpr int ring_bytes() {
  return by_copies<T, Tl>() ? rows_ahead<T, Tl, kArrays>() * kArrays * kScanThreads * Tl::V * static_cast<int>(sizeof(T)) : 0;
}
template <int kBytes> __device__ __forceinline__ void copy_ahead(uint32_t to, const void* from) {
  if constexpr (kBytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(to), "l"(from) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" :: "r"(to), "l"(from) : "memory");
}

// Walks the rows of a segment, backwards from its last one with kBack: f(t, row t of the arrays).
template <class T, class Tl, bool kBack, int kArrays, class F>
__device__ __forceinline__ void walk_rows(const Segment<Tl, kBack>& seg, int first, const T* (&base)[kArrays], const long long (&stride)[kArrays], F f) {
  constexpr int V = Tl::V, U = rows_ahead<T, Tl, kArrays>(), kBytes = V * sizeof(T);
  const int last = seg.last, n = last - first;
  const T* next[kArrays];
#pragma unroll
  for (int a = 0; a < kArrays; ++a) next[a] = base[a] + (kBack ? last - 1 : first) * stride[a];
  auto advance = [&] {
#pragma unroll
    for (int a = 0; a < kArrays; ++a) next[a] += kBack ? -stride[a] : stride[a];
  };
  if constexpr (by_copies<T, Tl>()) {
    extern __shared__ __align__(16) unsigned char ring[];
    // (a loop over single rows: unrolled over the ring, its code no longer fits the SM's nearest instruction cache)
    constexpr int kRow = kArrays * kScanThreads * kBytes;
    unsigned char* const mine = ring + threadIdx.x * kBytes;
    auto fetch = [&](unsigned char* to, bool there) {
      if (there) {
#pragma unroll
        for (int a = 0; a < kArrays; ++a) {
          const uint32_t place = smem_u32(to + a * kScanThreads * kBytes);
          if constexpr (Tl::kStrided) {
#pragma unroll
            for (int i = 0; i < V; ++i) if (i < seg.count) copy_ahead<4>(place + i * 4, next[a] + Tl::apart(i));
          } else {
            copy_ahead<kBytes>(place, next[a]);
          }
        }
        advance();
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for (int u = 0; u < U; ++u) fetch(mine + u * kRow, u < n);
    int slot = 0;
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      unsigned char* const at = mine + slot;
      slot = slot == (U - 1) * kRow ? 0 : slot + kRow;
      asm volatile("cp.async.wait_group %0;" :: "n"(U - 1) : "memory");
      Raw<T, V> row[kArrays];
#pragma unroll
      for (int a = 0; a < kArrays; ++a) row[a].load(reinterpret_cast<const T*>(at + a * kScanThreads * kBytes));
      fetch(at, i + U < n);
      f(kBack ? last - 1 - i : first + i, row);
    }
  } else {
    Raw<T, V> now[U][kArrays], ahead[U][kArrays];
    auto fetch = [&](Raw<T, V> (&to)[U][kArrays], int i0) {
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + u < n) {
#pragma unroll
          for (int a = 0; a < kArrays; ++a) to[u][a].gather(next[a], Tl::apart(1), seg.count);
          advance();
        }
    };
    fetch(now, 0);
    for (int i0 = 0; i0 < n; i0 += U) {
      fetch(ahead, i0 + U);
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + u < n) f(kBack ? last - 1 - (i0 + u) : first + i0 + u, now[u]);
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int a = 0; a < kArrays; ++a) now[u][a] = ahead[u][a];
    }
  }
}

// What the rows of a segment do to the state in front of them.  All threads call.  `rows`: x, or the rows' own gradients (which may be left out).
template <class T, class Tl, bool kBack>
__device__ __forceinline__ void run_of_segment(const ScanShape& p, const ScanSplit& s, const Segment<Tl, kBack>& seg, const void* rows, long long rows_stride, const float* edge,
                                               Run (&run)[Tl::V]) {
  constexpr int V = Tl::V;
  Row<V> a = Row<V>::all(1.f), lost = Row<V>::all(0.f), b = Row<V>::all(0.f);    // lost: 1 - a
  bool starts = false;
#pragma unroll
  for (int i = 0; i < V; ++i) run[i] = nothing();
  const bool plain = all_plain(p, seg, kBack ? seg.first : seg.first - 1, kBack ? seg.last + 1 : seg.last);
  if (!seg.there || seg.first >= seg.last) return;
  auto begin = [&](int sequence) {
    starts = true;
    b = edge != nullptr && sequence >= 0 ? Tl::load(edge + static_cast<long long>(sequence) * p.channels + seg.col, seg.count) : Row<V>::all(0.f);
  };
  const bool none = kBack && rows == nullptr;
  auto take_row = [&](const Raw<T, V> (&row)[2], auto any) {
    constexpr bool kAny = decltype(any)::value;
    Row<V> power, take;
    gates_of<T, V>(row[0].get(), power, take);
    lost = fused(take, a, lost);
    a = fade<false>(a, power, take);
    if constexpr (kBack) b = fade<kAny>(none ? b : b + row[1].get(), power, take); else b = follow<kAny>(b, row[1].get(), power, take);
  };
  const T* base[2] = {static_cast<const T*>(p.gate) + seg.col, static_cast<const T*>(none ? p.gate : rows) + seg.col};
  const long long stride[2] = {p.gate_stride, none ? p.gate_stride : rows_stride};
  bool bad = false;              // a number that is not finite was met
  auto sequences = [&](auto any) {
    SequenceWalk walk(p, kBack ? seg.last : seg.first - 1);
    int previous = walk.at(p, kBack ? seg.last : seg.first - 1);
    walk_rows<T, Tl, kBack, 2>(seg, seg.first, base, stride, [&](int t, Raw<T, V> (&row)[2]) {
      const int sequence = walk.at(p, t);
      if (sequence != previous || sequence < 0) { bad = bad || !finite(b, seg.count); begin(sequence); }
      if (sequence >= 0) take_row(row, any);
      previous = sequence;
    });
  };
  if (plain) {
    if (p.offsets == nullptr && seg.part == (kBack ? s.parts - 1 : 0)) begin(seg.sequence);
    walk_rows<T, Tl, kBack, 2>(seg, seg.first, base, stride, [&](int, Raw<T, V> (&row)[2]) { take_row(row, std::false_type{}); });
  } else {
    sequences(std::false_type{});
  }
  if (bad || !finite(b, seg.count)) {
    a = Row<V>::all(1.f); lost = b = Row<V>::all(0.f);
    starts = false;
    sequences(std::true_type{});
  }
#pragma unroll
  for (int i = 0; i < V; ++i) run[i] = starts ? Run{-0.f, 1.f, b.f[i]} : Run{a.f[i], lost.f[i], b.f[i]};
}

// From the runs of a block's segments: of those before each thread's own.  All threads call; the ring is not in use.
template <class Tl>
__device__ __forceinline__ void runs_before(const Run (&own)[Tl::V], Run (&before)[Tl::V]) {
  constexpr int V = Tl::V;
  extern __shared__ __align__(16) unsigned char ring[];
  Run* runs = reinterpret_cast<Run*>(ring);                    // [SEGS][COLS]
  __shared__ Run parts[Tl::PARTS][Tl::COLS];
  const int seg = threadIdx.x / Tl::LANES, side = threadIdx.x % Tl::LANES;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < V; ++i) runs[seg * Tl::COLS + Tl::place(side, i)] = own[i];
  __syncthreads();
  const int ch = threadIdx.x % Tl::COLS, part = threadIdx.x / Tl::COLS;
  constexpr int kEach = Tl::SEGS / Tl::PARTS;
  Run run = nothing();
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    Run* at = runs + (part * kEach + i) * Tl::COLS + ch;
    const Run r = *at;
    *at = run;
    run = i == 0 ? r : join(run, r);
  }
  parts[part][ch] = run;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < V; ++i) {
    run = nothing();
#pragma unroll
    for (int q = 0; q < Tl::PARTS - 1; ++q)
      if (q < seg / kEach) run = q == 0 ? parts[q][Tl::place(side, i)] : join(run, parts[q][Tl::place(side, i)]);
    before[i] = join(run, runs[seg * Tl::COLS + Tl::place(side, i)]);
  }
  __syncthreads();               // the ring may be filled again
}

// Leaves, of every segment, the run of the segments before it in its block; and of every block the run of all.
template <class T, class Tl, bool kBack>
__global__ void __launch_bounds__(kScanThreads, kScanBlocks) scan_runs_kernel(const ScanShape p, const ScanSplit s, const void* rows, long long rows_stride, const float* edge) {
  constexpr int V = Tl::V;
  grid_release();
  const int block = blockIdx.x / s.tiles, tile = blockIdx.x - block * s.tiles;
  const Segment<Tl, kBack> seg(p, s, block, tile);
  Run run[V], before[V];
  run_of_segment<T, Tl, kBack>(p, s, seg, rows, rows_stride, edge, run);
  runs_before<Tl>(run, before);
  if (!seg.there) return;
  float fa[V], fb[V];
  const long long at = static_cast<long long>(seg.order) * p.channels + seg.col;
#pragma unroll
  for (int i = 0; i < V; ++i) { fa[i] = factor_of(before[i]); fb[i] = before[i].b; }
  Tl::store(s.factors + at, Row<V>::of(fa), seg.count);
  Tl::store(s.sums + at, Row<V>::of(fb), seg.count);
  if (seg.order % Tl::SEGS != Tl::SEGS - 1) return;            // (nobody follows a block that is not full)
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const Run r = join(before[i], run[i]);
    fa[i] = factor_of(r); fb[i] = r.b;
  }
  const long long block_at = static_cast<long long>(block) * p.channels + seg.col;
  Tl::store(s.block_factors + block_at, Row<V>::of(fa), seg.count);
  Tl::store(s.block_sums + block_at, Row<V>::of(fb), seg.count);
}

// The state in front of each thread's segment.  All threads call.
template <class T, class Tl, bool kBack>
__device__ __forceinline__ Row<Tl::V> state_before(const ScanShape& p, const ScanSplit& s, const Segment<Tl, kBack>& seg, int block, int tile, const void* rows, long long rows_stride,
                                               const float* edge) {
  constexpr int V = Tl::V;
  if (s.parts == 1) return Row<V>::all(0.f);
  if (s.within) {                                // no sequence goes on in another block
    Run run[V], before[V];
    run_of_segment<T, Tl, kBack>(p, s, seg, rows, rows_stride, edge, run);
    runs_before<Tl>(run, before);
    float f[V];
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = before[i].b;
    return Row<V>::of(f);
  }
  __shared__ Run parts[Tl::PARTS][Tl::COLS];
  const int ch = threadIdx.x % Tl::COLS, part = threadIdx.x / Tl::COLS, col = tile * Tl::COLS + ch;
  // the first block that the sequence of this block's first segment has a part in
  const int order0 = block * Tl::SEGS, index0 = kBack ? s.segments - 1 - order0 : order0;
  int from = block;
  if (p.offsets == nullptr) {
    const int sequence = index0 / s.parts;
    from = (kBack ? s.segments - (sequence + 1) * s.parts : sequence * s.parts) / Tl::SEGS;
  } else {
    const int edge_row = kBack ? min(index0 * s.rows + s.rows, p.rows) : index0 * s.rows;      // the rows on both sides of it: of one sequence?
    SequenceWalk walk(p, edge_row - 1);
    const int i = walk.at(p, edge_row - 1);
    if (i >= 0 && walk.all_within(p, edge_row + 1)) {
      const long long far = kBack ? min(max(walk.behind, 1ll), static_cast<long long>(p.rows)) - 1 : max(walk.first, 0ll);
      const int segment = static_cast<int>(far / s.rows);
      from = (kBack ? s.segments - 1 - segment : segment) / Tl::SEGS;
    }
  }
  const int n = max(block - from, 0), begin = from + n * part / Tl::PARTS, end = from + n * (part + 1) / Tl::PARTS;
  Run run = nothing();
  if (col < p.channels) {
#pragma unroll 8
    for (int k = begin; k < end; ++k) {
      const long long at = static_cast<long long>(k) * p.channels + col;
      run = join(run, run_of(s.block_factors[at], s.block_sums[at]));
    }
  }
  parts[part][ch] = run;
  __syncthreads();
  if (!seg.there) return Row<V>::all(0.f);
  const int side = threadIdx.x % Tl::LANES;
  const long long at = static_cast<long long>(seg.order) * p.channels + seg.col;
  float fa[V], fb[V], f[V];
  Tl::load(s.factors + at, seg.count).get(fa);
  Tl::load(s.sums + at, seg.count).get(fb);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float state = parts[0][Tl::place(side, i)].b;
#pragma unroll
    for (int q = 1; q < Tl::PARTS; ++q) state = apply(parts[q][Tl::place(side, i)], state);
    f[i] = apply(run_of(fa[i], fb[i]), state);
  }
  return Row<V>::of(f);
}

// Sequences without rows hand their state on (`from` to `to`); offsets that are none are reported.
template <class Tl>
__device__ __forceinline__ void empty_sequences(const ScanShape& p, const float* from, float* to, bool report) {
  if (p.offsets == nullptr && p.length > 0) return;
  constexpr int V = Tl::kStrided ? 1 : Tl::V;
  const int vectors = p.channels / V;
  const long long all = static_cast<long long>(p.sequences) * vectors;
  for (long long i = static_cast<long long>(blockIdx.x) * kScanThreads + threadIdx.x; i < all; i += static_cast<long long>(gridDim.x) * kScanThreads) {
    const int s = static_cast<int>(i / vectors), vector = static_cast<int>(i - static_cast<long long>(s) * vectors);
    const long long a = p.offsets != nullptr ? offset_of(p, s) : 0, b = p.offsets != nullptr ? offset_of(p, s + 1) : 0;
    if (a < 0 || b < a || b > p.rows) {
      if (report && vector == 0)
        report_note(p.status, kStatusBadOffsets, kKernelScan, 0, p.rank, s, static_cast<int>(min(max(a, -1ll << 31), (1ll << 31) - 1)),
                    static_cast<int>(min(max(b, -1ll << 31), (1ll << 31) - 1)));
      continue;
    }
    if (a != b || to == nullptr) continue;
    const long long at = static_cast<long long>(s) * p.channels + vector * V;
    store_state<V>(to + at, from != nullptr ? load_state<V>(from + at) : Row<V>::all(0.f));
  }
}

template <class T, class Tl>
__global__ void __launch_bounds__(kScanThreads, kScanBlocks) scan_forward_kernel(const ScanParams p, const ScanSplit s) {
  constexpr int V = Tl::V;
  grid_wait();
  empty_sequences<Tl>(p, p.initial, p.final_state, true);
  // (from the last block: what was read last is still in L2)
  const int unit = gridDim.x - 1 - blockIdx.x, block = unit / s.tiles, tile = unit - block * s.tiles;
  const Segment<Tl, false> seg(p, s, block, tile);
  Row<V> h = state_before<T, Tl, false>(p, s, seg, block, tile, p.x, p.x_stride, p.initial);
  const bool plain = all_plain(p, seg, seg.first - 1, seg.last + 1);
  if (!seg.there || seg.first >= seg.last) return;
  auto state_at = [&](int sequence) { return static_cast<long long>(sequence) * p.channels + seg.col; };
  auto begin = [&](int sequence) { h = p.initial != nullptr ? Tl::load(p.initial + state_at(sequence), seg.count) : Row<V>::all(0.f); };
  auto step = [&](const Raw<T, V> (&row)[2], auto any) {
    Row<V> power, take;
    gates_of<T, V>(row[0].get(), power, take);
    h = follow<decltype(any)::value>(h, row[1].get(), power, take);
  };
  const T* base[2] = {static_cast<const T*>(p.gate) + seg.col, static_cast<const T*>(p.x) + seg.col};
  const long long stride[2] = {p.gate_stride, p.x_stride};
  T* out = static_cast<T*>(p.h) + seg.col;
  const Row<V> before = h;
  bool bad = false;              // a number that is not finite was met
  auto sequences = [&](auto any) {
    SequenceWalk walk(p, seg.first - 1);
    int previous = walk.at(p, seg.first - 1), sequence = walk.at(p, seg.first);
    walk_rows<T, Tl, false, 2>(seg, seg.first, base, stride, [&](int t, Raw<T, V> (&row)[2]) {
      const int behind = walk.at(p, t + 1);
      if (sequence != previous || sequence < 0) { bad = bad || !finite(h, seg.count); h = Row<V>::all(0.f); }
      if (sequence >= 0) {
        if (sequence != previous) begin(sequence);
        step(row, any);
        if (p.final_state != nullptr && behind != sequence) Tl::store(p.final_state + state_at(sequence), h, seg.count);
      }
      Tl::template store_rounded<T>(out + static_cast<long long>(t) * p.channels, h, seg.count);
      previous = sequence;
      sequence = behind;
    });
  };
  if (plain) {
    const bool dense = p.offsets == nullptr;
    if (dense && seg.part == 0) begin(seg.sequence);
    walk_rows<T, Tl, false, 2>(seg, seg.first, base, stride, [&](int t, Raw<T, V> (&row)[2]) {
      step(row, std::false_type{});
      Tl::template store_rounded<T>(out + static_cast<long long>(t) * p.channels, h, seg.count);
    });
    if (dense && p.final_state != nullptr && seg.last == (seg.sequence + 1) * p.length) Tl::store(p.final_state + state_at(seg.sequence), h, seg.count);
  } else {
    sequences(std::false_type{});
  }
  if (bad || !finite(h, seg.count)) {       // again, all of it
    h = before;
    sequences(std::true_type{});
  }
}

// kGate: with the gate's gradient, for which x and h of the row before are read too: h as it was returned, for bf16 rounded by up to 2^-8 of itself (against 64 bits
// dgate of 8192 rows of 2048 is 1.8e-3 off in 2-norm, where its own rounding is 1.7e-3).  Its fp32 values would be a third array more to write and read; the state that is
// carried on, and the gradient that is carried back, are fp32.
template <class T, class Tl, bool kGate>
__global__ void __launch_bounds__(kScanThreads, 6) scan_backward_kernel(const ScanGradParams p, const ScanSplit s) {
  constexpr int V = Tl::V;
  grid_wait();
  empty_sequences<Tl>(p, p.dfinal, p.dinitial, false);
  const int unit = gridDim.x - 1 - blockIdx.x, block = unit / s.tiles, tile = unit - block * s.tiles;
  const Segment<Tl, true> seg(p, s, block, tile);
  Row<V> back = state_before<T, Tl, true>(p, s, seg, block, tile, p.dh, p.dh_stride, p.dfinal);     // keep_{t+1} g_{t+1}
  const bool plain = all_plain(p, seg, seg.first - 1, seg.last + 1);
  if (!seg.there || seg.first >= seg.last) return;
  auto state_at = [&](int sequence) { return static_cast<long long>(sequence) * p.channels + seg.col; };
  const bool none = p.dh == nullptr;
  // one row, whose state before is h
  auto step = [&](auto any, int t, const Row<V>& gate, const Row<V>& dh, const Row<V>& x, const Row<V>& h) {
    Row<V> power, take;
    gates_of<T, V>(gate, power, take);
    const Row<V> g = none ? back : back + dh;
    const long long at = static_cast<long long>(t) * p.channels + seg.col;
    if (p.dx != nullptr) Tl::template store_rounded<T>(static_cast<T*>(p.dx) + at, take * g, seg.count);
    if constexpr (kGate) Tl::template store_rounded<T>(static_cast<T*>(p.dgate) + at, g * (power * take * take) * fused(Row<V>::all(-1.f), x, h), seg.count);
    back = fade<decltype(any)::value>(g, power, take);
  };
  auto outside = [&](int t) {
    const long long at = static_cast<long long>(t) * p.channels + seg.col;
    if (p.dx != nullptr) Tl::template store_rounded<T>(static_cast<T*>(p.dx) + at, Row<V>::all(0.f), seg.count);
    if constexpr (kGate) Tl::template store_rounded<T>(static_cast<T*>(p.dgate) + at, Row<V>::all(0.f), seg.count);
    back = Row<V>::all(0.f);
  };
  auto begin = [&](int sequence) { back = p.dfinal != nullptr ? Tl::load(p.dfinal + state_at(sequence), seg.count) : Row<V>::all(0.f); };
  auto initial = [&](int sequence) { return p.initial != nullptr ? Tl::load(p.initial + state_at(sequence), seg.count) : Row<V>::all(0.f); };

  constexpr int kArrays = kGate ? 4 : 2;
  const T* gate = static_cast<const T*>(p.gate) + seg.col;
  const T* dh = none ? gate : static_cast<const T*>(p.dh) + seg.col;
  const T *base[kArrays];
  long long stride[kArrays];
  base[0] = gate; base[1] = dh; stride[0] = p.gate_stride; stride[1] = none ? p.gate_stride : p.dh_stride;
  // The state before a row is the row before's result; before the first row of all nothing lies, and the walk must not look there.
  int first = seg.first;
  if constexpr (kGate) {
    base[2] = static_cast<const T*>(p.x) + seg.col; stride[2] = p.x_stride;
    base[3] = static_cast<const T*>(p.h) + seg.col - p.channels; stride[3] = p.channels;
    if (first == 0) first = 1;
  }
  const Row<V> zero = Row<V>::all(0.f);
  auto zeroth = [&](auto any, const Row<V>& h) {           // row 0, where it was left out of the walk
    Raw<T, V> g, d, x;
    auto load = [&](Raw<T, V>& to, const T* from) {
      if constexpr (Tl::kStrided) to.gather(from, Tl::apart(1), seg.count); else to.load(from);
    };
    load(g, base[0]); load(d, base[1]);
    if constexpr (kGate) load(x, base[2]); else x = g;
    step(any, 0, g.get(), d.get(), x.get(), h);
  };
  const Row<V> beyond = back;
  bool bad = false;              // a number that is not finite was met
  auto sequences = [&](auto any) {
    SequenceWalk walk(p, seg.last);
    int behind = walk.at(p, seg.last), sequence = walk.at(p, seg.last - 1);
    auto row_of = [&](int t, auto calculate) {
      const int previous = walk.at(p, t - 1);
      if (sequence != behind || sequence < 0) bad = bad || !finite(back, seg.count);
      if (sequence >= 0) {
        if (sequence != behind) begin(sequence);
        calculate(sequence != previous);
        if (sequence != previous && p.dinitial != nullptr) Tl::store(p.dinitial + state_at(sequence), back, seg.count);
      } else {
        outside(t);
      }
      behind = sequence;
      sequence = previous;
    };
    walk_rows<T, Tl, true, kArrays>(seg, first, base, stride, [&](int t, Raw<T, V> (&row)[kArrays]) {
      row_of(t, [&](bool start) {
        if constexpr (kGate) step(any, t, row[0].get(), row[1].get(), row[2].get(), start ? initial(sequence) : row[3].get());
        else step(any, t, row[0].get(), row[1].get(), zero, zero);
      });
    });
    if (first > seg.first) row_of(0, [&](bool) { zeroth(any, initial(sequence)); });
  };
  if (plain) {
    constexpr std::false_type kAny{};
    const bool dense = p.offsets == nullptr;
    if (dense && seg.part == s.parts - 1) begin(seg.sequence);
    const int start = dense ? seg.sequence * p.length : -1;
    walk_rows<T, Tl, true, kArrays>(seg, first, base, stride, [&](int t, Raw<T, V> (&row)[kArrays]) {
      if constexpr (kGate) step(kAny, t, row[0].get(), row[1].get(), row[2].get(), t == start ? initial(seg.sequence) : row[3].get());
      else step(kAny, t, row[0].get(), row[1].get(), zero, zero);
    });
    if (first > seg.first) zeroth(kAny, initial(0));
    if (dense && seg.first == start && p.dinitial != nullptr) Tl::store(p.dinitial + state_at(seg.sequence), back, seg.count);
  } else {
    sequences(std::false_type{});
  }
  if (bad || !finite(back, seg.count)) {    // again, all of it
    back = beyond;
    sequences(std::true_type{});
  }
}

template <class T, int V>
__global__ void __launch_bounds__(kScanThreads) scan_step_kernel(const ScanStepParams p) {
  const int vectors = p.channels / V;
  const long long i = static_cast<long long>(blockIdx.x) * kScanThreads + threadIdx.x, row = i / vectors;
  if (row >= p.rows) return;
  const int col = static_cast<int>(i - row * vectors) * V;
  Raw<T, V> gate, x;
  gate.load(static_cast<const T*>(p.gate) + row * p.gate_stride + col);
  x.load(static_cast<const T*>(p.x) + row * p.x_stride + col);
  float* state = p.state + row * p.state_stride + col;
  Row<V> power, take;
  gates_of<T, V>(gate.get(), power, take);
  const Row<V> h = follow<true>(load_state<V>(state), x.get(), power, take);
  store_state<V>(state, h);
  store_row<T, V>(static_cast<T*>(p.h) + row * p.channels + col, h);
}

// Channels a thread takes at a time: 16 bytes, or 4, or one, as all rows allow it.
int vector_of(int half, int channels, std::initializer_list<std::pair<const void*, long long>> arrays, std::initializer_list<const void*> states) {
  auto fits = [&](int bytes) {
    const int v = bytes / (half ? 2 : 4);
    if (channels % v != 0) return false;
    for (const auto& a : arrays)
      if (reinterpret_cast<uintptr_t>(a.first) % bytes != 0 || (a.first != nullptr && a.second % v != 0)) return false;
    for (const void* q : states)
      if (reinterpret_cast<uintptr_t>(q) % (v >= 4 ? 16 : v * 4) != 0) return false;
    return true;
  };
  if (fits(16)) return half ? 8 : 4;
  return half && fits(4) ? 2 : 1;
}
int vector_of(const ScanParams& p) { return vector_of(p.half, p.channels, {{p.gate, p.gate_stride}, {p.x, p.x_stride}}, {p.initial}); }
int vector_of(const ScanGradParams& p) {
  return vector_of(p.half, p.channels, {{p.gate, p.gate_stride}, {p.x, p.x_stride}, {p.dh, p.dh_stride}}, {p.initial, p.dfinal});
}
template <class F>
cudaError_t by_tile(int half, int vec, F f) {
  if (half) {
    if (vec == 8) return f(__nv_bfloat16{}, Tile<8, false>{});
    if (vec == 2) return f(__nv_bfloat16{}, Tile<2, false>{});
    return f(__nv_bfloat16{}, Tile<4, true>{});
  }
  if (vec == 4) return f(float{}, Tile<4, false>{});
  return f(float{}, Tile<4, true>{});
}

ScanSplit split_of(const ScanShape& p, int vec, int sms, bool back) {
  ScanSplit s{};
  const long long sequences = p.offsets == nullptr ? p.sequences : 1, length = p.offsets == nullptr ? p.length : p.rows;
  const int lanes = vec >= 4 ? 8 : 32, segs = kScanThreads / lanes, cols = lanes * (vec == 1 ? 4 : vec);
  s.tiles = (p.channels + cols - 1) / cols;
  const long long vectors = static_cast<long long>(s.tiles) * lanes;
  // Threads that are enough to keep memory busy, and 16 to 32 rows a segment at least.  One sequence of 131072 rows of 1024 channels, with 384 and 1200 vectors of 16
  // bytes an SM: forward 232 and 260 us, backward 470 and 396.
  const long long enough = static_cast<long long>(sms) * (vec == 2 ? 1536 : vec == 1 ? 768 : back ? 1200 : 384);
  long long parts = 1;
  // (bf16 channels off the boundaries, which come through registers: 7488 rows of 1001 in 9 sequences with gradients in segments of 32 and 16 rows 174 and 136 us of kernels;
  // fp32 ones 151 and 149, as one sequence 133 and 142)
  const long long least = vec == 1 && p.half ? 16 : 32;
  while (sequences * vectors * parts < enough && length > least * parts) parts *= 2;
  // (short calls: 4096 rows of 1024 channels in segments of 32 and 16 rows forward 21.5 and 19.5 us, backward 29.7 and 25.7; 8192 rows of 2048 backward 58.6 and 65.6)
  while (sequences * vectors * parts < sms * 256ll && length > 16 * parts) parts *= 2;
  s.rows = static_cast<int>((length + parts - 1) / parts);
  if (s.rows < 1) s.rows = 1;
  s.parts = static_cast<int>(length > 0 ? (length + s.rows - 1) / s.rows : 1);
  s.segments = static_cast<int>(sequences * s.parts);
  s.blocks = (s.segments + segs - 1) / segs;
  s.within = s.blocks <= 1 || segs % s.parts == 0;
  return s;
}

template <auto kKernel, class... Args>
cudaError_t launch(dim3 grid, int smem, bool early, cudaStream_t stream, const Args&... args) {
  static std::atomic<bool> configured[64];       // the shared-memory limit is an attribute of the function on a device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (smem > 0 && !configured[dev].load(std::memory_order_acquire)) {
    if ((e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) != cudaSuccess) return e;
    // Kernels that follow each other should not want another split of the SM's memory each: changing it cost 16 us a call (4096 rows of 1024
    // channels forward 38 -> 21.5 us).
    if ((e = cudaFuncSetAttribute(kKernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared)) != cudaSuccess) return e;
    configured[dev].store(true, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kScanThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = early ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kKernel, args...);
}
void lay_out(ScanSplit& s, int channels, void* space) {
  s.factors = static_cast<float*>(space);
  s.sums = s.factors + static_cast<long long>(s.segments) * channels;
  s.block_factors = s.sums + static_cast<long long>(s.segments) * channels;
  s.block_sums = s.block_factors + static_cast<long long>(s.blocks) * channels;
}
// Blocks of the walks: their ring, or the runs in its place.
template <class T, class Tl, int kArrays> constexpr int walk_bytes() {
  return std::max(ring_bytes<T, Tl, kArrays>(), Tl::SEGS * Tl::COLS * static_cast<int>(sizeof(Run)));
}

}  // namespace

ScanSplit scan_split(const ScanParams& p, int sms) { return split_of(p, vector_of(p), sms, false); }
ScanSplit scan_split(const ScanGradParams& p, int sms) { return split_of(p, vector_of(p), sms, true); }
long long scan_space(const ScanSplit& s, int channels) { return s.within ? 0 : 8ll * (static_cast<long long>(s.segments) + s.blocks) * channels; }

cudaError_t launch_scan_forward(const ScanParams& p, ScanSplit s, void* space, cudaStream_t stream) {
  return by_tile(p.half, vector_of(p), [&](auto type, auto tile) {
    using T = decltype(type);
    using Tl = decltype(tile);
    constexpr int smem = walk_bytes<T, Tl, 2>();
    const dim3 grid(static_cast<unsigned>(std::max(1, s.blocks * s.tiles)));
    if (!s.within) {
      lay_out(s, p.channels, space);
      const cudaError_t e = launch<scan_runs_kernel<T, Tl, false>>(grid, smem, false, stream, static_cast<const ScanShape&>(p), s, p.x, p.x_stride, p.initial);
      if (e != cudaSuccess) return e;
    }
    return launch<scan_forward_kernel<T, Tl>>(grid, smem, !s.within, stream, p, s);
  });
}

cudaError_t launch_scan_backward(const ScanGradParams& p, ScanSplit s, void* space, cudaStream_t stream) {
  return by_tile(p.half, vector_of(p), [&](auto type, auto tile) {
    using T = decltype(type);
    using Tl = decltype(tile);
    constexpr int smem = walk_bytes<T, Tl, 2>();
    const dim3 grid(static_cast<unsigned>(std::max(1, s.blocks * s.tiles)));
    if (!s.within) {
      lay_out(s, p.channels, space);
      const cudaError_t e = launch<scan_runs_kernel<T, Tl, true>>(grid, smem, false, stream, static_cast<const ScanShape&>(p), s, p.dh, p.dh_stride, p.dfinal);
      if (e != cudaSuccess) return e;
    }
    if (p.dgate == nullptr) return launch<scan_backward_kernel<T, Tl, false>>(grid, smem, !s.within, stream, p, s);
    return launch<scan_backward_kernel<T, Tl, true>>(grid, walk_bytes<T, Tl, 4>(), !s.within, stream, p, s);
  });
}

cudaError_t launch_scan_step(const ScanStepParams& p, cudaStream_t stream) {
  const int vec = vector_of(p.half, p.channels, {{p.gate, p.gate_stride}, {p.x, p.x_stride}, {nullptr, 0}}, {p.state, reinterpret_cast<const void*>(p.state_stride * 4)});
  const long long threads = static_cast<long long>(p.rows) * (p.channels / vec);
  const dim3 grid(static_cast<unsigned>((threads + kScanThreads - 1) / kScanThreads));
  if (!p.half) return vec == 4 ? launch<scan_step_kernel<float, 4>>(grid, 0, false, stream, p) : launch<scan_step_kernel<float, 1>>(grid, 0, false, stream, p);
  if (vec == 8) return launch<scan_step_kernel<__nv_bfloat16, 8>>(grid, 0, false, stream, p);
  return vec == 2 ? launch<scan_step_kernel<__nv_bfloat16, 2>>(grid, 0, false, stream, p) : launch<scan_step_kernel<__nv_bfloat16, 1>>(grid, 0, false, stream, p);
}

}  // namespace sep

// Normalisation of rows, with the residual stream added on the way, and its gradients.
//
//   s = x + residual;  u = (s - mean s) / sqrt(var s + eps);  y = u * weight + bias        (without `center` the mean is taken as 0)
//   d = dy * weight;   dx = (d - mean d - u * mean(d u)) / deviation + dsum;  dweight = sum over rows of dy u;  dbias = sum of dy
//
// Both passes are bound by memory: x, residual, y and sum once, x, residual and three gradients once.  Rows of up to 8192 columns stay in registers: a
// group of threads holds a row, each K vectors of it, and gets the sums of the whole row over shared memory.  Blocks stay for all rows of theirs, whose
// arrays come by asynchronous copies into places of each thread's own, a row or more ahead; so the sums over rows stay in registers too, and leave
// as one row a block, which a small kernel adds up.  Longer rows are read again for each of their passes.
// All sums are fp32, in a fixed order (a repeated call gives the same bits).
#include <atomic>
#include <type_traits>

#include "norm.h"
#include "ptx.cuh"
#include "rows.cuh"

namespace sep {

namespace {

constexpr int kRowThreads = 256;                 // of a block that takes one row at a time
constexpr int kColumnThreads = 32, kColumnRows = 8;

__device__ __forceinline__ float load_weight(const void* w, int type, int i) {
  return type == kNormHalf ? __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]) : static_cast<const float*>(w)[i];
}
__device__ __forceinline__ void store_weight(void* w, int type, int i, float v) {
  if (type == kNormHalf) static_cast<__nv_bfloat16*>(w)[i] = __float2bfloat16_rn(v); else static_cast<float*>(w)[i] = v;
}

__device__ __forceinline__ float2 warp_sum(float2 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  return v;
}
// Every thread of the block gets the sums; `scratch` holds one entry a warp.
__device__ __forceinline__ float2 block_sum(float2 v, float2* scratch) {
  v = warp_sum(v);
  __syncthreads();               // the sums before these have been read
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  float2 s = make_float2(0.f, 0.f);
  for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) { s.x += scratch[w].x; s.y += scratch[w].y; }
  return s;
}

constexpr int kMostColumns = 8192;               // of rows that stay in registers: 512 threads of 16
constexpr int kGroupThreads = 256;               // of a block, where a row takes no more

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A block's threads in groups of `threads` (a multiple of 32, up to 512) for a row each; a thread takes vectors lane, lane + threads, ... of it.
struct Group {
  int threads, lane, index, count;
  __device__ __forceinline__ explicit Group(int t) : threads(t), lane(threadIdx.x % t), index(threadIdx.x / t), count(blockDim.x / t) {}
  // Every thread of a group gets its sums.  All of the block call, each time with the next of three buffers.
  template <class Sum>
  __device__ __forceinline__ Sum sum(Sum v, float2 (*scratch)[16], int& turn) const {
    v = warp_sum(v);
    if (threads == 32) return v;
    Sum* mine = reinterpret_cast<Sum*>(scratch[turn]);
    turn = turn == 2 ? 0 : turn + 1;
    if ((threadIdx.x & 31) == 0) mine[threadIdx.x >> 5] = v;
    __syncthreads();
    // (the warps' sums like a warp's: one after another they took 500 cycles a row of 14 warps)
    const int warps = threads >> 5, w = threadIdx.x & 31;
    v = Sum{};
    if (w < warps) v = mine[index * warps + w];
    return warp_sum(v);
  }
};
template <int V> __device__ __forceinline__ float across(const Row<V>& r) {
  float f[V], s = 0.f;
  r.get(f);
#pragma unroll
  for (int i = 0; i < V; ++i) s = i == 0 ? f[0] : s + f[i];
  return s;
}

// Rows that are on their way, kArrays arrays of each, some of which may be left out (null).  bf16 taken one by one, 2 bytes, come through registers.
template <class T, int V, int K, int kThreads, bool kFull, int kArrays>
struct RowsAhead {
  static constexpr bool kCopies = sizeof(T) * V >= 4;
  static constexpr int kBytes = kCopies ? sizeof(T) * V : 4;
  int ahead;                     // rows that the ring holds: 2, or 1 where two do not fit
  static constexpr int kPlane = kThreads * kBytes, kRow = kArrays * K * kPlane;        // bytes of a vector of all threads, of a row of the ring
  unsigned char *mine, *other;   // this thread's place in the row that is worked on, and in the one behind it
  int left;                      // this thread's vectors
  int columns;                   // between a thread's vectors
  const T* next[kArrays];        // this thread's first vector of the next row to fetch
  long long step[kArrays];

  __device__ __forceinline__ RowsAhead(int ahead, unsigned char* ring, const Group& g, int vectors) : ahead(ahead) {
    mine = ring + threadIdx.x * kBytes;
    other = ahead == 2 ? mine + kRow : mine;
    columns = g.threads * V;
    left = (vectors - g.lane + g.threads - 1) / g.threads;
  }
  __device__ __forceinline__ bool in(int k) const { return kFull || k < left; }
  __device__ __forceinline__ void turn() { unsigned char* t = mine; mine = other; other = t; }
  __device__ __forceinline__ void array(int a, const void* base, long long stride, long long first, long long rows, int column) {
    next[a] = base != nullptr ? static_cast<const T*>(base) + first * stride + column : nullptr;
    step[a] = rows * stride;
  }
  // into the row that has been worked on
  __device__ __forceinline__ void fetch(bool there) { fetch(mine, there); }
  __device__ __forceinline__ void fetch(unsigned char* to, bool there) {
    if (there) {
#pragma unroll
      for (int a = 0; a < kArrays; ++a) {
        if (next[a] == nullptr) continue;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          if (!in(k)) continue;
          unsigned char* place = to + (a * K + k) * kPlane;
          const T* from = next[a] + k * columns;
          if constexpr (!kCopies) *reinterpret_cast<float*>(place) = to_float(*from);
          else if constexpr (kBytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(smem_u32(place)), "l"(from) : "memory");
          else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" :: "r"(smem_u32(place)), "l"(from) : "memory");
        }
        next[a] += step[a];
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  __device__ __forceinline__ void wait() const {
    if (ahead == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else asm volatile("cp.async.wait_group 0;" ::: "memory");
  }
  __device__ __forceinline__ Row<V> get(int a, int k) const {
    const unsigned char* place = mine + (a * K + k) * kPlane;
    if constexpr (!kCopies) return Row<V>::all(*reinterpret_cast<const float*>(place));
    else { Raw<T, V> raw; raw.load(reinterpret_cast<const T*>(place)); return raw.get(); }
  }
};

// V numbers of weight or bias, from L1 for every row but the first: in registers they would cost half of the threads that an SM holds.
template <int V>
__device__ __forceinline__ Row<V> load_weights(const void* w, int type, int at) {
  if (type == kNormHalf) {
    Raw<__nv_bfloat16, V> raw;
    raw.load(static_cast<const __nv_bfloat16*>(w) + at);
    return raw.get();
  }
  return load_state<V>(static_cast<const float*>(w) + at);
}

template <class T, int V, int K, int kThreads, bool kFull>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) norm_forward_kernel(const NormParams p, int group_threads, int ahead) {
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ float2 scratch[3][16];
  const Group g(group_threads);
  const float inv = 1.f / static_cast<float>(p.hidden);
  const long long step = static_cast<long long>(gridDim.x) * g.count, first = static_cast<long long>(blockIdx.x) * g.count + g.index;
  RowsAhead<T, V, K, kThreads, kFull, 2> rows(ahead, ring, g, p.hidden / V);
  rows.array(0, p.x, p.x_stride, first, step, g.lane * V);
  rows.array(1, p.residual, p.residual_stride, first, step, g.lane * V);
  rows.fetch(rows.mine, first < p.rows);
  if (ahead == 2) rows.fetch(rows.other, first + step < p.rows);
  T* y = static_cast<T*>(p.y) + first * p.hidden + g.lane * V;
  T* sum = p.sum != nullptr ? static_cast<T*>(p.sum) + first * p.hidden + g.lane * V : nullptr;
  int turn = 0;
  // (all groups of a block take as many turns as its first one, for the barriers)
  for (long long row = first, lead = first - g.index; lead < p.rows; row += step, lead += step, y += step * p.hidden, rows.turn()) {
    const bool there = row < p.rows;
    rows.wait();
    Row<V> s[K], total = Row<V>::all(0.f);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      s[k] = Row<V>::all(0.f);
      if (there && rows.in(k)) {
        s[k] = rows.get(0, k);
        if (p.residual != nullptr) {
          s[k] = s[k] + rows.get(1, k);
          store_row<T, V>(sum + k * rows.columns, s[k]);
        }
        total = total + s[k];
      }
    }
    if (sum != nullptr) sum += step * p.hidden;
    rows.fetch(row + ahead * step < p.rows);
    float mean = 0.f;
    if (p.center) mean = g.sum(across(total), scratch, turn) * inv;
    const Row<V> minus = Row<V>::all(-mean);
    total = Row<V>::all(0.f);
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (rows.in(k)) {
        s[k] = s[k] + minus;
        total = fused(s[k], s[k], total);
      }
    const float rstd = rsqrtf(g.sum(across(total), scratch, turn) * inv + p.eps);
    if (!there) continue;
    if (p.stats != nullptr && g.lane == 0) p.stats[row] = make_float2(mean, rstd);
    const Row<V> scale = Row<V>::all(rstd);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!rows.in(k)) continue;
      Row<V> u = s[k] * scale;
      const int at = g.lane * V + k * rows.columns;
      if (p.weight != nullptr && p.bias != nullptr) u = fused(u, load_weights<V>(p.weight, p.weight_type, at), load_weights<V>(p.bias, p.weight_type, at));
      else if (p.weight != nullptr) u = u * load_weights<V>(p.weight, p.weight_type, at);
      else if (p.bias != nullptr) u = u + load_weights<V>(p.bias, p.weight_type, at);
      store_row<T, V>(y + k * rows.columns, u);
    }
  }
}

template <class T, int V, int K, int kThreads, bool kFull>
__global__ void __launch_bounds__(kThreads, 512 / kThreads) norm_backward_kernel(const NormGradParams p, int group_threads, int ahead) {
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ float2 scratch[3][16];
  const Group g(group_threads);
  const float inv = 1.f / static_cast<float>(p.hidden);
  const long long step = static_cast<long long>(gridDim.x) * g.count, first = static_cast<long long>(blockIdx.x) * g.count + g.index;
  RowsAhead<T, V, K, kThreads, kFull, 4> rows(ahead, ring, g, p.hidden / V);
  rows.array(0, p.x, p.x_stride, first, step, g.lane * V);
  rows.array(1, p.dy, p.dy_stride, first, step, g.lane * V);
  rows.array(2, p.residual, p.residual_stride, first, step, g.lane * V);
  rows.array(3, p.dsum, p.dsum_stride, first, step, g.lane * V);
  rows.fetch(rows.mine, first < p.rows);
  if (ahead == 2) rows.fetch(rows.other, first + step < p.rows);
  Row<V> dw[K], db[K];
#pragma unroll
  for (int k = 0; k < K; ++k) dw[k] = db[k] = Row<V>::all(0.f);
  T* dx = p.dx != nullptr ? static_cast<T*>(p.dx) + first * p.hidden + g.lane * V : nullptr;
  float2 next_stats = first < p.rows ? p.stats[first] : make_float2(0.f, 0.f);
  int turn = 0;
  for (long long row = first, lead = first - g.index; lead < p.rows; row += step, lead += step, rows.turn()) {
    const bool there = row < p.rows;
    const float2 st = next_stats;
    if (row + step < p.rows) next_stats = p.stats[row + step];
    rows.wait();
    const Row<V> minus = Row<V>::all(-st.x), scale = Row<V>::all(st.y);
    Row<V> u[K], d[K], sum_d = Row<V>::all(0.f), sum_du = Row<V>::all(0.f);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!there || !rows.in(k)) continue;
      u[k] = rows.get(0, k);
      if (p.residual != nullptr) u[k] = u[k] + rows.get(2, k);
      u[k] = (u[k] + minus) * scale;
      d[k] = rows.get(1, k);
      dw[k] = fused(d[k], u[k], dw[k]);
      db[k] = db[k] + d[k];
      if (p.weight != nullptr) d[k] = d[k] * load_weights<V>(p.weight, p.weight_type, g.lane * V + k * rows.columns);
      sum_d = sum_d + d[k];
      sum_du = fused(d[k], u[k], sum_du);
    }
    if (dx != nullptr) {
      const float2 sums = g.sum(make_float2(across(sum_d), across(sum_du)), scratch, turn);
      const Row<V> minus_d = Row<V>::all(p.center ? -sums.x * inv : 0.f), minus_du = Row<V>::all(-sums.y * inv);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (!there || !rows.in(k)) continue;
        const Row<V> v = fused(u[k], minus_du, d[k] + minus_d);
        store_row<T, V>(dx + k * rows.columns, p.dsum != nullptr ? fused(v, scale, rows.get(3, k)) : v * scale);
      }
      dx += step * p.hidden;
    }
    rows.fetch(row + ahead * step < p.rows);
  }
  if (p.parts == nullptr) return;
  // the groups' sums, one after another, in place of the ring
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  float* all = reinterpret_cast<float*>(ring);
  for (int q = g.count - 1; q >= 0; --q) {
    __syncthreads();
    if (g.index != q) continue;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!rows.in(k)) continue;
      const int at = g.lane * V + k * rows.columns;
      if (q < g.count - 1) {
        dw[k] = dw[k] + load_state<V>(all + at);
        db[k] = db[k] + load_state<V>(all + p.hidden + at);
      }
      float* to = q > 0 ? all : p.parts + static_cast<long long>(blockIdx.x) * p.hidden;
      store_state<V>(to + at, dw[k]);
      store_state<V>(to + (q > 0 ? static_cast<long long>(p.hidden) : static_cast<long long>(gridDim.x) * p.hidden) + at, db[k]);
    }
  }
}

// A row of any length, read again from L2 for each of its passes.
template <class T>
__global__ void __launch_bounds__(kRowThreads) norm_forward_any_kernel(const NormParams p) {
  __shared__ float2 scratch[kRowThreads / 32];
  const float inv = 1.f / static_cast<float>(p.hidden);
  for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + r * p.x_stride;
    const T* add = p.residual != nullptr ? static_cast<const T*>(p.residual) + r * p.residual_stride : nullptr;
    auto value = [&](int i) { return to_float(x[i]) + (add != nullptr ? to_float(add[i]) : 0.f); };
    float mean = 0.f;
    if (p.center) {
      float2 a = make_float2(0.f, 0.f);
      for (int i = threadIdx.x; i < p.hidden; i += kRowThreads) a.x += value(i);
      mean = block_sum(a, scratch).x * inv;
    }
    float2 q = make_float2(0.f, 0.f);
    for (int i = threadIdx.x; i < p.hidden; i += kRowThreads) { const float v = value(i) - mean; q.x = fmaf(v, v, q.x); }
    const float rstd = rsqrtf(block_sum(q, scratch).x * inv + p.eps);
    if (p.stats != nullptr && threadIdx.x == 0) p.stats[r] = make_float2(mean, rstd);
    T* y = static_cast<T*>(p.y) + r * p.hidden;
    T* sum = p.sum != nullptr ? static_cast<T*>(p.sum) + r * p.hidden : nullptr;
    for (int i = threadIdx.x; i < p.hidden; i += kRowThreads) {
      const float v = value(i);
      float u = (v - mean) * rstd;
      if (p.weight != nullptr) u *= load_weight(p.weight, p.weight_type, i);
      if (p.bias != nullptr) u += load_weight(p.bias, p.weight_type, i);
      y[i] = from_float<T>(u);
      if (sum != nullptr) sum[i] = from_float<T>(v);
    }
  }
}

template <class T>
__global__ void __launch_bounds__(kRowThreads) norm_dx_any_kernel(const NormGradParams p) {
  __shared__ float2 scratch[kRowThreads / 32];
  const float inv = 1.f / static_cast<float>(p.hidden);
  for (long long r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + r * p.x_stride;
    const T* add = p.residual != nullptr ? static_cast<const T*>(p.residual) + r * p.residual_stride : nullptr;
    const T* dy = static_cast<const T*>(p.dy) + r * p.dy_stride;
    const T* dsum = p.dsum != nullptr ? static_cast<const T*>(p.dsum) + r * p.dsum_stride : nullptr;
    const float2 st = p.stats[r];
    auto unit = [&](int i) { return ((add != nullptr ? to_float(x[i]) + to_float(add[i]) : to_float(x[i])) - st.x) * st.y; };
    auto down = [&](int i) { const float g = to_float(dy[i]); return p.weight != nullptr ? g * load_weight(p.weight, p.weight_type, i) : g; };
    float2 a = make_float2(0.f, 0.f);
    for (int i = threadIdx.x; i < p.hidden; i += kRowThreads) { const float d = down(i); a.x += d; a.y = fmaf(d, unit(i), a.y); }
    a = block_sum(a, scratch);
    const float mean_d = p.center ? a.x * inv : 0.f, mean_du = a.y * inv;
    T* dx = static_cast<T*>(p.dx) + r * p.hidden;
    for (int i = threadIdx.x; i < p.hidden; i += kRowThreads) {
      float v = st.y * (down(i) - mean_d - unit(i) * mean_du);
      if (dsum != nullptr) v += to_float(dsum[i]);
      dx[i] = from_float<T>(v);
    }
  }
}

// Sums over the rows of a part, 32 columns a block.
template <class T>
__global__ void __launch_bounds__(kColumnThreads* kColumnRows) norm_dw_any_kernel(const NormGradParams p, int parts) {
  __shared__ float2 scratch[kColumnRows][kColumnThreads];
  const int i = blockIdx.x * kColumnThreads + threadIdx.x, part = blockIdx.y;
  const long long begin = p.rows * part / parts, end = p.rows * (part + 1) / parts;
  float2 a = make_float2(0.f, 0.f);
  if (i < p.hidden) {
    for (long long r = begin + threadIdx.y; r < end; r += kColumnRows) {
      const float g = to_float(static_cast<const T*>(p.dy)[r * p.dy_stride + i]);
      const float2 st = p.stats[r];
      float v = to_float(static_cast<const T*>(p.x)[r * p.x_stride + i]);
      if (p.residual != nullptr) v += to_float(static_cast<const T*>(p.residual)[r * p.residual_stride + i]);
      a.x = fmaf(g, (v - st.x) * st.y, a.x);
      a.y += g;
    }
  }
  scratch[threadIdx.y][threadIdx.x] = a;
  __syncthreads();
  if (threadIdx.y != 0 || i >= p.hidden) return;
  for (int k = 1; k < kColumnRows; ++k) { a.x += scratch[k][threadIdx.x].x; a.y += scratch[k][threadIdx.x].y; }
  p.parts[static_cast<long long>(part) * p.hidden + i] = a.x;
  p.parts[static_cast<long long>(parts + part) * p.hidden + i] = a.y;
}

constexpr int kJoinRows = 32;
__global__ void __launch_bounds__(kColumnThreads* kJoinRows) norm_join_kernel(const NormGradParams p, int parts) {
  __shared__ float scratch[kJoinRows][kColumnThreads];
  const int i = blockIdx.x * kColumnThreads + threadIdx.x;
  const float* from = p.parts + static_cast<long long>(blockIdx.y) * parts * p.hidden;
  grid_wait();
  void* out = blockIdx.y == 0 ? p.dweight : p.dbias;
  if (out == nullptr) return;
  float a = 0.f;
  if (i < p.hidden) {
#pragma unroll 4
    for (int k = threadIdx.y; k < parts; k += kJoinRows) a += from[static_cast<long long>(k) * p.hidden + i];
  }
  scratch[threadIdx.y][threadIdx.x] = a;
  __syncthreads();
  if (threadIdx.y != 0 || i >= p.hidden) return;
#pragma unroll
  for (int k = 1; k < kJoinRows; ++k) a += scratch[k][threadIdx.x];
  store_weight(out, p.weight_type, i, a);
}

int row_blocks(long long rows, int sms) { return static_cast<int>(rows < sms * 8ll ? rows : sms * 8ll); }

}  // namespace

namespace {

// The form that rows take: vectors of V, K of them a thread, `threads` threads a row; 0: rows too long to stay in registers.
struct Form { int vec, each, threads; };
Form form_of(int half, int hidden, bool sixteen, bool four) {
  Form f{};
  if (hidden > kMostColumns) return f;
  f.vec = sixteen ? (half ? 8 : 4) : half && four ? 2 : 1;
  const int vectors = hidden / f.vec;
  // Few vectors a thread keep short rows of single numbers and pairs from waiting for one another's loads: 1777 rows of 1001 fp32 columns with 16 a
  // thread 19.5 us forward, with 4 8.8.  (Whole vectors the other way: 8192 rows of 2048 with one a thread 32.9, with two 27.9.)
  f.each = vectors <= 32 ? 1 : f.vec == 1 && vectors <= 1024 ? 4 : f.vec == 2 && vectors <= 512 ? 2 : 16 / f.vec;
  f.threads = (vectors + f.each - 1) / f.each;                 // whole warps; more than half of them, a block that is not full
  f.threads = (f.threads + 31) / 32 * 32;
  return f;
}
// Whether all rows and the weights begin on boundaries of 16 bytes (and of 4).
struct Boundaries {
  bool sixteen, four;
  Boundaries(int half, int hidden) { const int size = half ? 2 : 4; sixteen = hidden * size % 16 == 0; four = hidden * size % 4 == 0; }
  void rows(const void* base, long long stride, int half) {
    if (base == nullptr) return;
    const auto at = reinterpret_cast<uintptr_t>(base) | static_cast<uintptr_t>(stride * (half ? 2 : 4));
    sixteen = sixteen && at % 16 == 0; four = four && at % 4 == 0;
  }
  // (fp32 weights beside pairs of bf16 rows are read 8 bytes at a time)
  void weights(const void* w) { sixteen = sixteen && reinterpret_cast<uintptr_t>(w) % 16 == 0; four = four && reinterpret_cast<uintptr_t>(w) % 8 == 0; }
};
Form form_of(const NormParams& p) {
  const int half = p.type == kNormHalf;
  Boundaries b(half, p.hidden);
  b.rows(p.x, p.x_stride, half); b.rows(p.residual, p.residual_stride, half); b.weights(p.weight); b.weights(p.bias);
  return form_of(half, p.hidden, b.sixteen, b.four);
}
Form form_of(const NormGradParams& p) {
  const int half = p.type == kNormHalf;
  Boundaries b(half, p.hidden);
  b.rows(p.x, p.x_stride, half); b.rows(p.residual, p.residual_stride, half); b.rows(p.dy, p.dy_stride, half); b.rows(p.dsum, p.dsum_stride, half);
  b.weights(p.weight);
  return form_of(half, p.hidden, b.sixteen, b.four);
}
int threads_of(const Form& f) { return f.threads > kGroupThreads ? f.threads : kGroupThreads / f.threads * f.threads; }
int blocks_of(const Form& f, long long rows, int sms, int resident) {
  const long long groups = threads_of(f) / f.threads, most = (rows + groups - 1) / groups, all = static_cast<long long>(sms) * resident;
  return static_cast<int>(most < all ? most : all);
}
// Blocks that share an SM: as many as its registers (128 a thread in the backward, 64 in the forward) hold.  (Shared memory holds as many of bf16 rows in whole vectors; of fp32 rows, and of
// single numbers in rows above 1024 columns, 3 of 4 forward, 1 of 2 above 4096 columns, and 1 of 2 backward up to 4096: such a grid runs in two rounds.)
int resident_backward(const Form& f) { return threads_of(f) > kGroupThreads ? 1 : 2; }
int resident_forward(const Form& f) { return threads_of(f) > kGroupThreads ? 2 : 4; }

template <class F>
cudaError_t by_form(int half, const Form& f, F run) {
  using H = __nv_bfloat16;
  using std::integral_constant;
  auto with = [&](auto type, auto vec) {
    constexpr int V = decltype(vec)::value;
    if (f.each == 1) return run(type, vec, integral_constant<int, 1>{});
    if constexpr (V <= 2) { if (f.each == 4 / V) return run(type, vec, integral_constant<int, 4 / V>{}); }
    return run(type, vec, integral_constant<int, 16 / V>{});
  };
  if (!half) return f.vec == 4 ? with(float{}, integral_constant<int, 4>{}) : with(float{}, integral_constant<int, 1>{});
  return f.vec == 8 ? with(H{}, integral_constant<int, 8>{}) : f.vec == 2 ? with(H{}, integral_constant<int, 2>{}) : with(H{}, integral_constant<int, 1>{});
}
// Bytes of a ring of one row.
int ring_of(const Form& f, int half, int arrays) {
  const int bytes = f.vec * (half ? 2 : 4);
  return arrays * f.each * (f.threads > kGroupThreads ? 512 : kGroupThreads) * (bytes < 4 ? 4 : bytes);
}
constexpr int kMostRing = 160 * 1024;

template <auto kKernel, class Params>
cudaError_t launch_rows(const Params& p, const Form& f, int blocks, int smem, int ahead, cudaStream_t stream) {
  static std::atomic<bool> configured[64];       // the shared-memory limit is an attribute of the function on a device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[dev].load(std::memory_order_acquire)) {
    if ((e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostRing)) != cudaSuccess) return e;
    configured[dev].store(true, std::memory_order_release);
  }
  kKernel<<<blocks, threads_of(f), smem, stream>>>(p, f.threads, ahead);
  return cudaGetLastError();
}
}  // namespace

int norm_parts(const NormGradParams& p, int sms) {
  const Form f = form_of(p);
  if (f.threads > 0) return blocks_of(f, p.rows, sms, resident_backward(f));
  return static_cast<int>(p.rows < sms ? p.rows : sms);
}

cudaError_t launch_norm_forward(const NormParams& p, int sms, cudaStream_t stream) {
  const Form f = form_of(p);
  const int half = p.type == kNormHalf;
  if (f.threads > 0)
    return by_form(half, f, [&](auto type, auto vec, auto each) {
      using T = decltype(type);
      constexpr int V = decltype(vec)::value, K = decltype(each)::value;
      const int blocks = blocks_of(f, p.rows, sms, resident_forward(f)), ring = 2 * ring_of(f, half, 2);
      // (rows that all threads have K vectors of, such as those of 2048 and 7168 columns, without a look whether they do)
      constexpr bool kCan = V == 8 && K == 2;
      const bool full = kCan && f.threads * K * V == p.hidden;
      if constexpr (K * V == 16)                 // (with fewer numbers a thread a row takes no more than 256)
        if (f.threads > kGroupThreads)
          return full ? launch_rows<norm_forward_kernel<T, V, K, 512, kCan>>(p, f, blocks, ring, 2, stream)
                      : launch_rows<norm_forward_kernel<T, V, K, 512, false>>(p, f, blocks, ring, 2, stream);
      return full ? launch_rows<norm_forward_kernel<T, V, K, 256, kCan>>(p, f, blocks, ring, 2, stream)
                  : launch_rows<norm_forward_kernel<T, V, K, 256, false>>(p, f, blocks, ring, 2, stream);
    });
  const int blocks = row_blocks(p.rows, sms);
  if (half) norm_forward_any_kernel<__nv_bfloat16><<<blocks, kRowThreads, 0, stream>>>(p);
  else norm_forward_any_kernel<float><<<blocks, kRowThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_norm_backward(const NormGradParams& p, int sms, cudaStream_t stream) {
  const Form f = form_of(p);
  const int half = p.type == kNormHalf, parts = norm_parts(p, sms);
  cudaError_t e = cudaSuccess;
  if (f.threads > 0) {
    const int row = ring_of(f, half, 4), ahead = 2 * row <= kMostRing ? 2 : 1, ring = ahead * row, sums = p.hidden * 8;
    e = by_form(half, f, [&](auto type, auto vec, auto each) {
      using T = decltype(type);
      constexpr int V = decltype(vec)::value, K = decltype(each)::value;
      const int smem = ring > sums ? ring : sums;
      constexpr bool kCan = V == 8 && K == 2;
      const bool full = kCan && f.threads * K * V == p.hidden;
      if constexpr (K * V == 16)
        if (f.threads > kGroupThreads)
          return full ? launch_rows<norm_backward_kernel<T, V, K, 512, kCan>>(p, f, parts, smem, ahead, stream)
                      : launch_rows<norm_backward_kernel<T, V, K, 512, false>>(p, f, parts, smem, ahead, stream);
      return full ? launch_rows<norm_backward_kernel<T, V, K, 256, kCan>>(p, f, parts, smem, ahead, stream)
                  : launch_rows<norm_backward_kernel<T, V, K, 256, false>>(p, f, parts, smem, ahead, stream);
    });
  } else {
    const int blocks = row_blocks(p.rows, sms);
    if (p.dx != nullptr) {
      if (half) norm_dx_any_kernel<__nv_bfloat16><<<blocks, kRowThreads, 0, stream>>>(p);
      else norm_dx_any_kernel<float><<<blocks, kRowThreads, 0, stream>>>(p);
    }
    if (p.parts != nullptr) {
      const dim3 grid((p.hidden + kColumnThreads - 1) / kColumnThreads, parts), block(kColumnThreads, kColumnRows);
      if (half) norm_dw_any_kernel<__nv_bfloat16><<<grid, block, 0, stream>>>(p, parts);
      else norm_dw_any_kernel<float><<<grid, block, 0, stream>>>(p, parts);
    }
    e = cudaGetLastError();
  }
  if (e != cudaSuccess || p.parts == nullptr) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((p.hidden + kColumnThreads - 1) / kColumnThreads, 2);
  cfg.blockDim = dim3(kColumnThreads, kJoinRows);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, norm_join_kernel, p, parts);
}

}  // namespace sep

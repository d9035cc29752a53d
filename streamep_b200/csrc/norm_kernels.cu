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

namespace sep {

namespace {

constexpr int kRowThreads = 256;                 // of a block that takes one row at a time
constexpr int kColumnThreads = 32, kColumnRows = 8;

template <class T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

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

// V elements of a row, as they lie in memory.
template <class T, int V> __device__ __forceinline__ void unpack(const void* from, float (&f)[V]) {
  if constexpr (sizeof(T) * V == 16 && sizeof(T) == 2) {
    const uint4 v = *static_cast<const uint4*>(from);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { const float2 p = unpack_bf16x2(w[i]); f[2 * i] = p.x; f[2 * i + 1] = p.y; }
  } else if constexpr (sizeof(T) * V == 16) {
    const float4 v = *static_cast<const float4*>(from);
    f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
  } else if constexpr (sizeof(T) == 2 && V == 2) {
    const float2 p = unpack_bf16x2(*static_cast<const uint32_t*>(from));
    f[0] = p.x; f[1] = p.y;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = to_float(static_cast<const T*>(from)[i]);
  }
}
template <class T, int V> __device__ __forceinline__ void store(T* at, const float (&f)[V]) {
  if constexpr (sizeof(T) * V == 16 && sizeof(T) == 2)
    *reinterpret_cast<uint4*>(at) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  else if constexpr (sizeof(T) * V == 16) *reinterpret_cast<float4*>(at) = make_float4(f[0], f[1], f[2], f[3]);
  else if constexpr (sizeof(T) == 2 && V == 2) *reinterpret_cast<uint32_t*>(at) = pack_bf16x2(f[0], f[1]);
  else {
#pragma unroll
    for (int i = 0; i < V; ++i) at[i] = from_float<T>(f[i]);
  }
}
// V numbers of weight or bias (which lie on boundaries of 4 numbers where V >= 4).
template <int V> __device__ __forceinline__ void load_weights(const void* w, int type, int at, float (&f)[V]) {
  if constexpr (V == 8) {
    if (type == kNormHalf) { unpack<__nv_bfloat16, 8>(static_cast<const __nv_bfloat16*>(w) + at, f); return; }
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(w) + at + i);
      f[i] = v.x; f[i + 1] = v.y; f[i + 2] = v.z; f[i + 3] = v.w;
    }
  } else if constexpr (V == 4) {
    if (type == kNormFloat) { unpack<float, 4>(static_cast<const float*>(w) + at, f); return; }
    const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(w) + at);
    const float2 a = unpack_bf16x2(v.x), b = unpack_bf16x2(v.y);
    f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = load_weight(w, type, at + i);
  }
}

constexpr int kMostColumns = 8192;               // of rows that stay in registers: 512 threads of 16
constexpr int kGroupThreads = 256;               // of a block, where a row takes no more

// A block's threads in groups of `threads` (32 to 512) for a row each; a thread takes vectors lane, lane + threads, ... of it.
struct Group {
  int threads, lane, index, count;
  __device__ __forceinline__ explicit Group(int t) : threads(t), lane(threadIdx.x % t), index(threadIdx.x / t), count(blockDim.x / t) {}
  // Every thread of a group gets its sums.  All of the block call, each time with the next of three buffers.
  __device__ __forceinline__ float2 sum(float2 v, float2 (*scratch)[16], int& turn) const {
    v = warp_sum(v);
    if (threads == 32) return v;
    float2* mine = scratch[turn];
    turn = turn == 2 ? 0 : turn + 1;
    if ((threadIdx.x & 31) == 0) mine[threadIdx.x >> 5] = v;
    __syncthreads();
    float2 s = make_float2(0.f, 0.f);
    const int first = index * (threads >> 5);
    for (int w = 0; w < (threads >> 5); ++w) { s.x += mine[first + w].x; s.y += mine[first + w].y; }
    return s;
  }
};

// Arrays of a row ahead: `kArrays` of them, some of which may be left out (null).
template <class T, int V, int K, int kArrays>
struct RowsAhead {
  static constexpr bool kCopies = sizeof(T) * V >= 4;
  static constexpr int kBytes = sizeof(T) * V >= 4 ? sizeof(T) * V : 4;
  int ahead;                     // rows that the ring holds: 2, or 1 where two do not fit
  unsigned char* ring;
  const T* base[kArrays];
  long long stride[kArrays];
  __device__ __forceinline__ unsigned char* place(int slot, int a, int k) const { return ring + (((slot * kArrays + a) * K + k) * blockDim.x + threadIdx.x) * kBytes; }
  __device__ __forceinline__ void fetch(int slot, long long row, bool there, const Group& g, int vectors) const {
    if (there) {
#pragma unroll
      for (int a = 0; a < kArrays; ++a) {
        if (base[a] == nullptr) continue;
        const T* from = base[a] + row * stride[a];
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const int v = g.lane + k * g.threads;
          if (v >= vectors) continue;
          if constexpr (!kCopies) *reinterpret_cast<float*>(place(slot, a, k)) = to_float(from[v]);
          else if constexpr (kBytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(smem_u32(place(slot, a, k))), "l"(from + v * V) : "memory");
          else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" :: "r"(smem_u32(place(slot, a, k))), "l"(from + v * V) : "memory");
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  __device__ __forceinline__ void wait() const {
    if (ahead == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else asm volatile("cp.async.wait_group 0;" ::: "memory");
  }
  __device__ __forceinline__ void get(int slot, int a, int k, float (&f)[V]) const {
    if constexpr (!kCopies) f[0] = *reinterpret_cast<const float*>(place(slot, a, k));
    else unpack<T, V>(place(slot, a, k), f);
  }
};

template <class T, int V, int K>
__global__ void __launch_bounds__(512) norm_forward_kernel(const NormParams p, int group_threads, int ahead) {
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ float2 scratch[3][16];
  const Group g(group_threads);
  RowsAhead<T, V, K, 2> rows{ahead, ring, {static_cast<const T*>(p.x), static_cast<const T*>(p.residual)}, {p.x_stride, p.residual_stride}};
  const int vectors = p.hidden / V;
  const float inv = 1.f / static_cast<float>(p.hidden);
  const long long step = static_cast<long long>(gridDim.x) * g.count, first = static_cast<long long>(blockIdx.x) * g.count + g.index;
  int turn = 0;
  for (int i = 0; i < ahead; ++i) rows.fetch(i, first + i * step, first + i * step < p.rows, g, vectors);
  // (all groups of a block take as many turns as its first one, for the barriers)
  const long long turns = (p.rows - static_cast<long long>(blockIdx.x) * g.count + step - 1) / step;
  for (long long t = 0; t < turns; ++t) {
    const long long row = first + t * step;
    const bool there = row < p.rows;
    const int slot = ahead == 2 ? static_cast<int>(t & 1) : 0;
    rows.wait();
    float s[K][V];
    float2 sums = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int i = 0; i < V; ++i) s[k][i] = 0.f;
      if (there && g.lane + k * g.threads < vectors) {
        rows.get(slot, 0, k, s[k]);
        if (p.residual != nullptr) {
          float r[V];
          rows.get(slot, 1, k, r);
#pragma unroll
          for (int i = 0; i < V; ++i) s[k][i] += r[i];
        }
#pragma unroll
        for (int i = 0; i < V; ++i) sums.x += s[k][i];
      }
    }
    rows.fetch(slot, row + ahead * step, row + ahead * step < p.rows, g, vectors);
    float mean = 0.f;
    if (p.center) mean = g.sum(sums, scratch, turn).x * inv;
    sums.x = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (g.lane + k * g.threads < vectors) {
#pragma unroll
        for (int i = 0; i < V; ++i) { const float d = s[k][i] - mean; sums.x = fmaf(d, d, sums.x); }
      }
    const float rstd = rsqrtf(g.sum(sums, scratch, turn).x * inv + p.eps);
    if (!there) continue;
    if (p.stats != nullptr && g.lane == 0) p.stats[row] = make_float2(mean, rstd);
    T* y = static_cast<T*>(p.y) + row * p.hidden;
    T* sum = static_cast<T*>(p.sum) + row * p.hidden;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int at = (g.lane + k * g.threads) * V;
      if (at >= p.hidden) continue;
      if (p.sum != nullptr) store<T, V>(sum + at, s[k]);
      float w[V];
#pragma unroll
      for (int i = 0; i < V; ++i) s[k][i] = (s[k][i] - mean) * rstd;
      if (p.weight != nullptr) {
        load_weights<V>(p.weight, p.weight_type, at, w);
#pragma unroll
        for (int i = 0; i < V; ++i) s[k][i] *= w[i];
      }
      if (p.bias != nullptr) {
        load_weights<V>(p.bias, p.weight_type, at, w);
#pragma unroll
        for (int i = 0; i < V; ++i) s[k][i] += w[i];
      }
      store<T, V>(y + at, s[k]);
    }
  }
}

template <class T, int V, int K>
__global__ void __launch_bounds__(512) norm_backward_kernel(const NormGradParams p, int group_threads, int ahead) {
  extern __shared__ __align__(16) unsigned char ring[];
  __shared__ float2 scratch[3][16];
  const Group g(group_threads);
  RowsAhead<T, V, K, 4> rows{ahead, ring,
                                     {static_cast<const T*>(p.x), static_cast<const T*>(p.dy), static_cast<const T*>(p.residual), static_cast<const T*>(p.dsum)},
                                     {p.x_stride, p.dy_stride, p.residual_stride, p.dsum_stride}};
  const int vectors = p.hidden / V;
  const float inv = 1.f / static_cast<float>(p.hidden);
  const long long step = static_cast<long long>(gridDim.x) * g.count, first = static_cast<long long>(blockIdx.x) * g.count + g.index;
  int turn = 0;
  float dw[K][V], db[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) dw[k][i] = db[k][i] = 0.f;
  for (int i = 0; i < ahead; ++i) rows.fetch(i, first + i * step, first + i * step < p.rows, g, vectors);
  const long long turns = (p.rows - static_cast<long long>(blockIdx.x) * g.count + step - 1) / step;
  float2 next_stats = first < p.rows ? p.stats[first] : make_float2(0.f, 0.f);
  for (long long t = 0; t < turns; ++t) {
    const long long row = first + t * step;
    const bool there = row < p.rows;
    const int slot = ahead == 2 ? static_cast<int>(t & 1) : 0;
    const float2 st = next_stats;
    if (row + step < p.rows) next_stats = p.stats[row + step];
    rows.wait();
    float u[K][V], d[K][V];
    float2 sums = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!there || g.lane + k * g.threads >= vectors) continue;
      rows.get(slot, 0, k, u[k]);
      rows.get(slot, 1, k, d[k]);
      float w[V];
      if (p.residual != nullptr) {
        rows.get(slot, 2, k, w);
#pragma unroll
        for (int i = 0; i < V; ++i) u[k][i] += w[i];
      }
      if (p.weight != nullptr) load_weights<V>(p.weight, p.weight_type, (g.lane + k * g.threads) * V, w);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        u[k][i] = (u[k][i] - st.x) * st.y;
        dw[k][i] = fmaf(d[k][i], u[k][i], dw[k][i]);
        db[k][i] += d[k][i];
        if (p.weight != nullptr) d[k][i] *= w[i];
        sums.x += d[k][i];
        sums.y = fmaf(d[k][i], u[k][i], sums.y);
      }
    }
    if (p.dx != nullptr) {
      sums = g.sum(sums, scratch, turn);
      const float mean_d = p.center ? sums.x * inv : 0.f, mean_du = sums.y * inv;
      T* dx = static_cast<T*>(p.dx) + row * p.hidden;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int at = (g.lane + k * g.threads) * V;
        if (!there || at >= p.hidden) continue;
#pragma unroll
        for (int i = 0; i < V; ++i) d[k][i] = st.y * (d[k][i] - mean_d - u[k][i] * mean_du);
        if (p.dsum != nullptr) {
          float add[V];
          rows.get(slot, 3, k, add);
#pragma unroll
          for (int i = 0; i < V; ++i) d[k][i] += add[i];
        }
        store<T, V>(dx + at, d[k]);
      }
    }
    rows.fetch(slot, row + ahead * step, row + ahead * step < p.rows, g, vectors);
  }
  if (p.parts == nullptr) return;
  // the groups' sums, one after another, in place of the ring
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  float2* all = reinterpret_cast<float2*>(ring);
  for (int q = g.count - 1; q >= 0; --q) {
    __syncthreads();
    if (g.index != q) continue;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int at = (g.lane + k * g.threads) * V + i;
        if (at >= p.hidden) continue;
        if (q < g.count - 1) { const float2 v = all[at]; dw[k][i] += v.x; db[k][i] += v.y; }
        if (q > 0) all[at] = make_float2(dw[k][i], db[k][i]);
      }
    if (q > 0) continue;
    float* out_w = p.parts + static_cast<long long>(blockIdx.x) * p.hidden;
    float* out_b = p.parts + static_cast<long long>(gridDim.x + blockIdx.x) * p.hidden;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int at = (g.lane + k * g.threads) * V;
      if (at >= p.hidden) continue;
      if constexpr (V == 8) {
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
          *reinterpret_cast<float4*>(out_w + at + i) = make_float4(dw[k][i], dw[k][i + 1], dw[k][i + 2], dw[k][i + 3]);
          *reinterpret_cast<float4*>(out_b + at + i) = make_float4(db[k][i], db[k][i + 1], db[k][i + 2], db[k][i + 3]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) { out_w[at + i] = dw[k][i]; out_b[at + i] = db[k][i]; }
      }
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
  f.each = vectors <= 32 ? 1 : 16 / f.vec;
  f.threads = 32;
  while (f.threads * f.each < vectors) f.threads *= 2;
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
  void weights(const void* w) { sixteen = sixteen && reinterpret_cast<uintptr_t>(w) % 16 == 0; }
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
int threads_of(const Form& f) { return f.threads > kGroupThreads ? f.threads : kGroupThreads; }
int blocks_of(const Form& f, long long rows, int sms, int resident) {
  const long long groups = threads_of(f) / f.threads, most = (rows + groups - 1) / groups, all = static_cast<long long>(sms) * resident;
  return static_cast<int>(most < all ? most : all);
}
// Blocks that share an SM: as many as its registers (128 a thread in the backward, 64 in the forward) and shared memory hold.
int resident_backward(const Form& f) { return threads_of(f) > kGroupThreads ? 1 : 2; }
int resident_forward(const Form& f) { return (threads_of(f) > kGroupThreads ? 1 : 2) * (f.vec == 8 || f.each == 1 ? 2 : 1); }

template <class F>
cudaError_t by_form(int half, const Form& f, F run) {
  using H = __nv_bfloat16;
  using std::integral_constant;
  if (half) {
    if (f.vec == 8) return f.each == 1 ? run(H{}, integral_constant<int, 8>{}, integral_constant<int, 1>{}) : run(H{}, integral_constant<int, 8>{}, integral_constant<int, 2>{});
    if (f.vec == 2) return f.each == 1 ? run(H{}, integral_constant<int, 2>{}, integral_constant<int, 1>{}) : run(H{}, integral_constant<int, 2>{}, integral_constant<int, 8>{});
    return f.each == 1 ? run(H{}, integral_constant<int, 1>{}, integral_constant<int, 1>{}) : run(H{}, integral_constant<int, 1>{}, integral_constant<int, 16>{});
  }
  if (f.vec == 4) return f.each == 1 ? run(float{}, integral_constant<int, 4>{}, integral_constant<int, 1>{}) : run(float{}, integral_constant<int, 4>{}, integral_constant<int, 4>{});
  return f.each == 1 ? run(float{}, integral_constant<int, 1>{}, integral_constant<int, 1>{}) : run(float{}, integral_constant<int, 1>{}, integral_constant<int, 16>{});
}
// Bytes of a ring of one row.
int ring_of(const Form& f, int half, int arrays) {
  const int bytes = f.vec * (half ? 2 : 4);
  return arrays * f.each * threads_of(f) * (bytes < 4 ? 4 : bytes);
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
      return launch_rows<norm_forward_kernel<decltype(type), decltype(vec)::value, decltype(each)::value>>(p, f, blocks_of(f, p.rows, sms, resident_forward(f)), 2 * ring_of(f, half, 2), 2, stream);
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
      return launch_rows<norm_backward_kernel<decltype(type), decltype(vec)::value, decltype(each)::value>>(p, f, parts, ring > sums ? ring : sums, ahead, stream);
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

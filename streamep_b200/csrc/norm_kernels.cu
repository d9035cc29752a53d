// Normalisation of rows, with the residual stream added on the way, and its gradients.
//
//   s = x + residual;  u = (s - mean s) / sqrt(var s + eps);  y = u * weight + bias        (without `center` the mean is taken as 0)
//   d = dy * weight;   dx = (d - mean d - u * mean(d u)) / deviation + dsum;  dweight = sum over rows of dy u;  dbias = sum of dy
//
// Both passes are bound by memory.  All sums are fp32, in a fixed order (a repeated call gives the same bits).
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
    const T* dy = static_cast<const T*>(p.dy) + r * p.dy_stride;
    const T* dsum = p.dsum != nullptr ? static_cast<const T*>(p.dsum) + r * p.dsum_stride : nullptr;
    const float2 st = p.stats[r];
    auto unit = [&](int i) { return (to_float(x[i]) - st.x) * st.y; };
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
      a.x = fmaf(g, (to_float(static_cast<const T*>(p.x)[r * p.x_stride + i]) - st.x) * st.y, a.x);
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

__global__ void __launch_bounds__(kColumnThreads* kColumnRows) norm_join_kernel(const NormGradParams p, int parts) {
  __shared__ float2 scratch[kColumnRows][kColumnThreads];
  const int i = blockIdx.x * kColumnThreads + threadIdx.x;
  float2 a = make_float2(0.f, 0.f);
  if (i < p.hidden) {
    for (int k = threadIdx.y; k < parts; k += kColumnRows) {
      a.x += p.parts[static_cast<long long>(k) * p.hidden + i];
      a.y += p.parts[static_cast<long long>(parts + k) * p.hidden + i];
    }
  }
  scratch[threadIdx.y][threadIdx.x] = a;
  __syncthreads();
  if (threadIdx.y != 0 || i >= p.hidden) return;
  for (int k = 1; k < kColumnRows; ++k) { a.x += scratch[k][threadIdx.x].x; a.y += scratch[k][threadIdx.x].y; }
  if (p.dweight != nullptr) store_weight(p.dweight, p.weight_type, i, a.x);
  if (p.dbias != nullptr) store_weight(p.dbias, p.weight_type, i, a.y);
}

int row_blocks(long long rows, int sms) { return static_cast<int>(rows < sms * 8ll ? rows : sms * 8ll); }

}  // namespace

int norm_parts(long long rows, int hidden, int sms) {
  (void)hidden;
  return static_cast<int>(rows < sms ? rows : sms);
}

cudaError_t launch_norm_forward(const NormParams& p, int sms, cudaStream_t stream) {
  const int blocks = row_blocks(p.rows, sms);
  if (p.type == kNormHalf) norm_forward_any_kernel<__nv_bfloat16><<<blocks, kRowThreads, 0, stream>>>(p);
  else norm_forward_any_kernel<float><<<blocks, kRowThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_norm_backward(const NormGradParams& p, int sms, cudaStream_t stream) {
  const int blocks = row_blocks(p.rows, sms), parts = norm_parts(p.rows, p.hidden, sms);
  if (p.dx != nullptr) {
    if (p.type == kNormHalf) norm_dx_any_kernel<__nv_bfloat16><<<blocks, kRowThreads, 0, stream>>>(p);
    else norm_dx_any_kernel<float><<<blocks, kRowThreads, 0, stream>>>(p);
  }
  if (p.parts != nullptr) {
    const dim3 grid((p.hidden + kColumnThreads - 1) / kColumnThreads, parts), block(kColumnThreads, kColumnRows);
    if (p.type == kNormHalf) norm_dw_any_kernel<__nv_bfloat16><<<grid, block, 0, stream>>>(p, parts);
    else norm_dw_any_kernel<float><<<grid, block, 0, stream>>>(p, parts);
    norm_join_kernel<<<grid.x, block, 0, stream>>>(p, parts);
  }
  return cudaGetLastError();
}

}  // namespace sep

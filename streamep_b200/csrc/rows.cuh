// Vectors of a row in registers: loads and stores of bf16 and fp32, fp32 arithmetic.
#pragma once

#include <cuda_bf16.h>

#include "ptx.cuh"

namespace sep {

template <class T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// V numbers of a thread, of one row.  Sums and products are written out, so that the bits do not depend on what else a call computes.  (Two fp32 numbers an
// instruction, fma.rn.f32x2 and its like, save none here, where each pair has to be brought together first: a normalisation of 32768 rows of 7168 columns
// 298 -> 393 us, its gradients 432 -> 436, a recurrence of 8192 rows of 2048 channels with gradients 96 -> 94.)
template <int V> struct Row {
  float f[V];
  __device__ __forceinline__ static Row all(float v) {
    Row r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.f[i] = v;
    return r;
  }
  __device__ __forceinline__ void get(float (&o)[V]) const {
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = f[i];
  }
  __device__ __forceinline__ static Row of(const float (&o)[V]) {
    Row r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.f[i] = o[i];
    return r;
  }
};
template <int V> __device__ __forceinline__ Row<V> operator+(Row<V> a, const Row<V>& b) {
#pragma unroll
  for (int i = 0; i < V; ++i) a.f[i] = __fadd_rn(a.f[i], b.f[i]);
  return a;
}
template <int V> __device__ __forceinline__ Row<V> operator*(Row<V> a, const Row<V>& b) {
#pragma unroll
  for (int i = 0; i < V; ++i) a.f[i] = __fmul_rn(a.f[i], b.f[i]);
  return a;
}
template <int V> __device__ __forceinline__ Row<V> fused(const Row<V>& a, const Row<V>& b, Row<V> c) {
#pragma unroll
  for (int i = 0; i < V; ++i) c.f[i] = fmaf(a.f[i], b.f[i], c.f[i]);
  return c;
}

// V numbers of a row, as they lie in memory.
template <class T, int V> struct Raw;
template <> struct Raw<__nv_bfloat16, 8> {
  uint4 v;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ Row<8> get() const {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    Row<8> r;
#pragma unroll
    for (int i = 0; i < 4; ++i) { r.f[2 * i] = __uint_as_float(w[i] << 16); r.f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
    return r;
  }
};
template <> struct Raw<__nv_bfloat16, 2> {
  uint32_t v;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = *reinterpret_cast<const uint32_t*>(p); }
  __device__ __forceinline__ Row<2> get() const { return Row<2>{__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u)}; }
};
template <> struct Raw<__nv_bfloat16, 4> {
  uint2 v;
  // `count` numbers, `step` apart; zeros behind them
  __device__ __forceinline__ void gather(const __nv_bfloat16* p, int step, int count) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) u[i] = i < count ? *reinterpret_cast<const unsigned short*>(p + i * step) : 0u;
    v = make_uint2(u[0] | u[1] << 16, u[2] | u[3] << 16);
  }
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = *reinterpret_cast<const uint2*>(p); }
  __device__ __forceinline__ Row<4> get() const {
    return Row<4>{__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u)};
  }
};
template <> struct Raw<float, 4> {
  float4 v;
  __device__ __forceinline__ void gather(const float* p, int step, int count) {
    v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (count > 0) v.x = p[0];
    if (count > 1) v.y = p[step];
    if (count > 2) v.z = p[2 * step];
    if (count > 3) v.w = p[3 * step];
  }
  __device__ __forceinline__ void load(const float* p) { v = *reinterpret_cast<const float4*>(p); }
  __device__ __forceinline__ Row<4> get() const { return Row<4>{v.x, v.y, v.z, v.w}; }
};
template <class T> struct Raw<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = *p; }
  __device__ __forceinline__ Row<1> get() const { return Row<1>{to_float(v)}; }
};
template <class T, int V>
__device__ __forceinline__ void store_row(T* at, const Row<V>& row) {
  float f[V];
  row.get(f);
  if constexpr (V == 8) *reinterpret_cast<uint4*>(at) = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  else if constexpr (V == 2) *reinterpret_cast<uint32_t*>(at) = pack_bf16x2(f[0], f[1]);
  else if constexpr (V == 4) *reinterpret_cast<float4*>(at) = make_float4(f[0], f[1], f[2], f[3]);
  else *at = from_float<T>(f[0]);
}
template <int V>
__device__ __forceinline__ Row<V> load_state(const float* at) {
  float f[V];
  if constexpr (V >= 4) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const float4 v = *reinterpret_cast<const float4*>(at + i);
      f[i] = v.x; f[i + 1] = v.y; f[i + 2] = v.z; f[i + 3] = v.w;
    }
  } else if constexpr (V == 2) {
    const float2 v = *reinterpret_cast<const float2*>(at);
    f[0] = v.x; f[1] = v.y;
  } else {
    f[0] = *at;
  }
  return Row<V>::of(f);
}
template <int V>
__device__ __forceinline__ void store_state(float* at, const Row<V>& row) {
  float f[V];
  row.get(f);
  if constexpr (V >= 4) {
#pragma unroll
    for (int i = 0; i < V; i += 4) *reinterpret_cast<float4*>(at + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
  } else if constexpr (V == 2) {
    *reinterpret_cast<float2*>(at) = make_float2(f[0], f[1]);
  } else {
    *at = f[0];
  }
}

}  // namespace sep

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

constexpr int kThreads = 128;

template <class T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// sigmoid(gate) and sigmoid(-gate), each to its own last digits: the smaller one is computed, the other is its difference to 1.
struct Gate { float keep, take; };
__device__ __forceinline__ Gate gate_of(float g) {
  const float small = 1.f / (1.f + expf(fabsf(g)));
  return signbit(g) ? Gate{small, 1.f - small} : Gate{1.f - small, small};
}

// The rows of sequence `s`, within the rows that there are whatever the offsets say; these are checked where `report`.
struct Span { int begin, end; };
__device__ __forceinline__ long long offset_of(const ScanShape& p, int i) {
  return p.offsets_wide ? static_cast<const long long*>(p.offsets)[i] : static_cast<const int*>(p.offsets)[i];
}
__device__ __forceinline__ Span rows_of(const ScanShape& p, int s, bool report) {
  if (p.offsets == nullptr) return {s * p.length, (s + 1) * p.length};
  const long long begin = offset_of(p, s), end = offset_of(p, s + 1);
  if (begin < 0 || end < begin || end > p.rows) {
    if (report) report_note(p.status, kStatusBadOffsets, kKernelScan, 0, p.rank, s, static_cast<int>(begin), static_cast<int>(end));
    return {0, 0};
  }
  return {static_cast<int>(begin), static_cast<int>(end)};
}

// One thread walks one channel of one sequence.
template <class T>
__global__ void __launch_bounds__(kThreads) scan_forward_walk_kernel(const ScanParams p) {
  const int d = blockIdx.x * kThreads + threadIdx.x;
  for (int s = blockIdx.y; s < p.sequences; s += gridDim.y) {
    const Span span = rows_of(p, s, threadIdx.x == 0 && blockIdx.x == 0);
    if (d >= p.channels) continue;
    const long long state = static_cast<long long>(s) * p.channels + d;
    float h = p.initial != nullptr ? p.initial[state] : 0.f;
    for (long long t = span.begin; t < span.end; ++t) {
      const Gate g = gate_of(to_float(static_cast<const T*>(p.gate)[t * p.gate_stride + d]));
      h = fmaf(g.keep, h, g.take * to_float(static_cast<const T*>(p.x)[t * p.x_stride + d]));
      static_cast<T*>(p.h)[t * p.channels + d] = from_float<T>(h);
    }
    if (p.final_state != nullptr) p.final_state[state] = h;
  }
}

template <class T>
__global__ void __launch_bounds__(kThreads) scan_backward_walk_kernel(const ScanGradParams p) {
  const int d = blockIdx.x * kThreads + threadIdx.x;
  for (int s = blockIdx.y; s < p.sequences; s += gridDim.y) {
    const Span span = rows_of(p, s, false);
    if (d >= p.channels) continue;
    const long long state = static_cast<long long>(s) * p.channels + d;
    float carry = p.dfinal != nullptr ? p.dfinal[state] : 0.f;      // keep_{t+1} g_{t+1}
    for (long long t = span.end - 1; t >= span.begin; --t) {
      const Gate k = gate_of(to_float(static_cast<const T*>(p.gate)[t * p.gate_stride + d]));
      const float g = carry + (p.dh != nullptr ? to_float(static_cast<const T*>(p.dh)[t * p.dh_stride + d]) : 0.f);
      if (p.dx != nullptr) static_cast<T*>(p.dx)[t * p.channels + d] = from_float<T>(k.take * g);
      if (p.dgate != nullptr) {
        const float before = t > span.begin ? to_float(static_cast<const T*>(p.h)[(t - 1) * p.channels + d]) : p.initial != nullptr ? p.initial[state] : 0.f;
        const float x = to_float(static_cast<const T*>(p.x)[t * p.x_stride + d]);
        static_cast<T*>(p.dgate)[t * p.channels + d] = from_float<T>(g * (k.keep * k.take) * (before - x));
      }
      carry = __fmul_rn(k.keep, g);        // (not joined with the next addition: the bits do not depend on what else is asked for)
    }
    if (p.dinitial != nullptr) p.dinitial[state] = carry;
  }
}

template <class T>
__global__ void __launch_bounds__(kThreads) scan_step_kernel(const ScanStepParams p) {
  const int d = blockIdx.x * kThreads + threadIdx.x;
  if (d >= p.channels) return;
  for (long long s = blockIdx.y; s < p.rows; s += gridDim.y) {
    float* state = p.state + s * p.state_stride + d;
    const Gate g = gate_of(to_float(static_cast<const T*>(p.gate)[s * p.gate_stride + d]));
    const float h = fmaf(g.keep, *state, g.take * to_float(static_cast<const T*>(p.x)[s * p.x_stride + d]));
    *state = h;
    static_cast<T*>(p.h)[s * p.channels + d] = from_float<T>(h);
  }
}

dim3 walk_grid(int channels, int sequences) { return dim3((channels + kThreads - 1) / kThreads, sequences < 65535 ? sequences : 65535); }

}  // namespace

cudaError_t launch_scan_forward(const ScanParams& p, int sms, cudaStream_t stream) {
  (void)sms;
  // (packed sequences need not cover all rows)
  if (p.offsets != nullptr && p.rows > 0) {
    const cudaError_t e = cudaMemsetAsync(p.h, 0, static_cast<size_t>(p.rows) * p.channels * (p.half ? 2 : 4), stream);
    if (e != cudaSuccess) return e;
  }
  if (p.half) scan_forward_walk_kernel<__nv_bfloat16><<<walk_grid(p.channels, p.sequences), kThreads, 0, stream>>>(p);
  else scan_forward_walk_kernel<float><<<walk_grid(p.channels, p.sequences), kThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_scan_backward(const ScanGradParams& p, int sms, cudaStream_t stream) {
  (void)sms;
  if (p.offsets != nullptr && p.rows > 0) {
    for (void* out : {p.dx, p.dgate}) {
      const cudaError_t e = out != nullptr ? cudaMemsetAsync(out, 0, static_cast<size_t>(p.rows) * p.channels * (p.half ? 2 : 4), stream) : cudaSuccess;
      if (e != cudaSuccess) return e;
    }
  }
  if (p.half) scan_backward_walk_kernel<__nv_bfloat16><<<walk_grid(p.channels, p.sequences), kThreads, 0, stream>>>(p);
  else scan_backward_walk_kernel<float><<<walk_grid(p.channels, p.sequences), kThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_scan_step(const ScanStepParams& p, int sms, cudaStream_t stream) {
  (void)sms;
  if (p.half) scan_step_kernel<__nv_bfloat16><<<walk_grid(p.channels, p.rows), kThreads, 0, stream>>>(p);
  else scan_step_kernel<float><<<walk_grid(p.channels, p.rows), kThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace sep

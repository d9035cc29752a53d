// Operators over lists of tensors: sum of squares, scaling by the clipping factor, AdamW.
//
// All three are bound by memory: the norm reads every gradient once (2 or 4 bytes an element), clipping reads and writes them only where the
// norm is above the limit, AdamW on bf16 weights with master copies moves 28 bytes an element for about 20 operations.  A block
// takes a contiguous run of chunks (one search for its first tensor), every thread 16 bytes at a time and several loads in flight.
// Sums: fp32 in the four accumulators of a thread, doubles from there, in a fixed order (a repeated call gives the same bits).  A launch of 148 x 3
// blocks gives a thread n / 227328 of n elements (1220 at 277 M), so an accumulator adds up n / 7.3 M vectors of eight (bf16; four, fp32: n / 3.6 M): each
// addition is off by 2^-24 at most, the norm by half of that: 1e-6 at 277 M, 2e-5 at 5 G.
#include "list_kernels.h"
#include "ptx.cuh"

namespace sep {

namespace {

// The entry that chunk `c` belongs to: the last i with first[i] <= c (every entry has a chunk).
template <class List>
__device__ __forceinline__ int entry_of(const List& list, int c) {
  int lo = 0, hi = list.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (list.first[mid] <= c) lo = mid; else hi = mid - 1;
  }
  return lo;
}

struct Run { int begin, end; };
__device__ __forceinline__ Run run_of(int chunks, int block, int blocks) {
  return {static_cast<int>(static_cast<long long>(chunks) * block / blocks), static_cast<int>(static_cast<long long>(chunks) * (block + 1) / blocks)};
}

__device__ __forceinline__ float square_sum(uint4 v, bool half) {
  if (half) {
    const float2 a = unpack_bf16x2(v.x), b = unpack_bf16x2(v.y), c = unpack_bf16x2(v.z), d = unpack_bf16x2(v.w);
    return (fmaf(a.x, a.x, a.y * a.y) + fmaf(b.x, b.x, b.y * b.y)) + (fmaf(c.x, c.x, c.y * c.y) + fmaf(d.x, d.x, d.y * d.y));
  }
  const float a = __uint_as_float(v.x), b = __uint_as_float(v.y), c = __uint_as_float(v.z), d = __uint_as_float(v.w);
  return fmaf(a, a, b * b) + fmaf(c, c, d * d);
}
__device__ __forceinline__ float load_one(const void* base, long long i, bool half) {
  return half ? __bfloat162float(static_cast<const __nv_bfloat16*>(base)[i]) : static_cast<const float*>(base)[i];
}
__device__ __forceinline__ void store_one(void* base, long long i, bool half, float v) {
  if (half) static_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16_rn(v); else static_cast<float*>(base)[i] = v;
}

__device__ __forceinline__ double block_sum(double v, double* scratch) {
  for (int d = 16; d > 0; d >>= 1) v += __shfl_down_sync(0xffffffffu, v, d);
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
  for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) s += scratch[w];
  return s;                      // every thread has it
}

// A span of elements of one tensor, cut at 16-byte boundaries: [begin, head) and [tail, end) one by one, [head, tail) in vectors.
struct Span { long long begin, head, tail, end; };
__device__ __forceinline__ Span span_of(const void* base, long long begin, long long end, int width) {
  const int per = 16 / width;
  const long long off = static_cast<long long>(reinterpret_cast<uintptr_t>(base) / width % per);     // tensors start on whole elements
  long long head = (begin + off + per - 1) / per * per - off, tail = (end + off) / per * per - off;
  if (head > end) head = end;
  if (tail < head) tail = head;
  return {begin, head, tail, end};
}

__global__ void __launch_bounds__(kListThreads) list_squares_kernel(const __grid_constant__ NormList list, double* sums) {
  __shared__ double scratch[kListThreads / 32];
  grid_release();
  const Run run = run_of(list.chunks, blockIdx.x, gridDim.x);
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  if (run.begin < run.end) {
    int e = entry_of(list, run.begin);
    int c = run.begin;
    while (c < run.end) {
      while (e + 1 < list.count && list.first[e + 1] <= c) ++e;
      // all chunks of this tensor in the run at once
      const int stop = min(run.end, list.first[e + 1]);
      const unsigned long long word = list.length[e];
      const bool half = (word >> kListTypeShift) & kListHalf;
      const long long n = static_cast<long long>(word & kListLength);
      const long long begin = static_cast<long long>(c - list.first[e]) * list.chunk;
      const long long end = min(n, static_cast<long long>(stop - list.first[e]) * list.chunk);
      const void* base = list.data[e];
      const Span s = span_of(base, begin, end, half ? 2 : 4);
      for (long long i = s.begin + threadIdx.x; i < s.head; i += kListThreads) { const float v = load_one(base, i, half); acc[0] = fmaf(v, v, acc[0]); }
      for (long long i = s.tail + threadIdx.x; i < s.end; i += kListThreads) { const float v = load_one(base, i, half); acc[1] = fmaf(v, v, acc[1]); }
      const int per = half ? 8 : 4;
      const char* q = static_cast<const char*>(base) + s.head * (half ? 2 : 4);
      const long long vectors = (s.tail - s.head) / per;
      long long i = threadIdx.x;
      for (; i + 3 * kListThreads < vectors; i += 4 * kListThreads) {
        uint4 v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const uint4*>(q + (i + j * kListThreads) * 16);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] += square_sum(v[j], half);
      }
      for (; i < vectors; i += kListThreads) acc[0] += square_sum(*reinterpret_cast<const uint4*>(q + i * 16), half);
      c = stop;
    }
  }
  const double s = block_sum((static_cast<double>(acc[0]) + acc[1]) + (static_cast<double>(acc[2]) + acc[3]), scratch);
  if (threadIdx.x == 0) sums[blockIdx.x] = s;
}

// The sum of `count` doubles in a fixed order, the same in every block.
__device__ __forceinline__ double total_of(const double* sums, int count, double* scratch) {
  double v = 0.0;
  for (int i = threadIdx.x; i < count; i += blockDim.x) v += sums[i];
  return block_sum(v, scratch);
}

__global__ void __launch_bounds__(kListThreads) list_norm_kernel(const double* sums, int count, float* norm, double* total) {
  __shared__ double scratch[kListThreads / 32];
  grid_wait();
  const double s = total_of(sums, count, scratch);
  if (threadIdx.x == 0) { *norm = static_cast<float>(sqrt(s)); *total = s; }
}

// min(1, max_norm / (norm + 1e-6)); a NaN norm gives NaN
__device__ __forceinline__ float clip_factor(float norm, float max_norm) {
  const float f = max_norm / (norm + 1e-6f);
  return f > 1.f ? 1.f : f;
}

__device__ __forceinline__ uint32_t scale_pair(uint32_t u, float f) {
  const float2 v = unpack_bf16x2(u);
  return pack_bf16x2(v.x * f, v.y * f);
}
__device__ __forceinline__ uint4 scaled(uint4 v, float f, bool half) {
  if (half) return make_uint4(scale_pair(v.x, f), scale_pair(v.y, f), scale_pair(v.z, f), scale_pair(v.w, f));
  return make_uint4(__float_as_uint(__uint_as_float(v.x) * f), __float_as_uint(__uint_as_float(v.y) * f),
                    __float_as_uint(__uint_as_float(v.z) * f), __float_as_uint(__uint_as_float(v.w) * f));
}

__global__ void __launch_bounds__(kListThreads) list_scale_kernel(const __grid_constant__ NormList list, const double* sums, int num_sums, float* norm, float max_norm) {
  __shared__ double scratch[kListThreads / 32];
  grid_wait();
  float value;
  if (sums != nullptr) {
    value = static_cast<float>(sqrt(total_of(sums, num_sums, scratch)));
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm = value;
  } else {
    value = *norm;
  }
  const float f = clip_factor(value, max_norm);
  if (f == 1.f) return;
  // from the end of the list: what the norm read last is still in L2
  const Run run = run_of(list.chunks, static_cast<int>(gridDim.x - 1 - blockIdx.x), gridDim.x);
  if (run.begin >= run.end) return;
  int e = entry_of(list, run.begin);
  int c = run.begin;
  while (c < run.end) {
    while (e + 1 < list.count && list.first[e + 1] <= c) ++e;
    const int stop = min(run.end, list.first[e + 1]);
    const unsigned long long word = list.length[e];
    const bool half = (word >> kListTypeShift) & kListHalf;
    const long long n = static_cast<long long>(word & kListLength);
    const long long begin = static_cast<long long>(c - list.first[e]) * list.chunk;
    const long long end = min(n, static_cast<long long>(stop - list.first[e]) * list.chunk);
    void* base = list.data[e];
    const Span s = span_of(base, begin, end, half ? 2 : 4);
    for (long long i = s.begin + threadIdx.x; i < s.head; i += kListThreads) store_one(base, i, half, load_one(base, i, half) * f);
    for (long long i = s.tail + threadIdx.x; i < s.end; i += kListThreads) store_one(base, i, half, load_one(base, i, half) * f);
    const int per = half ? 8 : 4;
    char* q = static_cast<char*>(base) + s.head * (half ? 2 : 4);
    const long long vectors = (s.tail - s.head) / per;
    long long i = threadIdx.x;
    for (; i + 3 * kListThreads < vectors; i += 4 * kListThreads) {
      uint4 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const uint4*>(q + (i + j * kListThreads) * 16);
#pragma unroll
      for (int j = 0; j < 4; ++j) *reinterpret_cast<uint4*>(q + (i + j * kListThreads) * 16) = scaled(v[j], f, half);
    }
    for (; i < vectors; i += kListThreads) {
      uint4* at = reinterpret_cast<uint4*>(q + i * 16);
      *at = scaled(*at, f, half);
    }
    c = stop;
  }
}

struct Corrections { float step_size, inv_sqrt; };
__device__ __forceinline__ Corrections corrections_of(const AdamParams& p) {
  if (p.step == nullptr) return {p.step_size, p.inv_sqrt_correction};
  // 1 - beta^step = -expm1(step log beta): the exponent is rounded once, so the result keeps its digits however near 1 beta is
  const double t = static_cast<double>(*p.step);
  const float c1 = -expm1f(static_cast<float>(t * p.log_beta1)), c2 = -expm1f(static_cast<float>(t * p.log_beta2));
  return {p.lr / c1, 1.f / sqrtf(c2)};
}

struct Adam { float m, v, w; };
__device__ __forceinline__ Adam adam(const AdamParams& p, const Corrections& c, float g, float m, float v, float w) {
  m = fmaf(p.beta1, m, p.one_minus_beta1 * g);
  v = fmaf(p.beta2, v, p.one_minus_beta2 * g * g);
  w = w * p.keep - c.step_size * m / (sqrtf(v) * c.inv_sqrt + p.eps);
  return {m, v, w};
}
__device__ __forceinline__ float4 load_four(const void* base, long long i, bool half) {
  if (!half) return *reinterpret_cast<const float4*>(static_cast<const float*>(base) + i);
  const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(base) + i);
  const float2 a = unpack_bf16x2(u.x), b = unpack_bf16x2(u.y);
  return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ void store_four(void* base, long long i, bool half, float4 v) {
  if (!half) *reinterpret_cast<float4*>(static_cast<float*>(base) + i) = v;
  else *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(base) + i) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
}

__global__ void __launch_bounds__(kListThreads, 2) list_adamw_kernel(const __grid_constant__ AdamList list, const __grid_constant__ AdamParams p) {
  grid_wait();
  float f = 1.f;
  if (p.norm != nullptr) {
    const float norm = *p.norm;
    if (p.skip_nonfinite && !isfinite(norm)) return;
    if (p.max_norm >= 0.f) f = clip_factor(norm, p.max_norm);
  }
  const Corrections corrections = corrections_of(p);
  // from the end of the list: what the norm read last is still in L2
  for (long long last = list.chunks - static_cast<long long>(blockIdx.x) * list.window; last > 0; last -= static_cast<long long>(gridDim.x) * list.window) {
    const Run run = {static_cast<int>(max(last - list.window, 0ll)), static_cast<int>(last)};
    int e = entry_of(list, run.begin);
    int c = run.begin;
    while (c < run.end) {
      while (e + 1 < list.count && list.first[e + 1] <= c) ++e;
      const int stop = min(run.end, list.first[e + 1]);
      const unsigned long long word = list.length[e];
      const int flags = static_cast<int>(word >> kListTypeShift);
      const bool half = flags & kListHalf, grad_half = flags & kListGradHalf;
      // Vectors of four start `lead` elements into the tensor; these belong to its first chunk in addition, so that all others begin on a
      // boundary (with heads and tails in every chunk a packed list of 200 M odd elements took 1533 us instead of 1096).
      const int lead = flags >> kListHeadShift;
      const long long begin = c == list.first[e] ? 0 : lead + static_cast<long long>(c - list.first[e]) * list.chunk;
      const long long end = stop == list.first[e + 1] ? static_cast<long long>(word & kListLength) : lead + static_cast<long long>(stop - list.first[e]) * list.chunk;
      void* param = list.param[e];
      const void* grad = list.grad[e];
      float* m = list.exp_avg[e];
      float* v = list.exp_avg_sq[e];
      float* master = list.master[e];
      auto one = [&](long long i) {
        const Adam a = adam(p, corrections, load_one(grad, i, grad_half) * f, m[i], v[i], master != nullptr ? master[i] : load_one(param, i, half));
        m[i] = a.m; v[i] = a.v;
        if (master != nullptr) master[i] = a.w;
        store_one(param, i, half, a.w);
      };
      // what lies before the first vector and after the last goes one by one, and all of it where the entry's arrays have no boundary in common
      long long head = end, tail = end;
      if (!(flags & kListScalar)) {
        head = begin == 0 ? min(end, static_cast<long long>(lead)) : begin;
        tail = head + (end - head) / 4 * 4;
      }
      for (long long i = begin + threadIdx.x; i < head; i += kListThreads) one(i);
      for (long long i = tail + threadIdx.x; i < end; i += kListThreads) one(i);
      const long long step = 4 * kListThreads;
      long long i = head + 4 * threadIdx.x;
      auto four = [&](long long at, float4 g, float4 a, float4 b, float4 w) {
        const Adam r0 = adam(p, corrections, g.x * f, a.x, b.x, w.x), r1 = adam(p, corrections, g.y * f, a.y, b.y, w.y),
                   r2 = adam(p, corrections, g.z * f, a.z, b.z, w.z), r3 = adam(p, corrections, g.w * f, a.w, b.w, w.w);
        *reinterpret_cast<float4*>(m + at) = make_float4(r0.m, r1.m, r2.m, r3.m);
        *reinterpret_cast<float4*>(v + at) = make_float4(r0.v, r1.v, r2.v, r3.v);
        const float4 w4 = make_float4(r0.w, r1.w, r2.w, r3.w);
        if (master != nullptr) *reinterpret_cast<float4*>(master + at) = w4;
        store_four(param, at, half, w4);
      };
      for (; i + step < tail; i += 2 * step) {
        const float4 g0 = load_four(grad, i, grad_half), a0 = *reinterpret_cast<const float4*>(m + i), b0 = *reinterpret_cast<const float4*>(v + i);
        const float4 w0 = master != nullptr ? *reinterpret_cast<const float4*>(master + i) : load_four(param, i, half);
        const long long k = i + step;
        const float4 g1 = load_four(grad, k, grad_half), a1 = *reinterpret_cast<const float4*>(m + k), b1 = *reinterpret_cast<const float4*>(v + k);
        const float4 w1 = master != nullptr ? *reinterpret_cast<const float4*>(master + k) : load_four(param, k, half);
        four(i, g0, a0, b0, w0);
        four(k, g1, a1, b1, w1);
      }
      for (; i < tail; i += step)
        four(i, load_four(grad, i, grad_half), *reinterpret_cast<const float4*>(m + i), *reinterpret_cast<const float4*>(v + i),
             master != nullptr ? *reinterpret_cast<const float4*>(master + i) : load_four(param, i, half));
      c = stop;
    }
  }
}

// `early`: may prepare while the kernel before it drains (it waits before it reads anything).
template <class... Args, class... Values>
cudaError_t launch(void (*kernel)(Args...), int blocks, bool early, cudaStream_t stream, Values... values) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(kListThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  cfg.attrs = attr;
  if (early) {
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
  }
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<Args>(values)...);
}

}  // namespace

cudaError_t launch_list_squares(const NormList& list, double* sums, int blocks, cudaStream_t stream) {
  return launch(list_squares_kernel, blocks, false, stream, list, sums);
}
cudaError_t launch_list_norm(const double* sums, int count, float* norm, double* total, cudaStream_t stream) {
  return launch(list_norm_kernel, 1, true, stream, sums, count, norm, total);
}
cudaError_t launch_list_scale(const NormList& list, const double* sums, int num_sums, float* norm, float max_norm, int blocks, cudaStream_t stream) {
  return launch(list_scale_kernel, blocks, sums != nullptr, stream, list, sums, num_sums, norm, max_norm);
}
cudaError_t launch_list_adamw(const AdamList& list, const AdamParams& p, int blocks, cudaStream_t stream) {
  return launch(list_adamw_kernel, blocks, false, stream, list, p);
}

}  // namespace sep

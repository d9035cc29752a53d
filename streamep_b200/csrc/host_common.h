// What the host-side translation units share: argument checks that become Python exceptions, driver entry points, and
// tensor maps for TMA.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <torch/types.h>

#include <sstream>
#include <stdexcept>
#include <string>

namespace sep {

#define SEP_CUDA_CHECK(expr)                                                                        \
  do {                                                                                              \
    cudaError_t e__ = (expr);                                                                       \
    if (e__ != cudaSuccess) {                                                                       \
      std::ostringstream os__;                                                                      \
      os__ << "CUDA error " << cudaGetErrorName(e__) << " (" << cudaGetErrorString(e__) << ") at "  \
           << __FILE__ << ":" << __LINE__ << " in " #expr;                                          \
      throw std::runtime_error(os__.str());                                                         \
    }                                                                                               \
  } while (0)

#define SEP_ASSERT(cond, msg)                                                         \
  do {                                                                                \
    if (!(cond)) {                                                                    \
      std::ostringstream os__;                                                        \
      os__ << "streamep_b200: " << msg << " (" #cond ") at " << __FILE__ << ":" << __LINE__; \
      throw std::invalid_argument(os__.str());                                        \
    }                                                                                 \
  } while (0)

// ---------------------------------------------------------------------------------------------
// Driver entry points fetched at run time (the extension does not link libcuda).
// ---------------------------------------------------------------------------------------------
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

template <class Fn>
inline Fn driver_fn(const char* name) {
  void* fn = nullptr;
  cudaDriverEntryPointQueryResult q;
  SEP_CUDA_CHECK(cudaGetDriverEntryPoint(name, &fn, cudaEnableDefault, &q));
  if (q != cudaDriverEntryPointSuccess || fn == nullptr)
    throw std::runtime_error(std::string("streamep_b200: driver entry point not found: ") + name);
  return reinterpret_cast<Fn>(fn);
}

// 3-D tensor map (bf16 unless `type` says otherwise), 128-byte swizzle, OOB reads return zero.  dims/box are innermost-first.
inline CUtensorMap make_tmap(const void* base, uint64_t d0, uint64_t d1, uint64_t d2, uint64_t stride1_elems,
                             uint64_t stride2_elems, uint32_t b0, uint32_t b1,
                             CUtensorMapSwizzle swizzle = CU_TENSOR_MAP_SWIZZLE_128B,
                             CUtensorMapDataType type = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16) {
  static EncodeTiledFn encode = driver_fn<EncodeTiledFn>("cuTensorMapEncodeTiled");
  CUtensorMap m;
  const cuuint64_t width = type == CU_TENSOR_MAP_DATA_TYPE_FLOAT32 ? 4 : 2;
  cuuint64_t dims[3] = {d0, d1, d2};
  cuuint64_t strides[2] = {stride1_elems * width, stride2_elems * width};
  cuuint32_t box[3] = {b0, b1, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  SEP_ASSERT(reinterpret_cast<uintptr_t>(base) % 16 == 0, "TMA base address must be 16-byte aligned");
  SEP_ASSERT(strides[0] % 16 == 0 && strides[1] % 16 == 0, "TMA row pitch must be a multiple of 16 bytes");
  CUresult r = encode(&m, type, 3, const_cast<void*>(base), dims, strides, box, estr,
                      CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) throw std::runtime_error("streamep_b200: cuTensorMapEncodeTiled failed with code " + std::to_string(r));
  return m;
}

// Rows are read 16 bytes at a time.  A contiguous tensor may still start anywhere (a view of a flat buffer at an odd element,
// the gradient of an output that was concatenated behind something): such rows are copied to an aligned place first.
inline bool is_aligned(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
inline at::Tensor aligned_rows(const at::Tensor& t) { return !t.is_contiguous() || is_aligned(t) ? t : t.clone(); }

}  // namespace sep

// Host <-> kernel interface of the operators over lists of tensors (list_kernels.cu): global norm, clipping, AdamW.
//
// A list travels as a kernel argument (up to 32 KB of them), not through device memory: nothing to copy ahead of the
// launch, nothing to keep alive after it, and a captured launch holds its own list.  Tensors are cut into chunks of one size; a tensor
// has chunks [first[i], first[i + 1]).
#pragma once

#include <cuda_runtime.h>

namespace sep {

constexpr int kListTypeShift = 56;               // length word: elements, and flags from this bit on
constexpr unsigned long long kListLength = (1ull << kListTypeShift) - 1;
enum ListFlag : int {
  kListHalf = 1,                 // the tensor (AdamW: the parameter) is bf16, else fp32
  kListGradHalf = 2,             // AdamW: the gradient is bf16
  kListScalar = 4,               // AdamW: the tensors of this entry cannot be brought to 16-byte boundaries together
};
constexpr int kListHeadShift = 4;                // AdamW: flags >> 4 = elements before the first common boundary, in addition to those of the
                                                 // tensor's first chunk

constexpr int kNormEntries = 1024;
struct NormList {
  void* data[kNormEntries];
  unsigned long long length[kNormEntries];
  int first[kNormEntries + 1];
  int count, chunks, chunk;      // entries, chunks in all, elements of a chunk
};
constexpr int kAdamEntries = 512;
struct AdamList {
  void* param[kAdamEntries];
  const void* grad[kAdamEntries];
  float* exp_avg[kAdamEntries];
  float* exp_avg_sq[kAdamEntries];
  float* master[kAdamEntries];   // null: the parameter is updated itself
  unsigned long long length[kAdamEntries];
  int first[kAdamEntries + 1];
  int count, chunks, chunk;
  int window;                    // chunks that a block takes at a time
};

// One double per block: the sum of squares of its chunks.
cudaError_t launch_list_squares(const NormList& list, double* sums, int blocks, cudaStream_t stream);
// norm = sqrt(sum of sums), total = the sum
cudaError_t launch_list_norm(const double* sums, int count, float* norm, double* total, cudaStream_t stream);
// Multiplies by min(1, max_norm / (norm + 1e-6)).  `norm` is read, or (`sums` given) computed by every block and written by one.
cudaError_t launch_list_scale(const NormList& list, const double* sums, int num_sums, float* norm, float max_norm, int blocks, cudaStream_t stream);

struct AdamParams {
  float step_size;               // lr / (1 - beta1^step)
  float inv_sqrt_correction;     // 1 / sqrt(1 - beta2^step)
  const long long* step;         // optional: the step is this number on the device, and the two above are formed from it and these:
  float lr;
  double log_beta1, log_beta2;
  float beta1, one_minus_beta1, beta2, one_minus_beta2, eps, keep;   // keep = 1 - lr * weight_decay
  const float* norm;             // optional: the gradients' norm, and clipping by it (max_norm < 0: none)
  float max_norm;
  int skip_nonfinite;
};
cudaError_t launch_list_adamw(const AdamList& list, const AdamParams& p, int blocks, cudaStream_t stream);

constexpr int kListThreads = 512;
// what the registers of each kernel allow to be resident on an SM
constexpr int kNormBlocksPerSm = 3, kAdamBlocksPerSm = 2;

}  // namespace sep

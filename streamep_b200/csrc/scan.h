// Gated linear recurrence: launches of scan_kernels.cu.
#pragma once

#include <cuda_runtime.h>

#include "status.h"

namespace sep {

struct ScanShape {
  int half;                      // 1: x, gate, h and their gradients are bf16, 0: fp32
  int rows, channels;            // of all sequences together
  int sequences;
  int length;                    // rows of each sequence, where `offsets` is null
  const void* offsets;           // [sequences + 1] first rows of packed sequences, or null
  int offsets_wide;              // 1: int64, 0: int32
  long long x_stride, gate_stride;
  const void* x;
  const void* gate;
  const float* initial;          // [sequences, channels] or null (zeros)
  StatusBlock* status;
  int rank;
};
struct ScanParams : ScanShape {
  void* h;                       // [rows, channels]
  float* final_state;            // [sequences, channels] or null
};
struct ScanGradParams : ScanShape {
  const void* h;
  const void* dh;                // rows `dh_stride` apart; null: zeros
  long long dh_stride;
  const float* dfinal;           // or null
  void* dx;                      // or null
  void* dgate;                   // or null
  float* dinitial;               // or null
};
// How time is split: each sequence (packed ones: all rows) into `parts` segments of `rows` rows, of which a block takes a number side by side; and
// the workspace of their runs, where a sequence goes on in another block.
struct ScanSplit {
  int segments, parts, rows;
  int blocks, tiles;             // of segments, of channels
  int within;                    // 1: the segments of a sequence lie in one block
  float *factors, *sums;         // [segments][channels]
  float *block_factors, *block_sums;             // [blocks][channels]
};
ScanSplit scan_split(const ScanParams& p, int sms);
ScanSplit scan_split(const ScanGradParams& p, int sms);
long long scan_space(const ScanSplit& s, int channels);        // bytes, from a 16-byte boundary on
cudaError_t launch_scan_forward(const ScanParams& p, ScanSplit s, void* space, cudaStream_t stream);
cudaError_t launch_scan_backward(const ScanGradParams& p, ScanSplit s, void* space, cudaStream_t stream);

struct ScanStepParams {
  int half, rows, channels;
  long long x_stride, gate_stride, state_stride;
  const void* x;
  const void* gate;
  float* state;
  void* h;                       // [rows, channels]
};
cudaError_t launch_scan_step(const ScanStepParams& p, cudaStream_t stream);

}  // namespace sep

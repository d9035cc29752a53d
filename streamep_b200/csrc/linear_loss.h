// Host <-> kernel interface of the output projection with softmax cross entropy (linear_loss_kernels.cu).
#pragma once

#include <cuda.h>

#include "api.h"

namespace sep {

constexpr int kLossUnit = 256;        // rows and columns of a unit of work: one tile of a CTA pair
constexpr int kLossPart = 128;        // columns that one thread reduces: the softmax statistics come in parts of this many (narrow form: one
                                      // part for each quarter of every CTA)

// Kinds of work.  Forward: kLossStats.  Backward, for each piece of the vocabulary: kLossDz, then kLossDx and kLossDw.
enum LossKind : int { kLossStats = 0, kLossDz = 1, kLossDx = 2, kLossDw = 3 };

struct LossParams {
  int T, H, V;
  int narrow;                    // 1: tokens are the columns of a unit (see linear_loss_kernels.cu), `tile_tokens` of them
  int tile_tokens;               // tokens of a unit: 256, narrow: a multiple of 32
  int row_units;                 // ceil(T / tile_tokens)
  int stages, stage_bytes;       // narrow: the operand ring
  int dw_rows;                   // tokens of a k-block of dw: 64, or 32 where the ring's stages are too small for that
  int band;                      // row units that are walked together (see unit_of)
  // --- forward ---
  float2* parts;                 // [loss_forward_parts][T] maximum and sum of exp(z - maximum)
  float* target_logit;           // [T]
  const long long* targets;      // [T]
  long long ignore_index;
  int* zero; int zero_ints;      // memory that the forward kernel clears for the kernels after it
  // --- backward ---
  const float* top;              // [3][T] each token's largest logit, log2 of its sum of exp(z - largest), and its target's logit
  const float* row_scale;        // [T] upstream gradient of each token's loss, or null: 1
  const float* scale;            // [1] factor of every gradient, or null: 1 ...
  const float* scale2;           // [1] ... and another (1 / counted tokens)
  int piece;                     // columns of a piece, a multiple of 256
  int pieces, last_cols;         // how many, and the columns of the last
  int ahead;                     // pieces whose dz is computed before the first product is taken from one
  int buffers;                   // dz buffers in rotation, > ahead
  int split2;                    // 1: dz is kept as the sum of two bf16 numbers (short calls, narrow)
  int dx_direct;                 // 1: a dx unit is all there is of its place (one split, one piece) and stores bf16: no partial sums
  float* dx_parts;               // narrow: [splits][T][H] ...
  void* dx;                      // ... or [T, H] bf16
  int want_dx, want_dw;
  int splits;                    // reductions over a piece of the vocabulary into which a dx unit is split
  int split_blocks;              // k-blocks of each but the last
  int h_units;                   // ceil(H / 256)
  int dw_group;                  // column tiles of a dw unit
  int* claim;                    // next unit; zero on entry.  Null (forward): units are dealt out in turn
  int claim_lead;                // units that are claimed ahead of the one whose operands are being requested, beyond the next
  int* done;                     // epilogue warps that have finished units, zero on entry: [3][pieces] of a piece's dz / dx / dw,
                                 // then [pieces][piece / 256] of the dz of one column tile
  int dw_lead;                   // dw units of a piece that come before its dx units
  StatusBlock* status;
  int rank;
  unsigned long long wait_budget_ns;
};

struct LossMaps {                // CUtensorMap each: loads in boxes of 64 columns by 128 (k: K-major; narrow: x and dz by what a CTA
                                 // takes of the tokens) or 64 (mn) rows
  CUtensorMap x_k, x_mn, w_k, w_mn;
  CUtensorMap z_k, z_mn, z_out;
  CUtensorMap dw, dx;
};

void loss_narrow_ring(LossParams& p, bool backward);      // stages and stage_bytes of the narrow form (tile_tokens, split2, dw_rows given)
long long loss_forward_parts(const LossParams& p, int sms);
cudaError_t launch_loss_forward(const LossParams& p, const LossMaps& m, int sms, cudaStream_t stream);
cudaError_t launch_loss_backward(const LossParams& p, const LossMaps& m, int sms, cudaStream_t stream);
long long loss_backward_units(const LossParams& p);
// {kind, piece, unit row, unit column, split, first k-block, k-blocks} of backward unit `lin`
void loss_backward_unit(const LossParams& p, int lin, int (&out)[7]);

struct LossFinalParams {
  int T, V, num_parts;
  const float2* parts;
  const float* target_logit;
  const long long* targets;
  long long ignore_index;
  int mean, sum;                 // reduction (neither: per token)
  float* each;                   // [T] losses (scratch where they are reduced)
  float* top;                    // [3][T], as in LossParams
  float* loss;                   // [1] where they are reduced
  float* inv_count;              // [1] 1 / counted tokens (mean; 0 without any)
  int* ticket;                   // [1], zero on entry (cleared by the forward kernel)
  StatusBlock* status;
  int rank;
};
cudaError_t launch_loss_final(const LossFinalParams& p, cudaStream_t stream);

struct LossDxParams {
  int T, H, slots;
  int lanes;                     // threads that share the slots of an element: a power of two (set by the launcher)
  const float* parts;            // [slots][T][H]
  const float* scale;            // as in LossParams
  const float* scale2;
  void* dx;                      // [T, H] bf16
};
cudaError_t launch_loss_dx(const LossDxParams& p, cudaStream_t stream);

}  // namespace sep

// Launchers of the kernels over rows of logits (vocab_rows.cu); checked and called by vocab_rows_ops.cpp.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace bb {

constexpr int kMaxTop = 256;   // alternatives per row, and teacher entries per row
constexpr int kMaxVocab = 1 << 22;   // columns: bounds what a block notes about its slice in shared memory

enum class RowType { f32, f16, bf16 };

struct TokenArgs {
  const int64_t* tokens;   // [U, n] or null
  const float* temp;       // [U] or null
  double inv_temp1;        // 1 / T of every row when temp is null
  int U, V, n, k;
  long stride;             // elements between rows of the logits
  long vocab_start, vocab_total;
  float* logp;             // [U, n]: finished log-probs, or the tokens' x c when `open`
  float* entropy;          // [U] or null
  float* stats;            // [U, 3] or null: (R, 1/s, sum e t / s), or (R, s, sum e t) when `open`
  int64_t* top_ids;        // [U, k]
  float* top_logp;         // [U, k]: finished, or the raw logits when `open`
  const float* d_logp;     // [U, n]  (backward)
  const float* d_entropy;  // [U] or null
  bool open;               // a shard of the vocabulary: the sums are joined elsewhere
};

struct DistillArgs {
  const int64_t* ids;      // [U, K]
  const float* logq;       // [U, K]
  const float* weights;    // [U] or null
  const float* temp;       // [U] or null
  double inv_temp1;
  double scale;            // of the gradient: grad_scale / denom
  const float* num;        // null, or the gradient is for `scale` num / den instead, and stays where that is 1
  float den;
  int U, V, K;
  long stride;
  long vocab_start, vocab_total;
  bool tail, open;         // open: a shard of the vocabulary, the sums are joined elsewhere
  float* rows;             // [U] divergence, or null
  float* stats;            // [U, 2] (R, s) of the columns outside the given ids
  float* xc;               // [U, K] x c of the given ids in this shard, else 0
  float* coef;             // [U, 2] (R, factor of 2^(x c - R)) of the columns outside the given ids
  float* fix;              // [U, K] gradients of the given ids' columns
};

cudaError_t launch_token_logprob(RowType t, const void* logits, const TokenArgs& a, cudaStream_t stream);
cudaError_t launch_token_logprob_bwd(RowType t, const void* logits, void* grad, const TokenArgs& a,
                                     cudaStream_t stream);
// rows (+ grad unless null), or with a.open a shard's stats and xc
cudaError_t launch_distill(RowType t, const void* logits, void* grad, const DistillArgs& a, cudaStream_t stream);
cudaError_t launch_distill_finish(const DistillArgs& a, cudaStream_t stream);
cudaError_t launch_distill_grad(RowType t, const void* logits, void* grad, const DistillArgs& a, cudaStream_t stream);
cudaError_t launch_weighted_sum(const float* rows, const float* weights, int U, double inv_denom, float* out,
                                cudaStream_t stream);
cudaError_t launch_scale_unless_one(RowType t, void* x, long n, const float* num, float den, cudaStream_t stream);

}  // namespace bb

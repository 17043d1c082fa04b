// Tensor-core launches of the vocabulary cross entropy (xent_tc.cu).
#pragma once

#include "bwpp_cuda_internal.cuh"

// x [T, D] and vocabulary columns [v0, v0 + V) of the weight, both with row
// pitches of 16 bytes and 16-byte aligned bases.
struct XentOperands {
  const uint16_t *x, *w;
  uint32_t T, V, D, ldx, ldw;
  uint32_t v0, vocab;  // vocab: the whole vocabulary, targets are below it
  bool vocab_major;
  float scale;
};

// (maximum, sum of exponentials) in powers of two per row and 128 columns:
// part [ceil(V / 128)][T]; hit [T]: the target's logit where it is among the
// columns (target may be NULL).
int bwpp_xent_stats_launch(BwppCudaCtx *ctx, const XentOperands &o, const int32_t *target,
                           float2 *part, float *hit);
int bwpp_xent_combine_launch(BwppCudaCtx *ctx, const float2 *part, uint32_t nparts, const float *hit,
                             const int32_t *target, float *loss, float *lse, uint32_t T, uint32_t V);
// bf16 scale * dlogit [T, ld] of the columns.
int bwpp_xent_dlogit_launch(BwppCudaCtx *ctx, const XentOperands &o, const int32_t *target,
                            const float *lse, const float *dloss, uint16_t *dlogit, uint32_t ld);

// Tensor-core launches of the vocabulary cross entropy.

#pragma once

#include "bwpp_cuda_internal.cuh"

// ---- xent_tc.cu ----

// x [T, D] and vocabulary columns [v0, v0 + V) of the weight, both with row
// pitches of 16 bytes and 16-byte aligned bases.
struct XentOperands {
  const uint16_t *x, *w;
  uint32_t T, V, D, ldx, ldw;
  uint32_t v0, vocab;  // vocab: the whole vocabulary, targets are below it
  bool vocab_major;
  float scale;
};

// Few rows.  Their loss and gradients have no other rows' errors to average with,
// and they wait for W: up to so many, sums are shorter, a target's logit is kept
// apart from the others' sum, and dlogit is [2 * XENT_EXACT_ROWS, ld]: its rounded
// values, and in the second half what the rounding left.  Both halves are one row
// block of the gradients' products (dx) or two K blocks (dW).
constexpr uint32_t XENT_EXACT_ROWS = 64;
// (maximum, sum of exponentials) in powers of two per row and 128 columns:
// part [ceil(V / 128)][T]; hit [T]: the target's logit where it is among the
// columns, in powers of two as well (target may be NULL).  Few rows: the pair
// leaves the target out.
int bwpp_xent_stats_launch(BwppCudaCtx *ctx, const XentOperands &o, const int32_t *target,
                           float2 *part, float *hit);
int bwpp_xent_combine_launch(BwppCudaCtx *ctx, const float2 *part, uint32_t nparts, const float *hit,
                             const int32_t *target, float *loss, float *lse, uint32_t T, uint32_t V);
// bf16 scale * dlogit [T, ld] of the columns.  common: two floats as
// xent.cu's find_common writes them, or NULL.
int bwpp_xent_dlogit_launch(BwppCudaCtx *ctx, const XentOperands &o, const int32_t *target,
                            const float *lse, const float *dloss, const float *common,
                            uint16_t *dlogit, uint32_t ld);

// ---- xent_grad.cu ----

// C [M, N] = A [M, K] B [K, N] (+ add), bf16 operands, K-major or MN-major.
struct XentProduct {
  const uint16_t *a, *b;
  void *c;
  uint32_t M, N, K, lda, ldb, ldc;
  bool a_mn, b_mn;
  bool bf16;          // C bf16, else fp32
  bool guarded;       // what lies behind C's N columns is not to be written
  const float *factor; // device scalar that multiplies C, or NULL
  bool accumulate;    // add fp32 rows `add` (pitch ld_add; may be C)
  const void *add;
  uint32_t ld_add;
  uint32_t part_rows; // with K parts: rows from one part's C to the next, >= M
                      // rounded up to 256
};

// K parts of dx and dw, at most `most_dx` and `most_dw`, that a launch of both
// would best have.
int bwpp_xent_parts(BwppCudaCtx *ctx, const XentProduct &dx, const XentProduct &dw, uint32_t most_dx,
                    uint32_t most_dw, uint32_t *dx_parts, uint32_t *dw_parts);
// Either may be NULL.
int bwpp_xent_grad_launch(BwppCudaCtx *ctx, const XentProduct *dx, const XentProduct *dw,
                          uint32_t dx_parts, uint32_t dw_parts);
// out [rows, ld_out] = *factor (or 1) times the sum over parts, in order, of part
// + s * part_stride, and with second > 0 of what is `second` elements further.
int bwpp_xent_sum_parts_launch(BwppCudaCtx *ctx, const float *part, uint32_t parts,
                               size_t part_stride, size_t second, const float *factor, void *out,
                               uint32_t rows, uint32_t cols, uint32_t ld, uint32_t ld_out, int bf16);

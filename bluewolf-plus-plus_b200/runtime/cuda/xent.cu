// Softmax cross entropy over a vocabulary, from hidden states and the
// vocabulary weight, forward and gradient, without keeping the logits.
//
//   logit[t, v] = scale sum_d x[t, d] W[v, d]
//   lse[t] = log sum_v exp logit[t, v];   loss[t] = lse[t] - logit[t, target]
//   dlogit[t, v] = dloss[t] (exp(logit - lse) - [v == target])
//   dx = scale dlogit W;   dW = scale dlogit^T x
//
// The vocabulary goes by in pieces of C columns.  Forward: a piece's logits
// are one tensor-core product, folded into each row's running maximum, sum of
// exponentials and target logit.  Backward: a piece's logits are computed
// again (they were not kept), turned into bf16 dlogit, and two more products
// add the piece's share to dx and write its part of dW.
//
// A negative target ignores its row: loss 0, no share in any gradient (its x
// may hold anything, so the backward reads a copy of x with such rows zeroed:
// 0 * NaN would reach all of dW).  A target >= V reports BWPP_CUDA_ERR_ARG at
// the next bwpp_cuda_sync, its loss is NaN and its row is ignored.
//
// TMA wants row pitches of 16 bytes: x, W or gradients with others go through
// packed copies in scratch (a piece of W at a time).
#include <math.h>

#include "bwpp_cuda_internal.cuh"
#include "elem.cuh"
#include "rowwise.cuh"

int bwpp_gemm_launch_dt(BwppCudaCtx *ctx, const uint16_t *a, int a_mn, uint32_t lda,
                        const uint16_t *b, int b_mn, uint32_t ldb, void *c,
                        uint32_t ldc, uint32_t M, uint32_t N, uint32_t K,
                        const float *bias, int silu, const void *residual,
                        uint32_t ldr, int out_bf16, int force_simt, int ab_f16,
                        int out_f16, int res16);

namespace {

using bwpp_elem::aligned_to;
using bwpp_row::block_sum;

constexpr int kThreads = 256;

// dst[r, c] = src[r, c] of 16-bit elements; rows whose target is ignored
// become zero (target != NULL).
__global__ void __launch_bounds__(kThreads)
    pack_rows_kernel(const uint16_t *__restrict__ src, uint16_t *__restrict__ dst, uint32_t rows,
                     uint32_t cols, size_t ld_src, size_t ld_dst, const int32_t *target,
                     uint32_t V) {
  for (uint32_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const bool live = !target || (uint32_t)target[r] < V;
    for (uint32_t c = threadIdx.x; c < cols; c += kThreads)
      dst[r * ld_dst + c] = live ? src[r * ld_src + c] : (uint16_t)0;
  }
}

// Results from scratch into rows of any pitch.
__global__ void __launch_bounds__(kThreads)
    unpack_rows_kernel(const void *__restrict__ src, void *__restrict__ dst, uint32_t rows,
                       uint32_t cols, size_t ld_src, size_t ld_dst, int bf16) {
  for (uint32_t r = blockIdx.x; r < rows; r += gridDim.x)
    for (uint32_t c = threadIdx.x; c < cols; c += kThreads) {
      if (bf16)
        static_cast<uint16_t *>(dst)[r * ld_dst + c] =
            static_cast<const uint16_t *>(src)[r * ld_src + c];
      else
        static_cast<float *>(dst)[r * ld_dst + c] = static_cast<const float *>(src)[r * ld_src + c];
    }
}

// Folds the logits of vocabulary columns [v0, v0 + n) into the rows' state:
// [T] maximum, [T] sum of exponentials over it, [T] the target's logit.
__global__ void __launch_bounds__(kThreads)
    fold_kernel(const float *__restrict__ logits, uint32_t ld, uint32_t n, uint32_t v0, float scale,
                const int32_t *__restrict__ target, float *__restrict__ state, uint32_t T) {
  __shared__ float red[32];
  const uint32_t t = blockIdx.x;
  const float *row = logits + (size_t)t * ld;
  float m = -INFINITY;
  for (uint32_t c = threadIdx.x; c < n; c += kThreads) m = fmaxf(m, scale * row[c]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
  for (int w = 0; w < kThreads / 32; ++w) m = fmaxf(m, red[w]);
  const float before = v0 ? state[t] : -INFINITY;
  const float top = fmaxf(m, before);
  // rows of infinities: exp(-inf - -inf) is 0 here
  const float base = isinf(top) && top < 0 ? 0.0f : top;
  float s[1] = {0.0f};
  for (uint32_t c = threadIdx.x; c < n; c += kThreads) s[0] += expf(scale * row[c] - base);
  block_sum<1>(s, red);
  if (threadIdx.x == 0) {
    state[t] = top;
    state[T + t] = s[0] + (v0 ? state[T + t] * expf(before - base) : 0.0f);
    if (target) {
      const uint32_t at = (uint32_t)target[t] - v0;
      if ((uint32_t)target[t] >= v0 && at < n) state[2 * (size_t)T + t] = scale * row[at];
    }
  }
}

__global__ void __launch_bounds__(kThreads)
    finish_kernel(const float *__restrict__ state, const int32_t *__restrict__ target,
                  float *__restrict__ loss, float *__restrict__ lse, uint32_t T, uint32_t V,
                  int *status) {
  const uint32_t t = blockIdx.x * kThreads + threadIdx.x;
  if (t >= T) return;
  const float l = state[t] + logf(state[T + t]);
  if (lse) lse[t] = l;
  if (loss) {
    const int32_t y = target[t];
    float v = 0.0f;
    if (y >= 0) {
      v = l - state[2 * (size_t)T + t];
      if ((uint32_t)y >= V) {
        v = NAN;
        bwpp_report(status, BWPP_CUDA_ERR_ARG);
      }
    }
    loss[t] = v;
  }
}

// bf16 scale * dlogit of vocabulary columns [v0, v0 + n).
__global__ void __launch_bounds__(kThreads)
    dlogit_kernel(const float *__restrict__ logits, uint32_t ld, uint32_t n, uint32_t v0,
                  float scale, const int32_t *__restrict__ target, const float *__restrict__ lse,
                  const float *__restrict__ dloss, uint16_t *__restrict__ out, uint32_t ldo,
                  uint32_t V, int *status) {
  const uint32_t t = blockIdx.x;
  const int32_t y = target[t];
  const bool live = (uint32_t)y < V;
  if (y >= 0 && !live && threadIdx.x == 0) bwpp_report(status, BWPP_CUDA_ERR_ARG);
  const float l = lse[t], g = scale * (dloss ? dloss[t] : 1.0f);
  for (uint32_t c = threadIdx.x; c < n; c += kThreads) {
    const float p = expf(scale * logits[(size_t)t * ld + c] - l);
    const float d = live ? g * (v0 + c == (uint32_t)y ? p - 1.0f : p) : 0.0f;
    out[(size_t)t * ldo + c] = (uint16_t)(pack2_16<false>(d, 0.0f) & 0xFFFFu);
  }
}

inline uint32_t up8(uint32_t n) { return (n + 7) & ~7u; }
inline size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

// What a call keeps in scratch, as byte offsets.
struct Layout {
  uint32_t piece;             // vocabulary columns of a piece
  uint32_t dp;                // D rounded up
  size_t state, x, w, logits, dlogit, dx, dx16, dw, total;
};

// Vocabulary columns of a piece: about 2^26 logits at a time.
uint32_t piece_of(uint32_t T, uint32_t V) {
  uint64_t c = ((1ull << 26) / (T ? T : 1)) & ~255ull;
  if (c < 1024) c = 1024;
  const uint64_t all = ((uint64_t)V + 255) & ~255ull;
  return (uint32_t)(c < all ? c : all);
}

Layout layout_of(const BwppCudaXentParams &p, bool pack_x, bool pack_w, bool backward, bool stage_dx,
                 bool stage_dw) {
  Layout l{};
  l.piece = piece_of(p.T, p.V);
  l.dp = up8(p.D);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += up256(bytes);
    return here;
  };
  const size_t es = p.grads_bf16 ? 2 : 4;
  l.logits = take((size_t)p.T * l.piece * 4);
  if (!backward) l.state = take((size_t)p.T * 12);
  if (pack_x || backward) l.x = take((size_t)p.T * l.dp * 2);
  if (pack_w) l.w = take((size_t)l.piece * l.dp * 2);
  if (backward) {
    l.dlogit = take((size_t)p.T * l.piece * 2);
    if (stage_dx) {
      l.dx = take((size_t)p.T * l.dp * 4);
      l.dx16 = take((size_t)p.T * l.dp * 2);
    }
    if (stage_dw) l.dw = take((size_t)l.piece * l.dp * es);
  }
  l.total = at;
  return l;
}

int check(BwppCudaCtx *ctx, const BwppCudaXentParams *p) {
  if (!p) return bwpp_set_error(ctx, BWPP_CUDA_ERR_ARG, "xent: NULL params");
  if (p->V == 0 || p->D == 0 || p->V > 0x7fffffffu || p->T > 0x7fffffffu)
    return bwpp_set_error(ctx, BWPP_CUDA_ERR_ARG, "xent: V and D must be positive, V and T < 2^31");
  if (p->ldx < p->D || p->ldw < (p->w_vocab_major ? p->D : p->V))
    return bwpp_set_error(ctx, BWPP_CUDA_ERR_ARG, "xent: leading dim smaller than row");
  if (!isfinite(p->scale)) return bwpp_set_error(ctx, BWPP_CUDA_ERR_ARG, "xent: scale is not finite");
  return BWPP_CUDA_OK;
}

inline unsigned row_blocks(BwppCudaCtx *ctx, uint32_t rows) {
  const uint32_t most = (uint32_t)ctx->num_sms * 8;
  return rows < most ? rows : most;
}

// The piece [v0, v0 + n) of W as a GEMM operand.
struct Piece {
  const uint16_t *w;
  uint32_t ld;
};

int piece_w(BwppCudaCtx *ctx, const BwppCudaXentParams &p, const uint16_t *w, bool pack,
            uint16_t *scratch, uint32_t v0, uint32_t n, uint32_t ld_packed, Piece &out) {
  const uint16_t *src = w + (p.w_vocab_major ? (size_t)v0 * p.ldw : (size_t)v0);
  out = Piece{src, p.ldw};
  if (!pack) return BWPP_CUDA_OK;
  const uint32_t rows = p.w_vocab_major ? n : p.D, cols = p.w_vocab_major ? p.D : n;
  pack_rows_kernel<<<row_blocks(ctx, rows), kThreads, 0, ctx->stream>>>(src, scratch, rows, cols,
                                                                       p.ldw, ld_packed, nullptr, 0);
  BWPP_LAUNCH_CHECK(ctx, "xent pack");
  out = Piece{scratch, ld_packed};
  return BWPP_CUDA_OK;
}

bool needs_pack(const void *base, uint32_t ld) { return ld % 8 != 0 || !aligned_to(base, 16); }

}  // namespace

extern "C" {

size_t bwpp_cuda_xent_workspace_size(const BwppCudaXentParams *p, int backward) {
  if (!p || p->T == 0 || p->V == 0 || p->D == 0) return 0;
  return layout_of(*p, true, p->ldw % 8 != 0, backward != 0, true, true).total + BWPP_OP_SCRATCH_PAD;
}

int bwpp_cuda_xent_fwd_bf16(BwppCudaCtx *ctx, const uint16_t *x, const uint16_t *w,
                            const int32_t *target, float *loss, float *lse,
                            const BwppCudaXentParams *pp) {
  int rc = bwpp_ctx_enter(ctx);
  if (!rc) rc = check(ctx, pp);
  if (rc) return rc;
  const BwppCudaXentParams &p = *pp;
  if (p.T == 0) return BWPP_CUDA_OK;
  if (!x || !w || (loss && !target) || (!loss && !lse))
    return bwpp_set_error(ctx, BWPP_CUDA_ERR_ARG, "xent fwd: NULL buffer");
  const bool pack_x = needs_pack(x, p.ldx), pack_w = needs_pack(w, p.ldw);
  const Layout l = layout_of(p, pack_x, pack_w, false, false, false);
  uint8_t *scratch;
  rc = bwpp_op_scratch(ctx, l.total, "xent fwd", &scratch);
  if (rc) return rc;
  cudaStream_t s = ctx->stream;
  uint32_t ldx = p.ldx;
  if (pack_x) {
    uint16_t *xp = reinterpret_cast<uint16_t *>(scratch + l.x);
    pack_rows_kernel<<<row_blocks(ctx, p.T), kThreads, 0, s>>>(x, xp, p.T, p.D, p.ldx, l.dp, nullptr, 0);
    BWPP_LAUNCH_CHECK(ctx, "xent pack");
    x = xp;
    ldx = l.dp;
  }
  float *logits = reinterpret_cast<float *>(scratch + l.logits);
  float *state = reinterpret_cast<float *>(scratch + l.state);
  for (uint32_t v0 = 0; v0 < p.V; v0 += l.piece) {
    const uint32_t n = p.V - v0 < l.piece ? p.V - v0 : l.piece;
    Piece w1;
    rc = piece_w(ctx, p, w, pack_w, reinterpret_cast<uint16_t *>(scratch + l.w), v0, n,
                 p.w_vocab_major ? l.dp : l.piece, w1);
    if (!rc)
      rc = bwpp_gemm_launch_dt(ctx, x, 0, ldx, w1.w, p.w_vocab_major ? 0 : 1, w1.ld, logits, l.piece,
                               p.T, n, p.D, nullptr, 0, nullptr, 0, 0, 0, 0, 0, 0);
    if (rc) return rc;
    fold_kernel<<<p.T, kThreads, 0, s>>>(logits, l.piece, n, v0, p.scale, target, state, p.T);
    BWPP_LAUNCH_CHECK(ctx, "xent fold");
  }
  finish_kernel<<<(p.T + kThreads - 1) / kThreads, kThreads, 0, s>>>(state, target, loss, lse, p.T,
                                                                     p.V, ctx->status_word);
  BWPP_LAUNCH_CHECK(ctx, "xent finish");
  return BWPP_CUDA_OK;
}

int bwpp_cuda_xent_bwd_bf16(BwppCudaCtx *ctx, const uint16_t *x, const uint16_t *w,
                            const int32_t *target, const float *lse, const float *dloss, void *dx,
                            void *dw, const BwppCudaXentParams *pp) {
  int rc = bwpp_ctx_enter(ctx);
  if (!rc) rc = check(ctx, pp);
  if (rc) return rc;
  const BwppCudaXentParams &p = *pp;
  const uint32_t es = p.grads_bf16 ? 2 : 4;
  if ((dx && p.lddx < p.D) || (dw && p.lddw < (p.w_vocab_major ? p.D : p.V)))
    return bwpp_set_error(ctx, BWPP_CUDA_ERR_ARG, "xent bwd: leading dim smaller than row");
  cudaStream_t s = ctx->stream;
  if (p.T == 0) {  // no rows: dW is zero
    if (!dw) return BWPP_CUDA_OK;
    return bwpp_check_cuda(
        ctx,
        cudaMemset2DAsync(dw, (size_t)p.lddw * es, 0, (size_t)(p.w_vocab_major ? p.D : p.V) * es,
                          p.w_vocab_major ? p.V : p.D, s),
        "xent memset");
  }
  if (!dx && !dw) return BWPP_CUDA_OK;
  if (!x || !w || !target || !lse)
    return bwpp_set_error(ctx, BWPP_CUDA_ERR_ARG, "xent bwd: NULL buffer");
  const bool pack_w = needs_pack(w, p.ldw);
  const uint32_t piece = piece_of(p.T, p.V);
  const bool one = piece >= p.V;
  auto tma_out = [&](const void *q, uint32_t ld) { return (size_t)ld * es % 16 == 0 && aligned_to(q, 16); };
  // dx is summed over the pieces in fp32: in place where the caller's rows
  // are fp32 and TMA takes them
  const bool stage_dx = dx && (!tma_out(dx, p.lddx) || (p.grads_bf16 && !one));
  const bool stage_dw = dw && !tma_out(dw, p.lddw);
  const Layout l = layout_of(p, true, pack_w, true, stage_dx, stage_dw);
  uint8_t *scratch;
  rc = bwpp_op_scratch(ctx, l.total, "xent bwd", &scratch);
  if (rc) return rc;
  uint16_t *xp = reinterpret_cast<uint16_t *>(scratch + l.x);
  pack_rows_kernel<<<row_blocks(ctx, p.T), kThreads, 0, s>>>(x, xp, p.T, p.D, p.ldx, l.dp, target, p.V);
  BWPP_LAUNCH_CHECK(ctx, "xent pack");
  float *logits = reinterpret_cast<float *>(scratch + l.logits);
  uint16_t *dlogit = reinterpret_cast<uint16_t *>(scratch + l.dlogit);
  float *dx32 = reinterpret_cast<float *>(scratch + l.dx);
  for (uint32_t v0 = 0; v0 < p.V; v0 += piece) {
    const uint32_t n = p.V - v0 < piece ? p.V - v0 : piece;
    const bool last = v0 + n == p.V;
    Piece w1;
    rc = piece_w(ctx, p, w, pack_w, reinterpret_cast<uint16_t *>(scratch + l.w), v0, n,
                 p.w_vocab_major ? l.dp : piece, w1);
    if (!rc)
      rc = bwpp_gemm_launch_dt(ctx, xp, 0, l.dp, w1.w, p.w_vocab_major ? 0 : 1, w1.ld, logits, piece,
                               p.T, n, p.D, nullptr, 0, nullptr, 0, 0, 0, 0, 0, 0);
    if (rc) return rc;
    dlogit_kernel<<<p.T, kThreads, 0, s>>>(logits, piece, n, v0, p.scale, target, lse, dloss, dlogit,
                                           piece, p.V, ctx->status_word);
    BWPP_LAUNCH_CHECK(ctx, "xent dlogit");
    if (dx) {
      // dx (+)= dlogit W: the last piece leaves the sum in the caller's rows
      // where TMA can store them
      const bool to_user = !stage_dx || (last && tma_out(dx, p.lddx));
      const bool bf16_out = p.grads_bf16 && last;
      void *out = to_user ? dx : bf16_out ? static_cast<void *>(scratch + l.dx16) : dx32;
      const uint32_t ldo = to_user ? p.lddx : l.dp;
      const float *sum = v0 == 0 ? nullptr : stage_dx ? dx32 : static_cast<float *>(dx);
      rc = bwpp_gemm_launch_dt(ctx, dlogit, 0, piece, w1.w, p.w_vocab_major ? 1 : 0, w1.ld, out, ldo,
                               p.T, p.D, n, nullptr, 0, sum, stage_dx ? l.dp : p.lddx,
                               bf16_out ? 1 : 0, 0, 0, 0, 0);
      if (rc) return rc;
      if (!to_user && last) {
        unpack_rows_kernel<<<row_blocks(ctx, p.T), kThreads, 0, s>>>(out, dx, p.T, p.D, l.dp, p.lddx,
                                                                    p.grads_bf16);
        BWPP_LAUNCH_CHECK(ctx, "xent unpack");
      }
    }
    if (dw) {
      uint8_t *user = static_cast<uint8_t *>(dw) +
                      (p.w_vocab_major ? (size_t)v0 * p.lddw : (size_t)v0) * es;
      const uint32_t ld_staged = p.w_vocab_major ? l.dp : piece;
      void *out = stage_dw ? static_cast<void *>(scratch + l.dw) : user;
      const uint32_t ldo = stage_dw ? ld_staged : p.lddw;
      if (p.w_vocab_major)  // [n, D] = dlogit^T x
        rc = bwpp_gemm_launch_dt(ctx, dlogit, 1, piece, xp, 1, l.dp, out, ldo, n, p.D, p.T, nullptr, 0,
                                 nullptr, 0, p.grads_bf16 ? 1 : 0, 0, 0, 0, 0);
      else  // [D, n] = x^T dlogit
        rc = bwpp_gemm_launch_dt(ctx, xp, 1, l.dp, dlogit, 1, piece, out, ldo, p.D, n, p.T, nullptr, 0,
                                 nullptr, 0, p.grads_bf16 ? 1 : 0, 0, 0, 0, 0);
      if (rc) return rc;
      if (stage_dw) {
        const uint32_t rows = p.w_vocab_major ? n : p.D, cols = p.w_vocab_major ? p.D : n;
        unpack_rows_kernel<<<row_blocks(ctx, rows), kThreads, 0, s>>>(out, user, rows, cols, ldo,
                                                                      p.lddw, p.grads_bf16);
        BWPP_LAUNCH_CHECK(ctx, "xent unpack");
      }
    }
  }
  return BWPP_CUDA_OK;
}

}  // extern "C"

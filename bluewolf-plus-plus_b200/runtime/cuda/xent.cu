// Softmax cross entropy over a vocabulary, from hidden states and the
// vocabulary weight, forward and gradient, without keeping the logits.
//
//   logit[t, v] = scale sum_d x[t, d] W[v, d]
//   lse[t] = log sum_v exp logit[t, v];   loss[t] = lse[t] - logit[t, target]
//   dlogit[t, v] = dloss[t] (exp(logit - lse) - [v == target])
//   dx = scale dlogit W;   dW = scale dlogit^T x
//
// The products run on the tensor cores (xent_tc.cu): the forward's logits are
// folded into a (maximum, sum) pair per row and 128 columns in the product's
// epilogue.  The backward computes them again, a piece of the vocabulary at a
// time, and writes bf16 dlogit; one launch of two products (xent_grad.cu) adds
// the piece's share to dx (in fp32) and writes its part of dW.
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
#include "xent.cuh"

namespace {

using bwpp_elem::aligned_to;

constexpr int kThreads = 256;

// Copies between rows of any pitch and rows of 16 bytes in scratch, for the
// operands and results that TMA does not take as they are.  A warp takes
// kSpan consecutive elements of a row.  (A thread with eight elements of its
// own, as 2-byte accesses 16 bytes apart, took 60 us for 1001 x 10007 bf16.)
constexpr uint32_t kSpan = 256;

// The dloss that all live rows share, if they do: out = {scale * dloss, 1}, or
// {1, 0} where they differ.  The gradients' products then take p - hit, and this
// factor goes onto their results: with a mean loss, the usual one, a rounding
// of scale * dloss * (p - hit) would round the same mantissa, that of 1 / rows,
// in every row, up to 2^-8 of all targets' entries at once.
struct Common {
  const float *dloss;  // NULL: ones
  uint32_t T;
  float scale;
  float *out;          // NULL: not wanted
};

// One block.
__device__ __forceinline__ void find_common(const Common &a, const int32_t *target, uint32_t V) {
  __shared__ float lows[kThreads / 32], highs[kThreads / 32];
  float low = INFINITY, high = -INFINITY;
  bool odd = false;  // NaN: no two are alike
  constexpr uint32_t U = 16;  // loads in flight: the block is alone with its rows
  for (uint32_t t0 = threadIdx.x; t0 < a.T; t0 += U * kThreads) {
    uint32_t y[U];
    float g[U];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      const uint32_t t = t0 + u * kThreads;
      y[u] = t < a.T ? (uint32_t)target[t] : V;
      g[u] = t < a.T && a.dloss ? a.dloss[t] : 1.0f;
    }
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      if (y[u] >= V) continue;
      odd |= g[u] != g[u];
      low = fminf(low, g[u]);
      high = fmaxf(high, g[u]);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
    high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
  }
  if ((threadIdx.x & 31) == 0) {
    lows[threadIdx.x >> 5] = low;
    highs[threadIdx.x >> 5] = high;
  }
  odd = __syncthreads_or(odd);
  if (threadIdx.x) return;
  for (int w = 1; w < kThreads / 32; ++w) {
    low = fminf(low, lows[w]);
    high = fmaxf(high, highs[w]);
  }
  const bool same = !odd && low == high && low - low == 0.0f;  // one finite value
  a.out[0] = same ? a.scale * low : 1.0f;
  a.out[1] = same ? 1.0f : 0.0f;
}

// dst[r, c] = src[r, c] of 16-bit elements; dst's rows are filled up with zeros
// to a multiple of eight.  With targets, rows that are ignored become zero, and
// a target outside the vocabulary is reported.  again > 0: the rows have a
// second copy `again` rows below, and rows from `live_rows` on are zero.  The
// block in front of the rows' finds the common dloss: a launch of its own cost 2.7
// us, the block 1 us at 8192 rows (20 at 100000).
__global__ void __launch_bounds__(kThreads)
    pack_rows_kernel(const uint16_t *src, uint16_t *dst, uint32_t rows,
                     uint32_t cols, size_t ld_src, size_t ld_dst, int wide, const int32_t *target,
                     uint32_t V, uint32_t live_rows, uint32_t again, const Common common,
                     int *status) {
  dependent_wait();
  uint32_t block = blockIdx.x;
  if (common.out && block-- == 0) {
    find_common(common, target, V);
    return;
  }
  const uint32_t spans = (cols + kSpan - 1) / kSpan;
  const uint32_t i = (block * kThreads + threadIdx.x) / 32, lane = threadIdx.x & 31;
  if (i >= rows * spans) return;
  const uint32_t r = i / spans, c0 = (i - r * spans) * kSpan;
  bool live = r < live_rows;
  if (live && target) {
    const int32_t y = target[r];
    live = (uint32_t)y < V;
    if (y >= 0 && !live && c0 + lane == 0) bwpp_report(status, BWPP_CUDA_ERR_ARG);
  }
  const uint16_t *from = src + r * ld_src;
  uint16_t *to = dst + r * ld_dst;
  const uint32_t padded = (cols + 7) & ~7u;
  if (wide && c0 + kSpan <= cols) {
    const uint32_t c = c0 + lane * 8;
    const uint4 t = live ? *reinterpret_cast<const uint4 *>(from + c) : make_uint4(0u, 0u, 0u, 0u);
    *reinterpret_cast<uint4 *>(to + c) = t;
    if (again) *reinterpret_cast<uint4 *>(to + again * ld_dst + c) = t;
    return;
  }
  uint32_t v[kSpan / 64];
#pragma unroll
  for (uint32_t k = 0; k < kSpan / 64; ++k) {
    const uint32_t c = c0 + k * 64 + lane * 2;
    const uint32_t lo = live && c < cols ? from[c] : 0u;
    const uint32_t hi = live && c + 1 < cols ? from[c + 1] : 0u;
    v[k] = lo | hi << 16;
  }
#pragma unroll
  for (uint32_t k = 0; k < kSpan / 64; ++k) {
    const uint32_t c = c0 + k * 64 + lane * 2;
    if (c >= padded) continue;
    *reinterpret_cast<uint32_t *>(to + c) = v[k];
    if (again) *reinterpret_cast<uint32_t *>(to + again * ld_dst + c) = v[k];
  }
}

// Results from rows of 16 bytes in scratch into rows of any pitch.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    unpack_rows_kernel(const T *src, T *dst, uint32_t rows, uint32_t cols,
                       size_t ld_src, size_t ld_dst) {
  dependent_wait();
  const uint32_t spans = (cols + kSpan - 1) / kSpan;
  const uint32_t i = (blockIdx.x * kThreads + threadIdx.x) / 32, lane = threadIdx.x & 31;
  if (i >= rows * spans) return;
  const uint32_t r = i / spans, c0 = (i - r * spans) * kSpan;
  T v[kSpan / 32];
#pragma unroll
  for (uint32_t k = 0; k < kSpan / 32; ++k) {
    const uint32_t c = c0 + k * 32 + lane;
    if (c < cols) v[k] = src[r * ld_src + c];
  }
#pragma unroll
  for (uint32_t k = 0; k < kSpan / 32; ++k) {
    const uint32_t c = c0 + k * 32 + lane;
    if (c < cols) dst[r * ld_dst + c] = v[k];
  }
}

int pack_rows(BwppCudaCtx *ctx, const uint16_t *src, uint16_t *dst, uint32_t rows, uint32_t cols,
              uint32_t ld_src, uint32_t ld_dst, const int32_t *target, uint32_t V,
              uint32_t live_rows = 0xffffffffu, uint32_t again = 0, Common common = Common{}) {
  const uint32_t spans = (cols + kSpan - 1) / kSpan;
  const int wide = ld_src % 8 == 0 && aligned_to(src, 16);
  const uint32_t most = (1u << 25) / spans;  // rows of a launch: indices stay in 31 bits
  for (uint32_t r0 = 0; r0 < rows; r0 += most) {
    const uint32_t n = rows - r0 < most ? rows - r0 : most;
    const int rc = bwpp_check_cuda(
        ctx,
        bwpp_launch_dependent(pack_rows_kernel,
                              dim3((n * spans + kThreads / 32 - 1) / (kThreads / 32) + (common.out != nullptr)),
                              dim3(kThreads), 0, ctx->stream, src + (size_t)r0 * ld_src,
                              dst + (size_t)r0 * ld_dst, n, cols, ld_src, ld_dst, wide,
                              target ? target + r0 : nullptr, V, live_rows > r0 ? live_rows - r0 : 0, again,
                              common, ctx->status_word),
        "xent pack");
    if (rc) return rc;
    common.out = nullptr;  // the first launch found it, from all rows
  }
  return BWPP_CUDA_OK;
}

template <typename T>
int unpack_rows(BwppCudaCtx *ctx, const void *src, void *dst, uint32_t rows, uint32_t cols,
                uint32_t ld_src, uint32_t ld_dst) {
  const uint32_t spans = (cols + kSpan - 1) / kSpan;
  const uint32_t most = (1u << 25) / spans;
  for (uint32_t r0 = 0; r0 < rows; r0 += most) {
    const uint32_t n = rows - r0 < most ? rows - r0 : most;
    const int rc = bwpp_check_cuda(
        ctx,
        bwpp_launch_dependent(unpack_rows_kernel<T>,
                              dim3((n * spans + kThreads / 32 - 1) / (kThreads / 32)), dim3(kThreads), 0,
                              ctx->stream, static_cast<const T *>(src) + (size_t)r0 * ld_src,
                              static_cast<T *>(dst) + (size_t)r0 * ld_dst, n, cols, ld_src, ld_dst),
        "xent unpack");
    if (rc) return rc;
  }
  return BWPP_CUDA_OK;
}

inline uint32_t up8(uint32_t n) { return (n + 7) & ~7u; }
inline size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

// What a call keeps in scratch, as byte offsets.
struct Layout {
  uint32_t piece;             // vocabulary columns of a piece
  uint32_t dp;                // D rounded up
  // K parts of dx and of dW that scratch has room for, and the rows of one
  uint32_t dx_rows, dx_parts, dw_rows, dw_parts;
  uint32_t k_rows;            // backward: rows of x and dlogit in scratch
  size_t part, hit, x, w, dlogit, dx, dw, common, total;
};

// Equal pieces of about c columns, whole 256s, at least 1024.
uint32_t piece_of(uint64_t c, uint32_t V) {
  if (c < 1024) c = 1024;
  const uint64_t pieces = (V + c - 1) / c;
  return (uint32_t)((((uint64_t)V + pieces - 1) / pieces + 255) & ~255ull);
}

// K parts of a [rows, ld] product that fit 64 MB, at most eight.
uint32_t parts_that_fit(uint64_t rows, uint64_t ld) {
  const uint64_t fit = (64ull << 20) / (rows * ld * 4);
  return fit < 1 ? 1 : fit > 8 ? 8 : (uint32_t)fit;
}

// Vocabulary columns of a piece.  Backward: about 2^27 dlogit at a time (T 8192,
// V 32000, D 2048: 3300 us at 2^24, 2883 at 2^25, 2744 at 2^26, 2692 at 2^27,
// where dx is read and written back once; 2659 with all of them kept).
// Forward: the whole vocabulary, or about 2^25 weights at a time where they
// are packed.
Layout layout_of(const BwppCudaXentParams &p, bool pack_x, bool pack_w, bool backward, bool stage_dx,
                 bool stage_dw) {
  Layout l{};
  l.dp = up8(p.D);
  l.piece = backward ? piece_of((1ull << 27) / p.T, p.V)
                     : piece_of(pack_w ? (1ull << 25) / l.dp : (uint64_t)p.V, p.V);
  l.k_rows = p.T <= XENT_EXACT_ROWS ? 2 * XENT_EXACT_ROWS : p.T;
  l.dx_rows = (uint32_t)up256(l.k_rows);
  l.dx_parts = parts_that_fit(l.dx_rows, l.dp);
  l.dw_rows = (uint32_t)up256(p.w_vocab_major ? l.piece : p.D);
  l.dw_parts = parts_that_fit(l.dw_rows, p.w_vocab_major ? l.dp : l.piece);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += up256(bytes);
    return here;
  };
  const size_t es = p.grads_bf16 ? 2 : 4;
  if (pack_x || backward) l.x = take((size_t)(backward ? l.k_rows : p.T) * l.dp * 2);
  if (pack_w) l.w = take((size_t)l.piece * l.dp * 2);
  if (!backward) {
    l.part = take((((size_t)p.V + 127) / 128) * p.T * sizeof(float2));
    l.hit = take((size_t)p.T * 4);
  } else {
    l.common = take(2 * sizeof(float));
    l.dlogit = take((size_t)l.k_rows * l.piece * 2);
    if (stage_dx) l.dx = take((size_t)l.dx_parts * l.dx_rows * l.dp * 4);
    if (stage_dw || l.dw_parts > 1)
      l.dw = take((size_t)l.dw_parts * l.dw_rows * (p.w_vocab_major ? l.dp : l.piece) *
                  (l.dw_parts > 1 ? 4 : es));
  }
  l.total = at;
  return l;
}

// Sizes that the calls take: rounded up to tiles they stay below 2^31, as the
// 32-bit indices and TMA's coordinates need.
bool sizes_fit(const BwppCudaXentParams &p) {
  constexpr uint32_t most = 0x7ffffe00u;
  return p.V > 0 && p.D > 0 && p.V <= most && p.D <= most && p.T <= most;
}

int check(BwppCudaCtx *ctx, const BwppCudaXentParams *p) {
  if (!p) return bwpp_set_error(ctx, BWPP_CUDA_ERR_ARG, "xent: NULL params");
  if (!sizes_fit(*p))
    return bwpp_set_error(ctx, BWPP_CUDA_ERR_ARG,
                          "xent: V and D must be positive, T, V and D at most 2^31 - 512");
  if (p->ldx < p->D || p->ldw < (p->w_vocab_major ? p->D : p->V))
    return bwpp_set_error(ctx, BWPP_CUDA_ERR_ARG, "xent: leading dim smaller than row");
  if (!isfinite(p->scale)) return bwpp_set_error(ctx, BWPP_CUDA_ERR_ARG, "xent: scale is not finite");
  return BWPP_CUDA_OK;
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
  out = Piece{scratch, ld_packed};
  return pack_rows(ctx, src, scratch, rows, cols, p.ldw, ld_packed, nullptr, 0);
}

bool needs_pack(const void *base, uint32_t ld) { return ld % 8 != 0 || !aligned_to(base, 16); }

}  // namespace

extern "C" {

size_t bwpp_cuda_xent_workspace_size(const BwppCudaXentParams *p, int backward) {
  if (!p || p->T == 0 || !sizes_fit(*p)) return 0;
  // every copy that a call may need: which it makes depends on addresses as well
  return layout_of(*p, true, true, backward != 0, true, true).total + BWPP_OP_SCRATCH_PAD;
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
  uint32_t ldx = p.ldx;
  if (pack_x) {
    uint16_t *xp = reinterpret_cast<uint16_t *>(scratch + l.x);
    rc = pack_rows(ctx, x, xp, p.T, p.D, p.ldx, l.dp, nullptr, 0);
    if (rc) return rc;
    x = xp;
    ldx = l.dp;
  }
  float2 *part = reinterpret_cast<float2 *>(scratch + l.part);
  float *hit = reinterpret_cast<float *>(scratch + l.hit);
  for (uint32_t v0 = 0; v0 < p.V; v0 += l.piece) {
    const uint32_t n = p.V - v0 < l.piece ? p.V - v0 : l.piece;
    Piece w1;
    rc = piece_w(ctx, p, w, pack_w, reinterpret_cast<uint16_t *>(scratch + l.w), v0, n,
                 p.w_vocab_major ? l.dp : l.piece, w1);
    const XentOperands o{x, w1.w, p.T, n, p.D, ldx, w1.ld, v0, p.V, p.w_vocab_major != 0, p.scale};
    if (!rc)
      rc = bwpp_xent_stats_launch(ctx, o, loss ? target : nullptr, part + (size_t)(v0 / 128) * p.T, hit);
    if (rc) return rc;
  }
  return bwpp_xent_combine_launch(ctx, part, (p.V + 127) / 128, hit, target, loss, lse, p.T, p.V);
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
  if (p.T == 0) {  // no rows: dW is zero
    if (!dw) return BWPP_CUDA_OK;
    return bwpp_check_cuda(
        ctx,
        cudaMemset2DAsync(dw, (size_t)p.lddw * es, 0, (size_t)(p.w_vocab_major ? p.D : p.V) * es,
                          p.w_vocab_major ? p.V : p.D, ctx->stream),
        "xent memset");
  }
  if (!dx && !dw) return BWPP_CUDA_OK;
  if (!x || !w || !target || !lse)
    return bwpp_set_error(ctx, BWPP_CUDA_ERR_ARG, "xent bwd: NULL buffer");
  const bool pack_w = needs_pack(w, p.ldw);
  auto tma_out = [&](const void *q, uint32_t ld) { return (size_t)ld * es % 16 == 0 && aligned_to(q, 16); };
  const bool dx_out = dx && tma_out(dx, p.lddx), stage_dw = dw && !tma_out(dw, p.lddw);
  const Layout probe = layout_of(p, true, pack_w, true, true, true);
  const uint32_t piece = probe.piece, pieces = (p.V - 1) / piece + 1;
  const bool vm = p.w_vocab_major != 0;
  const uint32_t ld_w = pack_w ? (vm ? probe.dp : piece) : p.ldw;
  // The products of the piece [v0, v0 + n), with no addresses yet.
  auto products = [&](uint32_t n, XentProduct &px, XentProduct &pw) {
    px = XentProduct{};
    px.M = probe.k_rows;
    px.N = p.D;
    px.K = n;
    px.lda = piece;
    px.ldb = ld_w;
    px.b_mn = vm;  // W's rows are K here
    px.ldc = px.ld_add = probe.dp;
    px.part_rows = probe.dx_rows;
    pw = XentProduct{};
    pw.M = vm ? n : p.D;
    pw.N = vm ? p.D : n;
    pw.K = probe.k_rows;
    pw.lda = vm ? piece : probe.dp;
    pw.ldb = vm ? probe.dp : piece;
    pw.a_mn = pw.b_mn = true;
    pw.part_rows = probe.dw_rows;
  };
  XentProduct px, pw;
  products(piece < p.V ? piece : p.V, px, pw);
  // K parts, the same whether both gradients are wanted or one, so that each
  // comes out the same
  uint32_t dx_parts, dw_parts;
  rc = bwpp_xent_parts(ctx, px, pw, probe.dx_parts, probe.dw_parts, &dx_parts, &dw_parts);
  if (rc) return rc;
  // few rows: two bf16 for each dlogit, XENT_EXACT_ROWS apart, which are summed here
  const bool exact = p.T <= XENT_EXACT_ROWS;
  // dx is summed in scratch, unless the caller's rows take it: all of it in one
  // piece, or fp32 sums
  const bool one_sum = dx_out && dx_parts == 1 && !exact;
  const bool direct = one_sum && (pieces == 1 || !p.grads_bf16);
  const Layout l = layout_of(p, true, pack_w, true, dx && !direct, stage_dw);
  uint8_t *scratch;
  rc = bwpp_op_scratch(ctx, l.total, "xent bwd", &scratch);
  if (rc) return rc;
  uint16_t *xp = reinterpret_cast<uint16_t *>(scratch + l.x);
  float *common = exact ? nullptr : reinterpret_cast<float *>(scratch + l.common);
  rc = exact ? pack_rows(ctx, x, xp, XENT_EXACT_ROWS, p.D, p.ldx, l.dp, target, p.V, p.T, XENT_EXACT_ROWS)
             : pack_rows(ctx, x, xp, p.T, p.D, p.ldx, l.dp, target, p.V, p.T, 0,
                         Common{dloss, p.T, p.scale, common});
  if (rc) return rc;
  uint16_t *dlogit = reinterpret_cast<uint16_t *>(scratch + l.dlogit);
  for (uint32_t v0 = 0; v0 < p.V; v0 += piece) {
    const uint32_t n = p.V - v0 < piece ? p.V - v0 : piece;
    const bool last = v0 + n == p.V;
    Piece w1;
    rc = piece_w(ctx, p, w, pack_w, reinterpret_cast<uint16_t *>(scratch + l.w), v0, n,
                 vm ? l.dp : piece, w1);
    const XentOperands o{xp, w1.w, p.T, n, p.D, l.dp, w1.ld, v0, p.V, vm, p.scale};
    if (!rc) rc = bwpp_xent_dlogit_launch(ctx, o, target, lse, dloss, common, dlogit, piece);
    if (rc) return rc;
    products(n, px, pw);
    px.a = dlogit;
    px.b = w1.w;
    px.accumulate = v0 > 0;
    // the last piece leaves the sum in the caller's rows where it can
    const bool to_user = direct || (one_sum && last);
    px.add = direct ? dx : static_cast<void *>(scratch + l.dx);
    px.ld_add = direct ? p.lddx : l.dp;
    px.c = to_user ? dx : static_cast<void *>(scratch + l.dx);
    px.ldc = to_user ? p.lddx : l.dp;
    px.bf16 = to_user && last && p.grads_bf16;
    px.guarded = to_user;
    px.factor = to_user && last ? common : nullptr;
    uint8_t *user_w =
        dw ? static_cast<uint8_t *>(dw) + (vm ? (size_t)v0 * p.lddw : (size_t)v0) * es : nullptr;
    const bool own_w = stage_dw || dw_parts > 1;  // dW's part goes through scratch
    pw.a = vm ? dlogit : xp;
    pw.b = vm ? xp : dlogit;
    pw.c = own_w ? static_cast<void *>(scratch + l.dw) : static_cast<void *>(user_w);
    pw.ldc = own_w ? (vm ? l.dp : piece) : p.lddw;
    pw.bf16 = p.grads_bf16 && dw_parts == 1;
    pw.guarded = !own_w;
    pw.factor = dw_parts == 1 ? common : nullptr;
    rc = bwpp_xent_grad_launch(ctx, dx ? &px : nullptr, dw ? &pw : nullptr, dx_parts, dw_parts);
    if (!rc && dw && dw_parts > 1)
      rc = bwpp_xent_sum_parts_launch(ctx, static_cast<const float *>(pw.c), dw_parts,
                                      (size_t)l.dw_rows * pw.ldc, 0, common, user_w, pw.M, pw.N, pw.ldc,
                                      p.lddw, p.grads_bf16);
    else if (!rc && stage_dw)
      rc = p.grads_bf16 ? unpack_rows<uint16_t>(ctx, pw.c, user_w, pw.M, pw.N, pw.ldc, p.lddw)
                        : unpack_rows<float>(ctx, pw.c, user_w, pw.M, pw.N, pw.ldc, p.lddw);
    if (rc) return rc;
  }
  if (dx && !one_sum) {
    return bwpp_xent_sum_parts_launch(ctx, reinterpret_cast<const float *>(scratch + l.dx), dx_parts,
                                      (size_t)l.dx_rows * l.dp, exact ? XENT_EXACT_ROWS * (size_t)l.dp : 0,
                                      common, dx, p.T, p.D, l.dp, p.lddx, p.grads_bf16);
  }
  return BWPP_CUDA_OK;
}

}  // extern "C"

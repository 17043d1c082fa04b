// Rotary positions on q and k, forward and gradient, f16 / bf16 / fp32.
//
// Pair i of a head turns by position * f_i:
//   (y0, y1) = a (x0 cos - x1 sin, x1 cos + x0 sin)
// over pairs (i, i + R/2) or, interleaved, (2i, 2i + 1) of the first R
// columns of each head; the columns behind R are copied (left alone in place).
// The map is a rotation times the amplitude a, so its gradient is the same
// kernel turning back.
//
// Angles.  The table holds each frequency as a 64-bit fraction of a turn, and
// position * fraction mod 2^64 is the angle's fraction of a turn: the whole
// turns, which carry no information, drop out exactly for any 32-bit position
// (an fp32 product is 0.03 rad off at position 10^6).  The top 32 bits go to
// sincospif, whose argument is then within [-1, 1), rounded to fp32: results are off by
// 5.5e-8 of their norm, 4.2e-8 with 64-bit angles.
#include <math.h>

#include "bwpp_cuda_internal.cuh"
#include "elem.cuh"

namespace {

using bwpp_elem::aligned_to;
using bwpp_elem::Elem;
using bwpp_elem::Raw;

constexpr int kThreads = 256;

struct RopeArgs {
  BwppCudaRopeTable table;
  const void *q, *k;
  void *qo, *ko;
  const int32_t *positions;
  BwppCudaRopeParams p;
  uint32_t seq;     // p.seq, or tokens where it is 0
  uint32_t token0;  // first token of this launch
  uint32_t units;   // threads with work: tokens * slots * lanes
  uint32_t turn_slots, slots, lanes;
};

// Heads that a thread loads before it turns any: 128 bytes in flight.  (For
// 32768 tokens x 32 heads x 128 bf16: 109 us with one head, 90 with two, 82.5
// with four, 84 with eight.)
constexpr int batch_of(bool one_vector) { return one_vector ? 8 : 4; }

// A thread owns one slot (VEC pairs, or VEC columns behind R) of one token in
// heads lane, lane + lanes, ... of q and then of k: its sines and cosines are
// computed once for all of them, behind the first loads.
//
// SINGLE: at most one head of each, loaded together: q's and k's transfers are all
// that a thread has in flight, so its registers are few and the threads many.  The
// turns come from shared memory: a warp's slots are different addresses of the
// constant bank, read one after another for each head.  (89658 tokens, one head of
// 196 each, bf16: 105 us as one batch of q and one of k, 78 together, 46 with shared
// turns; with many heads a thread, shared turns were 1-8% slower.)
template <int DT, int VEC, bool IL, bool SINGLE>
__global__ void __launch_bounds__(kThreads) rope_kernel(const __grid_constant__ RopeArgs a) {
  using T = typename Elem<DT>::type;
  constexpr bool ONE = IL && VEC > 1;  // a vector holds both sides of its pairs
  constexpr int PAIRS = ONE ? VEC / 2 : VEC;
  constexpr int kBatch = batch_of(ONE);
  __shared__ uint64_t shared_turns[SINGLE ? BWPP_CUDA_ROPE_MAX_PAIRS : 1];
  if constexpr (SINGLE) {
    for (uint32_t i = threadIdx.x; i < a.table.pairs; i += kThreads) shared_turns[i] = a.table.turns[i];
    __syncthreads();
  }
  dependent_wait();
  const uint32_t id = blockIdx.x * kThreads + threadIdx.x;
  if (id >= a.units) return;
  const uint32_t per = a.slots * a.lanes;
  const uint32_t n = id / per, rem = id - n * per, t = a.token0 + n;
  const uint32_t lane = rem / a.slots, slot = rem - lane * a.slots;
  const uint32_t b = t / a.seq, s = t - b * a.seq;
  const bool turns = slot < a.turn_slots;
  const bool two = !ONE && turns;
  const uint32_t half = a.table.pairs;
  uint32_t c0, c1 = 0;  // columns of the slot's two vectors
  if (!turns) {
    c0 = 2 * half + (slot - a.turn_slots) * VEC;
  } else if (IL) {
    c0 = ONE ? slot * VEC : 2 * slot;
    c1 = c0 + 1;
  } else {
    c0 = slot * VEC;
    c1 = c0 + half;
  }
  float cs[PAIRS], sn[PAIRS];
  bool ready = !turns;
  auto angles = [&]() {
    const int64_t pos =
        a.positions ? (int64_t)a.positions[t] : (int64_t)a.p.pos0 + (int64_t)s;
    const float up = a.table.amplitude, side = a.p.inverse ? -up : up;
#pragma unroll
    for (int i = 0; i < PAIRS; ++i) {
      const uint64_t turn = (uint64_t)pos * (SINGLE ? shared_turns[slot * PAIRS + i] : a.table.turns[slot * PAIRS + i]);
      sincospif((float)(int32_t)(turn >> 32) * 0x1p-31f, &sn[i], &cs[i]);
      cs[i] *= up;
      sn[i] *= side;
    }
    ready = true;
  };
  if constexpr (SINGLE) {
    const uint32_t side = c1 - c0;
    auto at = [&](int head_major, uint32_t heads, size_t ld) {  // of this thread's head
      return c0 + (head_major ? ((size_t)b * heads + lane) * a.seq * ld + s * ld
                              : t * ld + (size_t)lane * a.p.head_dim);
    };
    const T *from[2] = {static_cast<const T *>(a.q) + at(a.p.head_major_in, a.p.heads_q, a.p.ldq),
                        static_cast<const T *>(a.k) + at(a.p.head_major_in, a.p.heads_k, a.p.ldk)};
    T *into[2] = {static_cast<T *>(a.qo) + at(a.p.head_major_out, a.p.heads_q, a.p.ldq_out),
                  static_cast<T *>(a.ko) + at(a.p.head_major_out, a.p.heads_k, a.p.ldk_out)};
    const bool in[2] = {lane < a.p.heads_q, lane < a.p.heads_k};
    Raw<DT, VEC> x[2], y[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (in[u]) x[u].load(from[u]);
      if (in[u] && two) y[u].load(from[u] + side);
    }
    if (turns) angles();
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      if (!in[u]) continue;
      if (turns) {
        float v[VEC];
        if constexpr (ONE) {
#pragma unroll
          for (int i = 0; i < PAIRS; ++i) {
            const float x0 = x[u].get(2 * i), x1 = x[u].get(2 * i + 1);
            v[2 * i] = x0 * cs[i] - x1 * sn[i];
            v[2 * i + 1] = x1 * cs[i] + x0 * sn[i];
          }
        } else {
          float w[VEC];
#pragma unroll
          for (int i = 0; i < VEC; ++i) {
            const float x0 = x[u].get(i), x1 = y[u].get(i);
            v[i] = x0 * cs[i] - x1 * sn[i];
            w[i] = x1 * cs[i] + x0 * sn[i];
          }
          y[u].set(w);
          y[u].store(into[u] + side);
        }
        x[u].set(v);
      }
      x[u].store(into[u]);
    }
    return;
  }
  auto pass = [&](const void *from, void *into, uint32_t heads, size_t ldi, size_t ldo) {
    const size_t di = a.p.head_major_in ? (size_t)a.seq * ldi : a.p.head_dim;
    const size_t dn = a.p.head_major_out ? (size_t)a.seq * ldo : a.p.head_dim;
    const T *src = static_cast<const T *>(from) + c0 +
                   (a.p.head_major_in ? (size_t)b * heads * di + s * ldi : t * ldi);
    T *dst = static_cast<T *>(into) + c0 +
             (a.p.head_major_out ? (size_t)b * heads * dn + s * ldo : t * ldo);
    const uint32_t side = c1 - c0;
    for (uint32_t h0 = lane; h0 < heads; h0 += kBatch * a.lanes) {
      Raw<DT, VEC> x[kBatch], y[ONE ? 1 : kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const uint32_t h = h0 + u * a.lanes;
        if (h < heads) {
          x[u].load(src + h * di);
          if constexpr (!ONE)
            if (two) y[u].load(src + h * di + side);
        }
      }
      if (!ready) angles();
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const uint32_t h = h0 + u * a.lanes;
        if (h >= heads) break;
        if (turns) {
          float v[VEC];
          if constexpr (ONE) {
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) {
              const float x0 = x[u].get(2 * i), x1 = x[u].get(2 * i + 1);
              v[2 * i] = x0 * cs[i] - x1 * sn[i];
              v[2 * i + 1] = x1 * cs[i] + x0 * sn[i];
            }
          } else {
            float w[VEC];
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              const float x0 = x[u].get(i), x1 = y[u].get(i);
              v[i] = x0 * cs[i] - x1 * sn[i];
              w[i] = x1 * cs[i] + x0 * sn[i];
            }
            y[u].set(w);
            y[u].store(dst + h * dn + side);
          }
          x[u].set(v);
        }
        x[u].store(dst + h * dn);
      }
    }
  };
  pass(a.q, a.qo, a.p.heads_q, a.p.ldq, a.p.ldq_out);
  pass(a.k, a.ko, a.p.heads_k, a.p.ldk, a.p.ldk_out);
}

template <int DT, int VEC>
int rope_launch(BwppCudaCtx *ctx, RopeArgs &a) {
  const BwppCudaRopeParams &p = a.p;
  const uint32_t R = 2 * a.table.pairs;
  const bool pairs_in_one = p.interleaved && VEC > 1;
  a.turn_slots = (pairs_in_one ? R : R / 2) / VEC;
  const bool in_place = a.qo == a.q && a.ko == a.k;
  a.slots = a.turn_slots + (in_place ? 0 : (p.head_dim - R) / VEC);
  // A thread per head and slot for few tokens, where latency counts; a thread
  // takes a batch of heads of q and of k where that still leaves 1024 threads
  // per SM (4084 tokens x 32 heads x 128 fp32: 33.7 us without, 23.2 with).  One or
  // two heads are no batch (65536 tokens x 2 + 2 heads of 128, interleaved bf16: 38.5
  // us as one, 29 as SINGLE; 4 + 1 heads: 39.8 and 52.9).
  const uint32_t kBatch = batch_of(pairs_in_one);
  a.lanes = p.heads_q > p.heads_k ? p.heads_q : p.heads_k;
  if (a.lanes > 2 && (uint64_t)p.tokens * a.slots * a.lanes > (uint64_t)ctx->num_sms * 1024 * kBatch)
    a.lanes = (a.lanes + kBatch - 1) / kBatch;
  const bool single = a.lanes >= p.heads_q && a.lanes >= p.heads_k;
  const uint64_t per = (uint64_t)a.slots * a.lanes;
  const uint64_t most = (1u << 30) / per;  // tokens of a launch: unit ids stay in 31 bits
  if (most == 0)
    return bwpp_set_error(ctx, BWPP_CUDA_ERR_UNSUPPORTED, "rope: heads * head_dim too large");
  for (uint64_t t0 = 0; t0 < p.tokens; t0 += most) {
    const uint64_t n = p.tokens - t0 < most ? p.tokens - t0 : most;
    a.token0 = (uint32_t)t0;
    a.units = (uint32_t)(n * per);
    const uint32_t grid = (a.units + kThreads - 1) / kThreads;
    auto kernel = single ? (p.interleaved ? rope_kernel<DT, VEC, true, true> : rope_kernel<DT, VEC, false, true>)
                         : (p.interleaved ? rope_kernel<DT, VEC, true, false> : rope_kernel<DT, VEC, false, false>);
    const int rc = bwpp_check_cuda(
        ctx, bwpp_launch_dependent(kernel, dim3(grid), dim3(kThreads), 0, ctx->stream, a), "rope");
    if (rc) return rc;
  }
  return BWPP_CUDA_OK;
}

template <int DT>
int rope(BwppCudaCtx *ctx, const void *q, const void *k, void *qo, void *ko,
         const int32_t *positions, const BwppCudaRopeTable *table, const BwppCudaRopeParams *pp) {
  int rc = bwpp_ctx_enter(ctx);
  if (rc) return rc;
  if (!table || !pp) return bwpp_set_error(ctx, BWPP_CUDA_ERR_ARG, "rope: NULL table or params");
  const BwppCudaRopeParams &p = *pp;
  const uint32_t R = 2 * table->pairs;
  if (table->pairs == 0 || table->pairs > BWPP_CUDA_ROPE_MAX_PAIRS || R > p.head_dim)
    return bwpp_set_error(ctx, BWPP_CUDA_ERR_ARG, "rope: table of %u pairs for head_dim %u",
                          table->pairs, p.head_dim);
  // a thread's head index steps past the last head, in 32 bits
  if (p.heads_q > 0x7fffffffu || p.heads_k > 0x7fffffffu)
    return bwpp_set_error(ctx, BWPP_CUDA_ERR_ARG, "rope: more than 2^31 - 1 heads");
  if (p.tokens == 0 || (p.heads_q == 0 && p.heads_k == 0)) return BWPP_CUDA_OK;
  if ((p.heads_q && (!q || !qo)) || (p.heads_k && (!k || !ko)))
    return bwpp_set_error(ctx, BWPP_CUDA_ERR_ARG, "rope: NULL buffer");
  const uint64_t rq = (uint64_t)p.heads_q * p.head_dim, rk = (uint64_t)p.heads_k * p.head_dim;
  if ((p.heads_q && (p.ldq < (p.head_major_in ? p.head_dim : rq) ||
                     p.ldq_out < (p.head_major_out ? p.head_dim : rq))) ||
      (p.heads_k && (p.ldk < (p.head_major_in ? p.head_dim : rk) ||
                     p.ldk_out < (p.head_major_out ? p.head_dim : rk))))
    return bwpp_set_error(ctx, BWPP_CUDA_ERR_ARG, "rope: leading dim smaller than row");
  const uint32_t seq = p.seq ? p.seq : p.tokens;
  if ((p.head_major_in || p.head_major_out) && p.tokens % seq)
    return bwpp_set_error(ctx, BWPP_CUDA_ERR_ARG, "rope: tokens is not a multiple of seq");
  const bool same = (p.head_major_in != 0) == (p.head_major_out != 0);
  if ((p.heads_q && q == qo && !(same && p.ldq == p.ldq_out)) ||
      (p.heads_k && k == ko && !(same && p.ldk == p.ldk_out)))
    return bwpp_set_error(ctx, BWPP_CUDA_ERR_ARG, "rope: in place needs one layout and pitch");
  RopeArgs a{};
  a.table = *table;
  a.q = q;
  a.k = p.heads_k ? k : q;
  a.qo = qo;
  a.ko = p.heads_k ? ko : qo;
  if (!p.heads_q) {
    a.q = k;
    a.qo = ko;
  }
  a.positions = positions;
  a.p = p;
  a.seq = seq;
  // the widest transfer that every address and the pairs' halves allow
  constexpr int ES = (int)sizeof(typename Elem<DT>::type);
  auto fits = [&](uint32_t v) {
    if (p.head_dim % v || (p.interleaved ? R : R / 2) % v || R % v) return false;
    if (p.heads_q && (p.ldq % v || p.ldq_out % v || !aligned_to(q, v * ES) || !aligned_to(qo, v * ES)))
      return false;
    if (p.heads_k && (p.ldk % v || p.ldk_out % v || !aligned_to(k, v * ES) || !aligned_to(ko, v * ES)))
      return false;
    return true;
  };
  if constexpr (ES == 2) {
    if (fits(8)) return rope_launch<DT, 8>(ctx, a);
  }
  if (fits(4)) return rope_launch<DT, 4>(ctx, a);
  if (fits(2)) return rope_launch<DT, 2>(ctx, a);
  return rope_launch<DT, 1>(ctx, a);
}

}  // namespace

extern "C" {

int bwpp_cuda_rope_table(BwppCudaRopeTable *out, const BwppCudaRopeConfig *cfg) {
  if (!out || !cfg) return BWPP_CUDA_ERR_ARG;
  const uint32_t R = cfg->rotary_dim;
  if (R == 0 || (R & 1) || R / 2 > BWPP_CUDA_ROPE_MAX_PAIRS) return BWPP_CUDA_ERR_ARG;
  if (!(cfg->base > 0) || !isfinite(cfg->base) || !(cfg->amplitude > 0) || !isfinite(cfg->amplitude))
    return BWPP_CUDA_ERR_ARG;
  const bool scaled = cfg->scaling != BWPP_CUDA_ROPE_NONE;
  if (scaled && (!(cfg->factor > 0) || !isfinite(cfg->factor))) return BWPP_CUDA_ERR_ARG;
  double base = cfg->base;
  switch (cfg->scaling) {
    case BWPP_CUDA_ROPE_NONE:
    case BWPP_CUDA_ROPE_LINEAR: break;
    case BWPP_CUDA_ROPE_BASE:
      if (R == 2) return BWPP_CUDA_ERR_ARG;  // one pair does not depend on the base
      base *= pow(cfg->factor, (double)R / (R - 2));
      if (!(base > 0) || !isfinite(base)) return BWPP_CUDA_ERR_ARG;
      break;
    case BWPP_CUDA_ROPE_PARTS:
      if (!(cfg->context > 0) || !isfinite(cfg->context) || !(cfg->high > cfg->low) ||
          !isfinite(cfg->high) || !isfinite(cfg->low))
        return BWPP_CUDA_ERR_ARG;
      break;
    default: return BWPP_CUDA_ERR_ARG;
  }
  const double two_pi = 6.283185307179586476925286766559;
  BwppCudaRopeTable t = {};
  t.pairs = R / 2;
  t.amplitude = cfg->amplitude;
  for (uint32_t i = 0; i < R / 2; ++i) {
    double f = pow(base, -2.0 * i / R);  // radians per position
    if (cfg->scaling == BWPP_CUDA_ROPE_LINEAR) f /= cfg->factor;
    if (cfg->scaling == BWPP_CUDA_ROPE_PARTS) {
      double keep = (cfg->context * f / two_pi - cfg->low) / (cfg->high - cfg->low);
      keep = keep < 0 ? 0 : keep > 1 ? 1 : keep;
      f = f * keep + f / cfg->factor * (1 - keep);
    }
    const double turn = f / two_pi;
    if (!isfinite(turn)) return BWPP_CUDA_ERR_ARG;
    // whole turns per position drop out; ldexp is exact, llrint would not fit
    const double frac = turn - floor(turn);
    t.turns[i] = (uint64_t)ldexp(frac, 64);
  }
  *out = t;
  return BWPP_CUDA_OK;
}

int bwpp_cuda_rope_bf16(BwppCudaCtx *ctx, const uint16_t *q, const uint16_t *k, uint16_t *q_out,
                        uint16_t *k_out, const int32_t *positions, const BwppCudaRopeTable *table,
                        const BwppCudaRopeParams *params) {
  return rope<BWPP_CUDA_DTYPE_BF16>(ctx, q, k, q_out, k_out, positions, table, params);
}

int bwpp_cuda_rope_f16(BwppCudaCtx *ctx, const uint16_t *q, const uint16_t *k, uint16_t *q_out,
                       uint16_t *k_out, const int32_t *positions, const BwppCudaRopeTable *table,
                       const BwppCudaRopeParams *params) {
  return rope<BWPP_CUDA_DTYPE_F16>(ctx, q, k, q_out, k_out, positions, table, params);
}

int bwpp_cuda_rope_f32(BwppCudaCtx *ctx, const float *q, const float *k, float *q_out, float *k_out,
                       const int32_t *positions, const BwppCudaRopeTable *table,
                       const BwppCudaRopeParams *params) {
  return rope<BWPP_CUDA_DTYPE_F32>(ctx, q, k, q_out, k_out, positions, table, params);
}

}  // extern "C"

// The junction between two blocks of a decoder, forward and gradient: the
// norm after a block, its gate and the scaled residual sum, and the norm
// before the next block, in one pass over the rows.
//
//   u  = b / rms(b) * gain_post  (norm_after; else u = b)
//   h' = scale_h h + scale_b gate u
//   y  = h' / rms(h') * gain_pre            rms(x) = sqrt(mean(x^2) + eps)
//
// Gradient, with g = gain_pre dy, hat = h' / rms(h'), bhat = b / rms(b):
//   dH = dh' + (g - hat mean(g hat)) / rms(h')
//   dh = scale_h dH,  e = scale_b dH,  dgate = sum e u,  du = gate e
//   db = (gain_post du - bhat mean(gain_post du bhat)) / rms(b)
//   dgain_post = sum du bhat,  dgain_pre = sum dy hat
// The statistics are recomputed from the rows, which are read anyway.
//
// h, h', gains and gates are fp32; b, y, db, dy are fp32, bf16 or f16.  All
// arithmetic is fp32; y and db are rounded once.  HBM-bound: a row is held in
// registers, read once and written once.
//
// Column sums (deterministic): a CTA walks a chunk of consecutive rows that
// share one gate row and keeps sum e bhat (or sum e b) and sum dy hat of its
// columns in registers, then writes one partial row per chunk.  A second
// kernel adds the partial rows in a fixed order: dgain_post weights each
// with its chunk's gate row, dgate adds those of its group.
#include <atomic>

#include "bwpp_cuda_internal.cuh"
#include "elem.cuh"
#include "rowwise.cuh"

namespace {

using bwpp_elem::aligned_to;
using bwpp_elem::Elem;
using bwpp_elem::Raw;
using bwpp_row::block_sum;

constexpr int F32 = BWPP_CUDA_DTYPE_F32;

struct JunctionArgs {
  BwppCudaJunctionParams p;  // gate_rows > 0
  const float *h;            // forward: h; backward: h'
  const void *b;
  const float *gain_post, *gate, *gain_pre;
  float *h_out;              // forward: h'
  void *y;                   // forward
  const float *dh_out;       // backward from here on
  const void *dy;
  float *dh;
  void *db;
  float *dgate;              // written by the row kernel when gate_rows == 1
  float *part_post, *part_pre;  // [chunks][cols] or NULL
  uint32_t chunk_rows, chunks_per_group, group_rows;
};

// Sums NV values over the TPR threads of a row.
template <int TPR, int NV>
__device__ __forceinline__ void row_sum(float (&v)[NV], float *red) {
  if constexpr (TPR <= 32) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int o = TPR / 2; o > 0; o >>= 1) v[j] += __shfl_xor_sync(0xffffffffu, v[j], o);
  } else {
    block_sum<NV>(v, red);
  }
}

template <int VEC>
__device__ __forceinline__ void load_gain(const float *g, uint32_t c, float (&o)[VEC]) {
  if (!g) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) o[e] = 1.0f;
  } else if constexpr (VEC >= 4) {
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) {
      const float4 t = *(reinterpret_cast<const float4 *>(g + c) + i);
      o[4 * i] = t.x; o[4 * i + 1] = t.y; o[4 * i + 2] = t.z; o[4 * i + 3] = t.w;
    }
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) o[e] = g[c + e];
  }
}

// Rows of up to 32 threads share a block of 128.
constexpr int block_threads(int tpr) { return tpr <= 32 ? 128 : tpr; }

// ---- forward -----------------------------------------------------------------

// TPR threads hold a row, thread t the vectors t, t + TPR, ... (NV of them).
template <int DT, int VEC, int NV, int TPR>
__global__ void __launch_bounds__(block_threads(TPR))
    junction_fwd_kernel(const __grid_constant__ JunctionArgs a) {
  using T = typename Elem<DT>::type;
  __shared__ float red[32];
  dependent_wait();
  const BwppCudaJunctionParams &p = a.p;
  const uint32_t at = blockIdx.x * (block_threads(TPR) / TPR) + threadIdx.x / TPR;
  const bool live = at < p.rows;  // threads past the last row go along with it
  const uint32_t r = live ? at : p.rows - 1;
  const uint32_t t = threadIdx.x % TPR;
  const float *h = a.h + (size_t)r * p.ldh;
  const T *b = static_cast<const T *>(a.b) + (size_t)r * p.ldb;
  const float *gate = a.gate ? a.gate + (size_t)(r / p.gate_rows) * p.ldgate : nullptr;
  Raw<F32, VEC> hv[NV];
  Raw<DT, VEC> bv[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const uint32_t c = (t + i * TPR) * VEC;
    if (c < p.cols) {
      hv[i].load(h + c);
      bv[i].load(b + c);
    } else {
      hv[i].zero();
      bv[i].zero();
    }
  }
  float rb = 1.0f;
  if (p.norm_after) {
    float ss[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) ss[0] += bv[i].get(e) * bv[i].get(e);
    row_sum<TPR, 1>(ss, red);
    rb = 1.0f / sqrtf(ss[0] / (float)p.cols + p.eps_post);
  }
  float ss[1] = {0.0f};
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const uint32_t c = (t + i * TPR) * VEC;
    if (c >= p.cols) continue;
    float gp[VEC], gt[VEC], v[VEC];
    load_gain<VEC>(p.norm_after ? a.gain_post : nullptr, c, gp);
    load_gain<VEC>(gate, c, gt);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float u = bv[i].get(e) * rb * gp[e];
      v[e] = p.scale_h * hv[i].get(e) + p.scale_b * (gt[e] * u);
      ss[0] += v[e] * v[e];
    }
    hv[i].set(v);
    if (live) hv[i].store(a.h_out + (size_t)r * p.ldh + c);
  }
  if (!a.y) return;
  row_sum<TPR, 1>(ss, red);
  const float rh = 1.0f / sqrtf(ss[0] / (float)p.cols + p.eps_pre);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const uint32_t c = (t + i * TPR) * VEC;
    if (c >= p.cols) continue;
    float gq[VEC], v[VEC];
    load_gain<VEC>(a.gain_pre, c, gq);
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = hv[i].get(e) * rh * gq[e];
    Raw<DT, VEC> o;
    o.set(v);
    if (live) o.store(static_cast<T *>(a.y) + (size_t)r * p.ldy + c);
  }
}

constexpr int kLoopThreads = 1024;

// Rows of any width, read again for each step (a thread keeps to its own
// columns, so it sees its own stores).
template <int DT>
__global__ void __launch_bounds__(kLoopThreads)
    junction_fwd_looped_kernel(const __grid_constant__ JunctionArgs a) {
  using T = typename Elem<DT>::type;
  __shared__ float red[32];
  dependent_wait();
  const BwppCudaJunctionParams &p = a.p;
  const uint32_t r = blockIdx.x;
  const float *h = a.h + (size_t)r * p.ldh;
  const T *b = static_cast<const T *>(a.b) + (size_t)r * p.ldb;
  const float *gate = a.gate ? a.gate + (size_t)(r / p.gate_rows) * p.ldgate : nullptr;
  float *ho = a.h_out + (size_t)r * p.ldh;
  Raw<DT, 1> x;
  float rb = 1.0f;
  if (p.norm_after) {
    float ss[1] = {0.0f};
    for (uint32_t c = threadIdx.x; c < p.cols; c += kLoopThreads) {
      x.load(b + c);
      ss[0] += x.get(0) * x.get(0);
    }
    block_sum<1>(ss, red);
    rb = 1.0f / sqrtf(ss[0] / (float)p.cols + p.eps_post);
  }
  float ss[1] = {0.0f};
  for (uint32_t c = threadIdx.x; c < p.cols; c += kLoopThreads) {
    x.load(b + c);
    float u = x.get(0) * rb;
    if (p.norm_after && a.gain_post) u *= a.gain_post[c];
    if (gate) u *= gate[c];
    const float v = p.scale_h * h[c] + p.scale_b * u;
    ho[c] = v;
    ss[0] += v * v;
  }
  if (!a.y) return;
  block_sum<1>(ss, red);
  const float rh = 1.0f / sqrtf(ss[0] / (float)p.cols + p.eps_pre);
  for (uint32_t c = threadIdx.x; c < p.cols; c += kLoopThreads) {
    const float v[1] = {ho[c] * rh * (a.gain_pre ? a.gain_pre[c] : 1.0f)};
    x.set(v);
    x.store(static_cast<T *>(a.y) + (size_t)r * p.ldy + c);
  }
}

// ---- backward ----------------------------------------------------------------

// The rows [first, last) of chunk k.
__device__ __forceinline__ void chunk_range(const JunctionArgs &a, uint32_t k, uint32_t &first,
                                            uint32_t &last) {
  const uint32_t g = k / a.chunks_per_group;
  const uint64_t begin = (uint64_t)g * a.group_rows;
  const uint64_t end = min(begin + a.group_rows, (uint64_t)a.p.rows);
  const uint64_t f = begin + (uint64_t)(k - g * a.chunks_per_group) * a.chunk_rows;
  first = (uint32_t)min(f, end);
  last = (uint32_t)min(f + a.chunk_rows, end);
}

// Sums NV values over the TPR threads of a row with one barrier; `red` may be
// used again once another barrier of the block has passed.
template <int TPR, int NV>
__device__ __forceinline__ void row_sum_once(float (&v)[NV], float (*red)[32]) {
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1)
      v[j] += __shfl_xor_sync(0xffffffffu, v[j], o);
  if constexpr (TPR > 32) {
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int j = 0; j < NV; ++j) red[j][threadIdx.x >> 5] = v[j];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      v[j] = red[j][0];
#pragma unroll
      for (int w = 1; w < TPR / 32; ++w) v[j] += red[j][w];
    }
  }
}

// Rows in registers: narrow ones, a warp each, and those that 16-byte pieces
// do not fit.  A row's loads are issued before the row in front of it is
// worked on; gains and the chunk's gate row stay in registers.
template <int DT, int VEC, int NV, int TPR>
__global__ void __launch_bounds__(block_threads(TPR))
    junction_bwd_kernel(const __grid_constant__ JunctionArgs a) {
  using T = typename Elem<DT>::type;
  constexpr int RPB = block_threads(TPR) / TPR;  // rows that a block works on together
  __shared__ float red[3][32], red1[1][32];
  dependent_wait();
  const BwppCudaJunctionParams &p = a.p;
  const uint32_t t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  uint32_t first, last;
  chunk_range(a, blockIdx.x, first, last);
  const float inv_c = 1.0f / (float)p.cols;
  const bool token = p.gate_rows == 1 && a.gate;
  // gain_pre, and gain_post times the chunk's gate row
  float gq[NV][VEC], gp[NV][VEC], acc_post[NV][VEC], acc_pre[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const uint32_t c = (t + i * TPR) * VEC;
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc_post[i][e] = acc_pre[i][e] = gq[i][e] = gp[i][e] = 0.0f;
    if (c >= p.cols || first >= last) continue;
    load_gain<VEC>(a.gain_pre, c, gq[i]);
    load_gain<VEC>(p.norm_after ? a.gain_post : nullptr, c, gp[i]);
    if (!token && a.gate) {
      float gt[VEC];
      load_gain<VEC>(a.gate + (size_t)(first / p.gate_rows) * p.ldgate, c, gt);
#pragma unroll
      for (int e = 0; e < VEC; ++e) gp[i][e] *= gt[e];
    }
  }

  Raw<F32, VEC> hn[NV], dn[NV];
  Raw<DT, VEC> bn[NV], yn[NV];
  auto fetch = [&](uint32_t r) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t c = (t + i * TPR) * VEC;
      hn[i].zero();
      dn[i].zero();
      bn[i].zero();
      yn[i].zero();
      if (c < p.cols && r < last) {
        if (a.dy) {
          hn[i].load(a.h + (size_t)r * p.ldh + c);
          yn[i].load(static_cast<const T *>(a.dy) + (size_t)r * p.ldy + c);
        }
        if (a.dh_out) dn[i].load(a.dh_out + (size_t)r * p.ldh + c);
        if (a.b) bn[i].load(static_cast<const T *>(a.b) + (size_t)r * p.ldb + c);
      }
    }
  };
  fetch(first + sub);
  for (uint32_t r0 = first; r0 < last; r0 += RPB) {
    const uint32_t r = r0 + sub;
    const bool live = r < last;  // the others go along: their rows read as zero
    Raw<F32, VEC> hv[NV], dv[NV];
    Raw<DT, VEC> bv[NV], yv[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      hv[i] = hn[i];
      dv[i] = dn[i];
      bv[i] = bn[i];
      yv[i] = yn[i];
    }
    fetch(r + RPB);
    float s[3] = {0.0f, 0.0f, 0.0f};  // sum h'^2, sum gain_pre dy h', sum b^2
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float hh = hv[i].get(e), bb = bv[i].get(e);
        s[0] += hh * hh;
        s[1] += gq[i][e] * yv[i].get(e) * hh;
        s[2] += bb * bb;
      }
    row_sum_once<TPR, 3>(s, red);
    const float rh = a.dy ? 1.0f / sqrtf(s[0] * inv_c + p.eps_pre) : 0.0f;
    const float m2 = rh * s[1] * inv_c;  // mean(g hat)
    const float rb = p.norm_after ? 1.0f / sqrtf(s[2] * inv_c + p.eps_post) : 1.0f;
    const float *gate = token && live ? a.gate + (size_t)r * p.ldgate : nullptr;
    float m[1] = {0.0f};  // sum gain_post du bhat
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t c = (t + i * TPR) * VEC;
      if (c >= p.cols || !live) continue;
      float gt[VEC], w[VEC], dg[VEC], gu[VEC];
      load_gain<VEC>(gate, c, gt);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float hat = hv[i].get(e) * rh, dy = yv[i].get(e);
        const float dH = dv[i].get(e) + rh * (gq[i][e] * dy - hat * m2);
        const float bh = bv[i].get(e) * rb, ee = p.scale_b * dH;
        gu[e] = gp[i][e] * gt[e] * ee;  // gain_post du
        acc_pre[i][e] += dy * hat;
        acc_post[i][e] += gt[e] * ee * bh;
        m[0] += gu[e] * bh;
        dg[e] = ee * bh * gp[i][e];
        w[e] = p.scale_h * dH;
      }
      if (token && a.dgate) {
        Raw<F32, VEC> o;
        o.set(dg);
        o.store(a.dgate + (size_t)r * p.ldgate + c);
      }
      if (a.dh) {
        Raw<F32, VEC> o;
        o.set(w);
        o.store(a.dh + (size_t)r * p.ldh + c);
      }
      dv[i].set(gu);  // in place of dh'
    }
    row_sum_once<TPR, 1>(m, red1);
    if (!a.db) continue;
    const float m1 = p.norm_after ? m[0] * inv_c : 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t c = (t + i * TPR) * VEC;
      if (c >= p.cols || !live) continue;
      float w[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) w[e] = rb * (dv[i].get(e) - bv[i].get(e) * rb * m1);
      Raw<DT, VEC> o;
      o.set(w);
      o.store(static_cast<T *>(a.db) + (size_t)r * p.ldb + c);
    }
  }

  // the chunk's partial rows; with several rows at a time, their warps' sums
  // are added in warp order
  auto write = [&](float (&acc)[NV][VEC], float *part) {
    if (!part) return;  // the same for the whole block
    part += (size_t)blockIdx.x * p.cols;
    if constexpr (RPB == 1) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const uint32_t c = (t + i * TPR) * VEC;
        if (c >= p.cols) continue;
#pragma unroll
        for (int e = 0; e < VEC; ++e) part[c + e] = acc[i][e];
      }
    } else {
      __shared__ float sums[RPB][NV * TPR * VEC];
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) sums[sub][(t + i * TPR) * VEC + e] = acc[i][e];
      __syncthreads();
      for (uint32_t c = threadIdx.x; c < p.cols; c += block_threads(TPR)) {
        float v = sums[0][c];
#pragma unroll
        for (int w = 1; w < RPB; ++w) v += sums[w][c];
        part[c] = v;
      }
    }
  };
  write(acc_post, a.part_post);
  write(acc_pre, a.part_pre);
}

// The same for rows of 16-byte pieces, staged through shared memory: bulk
// copies bring the rows of the next `stages` steps while this one is worked
// on, so the loads in flight do not depend on the registers of the threads
// that wait in the row's two reductions.  (32768 x 2048 bf16, 12 bytes read
// and 6 written per element: 327 us with loads in the loop, 263 with the next
// row's loads in registers, 205 staged, 5.9 TB/s)
//
// All threads of the block hold one row, thread t the four-element vectors t,
// t + TPR, ....  TOKEN: a gate row per row (staged too), and its gradient.
constexpr int kMaxStages = 3;

template <int DT, int NV, int TPR, bool TOKEN>
__global__ void __launch_bounds__(TPR)
    junction_bwd_staged_kernel(const __grid_constant__ JunctionArgs a, uint32_t stages, int *status) {
  using T = typename Elem<DT>::type;
  constexpr int W = TPR / 32;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ uint64_t full[kMaxStages];
  __shared__ float red[3][W], red1[W];
  __shared__ volatile int expired;  // a wait ran out: the whole block leaves
  const BwppCudaJunctionParams &p = a.p;
  const uint32_t t = threadIdx.x, lane = t & 31, warp = t >> 5;
  uint32_t first, last;
  chunk_range(a, blockIdx.x, first, last);
  const float inv_c = 1.0f / (float)p.cols;
  // a stage: h', dh', [gate], b, dy
  const uint32_t wide = p.cols * 4, narrow = p.cols * (uint32_t)sizeof(T);
  const uint32_t at_gate = 2 * wide, at_b = at_gate + (TOKEN ? wide : 0), at_y = at_b + narrow;
  const uint32_t stage_bytes = at_y + narrow;
  if (t == 0) {
    for (uint32_t s = 0; s < stages; ++s) mbar_init(&full[s], 1);
    expired = 0;
    fence_mbar_init();
  }
  __syncthreads();
  dependent_wait();
  auto fetch = [&](uint32_t r, uint32_t s) {  // one thread
    uint8_t *to = ring + s * stage_bytes;
    mbar_arrive_expect_tx(&full[s], (a.dy ? wide + narrow : 0) + (a.dh_out ? wide : 0) +
                                        (TOKEN ? wide : 0) + (a.b ? narrow : 0));
    if (a.dy) {
      bulk_load(to, a.h + (size_t)r * p.ldh, wide, &full[s]);
      bulk_load(to + at_y, static_cast<const T *>(a.dy) + (size_t)r * p.ldy, narrow, &full[s]);
    }
    if (a.dh_out) bulk_load(to + wide, a.dh_out + (size_t)r * p.ldh, wide, &full[s]);
    if (TOKEN) bulk_load(to + at_gate, a.gate + (size_t)r * p.ldgate, wide, &full[s]);
    if (a.b) bulk_load(to + at_b, static_cast<const T *>(a.b) + (size_t)r * p.ldb, narrow, &full[s]);
  };
  if (t == 0)
    for (uint32_t s = 0; s < stages && first + s < last; ++s) fetch(first + s, s);

  // gain_pre, and gain_post times the chunk's gate row
  float gq[NV][4], gp[NV][4], acc_post[NV][4], acc_pre[NV][4];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const uint32_t c = (t + i * TPR) * 4;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc_post[i][e] = acc_pre[i][e] = gq[i][e] = gp[i][e] = 0.0f;
    if (c >= p.cols || first >= last) continue;
    load_gain<4>(a.gain_pre, c, gq[i]);
    load_gain<4>(p.norm_after ? a.gain_post : nullptr, c, gp[i]);
    if (!TOKEN && a.gate) {
      float gt[4];
      load_gain<4>(a.gate + (size_t)(first / p.gate_rows) * p.ldgate, c, gt);
#pragma unroll
      for (int e = 0; e < 4; ++e) gp[i][e] *= gt[e];
    }
  }

  uint32_t stage = 0, phase = 0;
  for (uint32_t r = first; r < last; ++r) {
    if (!mbar_wait(&full[stage], phase, status)) expired = 1;
    const uint8_t *row = ring + stage * stage_bytes;
    float hv[NV][4], dv[NV][4], gt[NV][4];
    Raw<DT, 4> bv[NV], yv[NV];
    float s[3] = {0.0f, 0.0f, 0.0f};  // sum h'^2, sum gain_pre dy h', sum b^2
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t c = (t + i * TPR) * 4;
      bv[i].zero();
      yv[i].zero();
#pragma unroll
      for (int e = 0; e < 4; ++e) hv[i][e] = dv[i][e] = gt[i][e] = 0.0f;
      if (c >= p.cols) continue;
      auto quad = [&](uint32_t at, float (&o)[4]) {
        const float4 v = *reinterpret_cast<const float4 *>(row + at + c * 4);
        o[0] = v.x; o[1] = v.y; o[2] = v.z; o[3] = v.w;
      };
      if (a.dy) {
        quad(0, hv[i]);
        yv[i].load_shared(row + at_y + c * sizeof(T));
      }
      if (a.dh_out) quad(wide, dv[i]);
      if (TOKEN) quad(at_gate, gt[i]);
      if (a.b) bv[i].load_shared(row + at_b + c * sizeof(T));
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float bb = bv[i].get(e);
        s[0] += hv[i][e] * hv[i][e];
        s[1] += gq[i][e] * yv[i].get(e) * hv[i][e];
        s[2] += bb * bb;
      }
    }
#pragma unroll
    for (int j = 0; j < 3; ++j) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s[j] += __shfl_xor_sync(0xffffffffu, s[j], o);
      if (lane == 0) red[j][warp] = s[j];
    }
    __syncthreads();  // every thread holds its part of the row: the stage is free
    if (expired) {
      if (t == 0)  // the copies still in flight, each with a limit again
        for (uint32_t k = 1; k < stages && r + k < last; ++k)
          mbar_wait(&full[(stage + k) % stages], phase ^ (stage + k >= stages ? 1u : 0u), status);
      break;
    }
    if (t == 0 && r + stages < last) fetch(r + stages, stage);
    if (++stage == stages) {
      stage = 0;
      phase ^= 1;
    }
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      s[j] = red[j][0];
#pragma unroll
      for (int w = 1; w < W; ++w) s[j] += red[j][w];
    }
    const float rh = a.dy ? 1.0f / sqrtf(s[0] * inv_c + p.eps_pre) : 0.0f;
    const float m2 = rh * s[1] * inv_c;  // mean(g hat)
    const float rb = p.norm_after ? 1.0f / sqrtf(s[2] * inv_c + p.eps_post) : 1.0f;
    float m = 0.0f;  // sum gain_post du bhat
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t c = (t + i * TPR) * 4;
      if (c >= p.cols) continue;
      float w[4], dg[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float hat = hv[i][e] * rh, dy = yv[i].get(e);
        const float dH = dv[i][e] + rh * (gq[i][e] * dy - hat * m2);
        const float bh = bv[i].get(e) * rb, ee = p.scale_b * dH;
        const float gu = (TOKEN ? gp[i][e] * gt[i][e] : gp[i][e]) * ee;  // gain_post du
        acc_pre[i][e] += dy * hat;
        acc_post[i][e] += (TOKEN ? ee * gt[i][e] : ee) * bh;
        m += gu * bh;
        dg[e] = ee * bh * gp[i][e];
        w[e] = p.scale_h * dH;
        dv[i][e] = gu;
      }
      if (TOKEN && a.dgate) {
        Raw<F32, 4> o;
        o.set(dg);
        o.store(a.dgate + (size_t)r * p.ldgate + c);
      }
      if (a.dh) {
        Raw<F32, 4> o;
        o.set(w);
        o.store(a.dh + (size_t)r * p.ldh + c);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
    if (lane == 0) red1[warp] = m;
    __syncthreads();
    if (!a.db) continue;
    float m1 = 0.0f;
    if (p.norm_after) {
#pragma unroll
      for (int w = 0; w < W; ++w) m1 += red1[w];
      m1 *= inv_c;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t c = (t + i * TPR) * 4;
      if (c >= p.cols) continue;
      float w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = rb * (dv[i][e] - bv[i].get(e) * rb * m1);
      Raw<DT, 4> o;
      o.set(w);
      o.store(static_cast<T *>(a.db) + (size_t)r * p.ldb + c);
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const uint32_t c = (t + i * TPR) * 4;
    if (c >= p.cols) continue;
    const size_t at = (size_t)blockIdx.x * p.cols + c;
    if (a.part_post)
      *reinterpret_cast<float4 *>(a.part_post + at) =
          make_float4(acc_post[i][0], acc_post[i][1], acc_post[i][2], acc_post[i][3]);
    if (a.part_pre)
      *reinterpret_cast<float4 *>(a.part_pre + at) =
          make_float4(acc_pre[i][0], acc_pre[i][1], acc_pre[i][2], acc_pre[i][3]);
  }
}

template <int DT>
__global__ void __launch_bounds__(kLoopThreads)
    junction_bwd_looped_kernel(const __grid_constant__ JunctionArgs a) {
  using T = typename Elem<DT>::type;
  __shared__ float red[3 * 32];
  dependent_wait();
  const BwppCudaJunctionParams &p = a.p;
  uint32_t first, last;
  chunk_range(a, blockIdx.x, first, last);
  const float inv_c = 1.0f / (float)p.cols;
  float *pp = a.part_post ? a.part_post + (size_t)blockIdx.x * p.cols : nullptr;
  float *pq = a.part_pre ? a.part_pre + (size_t)blockIdx.x * p.cols : nullptr;
  for (uint32_t c = threadIdx.x; c < p.cols; c += kLoopThreads) {
    if (pp) pp[c] = 0.0f;
    if (pq) pq[c] = 0.0f;
  }
  for (uint32_t r = first; r < last; ++r) {
    const float *h = a.h + (size_t)r * p.ldh;
    const float *dho = a.dh_out ? a.dh_out + (size_t)r * p.ldh : nullptr;
    const T *b = a.b ? static_cast<const T *>(a.b) + (size_t)r * p.ldb : nullptr;
    const T *dyr = a.dy ? static_cast<const T *>(a.dy) + (size_t)r * p.ldy : nullptr;
    const float *gate = a.gate ? a.gate + (size_t)(r / p.gate_rows) * p.ldgate : nullptr;
    Raw<DT, 1> x;
    float s[3] = {0.0f, 0.0f, 0.0f};
    for (uint32_t c = threadIdx.x; c < p.cols; c += kLoopThreads) {
      if (dyr) {
        x.load(dyr + c);
        s[0] += h[c] * h[c];
        s[1] += (a.gain_pre ? a.gain_pre[c] : 1.0f) * x.get(0) * h[c];
      }
      if (b) {
        x.load(b + c);
        s[2] += x.get(0) * x.get(0);
      }
    }
    block_sum<3>(s, red);
    const float rh = dyr ? 1.0f / sqrtf(s[0] * inv_c + p.eps_pre) : 0.0f;
    const float m2 = rh * s[1] * inv_c;
    const float rb = p.norm_after ? 1.0f / sqrtf(s[2] * inv_c + p.eps_post) : 1.0f;
    auto dH_of = [&](uint32_t c, float &dyhat) {
      float v = dho ? dho[c] : 0.0f;
      dyhat = 0.0f;
      if (dyr) {
        Raw<DT, 1> z;
        z.load(dyr + c);
        const float hat = h[c] * rh;
        v += rh * ((a.gain_pre ? a.gain_pre[c] : 1.0f) * z.get(0) - hat * m2);
        dyhat = z.get(0) * hat;
      }
      return v;
    };
    const bool gained = p.norm_after && a.gain_post;
    float m[1] = {0.0f};
    if (p.norm_after && b) {
      for (uint32_t c = threadIdx.x; c < p.cols; c += kLoopThreads) {
        float unused;
        const float du = p.scale_b * dH_of(c, unused) * (gate ? gate[c] : 1.0f);
        x.load(b + c);
        m[0] += (gained ? a.gain_post[c] : 1.0f) * du * (x.get(0) * rb);
      }
      block_sum<1>(m, red);
    }
    const float m1 = m[0] * inv_c;
    for (uint32_t c = threadIdx.x; c < p.cols; c += kLoopThreads) {
      float dyhat;
      const float dH = dH_of(c, dyhat), ee = p.scale_b * dH;
      const float du = ee * (gate ? gate[c] : 1.0f), gp = gained ? a.gain_post[c] : 1.0f;
      if (pq) pq[c] += dyhat;
      if (b) {
        x.load(b + c);
        const float bh = x.get(0) * rb;
        if (pp) pp[c] += (p.gate_rows == 1 ? du : ee) * bh;
        if (a.dgate) a.dgate[(size_t)r * p.ldgate + c] = ee * bh * gp;
        const float w[1] = {rb * (gp * du - bh * m1)};
        x.set(w);
      } else {
        const float w[1] = {du};
        x.set(w);
      }
      if (a.db) x.store(static_cast<T *>(a.db) + (size_t)r * p.ldb + c);
      if (a.dh) a.dh[(size_t)r * p.ldh + c] = p.scale_h * dH;
    }
  }
}

// Sums of the chunks' partial rows.  blockIdx.x: 0 dgain_post, 1 dgain_pre,
// 2 + g dgate of group g; blockIdx.y: 32 columns, one per lane.  Warp w adds
// rows w, w + 32, ... in order, then a thread per column adds the 32 warps'
// sums in warp order.  A block per group and 32 columns, however few partial rows the
// group has: 32768 x 2048 bf16 take 4.7 ms with a gate for every two rows, 1.3 for eight,
// 0.37 for 64, 0.28 for 2048.
struct JunctionSums {
  const float *part_post, *part_pre;
  const float *gain_post, *gate;
  float *dgain_post, *dgain_pre, *dgate;
  uint32_t chunks, chunks_per_group, cols, ldgate;
  int weighted;  // dgain_post: weight the partial rows with their gate rows
};

constexpr int kSumWarps = 32;
__global__ void __launch_bounds__(32 * kSumWarps) junction_sums_kernel(const JunctionSums a) {
  const uint32_t job = blockIdx.x;
  float *out = job == 0 ? a.dgain_post : job == 1 ? a.dgain_pre : a.dgate;
  dependent_wait();
  if (!out) return;
  __shared__ float sums[kSumWarps][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t c = blockIdx.y * 32 + lane;
  const float *part = job == 1 ? a.part_pre : a.part_post;
  const uint32_t begin = job < 2 ? 0 : (job - 2) * a.chunks_per_group;
  const uint32_t end = job < 2 ? a.chunks : begin + a.chunks_per_group;
  // rows k, k + kSumWarps, ... below `to`, eight loads in flight; `weight(k)`
  // is NULL or the gate row of chunk k
  auto add = [&](uint32_t k, uint32_t to, auto weight) {
    constexpr int U = 8;
    float sum = 0.0f;
    for (; k < to; k += U * kSumWarps) {
      float v[U], w[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t at = k + u * kSumWarps;
        const float *g = weight(at);
        v[u] = at < to ? part[(size_t)at * a.cols + c] : 0.0f;
        w[u] = g && at < to ? g[c] : 1.0f;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) sum += v[u] * w[u];
    }
    return sum;
  };
  auto plain = [](uint32_t) { return (const float *)nullptr; };
  float acc = 0.0f;
  if (c < a.cols) {
    if (job || !a.weighted) {
      acc = add(begin + warp, end, plain);
    } else if (a.chunks_per_group >= (uint32_t)kSumWarps) {
      // groups that keep every warp busy: one weight for each
      for (uint32_t k = 0, g = 0; k < a.chunks; k += a.chunks_per_group, ++g) {
        const float w = a.gate[(size_t)g * a.ldgate + c];
        acc += w * add(k + warp, k + a.chunks_per_group, plain);
      }
    } else {
      acc = add(warp, a.chunks,
                [&](uint32_t k) { return a.gate + (size_t)(k / a.chunks_per_group) * a.ldgate; });
    }
  }
  sums[warp][lane] = acc;
  __syncthreads();
  if (warp == 0 && c < a.cols) {
    float v = sums[0][lane];
    for (int w = 1; w < kSumWarps; ++w) v += sums[w][lane];
    if (job >= 2) {
      if (a.gain_post) v *= a.gain_post[c];
      out[(size_t)(job - 2) * a.ldgate + c] = v;
    } else {
      out[c] = v;
    }
  }
}

// ---- host ----------------------------------------------------------------------

struct Chunks {
  uint32_t group_rows, groups, chunk_rows, per_group, chunks;
};

// A chunk holds consecutive rows of one group (rows that share a gate row and
// whose dgate is summed), about `per_sm` chunks per SM (at most kMaxPerSm,
// which the scratch is sized for).
constexpr uint32_t kMaxPerSm = 12;
bool make_chunks(BwppCudaCtx *ctx, uint32_t rows, uint32_t gate_rows, uint32_t per_sm, Chunks &k) {
  k.group_rows = gate_rows <= 1 || gate_rows > rows ? rows : gate_rows;
  k.groups = (uint32_t)(((uint64_t)rows + k.group_rows - 1) / k.group_rows);
  const uint32_t want = (uint32_t)ctx->num_sms * per_sm;
  k.chunk_rows = (uint32_t)(((uint64_t)rows + want - 1) / want);
  k.per_group = (uint32_t)(((uint64_t)k.group_rows + k.chunk_rows - 1) / k.chunk_rows);
  const uint64_t n = (uint64_t)k.groups * k.per_group;
  k.chunks = (uint32_t)n;
  return n < (1u << 31) - 2;
}

constexpr uint32_t kMostSize = 0x7fffffffu;

int check_args(BwppCudaCtx *ctx, const BwppCudaJunctionParams *p, bool has_b, bool has_gate,
               bool has_y) {
  if (!p) return bwpp_set_error(ctx, BWPP_CUDA_ERR_ARG, "junction: NULL params");
  if (p->ldh < p->cols || (has_b && p->ldb < p->cols) || (has_gate && p->ldgate < p->cols) ||
      (has_y && p->ldy < p->cols))
    return bwpp_set_error(ctx, BWPP_CUDA_ERR_ARG, "junction: leading dim smaller than row");
  // a column index steps past the row's end by up to a block's threads, in 32 bits
  if (p->rows > kMostSize || p->cols > kMostSize)
    return bwpp_set_error(ctx, BWPP_CUDA_ERR_ARG, "junction: more than 2^31 - 1 rows or columns");
  return BWPP_CUDA_OK;
}

// Whether all of a's tensors take eight-element transfers.
template <int DT>
bool vectors(const JunctionArgs &a) {
  const BwppCudaJunctionParams &p = a.p;
  if (p.cols % 8 || p.ldh % 8 || p.ldb % 8 || p.ldy % 8 || (a.gate && p.ldgate % 8)) return false;
  for (const void *q : {(const void *)a.h, a.b, (const void *)a.gain_post, (const void *)a.gate,
                        (const void *)a.gain_pre, (const void *)a.h_out, (const void *)a.y,
                        (const void *)a.dh_out, a.dy, (const void *)a.dh, (const void *)a.db,
                        (const void *)a.dgate})
    if (!aligned_to(q, 16)) return false;
  return true;
}

template <int DT>
int launch_fwd(BwppCudaCtx *ctx, const JunctionArgs &a) {
  const uint32_t cols = a.p.cols;
  cudaStream_t s = ctx->stream;
  cudaError_t rc;
  // Few threads with more of the row each keep more bytes in flight per SM and
  // have less to wait for at the row's two reductions (32768 x 2048 bf16: 147 us
  // with 256 threads, 130 with 128, 127 with 64, 140 with a warp); many threads
  // finish a single row sooner (3.1 us with 256, 4.5 with 64).
  const bool many = a.p.rows > (uint32_t)ctx->num_sms * 4;
#define BWPP_FWD(VEC, NV, TPR)                                                             \
  rc = bwpp_launch_dependent(                                                              \
      junction_fwd_kernel<DT, VEC, NV, TPR>,                                               \
      dim3((a.p.rows + block_threads(TPR) / TPR - 1) / (block_threads(TPR) / TPR)),        \
      dim3(block_threads(TPR)), 0, s, a)
  if (vectors<DT>(a)) {
    if (cols <= 64) BWPP_FWD(8, 1, 8);
    else if (cols <= 128) BWPP_FWD(8, 1, 16);
    else if (cols <= 256) BWPP_FWD(8, 1, 32);
    else if (cols <= 512) BWPP_FWD(8, 2, 32);
    else if (cols <= 1024 && many) BWPP_FWD(8, 2, 64);
    else if (cols <= 1024) BWPP_FWD(8, 1, 128);
    else if (cols <= 2048 && many) BWPP_FWD(8, 4, 64);
    else if (cols <= 2048) BWPP_FWD(8, 1, 256);
    else if (cols <= 4096 && many) BWPP_FWD(8, 4, 128);
    else if (cols <= 4096) BWPP_FWD(8, 2, 256);
    else if (cols <= 6144 && many) BWPP_FWD(8, 3, 256);
    else if (cols <= 8192 && many) BWPP_FWD(8, 4, 256);
    else if (cols <= 8192) BWPP_FWD(8, 2, 512);
    else if (cols <= 12288) BWPP_FWD(8, 3, 512);
    else if (cols <= 16384) BWPP_FWD(8, 4, 512);
    else rc = bwpp_launch_dependent(junction_fwd_looped_kernel<DT>, dim3(a.p.rows), dim3(kLoopThreads), 0, s, a);
  } else {
    if (cols <= 64) BWPP_FWD(1, 8, 8);
    else if (cols <= 128) BWPP_FWD(1, 8, 16);
    else if (cols <= 256) BWPP_FWD(1, 8, 32);
    else if (cols <= 512) BWPP_FWD(1, 8, 64);
    else if (cols <= 1024) BWPP_FWD(1, 8, 128);
    else if (cols <= 2048) BWPP_FWD(1, 8, 256);
    else if (cols <= 4096) BWPP_FWD(1, 8, 512);
    else if (cols <= 16384) BWPP_FWD(1, 16, 1024);
    else rc = bwpp_launch_dependent(junction_fwd_looped_kernel<DT>, dim3(a.p.rows), dim3(kLoopThreads), 0, s, a);
  }
#undef BWPP_FWD
  return bwpp_check_cuda(ctx, rc, "junction fwd");
}

// How the backward takes a row width: CTAs per SM, and for rows staged in shared
// memory the stages (else 0) and the shared memory that a CTA asks for.
struct Plan {
  uint32_t stages, per_sm, bytes;
};

// An instantiation of the staged kernel on a device: the CTAs that an SM's registers
// and warps hold, and above 16 bits a CTA's shared memory besides what it asks for.  0: not
// asked yet.  One word, as contexts on several threads may ask at once.
std::atomic<uint32_t> g_staged_fit[64][32] = {};
constexpr uint32_t kSharedOfSm = 228 * 1024, kSharedOfCta = 227 * 1024;  // sm_100: 1 KB of a CTA is the system's
constexpr uint32_t kSharedUnit = 128;                                   // in which it is given out

// The instantiation for rows of `cols` columns: f(kernel, threads, its number).
template <int DT, bool TOKEN, typename F>
int with_staged(uint32_t cols, F f) {
  constexpr int n = DT * 2 + (TOKEN ? 1 : 0);
  if (cols <= 512) return f(junction_bwd_staged_kernel<DT, 2, 64, TOKEN>, 64, n);
  if (cols <= 1024) return f(junction_bwd_staged_kernel<DT, 2, 128, TOKEN>, 128, n + 6);
  if (cols <= 2048) return f(junction_bwd_staged_kernel<DT, 2, 256, TOKEN>, 256, n + 12);
  if (cols <= 4096) return f(junction_bwd_staged_kernel<DT, 4, 256, TOKEN>, 256, n + 18);
  return f(junction_bwd_staged_kernel<DT, 4, 512, TOKEN>, 512, n + 24);
}

// The plan of a staged row; stages 0 where two of them do not fit.
template <int DT, bool TOKEN>
int plan_staged(BwppCudaCtx *ctx, uint32_t cols, Plan &g) {
  g = Plan{0, 0, 0};
  if (ctx->device >= 64)
    return bwpp_set_error(ctx, BWPP_CUDA_ERR_UNSUPPORTED, "junction: device index >= 64");
  return with_staged<DT, TOKEN>(cols, [&](auto kern, int threads, int id) {
    uint32_t fit = g_staged_fit[ctx->device][id].load();
    if (!fit) {
      cudaFuncAttributes at;
      int n = 0;
      cudaError_t e = cudaFuncGetAttributes(&at, kern);
      if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, threads, 0);
      const uint32_t own = e == cudaSuccess ? ((uint32_t)at.sharedSizeBytes + kSharedUnit - 1) & ~(kSharedUnit - 1) : 0;
      if (e == cudaSuccess)
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(kSharedOfCta - own));
      const int rc = bwpp_check_cuda(ctx, e, "junction smem attribute");
      if (rc) return rc;
      fit = (uint32_t)n | (kSharedOfSm - kSharedOfCta + own) << 16;
      g_staged_fit[ctx->device][id].store(fit);
    }
    const uint32_t by_regs = fit & 0xffffu, fixed = fit >> 16;
    const uint32_t row = cols * (8 + (TOKEN ? 4 : 0) + 2 * (uint32_t)sizeof(typename Elem<DT>::type));
    // 16 warps per SM hide a row's two reductions (32768 x 2048 bf16: 323 us with
    // one CTA of 8 warps, 205 with two, 218 with three, 227 with four; 8192 x 2560
    // bf16: 115 us with one CTA of 16 warps, 77 with two of 8); two or more stages
    // make no difference then.  Rows of two warps have less to do between their
    // reductions and take all the CTAs that are resident, 12 at most (32768 x 512
    // bf16: 62.8 us with 12, 65.4 with 11, 60.1 with 10; x 384: 53.3, 57.2, 54.3).
    // Chunks for more than are resident leave a second round that is nearly empty:
    // planned as 12 where 11 fit, 32768 x 512 took 72.5 us, fp32 with a gate per token,
    // where 10 fit, 8000 x 512 33.8 instead of 29.0.
    const uint32_t want = cols <= 512 ? kMaxPerSm : cols <= 1024 ? 4 : cols <= 4096 ? 2 : 1;
    for (uint32_t per = want < by_regs ? want : by_regs; per >= 1; --per) {
      // A CTA asks for its whole share of shared memory: one more on an SM would
      // leave another SM with one less, which happens when the kernel in front still
      // holds SMs as these are placed (32768 x 2048 bf16: 263 us instead of 211).
      const uint32_t bytes = (kSharedOfSm / per & ~(kSharedUnit - 1)) - fixed;
      if (bytes / row < 2) continue;
      g.per_sm = per;
      g.bytes = bytes;
      g.stages = bytes / row < (uint32_t)kMaxStages ? bytes / row : (uint32_t)kMaxStages;
      break;
    }
    return (int)BWPP_CUDA_OK;
  });
}

template <int DT>
int plan_bwd(BwppCudaCtx *ctx, const JunctionArgs &a, Plan &g) {
  const uint32_t cols = a.p.cols;
  const bool vec = vectors<DT>(a);
  if (vec && cols > 256 && cols <= 8192) {
    const int rc = a.p.gate_rows == 1 && a.gate ? plan_staged<DT, true>(ctx, cols, g)
                                                : plan_staged<DT, false>(ctx, cols, g);
    if (rc || g.stages) return rc;
  }
  // threads of a block: 128 (VEC 8, or up to 128 columns), then a fourth of the
  // columns up to 512; 72 to 80 registers a thread, 128 in the widest and with VEC 8.
  // No more than are resident (4055 x 1003 fp32 took 23.0 us with the 3 that fit,
  // 26.8 with 4)
  const uint32_t per = vec && cols <= 256 ? 4 : cols <= 128 ? 6 : cols <= 256 ? 12 : cols <= 512 ? 6
                       : cols <= 1024 ? 3 : cols <= 4096 ? 1 : 2;
  g = Plan{0, per, 0};
  return BWPP_CUDA_OK;
}

template <int DT, bool TOKEN>
int launch_staged(BwppCudaCtx *ctx, const JunctionArgs &a, uint32_t chunks, const Plan &g) {
  return with_staged<DT, TOKEN>(a.p.cols, [&](auto kern, int threads, int) {
    return bwpp_check_cuda(ctx,
                           bwpp_launch_dependent(kern, dim3(chunks), dim3(threads), g.bytes, ctx->stream, a,
                                                 g.stages, ctx->status_word),
                           "junction bwd");
  });
}

template <int DT>
int launch_bwd(BwppCudaCtx *ctx, const JunctionArgs &a, uint32_t chunks, const Plan &g) {
  const uint32_t cols = a.p.cols;
  cudaStream_t s = ctx->stream;
  if (g.stages)
    return a.p.gate_rows == 1 && a.gate ? launch_staged<DT, true>(ctx, a, chunks, g)
                                        : launch_staged<DT, false>(ctx, a, chunks, g);
  cudaError_t rc;
#define BWPP_BWD(VEC, NV, TPR)                                                              \
  rc = bwpp_launch_dependent(junction_bwd_kernel<DT, VEC, NV, TPR>, dim3(chunks),           \
                             dim3(block_threads(TPR)), 0, s, a)
  if (vectors<DT>(a) && cols <= 256) {
    if (cols <= 64) BWPP_BWD(8, 1, 8);
    else if (cols <= 128) BWPP_BWD(8, 1, 16);
    else BWPP_BWD(8, 1, 32);
  } else {
    if (cols <= 64) BWPP_BWD(1, 4, 16);
    else if (cols <= 128) BWPP_BWD(1, 4, 32);
    else if (cols <= 256) BWPP_BWD(1, 4, 64);
    else if (cols <= 512) BWPP_BWD(1, 4, 128);
    else if (cols <= 1024) BWPP_BWD(1, 4, 256);
    else if (cols <= 2048) BWPP_BWD(1, 4, 512);
    else if (cols <= 4096) BWPP_BWD(1, 8, 512);
    else rc = bwpp_launch_dependent(junction_bwd_looped_kernel<DT>, dim3(chunks), dim3(kLoopThreads), 0, s, a);
  }
#undef BWPP_BWD
  return bwpp_check_cuda(ctx, rc, "junction bwd");
}

template <int DT>
int junction_fwd(BwppCudaCtx *ctx, const float *h, const void *b, const float *gain_post,
                 const float *gate, const float *gain_pre, float *h_out, void *y,
                 const BwppCudaJunctionParams *p) {
  int rc = bwpp_ctx_enter(ctx);
  if (!rc) rc = check_args(ctx, p, true, gate != nullptr, y != nullptr);
  if (rc) return rc;
  if (p->rows == 0 || p->cols == 0) return BWPP_CUDA_OK;
  if (!h || !b || !h_out) return bwpp_set_error(ctx, BWPP_CUDA_ERR_ARG, "junction: NULL buffer");
  JunctionArgs a{};
  a.p = *p;
  if (a.p.gate_rows == 0) a.p.gate_rows = a.p.rows;
  if (!y) a.p.ldy = 0;
  a.h = h;
  a.b = b;
  a.gain_post = gain_post;
  a.gate = gate;
  a.gain_pre = gain_pre;
  a.h_out = h_out;
  a.y = y;
  return launch_fwd<DT>(ctx, a);
}

template <int DT>
int junction_bwd(BwppCudaCtx *ctx, const float *h_out, const void *b, const float *gain_post,
                 const float *gate, const float *gain_pre, const float *dh_out, const void *dy,
                 float *dh, void *db, float *dgain_post, float *dgate, float *dgain_pre,
                 const BwppCudaJunctionParams *p) {
  int rc = bwpp_ctx_enter(ctx);
  if (!rc) rc = check_args(ctx, p, b || db, gate || dgate, dy != nullptr);
  if (rc) return rc;
  if (dgate && !gate)
    return bwpp_set_error(ctx, BWPP_CUDA_ERR_ARG, "junction bwd: dgate without a gate");
  if (dgain_post && !p->norm_after)
    return bwpp_set_error(ctx, BWPP_CUDA_ERR_ARG, "junction bwd: dgain_post without norm_after");
  if (p->cols == 0) return BWPP_CUDA_OK;
  cudaStream_t s = ctx->stream;
  if (p->rows == 0) {
    if (dgain_post)
      rc = bwpp_check_cuda(ctx, cudaMemsetAsync(dgain_post, 0, sizeof(float) * p->cols, s), "memset");
    if (!rc && dgain_pre)
      rc = bwpp_check_cuda(ctx, cudaMemsetAsync(dgain_pre, 0, sizeof(float) * p->cols, s), "memset");
    if (!rc && dgate && p->gate_rows == 0)  // one gate for all rows: there without rows too
      rc = bwpp_check_cuda(ctx, cudaMemsetAsync(dgate, 0, sizeof(float) * p->cols, s), "memset");
    return rc;
  }
  // b is read where the norm's, the gate's or the gain's gradient needs it
  const bool need_b = (db && p->norm_after) || dgain_post || dgate;
  if ((dy && !h_out) || (need_b && !b))
    return bwpp_set_error(ctx, BWPP_CUDA_ERR_ARG, "junction bwd: NULL buffer");
  if (db && db == b)
    return bwpp_set_error(ctx, BWPP_CUDA_ERR_ARG, "junction bwd: db may not be b");
  JunctionArgs a{};
  a.p = *p;
  if (a.p.gate_rows == 0) a.p.gate_rows = a.p.rows;
  if (!dy) a.p.ldy = 0;
  if (!b && !db) a.p.ldb = 0;
  a.h = h_out;
  a.b = need_b ? b : nullptr;
  a.gain_post = gain_post;
  a.gate = gate;
  a.gain_pre = gain_pre;
  a.dh_out = dh_out;
  a.dy = dy;
  a.dh = dh;
  a.db = db;
  const bool per_row = a.p.gate_rows == 1;
  a.dgate = per_row ? dgate : nullptr;
  Plan g;
  rc = plan_bwd<DT>(ctx, a, g);
  if (rc) return rc;
  Chunks k;
  if (!make_chunks(ctx, a.p.rows, a.p.gate_rows, g.per_sm, k))
    return bwpp_set_error(ctx, BWPP_CUDA_ERR_UNSUPPORTED, "junction bwd: too many gate rows");
  a.chunk_rows = k.chunk_rows;
  a.chunks_per_group = k.per_group;
  a.group_rows = k.group_rows;
  const bool sum_post = dgain_post || (dgate && !per_row);
  const bool sums = sum_post || dgain_pre;
  if (sums) {
    if ((a.p.cols - 1) / 32 >= 65535)  // blocks of 32 columns in a grid's second dimension
      return bwpp_set_error(ctx, BWPP_CUDA_ERR_UNSUPPORTED, "junction bwd: row too wide");
    uint8_t *scratch;
    const size_t part = (size_t)k.chunks * a.p.cols;
    rc = bwpp_op_scratch(ctx, 2 * part * sizeof(float), "junction bwd", &scratch);
    if (rc) return rc;
    if (sum_post) a.part_post = reinterpret_cast<float *>(scratch);
    if (dgain_pre) a.part_pre = reinterpret_cast<float *>(scratch) + part;
  }
  rc = launch_bwd<DT>(ctx, a, k.chunks, g);
  if (rc) return rc;
  if (sums) {
    JunctionSums q{};
    q.part_post = a.part_post;
    q.part_pre = a.part_pre;
    q.gain_post = a.p.norm_after ? gain_post : nullptr;
    q.gate = gate;
    q.dgain_post = dgain_post;
    q.dgain_pre = dgain_pre;
    q.dgate = per_row ? nullptr : dgate;
    q.chunks = k.chunks;
    q.chunks_per_group = k.per_group;
    q.cols = a.p.cols;
    q.ldgate = a.p.ldgate;
    q.weighted = gate && !per_row;
    const dim3 grid(2 + (q.dgate ? k.groups : 0), (a.p.cols + 31) / 32);
    rc = bwpp_check_cuda(
        ctx, bwpp_launch_dependent(junction_sums_kernel, grid, dim3(32 * kSumWarps), 0, s, q),
        "junction sums");
    if (rc) return rc;
  }
  return BWPP_CUDA_OK;
}

}  // namespace

extern "C" {

size_t bwpp_cuda_junction_bwd_workspace_size(BwppCudaCtx *ctx, uint32_t rows, uint32_t cols,
                                             uint32_t gate_rows) {
  if (!ctx || rows == 0 || cols == 0 || rows > kMostSize || cols > kMostSize) return 0;
  Chunks k;
  if (!make_chunks(ctx, rows, gate_rows ? gate_rows : rows, kMaxPerSm, k)) return 0;
  return 2 * (size_t)k.chunks * cols * sizeof(float) + BWPP_OP_SCRATCH_PAD;
}

#define BWPP_JUNCTION(SUFFIX, DT, T)                                                             \
  int bwpp_cuda_junction_fwd_##SUFFIX(BwppCudaCtx *ctx, const float *h, const T *b,              \
                                      const float *gain_post, const float *gate,                 \
                                      const float *gain_pre, float *h_out, T *y,                 \
                                      const BwppCudaJunctionParams *params) {                    \
    return junction_fwd<DT>(ctx, h, b, gain_post, gate, gain_pre, h_out, y, params);             \
  }                                                                                              \
  int bwpp_cuda_junction_bwd_##SUFFIX(                                                           \
      BwppCudaCtx *ctx, const float *h_out, const T *b, const float *gain_post,                  \
      const float *gate, const float *gain_pre, const float *dh_out, const T *dy, float *dh,     \
      T *db, float *dgain_post, float *dgate, float *dgain_pre,                                  \
      const BwppCudaJunctionParams *params) {                                                    \
    return junction_bwd<DT>(ctx, h_out, b, gain_post, gate, gain_pre, dh_out, dy, dh, db,        \
                            dgain_post, dgate, dgain_pre, params);                               \
  }
BWPP_JUNCTION(f32, BWPP_CUDA_DTYPE_F32, float)
BWPP_JUNCTION(bf16, BWPP_CUDA_DTYPE_BF16, uint16_t)
BWPP_JUNCTION(f16, BWPP_CUDA_DTYPE_F16, uint16_t)
#undef BWPP_JUNCTION

}  // extern "C"

// The logits of the vocabulary cross entropy on the tensor cores, used up in
// the epilogue: they never reach memory.
//
// logit[t, v] = scale sum_d x[t, d] W[v, d], in tiles of 256 rows x 256
// vocabulary columns (a CTA pair, cta_group::2) or 128 x 256 (one CTA, where a
// pair would have too few rows).  Persistent, warp-specialised like the GEMM (gemm.cu): warp 0
// feeds a ring of operand stages by TMA, one thread of warp 1 issues
// tcgen05.mma, warps 2..9 drain the accumulator; two TMEM accumulators, so the
// epilogue of a tile runs beside the next tile's main loop.
//
// FWD.  An epilogue thread owns a row of the tile and 128 of its columns: the
// running maximum and sum of 2^(logit log2 e - maximum) stay in registers over
// its four 32-column chunks and leave as one (maximum, sum) pair per row and
// 128 columns, 8 bytes for every 512 of logits.  xent_combine_kernel folds a
// row's pairs.  The thread that meets the row's target writes its logit, which
// stays out of the pair where there are few rows.
// Backward.  The epilogue turns the logits into bf16 scale g (p - hit) (or p -
// hit, where all rows have the same g: its mantissa would be rounded the same
// way in every row) and stores the tile by TMA: 2 bytes a logit, read by the two
// gradient products.  That rounding is what the gradients are off by besides their
// own: 1.0e-3 of their norm with one dloss, 1.8e-3 with rows' own (T 4096, V 16000,
// D 1024); value and rest, as few rows have it, leave 3e-6 and would double the products.
//
// Exponentials are ex2.approx (2 ulp; below 2^-126 they are zero): one per logit, 128 x 256 of them for a
// tile are 2048 cycles of an SM's MUFU, against 128 cycles of MMA for every 16
// of D: below D = 256 the exponentials set the pace, above it the products.
//
// Every wait is bounded as in the GEMM.
#include "bwpp_cuda_internal.cuh"
#include "xent.cuh"

namespace {

constexpr int BM = 128, BN = 256, BK = 64;
constexpr int A_STAGE = BM * BK * 2;
constexpr int B_BOX = 64 * BK * 2;  // 64 vocabulary columns x 64 of D
constexpr int EPI_WARPS = 8;
constexpr int EPI_BUF = 32 * 128;   // 32 rows x 64 bf16
constexpr int THREADS = 64 + 32 * EPI_WARPS;
constexpr uint32_t TMEM_COLS = 2 * BN;
constexpr uint32_t MANY_CHUNK = 16;  // K blocks of a sum, many rows (see EXACT)

template <bool PAIR>
struct Cfg {
  static constexpr int STAGES = PAIR ? 6 : 4;
  static constexpr int B_STAGE = (PAIR ? 128 : 256) * BK * 2;
  static constexpr int OFF_B = STAGES * A_STAGE;
  static constexpr int OFF_C = OFF_B + STAGES * B_STAGE;
  static constexpr int OFF_BAR = OFF_C + EPI_WARPS * EPI_BUF;
  static constexpr int SMEM = OFF_BAR + 256 + 1024;  // slack: 1024-byte alignment
  static constexpr uint32_t TILE_M = PAIR ? 2 * BM : BM;
  static_assert(SMEM <= 232448, "exceeds the 227 KB opt-in limit");
  static_assert((2 * STAGES + 5) * 8 + 8 <= 256, "barrier block");
};

struct XentTile {
  uint32_t T, V, D;     // V: columns of this launch
  uint32_t v0;          // vocabulary index of column 0
  float c;              // scale * log2(e)
  const int32_t *target;
  uint32_t chunk;       // EXACT: K blocks of a sum
  // FWD
  float2 *part;         // [ceil(V / 128)][T]
  float *hit;           // [T] logit of the target, in powers of two like the pairs
  bool apart;           // EXACT: the pairs leave the target out
  // backward
  const float *lse, *dloss;
  const float *common;  // [2]: not 0 where all rows have one dloss, which then is
                        // a factor of the results; NULL: rows have their own
  float scale;
  uint32_t vocab;       // targets below it are live
  // items [0, whole) are tiles, from there on each remaining tile is cut into
  // two of 128 columns, so that a short last round spreads over twice the workers
  uint32_t whole, items;
  uint32_t group;       // row blocks that pass the columns together
  uint32_t x_rows;      // rows of x that a CTA loads for a tile: a box of the tensor map
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Maximum and sum of exponentials over it of 2 P logits in powers of two,
// folded into (m, s).  Paired fp32 operations, and max of three: the epilogue
// warps share their issue slots with the thread that feeds the tensor core.
template <int P>
__device__ __forceinline__ void fold_logits(uint64_t (&t)[P], float &m, float &s) {
  float top = m;
#pragma unroll
  for (int j = 0; j < P; ++j) {
    float x, y;
    f2unpack(t[j], x, y);
    asm("max.f32 %0, %0, %1, %2;" : "+f"(top) : "f"(x), "f"(y));
  }
  // only -inf so far, or +inf: the exponentials are taken against 0
  const float base = fabsf(top) == INFINITY ? 0.0f : top;
  s *= ex2(m - base);
  const uint64_t less = f2pack(-base, -base);
  uint64_t sum[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
  for (int j = 0; j < P; ++j) {
    float x, y;
    f2unpack(f2add(t[j], less), x, y);
    sum[j & 3] = f2add(sum[j & 3], f2pack(ex2(x), ex2(y)));
  }
  float x, y;
  f2unpack(f2add(f2add(sum[0], sum[1]), f2add(sum[2], sum[3])), x, y);
  s += x + y;
  m = top;
}

// Columns from `end` on drop out.
template <int P>
__device__ __forceinline__ void mask_logits(uint64_t (&t)[P], uint32_t col, uint32_t end) {
  if (col + 2 * P <= end) return;
#pragma unroll
  for (int j = 0; j < P; ++j) {
    float x, y;
    f2unpack(t[j], x, y);
    if (col + 2 * j >= end) x = -INFINITY;
    if (col + 2 * j + 1 >= end) y = -INFINITY;
    t[j] = f2pack(x, y);
  }
}

// Column `at` of these; drop: it becomes -inf.
template <int P>
__device__ __forceinline__ float pick_logit(uint64_t (&t)[P], uint32_t at, bool drop) {
  float h = 0.0f;
#pragma unroll
  for (int j = 0; j < P; ++j) {
    float x, y;
    f2unpack(t[j], x, y);
    if (at == 2u * j) {
      h = x;
      if (drop) x = -INFINITY;
    }
    if (at == 2u * j + 1) {
      h = y;
      if (drop) y = -INFINITY;
    }
    t[j] = f2pack(x, y);
  }
  return h;
}

// Tiles go down the row blocks of a group, then to the next 256 columns.
__device__ __forceinline__ void tile_at(uint32_t i, uint32_t group, uint32_t tiles_m,
                                        uint32_t tiles_n, uint32_t &mb, uint32_t &nb) {
  const uint32_t per_group = group * tiles_n, g = i / per_group, first = g * group;
  const uint32_t gm = min(group, tiles_m - first), r = i - g * per_group;
  mb = first + r % gm;
  nb = r / gm;
}

// Item i: its row block, first column and width.
__device__ __forceinline__ void item_at(const XentTile &a, uint32_t i, uint32_t tiles_m,
                                        uint32_t tiles_n, uint32_t &mb, uint32_t &col,
                                        uint32_t &width) {
  const bool half = i >= a.whole;
  const uint32_t j = i - a.whole;
  uint32_t nb;
  tile_at(half ? a.whole + j / 2 : i, a.group, tiles_m, tiles_n, mb, nb);
  width = half ? BN / 2 : BN;
  col = nb * BN + (half ? (j & 1) * (BN / 2) : 0);
}

// EXACT: the sums over D are cut into chunks of `chunk` K blocks, each summed in
// TMEM from zero and added to the others in registers.  The tensor core
// truncates its running sum at each addition, and the errors, all towards zero,
// grow with the length of a sum: lse at D = 4096 was off by 2e-6 of its value in
// one sum, by 7e-7 in chunks of 16 blocks.  A few rows, which wait for W anyway,
// take chunks of two: the loss of one token has no others to average with, and
// at 512 to 2048 of D it went from 7e-6 to at most 2e-6 of its value.
// EXACT, backward: dlogit leaves as two bf16, its rounded value and what the
// rounding left, XENT_EXACT_ROWS below.  A gradient of few rows is mostly its targets'
// entries times rows of W or x, so their rounding, up to 2^-8 of them, would be
// its error; and 1 - p of a sure target is a difference, hence the chunks.
template <bool B_MN, bool PAIR, bool FWD, bool EXACT>
__global__ void __launch_bounds__(THREADS, 1)
    xent_tc_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
                   const __grid_constant__ CUtensorMap tmOut, const XentTile a, int *status) {
  using C = Cfg<PAIR>;
  constexpr int STAGES = C::STAGES;
  constexpr uint32_t IDESC = make_idesc_bf16_f32(C::TILE_M, BN, 0u, B_MN ? 1u : 0u);
  constexpr uint32_t IDESC_HALF = make_idesc_bf16_f32(C::TILE_M, BN / 2, 0u, B_MN ? 1u : 0u);
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t *smem = smem_raw + ((1024u - (raw & 1023u)) & 1023u);
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + C::OFF_BAR);
  uint64_t *empty = full + STAGES;
  uint64_t *tfull = empty + STAGES;
  uint64_t *tempty = tfull + 2;
  uint64_t *drain = tempty + 2;
  uint32_t *tmem_holder = reinterpret_cast<uint32_t *>(drain + 1);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_holder + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_ctarank() : 0u;
  const uint32_t worker = PAIR ? cluster_id_x() : blockIdx.x;
  const uint32_t workers = PAIR ? cluster_count_x() : gridDim.x;
  const uint32_t tiles_m = (a.T + C::TILE_M - 1) / C::TILE_M, tiles_n = (a.V + BN - 1) / BN;
  const uint32_t num_kb = (a.D + BK - 1) / BK;
  const uint32_t chunk = PAIR ? MANY_CHUNK : a.chunk;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&tfull[i], 1);
      mbar_init(&tempty[i], PAIR ? 2 * EPI_WARPS : EPI_WARPS);
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_mbar_init();
    prefetch_tmap(&tmX);
    prefetch_tmap(&tmW);
    if (!FWD) prefetch_tmap(&tmOut);
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      tmem_alloc_pair(tmem_holder, TMEM_COLS);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(tmem_holder, TMEM_COLS);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  if constexpr (PAIR) cluster_sync_all(); else __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  dependent_wait();

  if (warp == 0) {
    if (lane == 0) {
      uint32_t stage = 0, phase = 0;
      for (uint32_t i = worker; i < a.items && !*abort_flag; i += workers) {
        uint32_t mb, col, width;
        item_at(a, i, tiles_m, tiles_n, mb, col, width);
        const uint32_t mine = PAIR ? width / 2 : width;  // columns that this CTA loads
        const int32_t row0 = (int32_t)(mb * C::TILE_M + rank * BM);
        const int32_t col0 = (int32_t)(col + rank * mine);
        for (uint32_t kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1, status)) {
            *abort_flag = 1;
            break;
          }
          // both CTAs' bytes count on rank 0's barrier
          if (rank == 0)
            mbar_arrive_expect_tx(&full[stage], (PAIR ? 2 : 1) * ((a.x_rows + mine) * BK * 2));
          uint32_t fbar = 0;
          if constexpr (PAIR) fbar = cluster_addr(&full[stage], 0);
          auto load = [&](void *dst, const CUtensorMap *map, int32_t x, int32_t y) {
            if constexpr (PAIR) tma_load_2d_pair(dst, map, fbar, x, y);
            else tma_load_2d(dst, map, &full[stage], x, y);
          };
          const int32_t k0 = (int32_t)(kb * BK);
          uint8_t *sb = smem + C::OFF_B + stage * C::B_STAGE;
          load(smem + stage * A_STAGE, &tmX, k0, row0);
          for (uint32_t j = 0; j < mine / 64; ++j) {
            if (B_MN) load(sb + j * B_BOX, &tmW, col0 + (int32_t)j * 64, k0);
            else load(sb + j * B_BOX, &tmW, k0, col0 + (int32_t)j * 64);
          }
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      auto commit = [&](uint64_t *bar) {
        if constexpr (PAIR) {
          tc_commit_pair(smem_u32(bar));
          tc_commit_pair(cluster_addr(bar, 1));
        } else {
          tc_commit(bar);
        }
      };
      uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0;
      for (uint32_t i = worker; i < a.items && !*abort_flag; i += workers) {
        if (!mbar_wait(&tempty[acc], acc_phase ^ 1, status)) {
          *abort_flag = 1;
          break;
        }
        tc_fence_after();
        uint32_t mb, col, width;
        item_at(a, i, tiles_m, tiles_n, mb, col, width);
        const uint32_t idesc = width == BN ? IDESC : IDESC_HALF;
        bool ok = true;
        uint32_t first_kb = 0;  // of the running sum
        for (uint32_t kb = 0; kb < num_kb; ++kb) {
          if (EXACT && kb - first_kb == chunk) {  // the next accumulator takes over
            first_kb = kb;
            commit(&tfull[acc]);
            acc ^= 1;
            if (acc == 0) acc_phase ^= 1;
            if (!mbar_wait(&tempty[acc], acc_phase ^ 1, status)) {
              *abort_flag = 1;
              ok = false;
              break;
            }
            tc_fence_after();
          }
          if (!mbar_wait(&full[stage], phase, status)) {
            *abort_flag = 1;
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a0 = smem_u32(smem + stage * A_STAGE);
          const uint32_t b0 = smem_u32(smem + C::OFF_B + stage * C::B_STAGE);
          // K-major: 16 of D are 32 bytes inside the 128-byte swizzle; MN-major:
          // 64-column atoms 8 KB apart, 16 rows of D are 2 KB
          const uint64_t ad = make_smem_desc(a0, 16, 1024, BWPP_SWIZZLE_128B);
          const uint64_t bd = make_smem_desc(b0, B_MN ? B_BOX : 16, 1024, BWPP_SWIZZLE_128B);
#pragma unroll
          for (int ks = 0; ks < BK / 16; ++ks) {
            const uint64_t as = desc_add(ad, ks * 32), bs = desc_add(bd, ks * (B_MN ? 2048 : 32));
            const uint32_t accum = kb != first_kb || ks != 0 ? 1u : 0u;
            if constexpr (PAIR) tc_mma_f16_ss_pair(tmem_base + acc * BN, as, bs, idesc, accum);
            else tc_mma_f16_ss(tmem_base + acc * BN, as, bs, idesc, accum);
          }
          commit(&empty[stage]);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (!ok) break;
        commit(&tfull[acc]);
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
      }
      // every MMA issued here has finished before TMEM is freed
      if constexpr (PAIR) tc_commit_pair(smem_u32(drain)); else tc_commit(drain);
      mbar_wait(drain, 0, status);
    }
  } else {
    const int q = warp & 3;            // TMEM lane quarter of this warp
    const int ew = warp - 2;
    const int sub = ew >> 2;           // columns [128 sub, 128 sub + 128) of the tile
    const uint32_t tq = (uint32_t)(q * 32) << 16;
    uint32_t acc = 0, acc_phase = 0;
    for (uint32_t i = worker; i < a.items && !*abort_flag; i += workers) {
      uint32_t mb, col, width;
      item_at(a, i, tiles_m, tiles_n, mb, col, width);
      const uint32_t row0 = mb * C::TILE_M + rank * BM + q * 32, row = row0 + lane;
      const uint32_t first = col + sub * 128;  // this warp's first column
      const uint32_t end = min(a.V, col + width);
      const bool live_row = row < a.T;
      // nothing of the tile is this warp's (EXACT dlogit has zeros behind its rows)
      const bool none = first >= end || row0 >= (!FWD && EXACT ? XENT_EXACT_ROWS : a.T);
      const int32_t target = live_row && a.target ? __ldcg(a.target + row) : -1;
      // the target's column within this warp's 128, or beyond them
      const uint32_t hit_col =
          target >= 0 ? (uint32_t)target - a.v0 - first : 0xffffffffu;
      float g = 0.0f, lse2 = 0.0f;
      if constexpr (!FWD) {
        if (live_row && (uint32_t)target < a.vocab) {
          const bool shared = a.common ? __ldcg(a.common + 1) != 0.0f : false;
          g = shared ? 1.0f : a.scale * (a.dloss ? __ldcg(a.dloss + row) : 1.0f);
          lse2 = __ldcg(a.lse + row) * 1.44269504f;
        }
      }
      const bool live = live_row && (uint32_t)target < a.vocab;
      auto release = [&]() {  // the accumulator has been read
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (PAIR) mbar_arrive_cluster(cluster_addr(&tempty[acc], 0));
          else mbar_arrive(&tempty[acc]);
        }
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
      };
      // 32 logits in powers of two less lse2 to dlogit in bf16, and, EXACT, to
      // what the rounding left
      auto to_dlogit = [&](const uint64_t (&t)[16], uint32_t at, uint32_t *out, uint32_t *rest) {
        float d[32];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          f2unpack(t[j], d[2 * j], d[2 * j + 1]);
          d[2 * j] = ex2(d[2 * j]);
          d[2 * j + 1] = ex2(d[2 * j + 1]);
        }
        if (at < 32u) {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (at == (uint32_t)j) d[j] -= 1.0f;
        }
        const uint64_t g2 = f2pack(g, g);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          float x, y;
          f2unpack(f2mul(f2pack(d[2 * j], d[2 * j + 1]), g2), x, y);
          const uint32_t both = pack2_16<false>(x, y);
          out[j] = live ? both : 0u;
          if constexpr (EXACT)
            rest[j] = live ? pack2_16<false>(x - __uint_as_float(both << 16),
                                             y - __uint_as_float(both & 0xFFFF0000u))
                           : 0u;
        }
      };
      // 32 rows x 64 columns of dlogit (128 bytes a row) from column c0
      auto put = [&](const uint32_t (&w)[32], uint32_t c0, uint32_t to_row) {
        uint8_t *stage_c = smem + C::OFF_C + ew * EPI_BUF;
        if (lane == 0) tma_store_wait_read<0>();
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 8; ++j)
          *reinterpret_cast<uint4 *>(stage_c + lane * 128 + ((j ^ (lane & 7)) << 4)) =
              make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          tma_store_2d(&tmOut, stage_c, (int32_t)c0, (int32_t)to_row);
          tma_store_commit();
        }
      };
      const uint64_t c2 = f2pack(a.c, a.c), l2 = f2pack(-lse2, -lse2);
      if constexpr (EXACT) {
        uint64_t v[64];  // pairs of columns
#pragma unroll
        for (int j = 0; j < 64; ++j) v[j] = 0ull;
        bool ok = true;
#pragma unroll 1
        for (uint32_t kb = 0; kb < num_kb; kb += chunk) {
          if (!mbar_wait(&tfull[acc], acc_phase, status)) {
            *abort_flag = 1;
            ok = false;
            break;
          }
          tc_fence_after();
          // 16 columns at a time: 32 more registers would not fit
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            if (none) break;
            uint32_t r[16];
            tmem_ld_32x32b_x16(tmem_base + tq + acc * BN + sub * 128 + k * 16, r);
            tc_wait_ld16(r);
#pragma unroll
            for (int j = 0; j < 8; ++j)
              v[8 * k + j] = f2add(v[8 * k + j], f2pack(__uint_as_float(r[2 * j]),
                                                        __uint_as_float(r[2 * j + 1])));
          }
          release();
        }
        if (!ok) break;
        if (none) continue;
        if constexpr (FWD) {
#pragma unroll
          for (int j = 0; j < 64; ++j) v[j] = f2mul(v[j], c2);
          if (hit_col < 128u) a.hit[row] = pick_logit(v, hit_col, !PAIR && a.apart);
          mask_logits(v, first, end);
          float m = -INFINITY, s = 0.0f;
          fold_logits(v, m, s);
          if (live_row) a.part[(size_t)(first / 128) * a.T + row] = make_float2(m, s);
        } else {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            if (first + k * 64 >= end) break;
            uint32_t out[32], rest[32];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint64_t t[16];
#pragma unroll
              for (int j = 0; j < 16; ++j) t[j] = f2fma(v[k * 32 + h * 16 + j], c2, l2);
              to_dlogit(t, hit_col - (k * 64 + h * 32), out + h * 16, rest + h * 16);
            }
            put(out, first + k * 64, row0);
            put(rest, first + k * 64, row0 + XENT_EXACT_ROWS);
          }
        }
        continue;
      }
      if (!mbar_wait(&tfull[acc], acc_phase, status)) {
        *abort_flag = 1;
        break;
      }
      tc_fence_after();
      const uint32_t taddr = tmem_base + tq + acc * BN + sub * 128;
      if constexpr (FWD) {
        if (!none) {
          float m = -INFINITY, s = 0.0f;
#pragma unroll 1
          for (int k = 0; k < 4; ++k) {
            const uint32_t cs = first + k * 32;
            if (cs >= end) break;
            uint32_t r[32];
            tmem_ld_32x32b_x32(taddr + k * 32, r);
            tc_wait_ld(r);
            uint64_t v[16];
#pragma unroll
            for (int j = 0; j < 16; ++j)
              v[j] = f2mul(f2pack(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])), c2);
            if (hit_col - k * 32 < 32u) a.hit[row] = pick_logit(v, hit_col - k * 32, false);
            mask_logits(v, cs, end);
            fold_logits(v, m, s);
          }
          if (live_row) a.part[(size_t)(first / 128) * a.T + row] = make_float2(m, s);
        }
      } else {
#pragma unroll 1
        for (int k = 0; k < 2; ++k) {
          const uint32_t cs = first + k * 64;
          if (none || cs >= end) break;
          uint32_t out[32];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t r[32];
            tmem_ld_32x32b_x32(taddr + k * 64 + h * 32, r);
            tc_wait_ld(r);
            uint64_t t[16];
#pragma unroll
            for (int j = 0; j < 16; ++j)
              t[j] = f2fma(f2pack(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])), c2, l2);
            to_dlogit(t, hit_col - (k * 64 + h * 32), out + h * 16, nullptr);
          }
          put(out, cs, row0);
        }
      }
      release();
    }
    if (!FWD && lane == 0) tma_store_wait_all<0>();
  }

  // every wait is bounded, so both CTAs of a pair arrive here
  tc_fence_before();
  if constexpr (PAIR) cluster_sync_all(); else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    if constexpr (PAIR) tmem_dealloc_pair(tmem_base, TMEM_COLS);
    else tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

__device__ __forceinline__ void fold_pair(float2 &x, float2 y) {
  const float top = fmaxf(x.x, y.x), base = fabsf(top) == INFINITY ? 0.0f : top;
  x.y = x.y * ex2(x.x - base) + y.y * ex2(y.x - base);
  x.x = top;
}

// lse and loss of row t from its folded pair.  APART: the pair leaves a live
// target out.  With h its logit and d = log2 of the others' sum less h, the loss is
// log(1 + 2^d): it keeps its digits where the target takes nearly all of the
// probability, and lse - h would lose them.
template <bool APART>
__device__ __forceinline__ void finish_row(uint32_t t, float2 x, const float *hit,
                                           const int32_t *target, float *loss, float *lse, uint32_t V,
                                           int *status) {
  const float ln2 = 0.693147181f, nan = __int_as_float(0x7fc00000), more = log2f(x.y);
  const int32_t y = loss ? target[t] : -1;
  float l = (x.x + more) * ln2, v = 0.0f;
  if (y >= 0) {
    if ((uint32_t)y < V) {
      // the maximum less the target's logit first: one near the other cancels
      const float h = hit[t], d = (x.x - h) + more;
      if (APART) {
        // equal ones may be infinite: then d is NaN, and so is the loss, but not lse
        const float others = x.x + more, both = h == others ? ln2 : log1pf(exp2f(-fabsf(d)));
        l = fmaxf(h, others) * ln2 + both;
        // an infinite logit of the target: inf - inf
        v = d > 0.0f ? d * ln2 + both : d == d && h < INFINITY ? both : nan;
      } else {
        v = d * ln2;
      }
    } else {
      v = nan;
      bwpp_report(status, BWPP_CUDA_ERR_ARG);
    }
  }
  if (lse) lse[t] = l;
  if (loss) loss[t] = v;
}

// Many rows, 32 a block: lane = row, warp w folds the row's pairs w, w + warps,
// ... and the warps' results meet in shared memory, in order.
constexpr int COMBINE_WARPS = 16;
__global__ void __launch_bounds__(32 * COMBINE_WARPS)
    xent_combine_kernel(const float2 *part, uint32_t nparts, const float *hit, const int32_t *target, float *loss,
                        float *lse, uint32_t T, uint32_t V, int *status) {
  __shared__ float2 got[COMBINE_WARPS][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t t = blockIdx.x * 32 + lane;
  dependent_wait();
  float2 x = make_float2(-INFINITY, 0.0f);
  if (t < T)
    for (uint32_t k = warp; k < nparts; k += COMBINE_WARPS) fold_pair(x, part[(size_t)k * T + t]);
  got[warp][lane] = x;
  __syncthreads();
  if (warp || t >= T) return;
  for (int w = 1; w < COMBINE_WARPS; ++w) fold_pair(x, got[w][lane]);
  finish_row<false>(t, x, hit, target, loss, lse, V, status);
}

// Few rows: a block a row, its threads share the pairs.
constexpr int FEW_THREADS = 256;
__global__ void __launch_bounds__(FEW_THREADS)
    xent_combine_few_kernel(const float2 *part, uint32_t nparts, const float *hit, const int32_t *target,
                            float *loss, float *lse, uint32_t T, uint32_t V, int *status) {
  __shared__ float2 got[FEW_THREADS / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t t = blockIdx.x;
  dependent_wait();
  float2 x = make_float2(-INFINITY, 0.0f);
  for (uint32_t k = threadIdx.x; k < nparts; k += FEW_THREADS) fold_pair(x, part[(size_t)k * T + t]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    fold_pair(x, make_float2(__shfl_xor_sync(0xffffffffu, x.x, o), __shfl_xor_sync(0xffffffffu, x.y, o)));
  if (lane == 0) got[warp] = x;
  __syncthreads();
  if (threadIdx.x) return;
  for (int w = 1; w < FEW_THREADS / 32; ++w) fold_pair(x, got[w]);
  finish_row<true>(t, x, hit, target, loss, lse, V, status);
}

bool g_smem_set[16][64] = {};
int g_pairs[16][64] = {};  // resident CTA pairs per device (0: not asked yet)

template <bool B_MN, bool PAIR, bool FWD, bool EXACT>
int launch(BwppCudaCtx *ctx, const CUtensorMap &tx, const CUtensorMap &tw, const CUtensorMap &to,
           const XentTile &a) {
  using C = Cfg<PAIR>;
  auto kern = xent_tc_kernel<B_MN, PAIR, FWD, EXACT>;
  const int v = (B_MN ? 1 : 0) + (PAIR ? 2 : 0) + (FWD ? 4 : 0) + (EXACT ? 8 : 0), dev = ctx->device;
  if (dev >= 64) return bwpp_set_error(ctx, BWPP_CUDA_ERR_UNSUPPORTED, "xent: device index >= 64");
  if (!g_smem_set[v][dev]) {
    const int rc = bwpp_check_cuda(
        ctx, cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM),
        "xent smem attribute");
    if (rc) return rc;
    g_smem_set[v][dev] = true;
  }
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = PAIR ? 2 : 1;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(ctx->num_sms & ~1), 1, 1);
  cfg.blockDim = dim3(THREADS, 1, 1);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = ctx->stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  uint32_t cap = (uint32_t)ctx->num_sms;
  if constexpr (PAIR) {
    int &pairs = g_pairs[v][dev];
    if (pairs == 0) {
      int n = 0;
      if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n <= 0) {
        (void)cudaGetLastError();
        pairs = -1;
      } else {
        pairs = n;
      }
    }
    if (pairs < 0) return BWPP_CUDA_ERR_UNSUPPORTED;
    cap = (uint32_t)pairs;
  }
  const uint64_t tiles = ((uint64_t)a.T + C::TILE_M - 1) / C::TILE_M * (((uint64_t)a.V + BN - 1) / BN);
  if (tiles >= 0x80000000ull) return bwpp_set_error(ctx, BWPP_CUDA_ERR_UNSUPPORTED, "xent: T * V too large");
  XentTile b = a;
  const uint32_t tail = (uint32_t)(tiles % cap);
  const bool halve = tail > 0 && 2 * tail <= cap;
  b.whole = (uint32_t)tiles - (halve ? tail : 0);
  b.items = (uint32_t)tiles + (halve ? tail : 0);
  // W is read from memory once per group of row blocks, whose 32 MB of x stay
  // in L2 (T 8192, V 32000, D 2048 over seconds: 1277 TFLOP/s with groups of 8
  // blocks, 1305 with 16, 1343 with all 32)
  const uint64_t block = (uint64_t)C::TILE_M * a.D * 2, fit = (32ull << 20) / block;
  const uint64_t blocks = ((uint64_t)a.T + C::TILE_M - 1) / C::TILE_M;
  b.group = (uint32_t)(fit < 8 ? 8 : fit > blocks ? blocks : fit);
  const uint32_t n = b.items < cap ? b.items : cap;
  cfg.gridDim = dim3((PAIR ? 2 : 1) * n, 1, 1);
  cfg.numAttrs = 2;
  int *status = ctx->status_word;
  return bwpp_check_cuda(ctx, cudaLaunchKernelEx(&cfg, kern, tx, tw, to, b, status),
                         FWD ? "xent logits" : "xent dlogit");
}

template <bool PAIR, bool FWD, bool EXACT>
int launch_layout(BwppCudaCtx *ctx, const CUtensorMap &tx, const CUtensorMap &tw, const CUtensorMap &to,
                  const XentTile &a, bool vocab_major) {
  return vocab_major ? launch<false, PAIR, FWD, EXACT>(ctx, tx, tw, to, a)
                     : launch<true, PAIR, FWD, EXACT>(ctx, tx, tw, to, a);
}

// CTA pairs, which load each column of W once for 256 rows (T 8192, V 32000, D 1024:
// 360 us, 425 with one CTA a tile; T 512: 31.9, 34.2), but for an odd number of
// blocks of 128 rows that is so small that the half of a pair without rows costs
// more: T 300, V 32000, D 4096: 110 us in pairs, 97 without; T 896, D 4096: 197 and
// 180 forward, 174 and 179 dlogit.
template <bool FWD, bool EXACT>
int launch_any(BwppCudaCtx *ctx, const CUtensorMap &tx, const CUtensorMap &tw, const CUtensorMap &to,
               const XentTile &a, bool vocab_major) {
  const uint32_t blocks = (a.T + BM - 1) / BM;
  if (blocks % 2 == 0 || blocks > (FWD ? 7u : 5u)) {
    const int rc = launch_layout<true, FWD, EXACT>(ctx, tx, tw, to, a, vocab_major);
    if (rc != BWPP_CUDA_ERR_UNSUPPORTED) return rc;
  }
  return launch_layout<false, FWD, EXACT>(ctx, tx, tw, to, a, vocab_major);
}

// K blocks of a sum (see EXACT).  At one token, V = 16384, D = 2048, chunks of two
// and of four take the same 15.5 us, of one 15.7.
uint32_t chunk_of(uint32_t T) { return T > XENT_EXACT_ROWS ? MANY_CHUNK : 2; }

// Rows of x in a load.  Few rows are loaded in a box of their own size (whole
// eights, a swizzle atom): the tile's other rows keep what shared memory holds,
// and nothing reads their logits.  (Rows filled with zeros past T cost one token
// 20.5 us instead of 18.4 at V 32000, D 1024, and 61 instead of 50 at D 4096.)
uint32_t x_box(uint32_t T) { return T < (uint32_t)BM ? (T + 7) & ~7u : (uint32_t)BM; }

int operand_maps(BwppCudaCtx *ctx, const XentOperands &o, CUtensorMap *tx, CUtensorMap *tw) {
  const auto BF = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const auto SW = CU_TENSOR_MAP_SWIZZLE_128B;
  int rc = bwpp_make_tmap_2d(ctx, tx, o.x, BF, o.D, o.T, (uint64_t)o.ldx * 2, BK, x_box(o.T), SW);
  if (!rc)
    rc = o.vocab_major ? bwpp_make_tmap_2d(ctx, tw, o.w, BF, o.D, o.V, (uint64_t)o.ldw * 2, BK, 64, SW)
                       : bwpp_make_tmap_2d(ctx, tw, o.w, BF, o.V, o.D, (uint64_t)o.ldw * 2, 64, BK, SW);
  return rc;
}

}  // namespace

int bwpp_xent_stats_launch(BwppCudaCtx *ctx, const XentOperands &o, const int32_t *target,
                           float2 *part, float *hit) {
  CUtensorMap tx, tw;
  const int rc = operand_maps(ctx, o, &tx, &tw);
  if (rc) return rc;
  XentTile a{};
  a.T = o.T;
  a.x_rows = x_box(o.T);
  a.V = o.V;
  a.D = o.D;
  a.v0 = o.v0;
  a.c = o.scale * 1.44269504f;
  a.scale = o.scale;
  a.target = target;
  a.part = part;
  a.hit = hit;
  const bool few = o.T <= XENT_EXACT_ROWS;
  a.apart = few;
  a.vocab = o.vocab;
  a.chunk = chunk_of(o.T);
  return few || o.D > a.chunk * BK
             ? launch_any<true, true>(ctx, tx, tw, tx, a, o.vocab_major)
             : launch_any<true, false>(ctx, tx, tw, tx, a, o.vocab_major);
}

int bwpp_xent_combine_launch(BwppCudaCtx *ctx, const float2 *part, uint32_t nparts, const float *hit,
                             const int32_t *target, float *loss, float *lse, uint32_t T, uint32_t V) {
  const bool few = T <= XENT_EXACT_ROWS;
  return bwpp_check_cuda(
      ctx,
      bwpp_launch_dependent(few ? xent_combine_few_kernel : xent_combine_kernel,
                            dim3(few ? T : (T + 31) / 32), dim3(few ? FEW_THREADS : 32 * COMBINE_WARPS),
                            0, ctx->stream, part, nparts, hit, target, loss, lse, T, V, ctx->status_word),
      "xent combine");
}

int bwpp_xent_dlogit_launch(BwppCudaCtx *ctx, const XentOperands &o, const int32_t *target,
                            const float *lse, const float *dloss, const float *common,
                            uint16_t *dlogit, uint32_t ld) {
  const bool exact = o.T <= XENT_EXACT_ROWS;
  CUtensorMap tx, tw, to;
  int rc = operand_maps(ctx, o, &tx, &tw);
  if (!rc)
    rc = bwpp_make_tmap_2d(ctx, &to, dlogit, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, o.V,
                           exact ? 2 * XENT_EXACT_ROWS : o.T, (uint64_t)ld * 2, 64, 32,
                           CU_TENSOR_MAP_SWIZZLE_128B);
  if (rc) return rc;
  XentTile a{};
  a.T = o.T;
  a.x_rows = x_box(o.T);
  a.V = o.V;
  a.D = o.D;
  a.v0 = o.v0;
  a.c = o.scale * 1.44269504f;
  a.scale = o.scale;
  a.target = target;
  a.lse = lse;
  a.dloss = dloss;
  a.common = common;
  a.chunk = chunk_of(o.T);
  a.vocab = o.vocab;
  // many rows: one sum over D, whose error in p (1e-5 at D = 4096) is far below the
  // rounding of dlogit
  return exact ? launch_layout<false, false, true>(ctx, tx, tw, to, a, o.vocab_major)
               : launch_any<false, false>(ctx, tx, tw, to, a, o.vocab_major);
}

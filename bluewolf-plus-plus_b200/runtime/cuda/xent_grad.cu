// The two products of the vocabulary cross entropy's gradient,
//   dx (+)= dlogit W      [T, D], K = the piece's vocabulary columns
//   dW    = dlogit^T x    (or its transpose), K = T
// in one persistent launch: all workers go through dx's tiles, then through
// dW's.  Either product alone leaves part of its last round idle (T 8192, D
// 2048: 3.46 rounds of 74 CTA pairs for dx); here the workers without a tile
// in dx's last round take as many tiles of dW ahead as one of dx takes time.
// (T 8192, V 32000, D 2048, a piece of 16384: 774 us, 1.42 PFLOP/s.  Half the
// workers on each product balance as well, but the tiles that run together then
// share less in L2: 830 us.)
// A product of few tiles with a long K is cut into K parts, each summed on its
// own in fp32; a last kernel adds the parts in order, so the result does not
// depend on which part ends first.
//
// The tile is the GEMM's (gemm.cu): 256 x 256 by a CTA pair (128 x 256 by one
// CTA), TMA-fed ring, one issuing thread, eight epilogue warps, two TMEM
// accumulators, bounded waits.  Operand layouts are the product's, not the
// kernel's: K-major or MN-major A and B per product.
#include <type_traits>

#include "bwpp_cuda_internal.cuh"
#include "xent.cuh"

namespace {

constexpr int BM = 128, BN = 256, BK = 64;
constexpr int A_STAGE = BM * BK * 2;
constexpr int BOX = 64 * BK * 2;
constexpr int EPI_WARPS = 8;
constexpr int EPI_BUF = 32 * 128;
constexpr int THREADS = 64 + 32 * EPI_WARPS;
constexpr uint32_t TMEM_COLS = 2 * BN;

template <bool PAIR>
struct Cfg {
  static constexpr int STAGES = PAIR ? 6 : 4;
  static constexpr int B_COLS = PAIR ? 128 : 256;  // columns of B that a CTA loads
  static constexpr int B_STAGE = B_COLS * BK * 2;
  static constexpr int OFF_B = STAGES * A_STAGE;
  static constexpr int OFF_C = OFF_B + STAGES * B_STAGE;
  static constexpr int OFF_BAR = OFF_C + EPI_WARPS * EPI_BUF;
  static constexpr int SMEM = OFF_BAR + 256 + 1024;
  static constexpr uint32_t TILE_M = PAIR ? 2 * BM : BM;
  static_assert(SMEM <= 232448, "exceeds the 227 KB opt-in limit");
  static_assert((2 * STAGES + 5) * 8 + 8 <= 256, "barrier block");
};

// One product C = A B of the launch.
struct Product {
  uint32_t M, N, K;
  uint32_t a_mn, b_mn;      // 1: MN-major operand
  uint32_t tiles_m, tiles_n, group;
  uint32_t parts, num_kb;   // K parts, K blocks in all
  uint32_t items;           // tiles * parts
  uint32_t part_rows;       // rows from one part's C to the next
  const float *add;         // fp32 rows added to C (pitch ld_add; may be C), or NULL
  uint32_t ld_add;
  const float *factor;      // multiplies C, or NULL
  uint32_t bf16;            // C is bf16, else fp32
  // TMA stores a row up to a multiple of 16 bytes, behind its last column as well:
  // it takes the columns below `whole`, and the few from there on are stored as they are
  uint32_t whole, ldc;
  void *c;
};

struct Maps {
  CUtensorMap a, b, c;
};

// The launch's products, dx (0) and dW (1), each possibly without items.
struct Work {
  Maps maps[2];
  Product product[2];
  uint32_t workers;
  uint32_t late;    // workers [0, late) have a tile in dx's last, partial round
  uint32_t ahead;   // tiles of dW that each other worker takes meanwhile
};

// The n-th item of a worker: its product and number; false past the last.
__device__ __forceinline__ bool nth_item(const Work &w, uint32_t worker, uint32_t n, uint32_t &which,
                                         uint32_t &item) {
  const uint32_t rounds = w.product[0].items / w.workers;
  const bool late = worker < w.late;
  const uint32_t mine = rounds + (late ? 1 : 0);
  if (n < mine) {
    which = 0;
    item = n * w.workers + worker;
    return true;
  }
  which = 1;
  uint32_t k = n - mine;
  const uint32_t others = w.workers - w.late;
  if (!late) {
    if (k < w.ahead) {
      item = k * others + worker - w.late;
      return item < w.product[1].items;
    }
    k -= w.ahead;
  }
  item = w.ahead * others + k * w.workers + worker;
  return item < w.product[1].items;
}

// Item i of product p: a tile and its K blocks [kb0, kb1).
__device__ __forceinline__ void item_at(const Product &p, uint32_t i, uint32_t &mb, uint32_t &nb,
                                        uint32_t &part, uint32_t &kb0, uint32_t &kb1) {
  const uint32_t tiles = p.tiles_m * p.tiles_n;
  part = i / tiles;
  const uint32_t t = i - part * tiles;
  const uint32_t per_group = p.group * p.tiles_n, g = t / per_group, first = g * p.group;
  const uint32_t gm = min(p.group, p.tiles_m - first), r = t - g * per_group;
  mb = first + r % gm;
  nb = r / gm;
  kb0 = (uint32_t)((uint64_t)part * p.num_kb / p.parts);
  kb1 = (uint32_t)((uint64_t)(part + 1) * p.num_kb / p.parts);
}

// f(A MN-major, B MN-major) with the layouts as compile-time constants: the
// loops that feed and issue have nothing to decide in them.
template <typename F>
__device__ __forceinline__ void by_layout(bool a_mn, bool b_mn, F f) {
  using yes = std::true_type;
  using no = std::false_type;
  if (a_mn) {
    if (b_mn) f(yes{}, yes{}); else f(yes{}, no{});
  } else {
    if (b_mn) f(no{}, yes{}); else f(no{}, no{});
  }
}

template <bool PAIR>
__global__ void __launch_bounds__(THREADS, 1)
    xent_grad_kernel(const __grid_constant__ Work work, int *status) {
  using C = Cfg<PAIR>;
  constexpr int STAGES = C::STAGES;
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
    for (int i = 0; i < 2; ++i) {
      if (!work.product[i].items) continue;
      prefetch_tmap(&work.maps[i].a);
      prefetch_tmap(&work.maps[i].b);
      prefetch_tmap(&work.maps[i].c);
    }
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
      uint32_t which, i;
      for (uint32_t n = 0; !*abort_flag && nth_item(work, worker, n, which, i); ++n) {
        const Product &p = work.product[which];
        uint32_t mb, nb, part, kb0, kb1;
        item_at(p, i, mb, nb, part, kb0, kb1);
        const CUtensorMap *ma = &work.maps[which].a, *mb_ = &work.maps[which].b;
        const int32_t row0 = (int32_t)(mb * C::TILE_M + rank * BM);
        const int32_t col0 = (int32_t)(nb * BN + rank * (PAIR ? C::B_COLS : 0));
        auto feed = [&](auto a_mn, auto b_mn) {
          for (uint32_t kb = kb0; kb < kb1; ++kb) {
            if (!mbar_wait(&empty[stage], phase ^ 1, status)) {
              *abort_flag = 1;
              break;
            }
            // both CTAs' bytes count on rank 0's barrier
            if (rank == 0)
              mbar_arrive_expect_tx(&full[stage], (PAIR ? 2 : 1) * (A_STAGE + C::B_STAGE));
            [[maybe_unused]] uint32_t fbar = 0;
            if constexpr (PAIR) fbar = cluster_addr(&full[stage], 0);
            auto load = [&](void *dst, const CUtensorMap *map, int32_t x, int32_t y) {
              if constexpr (PAIR) tma_load_2d_pair(dst, map, fbar, x, y);
              else tma_load_2d(dst, map, &full[stage], x, y);
            };
            const int32_t k0 = (int32_t)(kb * BK);
            uint8_t *sa = smem + stage * A_STAGE;
            uint8_t *sb = smem + C::OFF_B + stage * C::B_STAGE;
            if constexpr (a_mn) {
#pragma unroll
              for (int j = 0; j < BM / 64; ++j) load(sa + j * BOX, ma, row0 + j * 64, k0);
            } else {
              load(sa, ma, k0, row0);
            }
#pragma unroll
            for (int j = 0; j < C::B_COLS / 64; ++j) {
              if constexpr (b_mn) load(sb + j * BOX, mb_, col0 + j * 64, k0);
              else load(sb + j * BOX, mb_, k0, col0 + j * 64);
            }
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1;
            }
          }
        };
        by_layout(p.a_mn, p.b_mn, feed);
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
      uint32_t which, i;
      for (uint32_t n = 0; !*abort_flag && nth_item(work, worker, n, which, i); ++n) {
        const Product &p = work.product[which];
        uint32_t mb, nb, part, kb0, kb1;
        item_at(p, i, mb, nb, part, kb0, kb1);
        if (!mbar_wait(&tempty[acc], acc_phase ^ 1, status)) {
          *abort_flag = 1;
          break;
        }
        tc_fence_after();
        bool ok = true;
        auto multiply = [&](auto a_mn, auto b_mn) {
          constexpr uint32_t idesc = make_idesc_bf16_f32(C::TILE_M, BN, a_mn ? 1u : 0u, b_mn ? 1u : 0u);
          for (uint32_t kb = kb0; kb < kb1; ++kb) {
            if (!mbar_wait(&full[stage], phase, status)) {
              *abort_flag = 1;
              ok = false;
              break;
            }
            tc_fence_after();
            // K-major: 16 of K are 32 bytes inside the 128-byte swizzle; MN-major:
            // 64-element atoms 8 KB apart, 16 rows of K are 2 KB
            const uint64_t ad = make_smem_desc(smem_u32(smem + stage * A_STAGE), a_mn ? BOX : 16, 1024,
                                               BWPP_SWIZZLE_128B);
            const uint64_t bd = make_smem_desc(smem_u32(smem + C::OFF_B + stage * C::B_STAGE),
                                               b_mn ? BOX : 16, 1024, BWPP_SWIZZLE_128B);
#pragma unroll
            for (int ks = 0; ks < BK / 16; ++ks) {
              const uint64_t as = desc_add(ad, ks * (a_mn ? 2048 : 32));
              const uint64_t bs = desc_add(bd, ks * (b_mn ? 2048 : 32));
              const uint32_t accum = kb != kb0 || ks != 0 ? 1u : 0u;
              if constexpr (PAIR) tc_mma_f16_ss_pair(tmem_base + acc * BN, as, bs, idesc, accum);
              else tc_mma_f16_ss(tmem_base + acc * BN, as, bs, idesc, accum);
            }
            commit(&empty[stage]);
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1;
            }
          }
        };
        by_layout(p.a_mn, p.b_mn, multiply);
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
    const int q = warp & 3;   // TMEM lane quarter of this warp
    const int ew = warp - 2;
    const int sub = ew >> 2;  // the two warps of a quarter take alternate chunks
    uint8_t *stage_c = smem + C::OFF_C + ew * EPI_BUF;
    const uint32_t tq = (uint32_t)(q * 32) << 16;
    uint32_t acc = 0, acc_phase = 0;
    uint32_t which, i;
    for (uint32_t n = 0; !*abort_flag && nth_item(work, worker, n, which, i); ++n) {
      const Product &p = work.product[which];
      uint32_t mb, nb, part, kb0, kb1;
      item_at(p, i, mb, nb, part, kb0, kb1);
      const bool out16 = p.bf16 != 0;
      const uint32_t M = p.M, N = p.N, whole = p.whole;
      const CUtensorMap *mc = &work.maps[which].c;
      const uint32_t cw = out16 ? 64 : 32;  // columns of 128 bytes
      const uint32_t row0 = mb * C::TILE_M + rank * BM + q * 32, row = row0 + lane;
      const uint32_t out_row = part * p.part_rows + row0;
      const float *add = p.add && row < M ? p.add + (size_t)(out_row + lane) * p.ld_add : nullptr;
      const float factor = p.factor ? __ldcg(p.factor) : 1.0f;
      if (!mbar_wait(&tfull[acc], acc_phase, status)) {
        *abort_flag = 1;
        break;
      }
      tc_fence_after();
      for (uint32_t k = sub; k < BN / cw; k += 2) {
        const uint32_t c0 = nb * BN + k * cw;
        if (c0 >= N) break;
        uint32_t out[32];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (h && !out16) break;
          const uint32_t cs = c0 + h * 32;
          uint32_t r[32];
          tmem_ld_32x32b_x32(tmem_base + tq + acc * BN + k * cw + h * 32, r);
          tc_wait_ld(r);
          if (add) {
            if (cs + 32 <= N) {
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const float4 t = *reinterpret_cast<const float4 *>(add + cs + 4 * j);
                r[4 * j] = __float_as_uint(__uint_as_float(r[4 * j]) + t.x);
                r[4 * j + 1] = __float_as_uint(__uint_as_float(r[4 * j + 1]) + t.y);
                r[4 * j + 2] = __float_as_uint(__uint_as_float(r[4 * j + 2]) + t.z);
                r[4 * j + 3] = __float_as_uint(__uint_as_float(r[4 * j + 3]) + t.w);
              }
            } else {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (cs + j < N) r[j] = __float_as_uint(__uint_as_float(r[j]) + add[cs + j]);
            }
          }
          const uint64_t f2 = f2pack(factor, factor);
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            float x, y;
            f2unpack(f2mul(f2pack(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])), f2), x, y);
            if (out16) {
              out[h * 16 + j] = pack2_16<false>(x, y);
            } else {
              out[2 * j] = __float_as_uint(x);
              out[2 * j + 1] = __float_as_uint(y);
            }
          }
        }
        if (lane == 0) tma_store_wait_read<0>();
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 8; ++j)
          *reinterpret_cast<uint4 *>(stage_c + lane * 128 + ((j ^ (lane & 7)) << 4)) =
              make_uint4(out[4 * j], out[4 * j + 1], out[4 * j + 2], out[4 * j + 3]);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0 && row0 < M && c0 < whole) {
          tma_store_2d(mc, stage_c, (int32_t)c0, (int32_t)out_row);
          tma_store_commit();
        }
      }
      // the columns from `whole` on: in one 16-byte piece of each row, and in this warp's
      // last chunk if in one of its chunks, so they are still staged
      const uint32_t at = whole - nb * BN;
      if (whole < N && at < BN && (at / cw & 1) == (uint32_t)sub && row < M) {
        const uint32_t j = at % cw / (out16 ? 8 : 4);
        const uint4 t = *reinterpret_cast<const uint4 *>(stage_c + lane * 128 + ((j ^ (lane & 7)) << 4));
        const uint32_t w[4] = {t.x, t.y, t.z, t.w};
        const size_t to = (size_t)(out_row + lane) * p.ldc + whole;
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) {
          if (whole + e >= N) break;
          if (out16)
            static_cast<uint16_t *>(p.c)[to + e] = (uint16_t)(w[e / 2] >> (16 * (e & 1)));
          else if (e < 4)
            static_cast<float *>(p.c)[to + e] = __uint_as_float(w[e]);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (PAIR) mbar_arrive_cluster(cluster_addr(&tempty[acc], 0));
        else mbar_arrive(&tempty[acc]);
      }
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1;
    }
    if (lane == 0) tma_store_wait_all<0>();
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

// A product from its K parts, added in order, into rows of any pitch.  second: a
// part has two terms, so many elements apart.  A thread takes four columns (the
// parts' rows are padded to whole 32 bytes) and has four parts' loads in flight:
// 64 rows x 768 of eight parts took 7.2 us with eight columns and one part.
__global__ void __launch_bounds__(256)
    xent_sum_parts_kernel(const float *part, uint32_t parts, size_t part_stride, size_t second,
                          const float *factor, void *out, uint32_t rows, uint32_t cols, size_t ld,
                          size_t ld_out, int bf16, int wide) {
  dependent_wait();
  const uint32_t quads = (cols + 3) / 4;
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * quads) return;
  const uint32_t r = i / quads, c = (i - r * quads) * 4;
  const float f = factor ? *factor : 1.0f;
  const float *p = part + r * ld + c;
  float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  auto add = [&](float4 t) {
    v[0] += t.x;
    v[1] += t.y;
    v[2] += t.z;
    v[3] += t.w;
  };
  auto at = [](const float *q) { return *reinterpret_cast<const float4 *>(q); };
  uint32_t s = 0;
  for (; s + 4 <= parts; s += 4, p += 4 * part_stride) {
    float4 t[4], u[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      t[k] = at(p + k * part_stride);
      u[k] = second ? at(p + k * part_stride + second) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      add(make_float4(t[k].x + u[k].x, t[k].y + u[k].y, t[k].z + u[k].z, t[k].w + u[k].w));
  }
#pragma unroll 3
  for (; s < parts; ++s, p += part_stride) {
    const float4 t = at(p);
    const float4 u = second ? at(p + second) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    add(make_float4(t.x + u.x, t.y + u.y, t.z + u.z, t.w + u.w));
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] *= f;
  const size_t to = r * ld_out + c;
  if (wide && c + 4 <= cols) {  // whole quads at aligned places
    if (bf16)
      *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(out) + to) =
          make_uint2(pack2_16<false>(v[0], v[1]), pack2_16<false>(v[2], v[3]));
    else
      *reinterpret_cast<float4 *>(static_cast<float *>(out) + to) = make_float4(v[0], v[1], v[2], v[3]);
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (c + k >= cols) break;
    if (bf16)
      static_cast<uint16_t *>(out)[to + k] = (uint16_t)(pack2_16<false>(v[k], 0.0f) & 0xFFFFu);
    else
      static_cast<float *>(out)[to + k] = v[k];
  }
}

bool g_smem_set[2][64] = {};
int g_pairs[64] = {};  // resident CTA pairs per device (0: not asked yet, -1: none)

inline uint32_t ceil_div(uint32_t a, uint32_t b) { return (uint32_t)(((uint64_t)a + b - 1) / b); }

template <bool PAIR>
int prepare(BwppCudaCtx *ctx) {
  if (ctx->device >= 64)
    return bwpp_set_error(ctx, BWPP_CUDA_ERR_UNSUPPORTED, "xent: device index >= 64");
  bool &set = g_smem_set[PAIR][ctx->device];
  if (set) return BWPP_CUDA_OK;
  const int rc = bwpp_check_cuda(
      ctx,
      cudaFuncSetAttribute(xent_grad_kernel<PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           Cfg<PAIR>::SMEM),
      "xent smem attribute");
  set = rc == BWPP_CUDA_OK;
  return rc;
}

// Sets `pairs` to the CTA pairs that run together on ctx's device, or -1.
int resident_pairs(BwppCudaCtx *ctx, int *out) {
  int rc = prepare<true>(ctx);
  if (rc) return rc;
  int &pairs = g_pairs[ctx->device];
  *out = pairs;
  if (pairs) return BWPP_CUDA_OK;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(ctx->num_sms & ~1), 1, 1);
  cfg.blockDim = dim3(THREADS, 1, 1);
  cfg.dynamicSmemBytes = Cfg<true>::SMEM;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, xent_grad_kernel<true>, &cfg) != cudaSuccess || n <= 0) {
    (void)cudaGetLastError();
    n = -1;
  }
  *out = pairs = n;
  return n > 0 ? BWPP_CUDA_OK : prepare<false>(ctx);
}

int operand_map(BwppCudaCtx *ctx, CUtensorMap *map, const uint16_t *base, bool mn, uint32_t rows,
                uint32_t k, uint32_t ld, uint32_t box_rows) {
  const auto BF = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const auto SW = CU_TENSOR_MAP_SWIZZLE_128B;
  return mn ? bwpp_make_tmap_2d(ctx, map, base, BF, rows, k, (uint64_t)ld * 2, 64, BK, SW)
            : bwpp_make_tmap_2d(ctx, map, base, BF, k, rows, (uint64_t)ld * 2, BK, box_rows, SW);
}

int make_product(BwppCudaCtx *ctx, const XentProduct &s, uint32_t tile_m, uint32_t parts, Maps &m,
                 Product &p) {
  p = Product{};
  p.M = s.M;
  p.N = s.N;
  p.K = s.K;
  p.a_mn = s.a_mn ? 1 : 0;
  p.b_mn = s.b_mn ? 1 : 0;
  p.tiles_m = ceil_div(s.M, tile_m);
  p.tiles_n = ceil_div(s.N, BN);
  p.num_kb = ceil_div(s.K, BK);
  p.parts = parts;
  p.part_rows = s.part_rows;
  p.add = s.accumulate ? static_cast<const float *>(s.add) : nullptr;
  p.ld_add = s.ld_add;
  p.factor = s.factor;
  p.bf16 = s.bf16 ? 1 : 0;
  const uint32_t unit = s.bf16 ? 8 : 4;  // columns of 16 bytes
  p.whole = s.guarded ? s.N / unit * unit : s.N;
  p.ldc = s.ldc;
  p.c = s.c;
  const uint64_t items = (uint64_t)p.tiles_m * p.tiles_n * parts;
  if (items >= 0x80000000ull) return bwpp_set_error(ctx, BWPP_CUDA_ERR_UNSUPPORTED, "xent: too many tiles");
  p.items = (uint32_t)items;
  int rc = operand_map(ctx, &m.a, s.a, s.a_mn, s.M, s.K, s.lda, BM);
  if (!rc) rc = operand_map(ctx, &m.b, s.b, s.b_mn, s.N, s.K, s.ldb, 64);
  const uint64_t rows = parts > 1 ? (uint64_t)parts * s.part_rows : s.M;
  const uint32_t cols = p.whole ? p.whole : unit;  // without whole pieces the map is not used
  if (!rc)
    rc = s.bf16 ? bwpp_make_tmap_2d(ctx, &m.c, s.c, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, cols, rows,
                                    (uint64_t)s.ldc * 2, 64, 32, CU_TENSOR_MAP_SWIZZLE_128B)
                : bwpp_make_tmap_2d(ctx, &m.c, s.c, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, cols, rows,
                                    (uint64_t)s.ldc * 4, 32, 32, CU_TENSOR_MAP_SWIZZLE_128B);
  return rc;
}

// Row blocks that go through the columns together: the workers cover about two
// such groups at once (T 8192, V 32000, D 2048: 774 us a piece with 4 blocks,
// 781 with 9, 791 with 16).
uint32_t group_of(const Product &p, uint32_t workers) {
  if (2 * p.tiles_n <= workers) return workers / (2 * p.tiles_n);
  return 2 * p.tiles_m <= workers ? p.tiles_m : 6;
}

// A tile's time in K blocks; its epilogue counts as three.
uint32_t tile_time(uint32_t num_kb, uint32_t parts) { return ceil_div(num_kb, parts) + 3; }

}  // namespace

int bwpp_xent_parts(BwppCudaCtx *ctx, const XentProduct &dx, const XentProduct &dw, uint32_t most_dx,
                    uint32_t most_dw, uint32_t *dx_parts, uint32_t *dw_parts) {
  int pairs;
  const int rc = resident_pairs(ctx, &pairs);
  if (rc) return rc;
  const uint32_t cap = pairs > 0 ? (uint32_t)pairs : (uint32_t)ctx->num_sms;
  const uint32_t tile_m = pairs > 0 ? 2 * BM : BM;
  const uint64_t tx = (uint64_t)ceil_div(dx.M, tile_m) * ceil_div(dx.N, BN);
  const uint64_t tw = (uint64_t)ceil_div(dw.M, tile_m) * ceil_div(dw.N, BN);
  const uint32_t kx = ceil_div(dx.K, BK), kw = ceil_div(dw.K, BK);
  uint64_t best = ~0ull;
  *dx_parts = *dw_parts = 1;
  for (uint32_t s = 1; s <= most_dx && s <= kx; ++s)
    for (uint32_t q = 1; q <= most_dw && q <= kw; ++q) {
      const uint64_t late = tx * s % cap, cx = tile_time(kx, s), cw = tile_time(kw, q);
      const uint64_t ahead = late ? cx / cw * (cap - late) : 0;
      uint64_t t = (tx * s + cap - 1) / cap * cx;
      if (tw * q > ahead) t += (tw * q - ahead + cap - 1) / cap * cw;
      // parts' sums are written and read once more: worth an eighth of the time
      t = t * (8 + (s > 1) + (q > 1));
      if (t < best) {
        best = t;
        *dx_parts = s;
        *dw_parts = q;
      }
    }
  return BWPP_CUDA_OK;
}

int bwpp_xent_grad_launch(BwppCudaCtx *ctx, const XentProduct *dx, const XentProduct *dw,
                          uint32_t dx_parts, uint32_t dw_parts) {
  int pairs;
  int rc = resident_pairs(ctx, &pairs);
  if (rc) return rc;
  const uint32_t cap = pairs > 0 ? (uint32_t)pairs : (uint32_t)ctx->num_sms;
  const uint32_t tile_m = pairs > 0 ? 2 * BM : BM;
  // a last, short piece may have fewer K blocks than parts
  if (dx && dx_parts > ceil_div(dx->K, BK)) dx_parts = ceil_div(dx->K, BK);
  Work work{};
  Product &p0 = work.product[0], &p1 = work.product[1];
  if (dx) rc = make_product(ctx, *dx, tile_m, dx_parts, work.maps[0], p0);
  if (!rc && dw) rc = make_product(ctx, *dw, tile_m, dw_parts, work.maps[1], p1);
  if (rc) return rc;
  const uint64_t items = (uint64_t)p0.items + p1.items;
  const uint32_t n = items < cap ? (uint32_t)items : cap;
  work.workers = n;
  work.late = p0.items % n;
  if (work.late && dw)
    work.ahead = tile_time(p0.num_kb, p0.parts) / tile_time(p1.num_kb, p1.parts);
  if (dx) p0.group = group_of(p0, n);
  if (dw) p1.group = group_of(p1, n);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = pairs > 0 ? 2 : 1;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((pairs > 0 ? 2 : 1) * n, 1, 1);
  cfg.blockDim = dim3(THREADS, 1, 1);
  cfg.dynamicSmemBytes = pairs > 0 ? Cfg<true>::SMEM : Cfg<false>::SMEM;
  cfg.stream = ctx->stream;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  int *status = ctx->status_word;
  return bwpp_check_cuda(
      ctx,
      pairs > 0 ? cudaLaunchKernelEx(&cfg, xent_grad_kernel<true>, work, status)
                : cudaLaunchKernelEx(&cfg, xent_grad_kernel<false>, work, status),
      "xent gradient");
}

int bwpp_xent_sum_parts_launch(BwppCudaCtx *ctx, const float *part, uint32_t parts,
                               size_t part_stride, size_t second, const float *factor, void *out,
                               uint32_t rows, uint32_t cols, uint32_t ld, uint32_t ld_out, int bf16) {
  const uint32_t quads = (uint32_t)(((uint64_t)cols + 3) / 4), most = (1u << 30) / quads;
  const size_t es = bf16 ? 2 : 4;
  const int wide = ld_out % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & (4 * es - 1)) == 0;
  for (uint32_t r0 = 0; r0 < rows; r0 += most) {
    const uint32_t n = rows - r0 < most ? rows - r0 : most;
    uint8_t *to = static_cast<uint8_t *>(out) + (size_t)r0 * ld_out * es;
    const int rc = bwpp_check_cuda(
        ctx,
        bwpp_launch_dependent(xent_sum_parts_kernel, dim3((n * quads + 255) / 256), dim3(256), 0,
                              ctx->stream, part + (size_t)r0 * ld, parts, part_stride, second, factor, to,
                              n, cols, ld, ld_out, bf16, wide),
        "xent sum");
    if (rc) return rc;
  }
  return BWPP_CUDA_OK;
}

// Typed element access for row kernels whose tensors come as f16, bf16 or
// fp32: VEC consecutive elements as one transfer (two 16-byte ones for eight
// fp32), widened to fp32.  The template's type numbers are BwppCudaDType's.
#pragma once

#include "bwpp_cuda_internal.cuh"

namespace bwpp_elem {

template <int DT>
struct Elem {
  using type = uint16_t;
};
template <>
struct Elem<BWPP_CUDA_DTYPE_F32> {
  using type = float;
};

// VEC elements as they lie in memory.
template <int DT, int VEC>
struct Raw {
  static constexpr int BYTES = VEC * (int)sizeof(typename Elem<DT>::type);
  static constexpr int WORDS = BYTES < 4 ? 1 : BYTES / 4;
  uint32_t w[WORDS];

  __device__ __forceinline__ void load(const typename Elem<DT>::type *p) {
    if constexpr (BYTES >= 16) {
#pragma unroll
      for (int i = 0; i < BYTES / 16; ++i) {
        const uint4 t = __ldcs(reinterpret_cast<const uint4 *>(p) + i);
        w[4 * i] = t.x; w[4 * i + 1] = t.y; w[4 * i + 2] = t.z; w[4 * i + 3] = t.w;
      }
    } else if constexpr (BYTES == 8) {
      const uint2 t = __ldcs(reinterpret_cast<const uint2 *>(p));
      w[0] = t.x; w[1] = t.y;
    } else if constexpr (BYTES == 4) {
      w[0] = __ldcs(reinterpret_cast<const uint32_t *>(p));
    } else {
      w[0] = __ldcs(reinterpret_cast<const uint16_t *>(p));
    }
  }

  // From shared memory (VEC elements are 8 or 16 bytes).
  __device__ __forceinline__ void load_shared(const uint8_t *p) {
    static_assert(BYTES == 8 || BYTES == 16, "8 or 16 bytes");
    if constexpr (BYTES == 16) {
      const uint4 t = *reinterpret_cast<const uint4 *>(p);
      w[0] = t.x; w[1] = t.y; w[2] = t.z; w[3] = t.w;
    } else {
      const uint2 t = *reinterpret_cast<const uint2 *>(p);
      w[0] = t.x; w[1] = t.y;
    }
  }

  __device__ __forceinline__ void store(typename Elem<DT>::type *p) const {
    if constexpr (BYTES >= 16) {
#pragma unroll
      for (int i = 0; i < BYTES / 16; ++i)
        __stcs(reinterpret_cast<uint4 *>(p) + i,
               make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]));
    } else if constexpr (BYTES == 8) {
      __stcs(reinterpret_cast<uint2 *>(p), make_uint2(w[0], w[1]));
    } else if constexpr (BYTES == 4) {
      __stcs(reinterpret_cast<uint32_t *>(p), w[0]);
    } else {
      __stcs(reinterpret_cast<uint16_t *>(p), (uint16_t)w[0]);
    }
  }

  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) w[i] = 0u;
  }

  __device__ __forceinline__ float get(int i) const {
    if constexpr (DT == BWPP_CUDA_DTYPE_F32) return __uint_as_float(w[i]);
    else
      return load16<DT == BWPP_CUDA_DTYPE_F16>((uint16_t)(w[i / 2] >> (16 * (i & 1))));
  }

  // Rounded once, to nearest even.
  __device__ __forceinline__ void set(const float (&v)[VEC]) {
    if constexpr (DT == BWPP_CUDA_DTYPE_F32) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) w[i] = __float_as_uint(v[i]);
    } else if constexpr (VEC == 1) {
      w[0] = pack2_16<DT == BWPP_CUDA_DTYPE_F16>(v[0], 0.0f) & 0xFFFFu;
    } else {
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i)
        w[i] = pack2_16<DT == BWPP_CUDA_DTYPE_F16>(v[2 * i], v[2 * i + 1]);
    }
  }
};

inline bool aligned_to(const void *p, size_t bytes) {
  return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0;
}

}  // namespace bwpp_elem

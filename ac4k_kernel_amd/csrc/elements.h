// Vectors of eight elements of any of the three float types, at any element address, for the kernels that read and write whole rows.
#pragma once

#include "linear_common.h"

namespace ac4k {

template <int DT>
struct Vec8 {
  static constexpr int WORDS = DT == AC4K_DTYPE_FP32 ? 8 : 4;
  uint32_t w[WORDS];
};

template <int DT>
__device__ __forceinline__ void vec8_zero(Vec8<DT> &v) {
#pragma unroll
  for (int i = 0; i < Vec8<DT>::WORDS; ++i) v.w[i] = 0;
}

// all eight elements at p (element aligned: the target takes vector accesses at any address)
template <int DT>
__device__ __forceinline__ void vec8_load_all(Vec8<DT> &v, const void *p) {
  const u32x4 a = *static_cast<const u32x4_elem *>(p);
  v.w[0] = a.x, v.w[1] = a.y, v.w[2] = a.z, v.w[3] = a.w;
  if constexpr (DT == AC4K_DTYPE_FP32) {
    const u32x4 b = static_cast<const u32x4_elem *>(p)[1];
    v.w[4] = b.x, v.w[5] = b.y, v.w[6] = b.z, v.w[7] = b.w;
  }
}
template <int DT>
__device__ __forceinline__ void vec8_store_all(void *p, const Vec8<DT> &v) {
  static_cast<u32x4_elem *>(p)[0] = (u32x4){v.w[0], v.w[1], v.w[2], v.w[3]};
  if constexpr (DT == AC4K_DTYPE_FP32) static_cast<u32x4_elem *>(p)[1] = (u32x4){v.w[4], v.w[5], v.w[6], v.w[7]};
}

// the first n elements at p (0 < n < 8), zeros behind them: a piece each of four, two and one
template <int DT>
__device__ __forceinline__ void vec8_load_some(Vec8<DT> &v, const void *p, int n) {
  if constexpr (DT == AC4K_DTYPE_FP32) {
    const uint32_t *q = static_cast<const uint32_t *>(p);
    u32x4 a = {0, 0, 0, 0};
    u32x2 b = {0, 0};
    uint32_t c = 0;
    if (n & 4) a = *reinterpret_cast<const u32x4_elem *>(q);
    if (n & 2) b = *reinterpret_cast<const u32x2_elem *>(q + (n & 4));
    if (n & 1) c = q[n & 6];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t rest = (n & 2) && i % 4 < 2 ? b[i % 2] : i % 4 == (n & 2) ? c : 0;  // behind the piece of four, or from the start
      v.w[i] = i < 4 ? ((n & 4) ? a[i % 4] : rest) : ((n & 4) ? rest : 0);
    }
  } else {
    const uint16_t *q = static_cast<const uint16_t *>(p);
    u32x2 a = {0, 0};
    uint32_t b = 0, c = 0;
    if (n & 4) a = *reinterpret_cast<const u32x2_elem *>(q);
    if (n & 2) b = *reinterpret_cast<const u32_elem *>(q + (n & 4));
    if (n & 1) c = q[n & 6];
    const uint32_t first = (n & 2) ? b : c, second = (n & 2) ? c : 0;
    v.w[0] = (n & 4) ? a.x : first;
    v.w[1] = (n & 4) ? a.y : second;
    v.w[2] = (n & 4) ? first : 0;
    v.w[3] = (n & 4) ? second : 0;
  }
}
template <int DT>
__device__ __forceinline__ void vec8_store_some(void *p, const Vec8<DT> &v, int n) {
  if constexpr (DT == AC4K_DTYPE_FP32) {
    uint32_t *q = static_cast<uint32_t *>(p);
    if (n & 4) *reinterpret_cast<u32x4_elem *>(q) = (u32x4){v.w[0], v.w[1], v.w[2], v.w[3]};
    if (n & 2) *reinterpret_cast<u32x2_elem *>(q + (n & 4)) = (u32x2){(n & 4) ? v.w[4] : v.w[0], (n & 4) ? v.w[5] : v.w[1]};
    if (n & 1) q[n & 6] = (n & 4) ? ((n & 2) ? v.w[6] : v.w[4]) : ((n & 2) ? v.w[2] : v.w[0]);
  } else {
    uint16_t *q = static_cast<uint16_t *>(p);
    const uint32_t first = (n & 4) ? v.w[2] : v.w[0], second = (n & 4) ? v.w[3] : v.w[1];
    if (n & 4) *reinterpret_cast<u32x2_elem *>(q) = (u32x2){v.w[0], v.w[1]};
    if (n & 2) *reinterpret_cast<u32_elem *>(q + (n & 4)) = first;
    if (n & 1) q[n & 6] = (uint16_t)((n & 2) ? second : first);
  }
}

// elements [k, k + 8) of a row of K: what lies behind the row reads as zero and is not written
template <int DT>
__device__ __forceinline__ void vec8_load(Vec8<DT> &v, const void *row, int64_t k, int64_t K) {
  const char *p = static_cast<const char *>(row) + k * (int64_t)sizeof(typename Elem<DT>::T);
  if (k + 8 <= K) vec8_load_all(v, p);
  else if (k < K) vec8_load_some(v, p, (int)(K - k));
  else vec8_zero(v);
}
template <int DT>
__device__ __forceinline__ void vec8_store(void *row, const Vec8<DT> &v, int64_t k, int64_t K) {
  char *p = static_cast<char *>(row) + k * (int64_t)sizeof(typename Elem<DT>::T);
  if (k + 8 <= K) vec8_store_all(p, v);
  else if (k < K) vec8_store_some(p, v, (int)(K - k));
}

template <int DT>
__device__ __forceinline__ float vec8_get(const Vec8<DT> &v, int i) {
  if constexpr (DT == AC4K_DTYPE_FP32) return __uint_as_float(v.w[i]);
  else if constexpr (DT == AC4K_DTYPE_BF16) return i & 1 ? bf16_hi(v.w[i / 2]) : bf16_lo(v.w[i / 2]);
  else return (float)__builtin_bit_cast(f16x2, v.w[i / 2])[i & 1];
}
// rounded to the type once, to nearest even
template <int DT>
__device__ __forceinline__ void vec8_set(Vec8<DT> &v, const float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if constexpr (DT == AC4K_DTYPE_FP32) v.w[i] = __float_as_uint(f[i]);
    else if (i & 1) v.w[i / 2] = Elem<DT>::cvt2(f[i - 1], f[i]);
}

}  // namespace ac4k

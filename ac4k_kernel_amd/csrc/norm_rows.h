// The kernel of the norms of rows: rms_norm (norm.hip) and, with BLOCK, block_norm (block_norm.hip), whose rows are a sum with a gate and whose values are
// centred and modulated.
#pragma once

#include "elements.h"

namespace ac4k {

enum NormOut { NORM_PLAIN = 0, NORM_FP8 = 1, NORM_INT8 = 2, NORM_NVFP4 = 3, NORM_STATS = 4, NORM_NVFP4_SECOND = 5, NORM_NVFP4_ONE = 6 };

// Rows of block_norm come in two kernels: without a vector that is cut by the row's end there is half the code, which keeps a third fewer registers.
enum NormMode { NORM_ROWS = 0, NORM_BLOCK = 1, NORM_BLOCK_CUT = 2 };

// one of a block's vectors of K: the same for all rows (rows 0), or one for so many rows each
struct NormVector {
  const void *p;
  int64_t stride;
  uint32_t rows;
};
struct NormArgs {
  const void *x, *residual, *weight;
  void *sum;              // h, where there is a residual
  void *out;
  void *sf;
  float *gs;              // nvfp4: given (NORM_NVFP4) or found
  float *factors;         // r of each row, NORM_STATS -> NORM_NVFP4_SECOND
  float *maxima;          // max|y| of each workgroup, likewise
  int64_t rows, K, Kp, Rp;
  int64_t x_stride, residual_stride, sum_stride, out_stride;  // elements between rows
  double eps, inverse_K;
  int maxima_count;
  // of a block
  NormVector gate, scale, shift;
  const void *post;       // weight of the norm of x, or null
  float *means;           // of each row, the mean in two pieces, like factors
  float alpha;            // of the residual
  bool centred;           // layer norm
};

constexpr float NORM_LEAST = 0x1p-100f;  // a smaller maximum counts as zero

// Sum over groups of L lanes (16, 32 or 64), in every lane of the group.  (By lane shuffles through LDS, a row's chain of waits was half a microsecond longer.)
template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, (uint64_t)dpp_u32<CTRL>((uint32_t)(b >> 32)) << 32 | dpp_u32<CTRL>((uint32_t)b));
}
template <int L>
__device__ __forceinline__ double group_sum(double v) {
  v += dpp_f64<DPP_QUAD_XOR1>(v);
  v += dpp_f64<DPP_QUAD_XOR2>(v);
  v += dpp_f64<DPP_ROW_HALF_MIRROR>(v);
  v += dpp_f64<DPP_ROW_MIRROR>(v);
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  if constexpr (L == 32) {
    const uint32_t hi = (uint32_t)__builtin_amdgcn_ds_swizzle((int)(b >> 32), 0x401F), lo = (uint32_t)__builtin_amdgcn_ds_swizzle((int)b, 0x401F);  // xor 16
    v += __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
  }
  if constexpr (L == 64) {
    auto row = [&](int lane) {  // the sum of 16 lanes that this lane has
      return __builtin_bit_cast(double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(b >> 32), lane) << 32 |
                                            (uint32_t)__builtin_amdgcn_readlane((int)b, lane));
    };
    v = (row(0) + row(16)) + (row(32) + row(48));
  }
  return v;
}

// 1 / sqrt(x) to 2^-50: the hardware's estimate and two steps of Newton's method.  An error of 2^-50 crosses the middle of two fp32 numbers, 2^-24 apart, in
// one row of ten million at the most, and so does another order of the sum; a division behind a square root took twenty times the instructions.
__device__ __forceinline__ float norm_factor(double x) {
  const double e = __builtin_amdgcn_rsq(x);
  const double half = 0.5 * x * e;
  const double once = __builtin_fma(e, __builtin_fma(-half, e, 0.5), e);
  const double r = __builtin_fma(once, __builtin_fma(-0.5 * x * once, once, 0.5), once);
  return (float)(x > 0.0 && x < __builtin_inf() ? r : e);  // (1 / 0, 1 / inf and NaN)
}

// A row holds at most one vector that is cut by its end.  It is read and written apart from the others, once a row, so that the code for
// pieces of vectors stands once in a kernel and not behind every vector (kernels a third of the size).
template <int DT>
__device__ __forceinline__ void cut_load(Vec8<DT> &v, const void *row, int64_t k_cut, bool mine, int n) {
  vec8_zero(v);
  if (mine) vec8_load_some(v, static_cast<const typename Elem<DT>::T *>(row) + k_cut, n);
}
template <int DT>
__device__ __forceinline__ void row_vector(Vec8<DT> &v, const void *row, int64_t k, int64_t K, const Vec8<DT> &cut) {
  if (k + 8 <= K) vec8_load_all(v, static_cast<const typename Elem<DT>::T *>(row) + k);
  else if (k < K) v = cut;
  else vec8_zero(v);
}

// BW waves a workgroup, LPR lanes a row, NV vectors of eight elements a lane: K <= 8 * LPR * NV.  A workgroup takes rows_per_block rows, a
// multiple of the rows that it has lanes for.
template <int MODE, int DT, int WT, int OUT, int BW, int LPR, int NV>
__global__ __launch_bounds__(64 * BW) void norm_rows_kernel(NormArgs a, int rows_per_block) {
  using T = typename Elem<DT>::T;
  constexpr bool BLOCK = MODE != NORM_ROWS;
  constexpr int GROUPS = 64 * BW / LPR, WPR = LPR / 64;  // WPR: waves a row, 0 where a wave has several
  constexpr int IN_WAVE = LPR < 64 ? LPR : 64;
  constexpr bool NVFP4 = OUT == NORM_NVFP4 || OUT == NORM_NVFP4_SECOND || OUT == NORM_NVFP4_ONE;
  constexpr bool SUMS = OUT != NORM_NVFP4_SECOND;  // x is normalized here, not by an earlier launch
  __shared__ double part[BLOCK ? 2 : 1][WPR > 1 ? BLOCK ? 2 * BW : BW : 1];
  __shared__ uint32_t part_max[BW];
  __shared__ float lut[NVFP4 ? 128 : 1];
  const int tid = threadIdx.x, sub = tid % LPR, wave = tid >> 6;
  const int group = WPR == 0 ? tid / LPR : __builtin_amdgcn_readfirstlane(tid / LPR);
  float alpha = 0.0f;
  float rcp = 0.0f;  // for the table; it is in LDS behind the next barrier
  if constexpr (NVFP4) rcp = g_rcp_e4m3.v[tid & 127];
  if constexpr (OUT == NORM_NVFP4) {
    if (tid < 128) lut[tid] = rcp;
    __syncthreads();
    const float g = *a.gs;
    alpha = g < NORM_LEAST / 4096.0f ? 0.0f : 1.0f / g;  // (a negative scale, too: codes of the table below are those of positive ones)
  }
  auto block_max = [&](uint32_t m) {  // of every wave's m (uniform in a wave)
    if ((tid & 63) == 0) part_max[wave] = m;
    if (NVFP4 && tid < 128) lut[tid] = rcp;
    __syncthreads();
    uint32_t b = part_max[0];
#pragma unroll
    for (int i = 1; i < BW; ++i) b = umax32(b, part_max[i]);
    return b;
  };
  auto global_scale = [&](uint32_t bits) {
    float m = __uint_as_float(bits);
    if (m < NORM_LEAST) m = 0.0f;
    const float g = m * (1.0f / 2688.0f);
    alpha = g == 0.0f ? 0.0f : 1.0f / g;
    if (blockIdx.x == 0 && tid == 0) *a.gs = g;
  };
  const int cut = MODE == NORM_BLOCK ? 0 : (int)(a.K & 7);
  const int64_t k_cut = a.K - cut;
  const bool cut_mine = cut != 0 && (int)(k_cut / 8 % LPR) == sub;
  // the weights, once for all rows of the workgroup, and under way before the first row's sum is known; rows of eight vectors leave no
  // registers for them, and read them where they are used, as rows of blocks do all their vectors
  constexpr bool HELD = NV <= 4 && !BLOCK;
  static_assert(!BLOCK || NV <= 4, "a block's rows are at most 32768 elements");
  Vec8<WT> w[HELD ? NV : 1];
  const bool weighted = a.weight != nullptr;
  if (HELD && weighted) {
    Vec8<WT> w_cut;
    cut_load(w_cut, a.weight, k_cut, cut_mine, cut);
#pragma unroll
    for (int j = 0; j < (HELD ? NV : 0); ++j) row_vector(w[j], a.weight, (j * LPR + sub) * 8, a.K, w_cut);
  }
  const int Ks = (int)a.K;
  // BLOCK: vector k of one of a block's rows of K; behind the row it is zero with `zero`, otherwise any of the row's vectors or zero
  auto row_piece = [&](auto &v, const auto *p, int k, bool zero) {
    if constexpr (MODE == NORM_BLOCK) {
      vec8_load_all(v, p + (k < Ks ? k : Ks - 8));  // no branch
      if (zero) {
#pragma unroll
        for (uint32_t &w : v.w) w = k < Ks ? w : 0u;
      }
    } else {
      int at = k;
      asm("" : "+v"(at));  // compared here, not once for all pieces (whose masks spill scalar registers)
      vec8_load(v, p, at, Ks);
    }
  };
  // BLOCK: two sums over a row; parts of these and of the next ones lie apart, so that a barrier each time is enough
  int flip = 0;
  auto row_sums = [&](double &s, double &t) {
    s = group_sum<IN_WAVE>(s);
    t = group_sum<IN_WAVE>(t);
    if constexpr (WPR > 1) {
      if ((tid & 63) == 0) part[flip][wave] = s, part[flip][BW + wave] = t;
      __syncthreads();
      s = t = 0.0;
#pragma unroll
      for (int i = 0; i < WPR; ++i) s += part[flip][group * WPR + i], t += part[flip][BW + group * WPR + i];
      flip ^= 1;
    }
  };
  // BLOCK: mean (in two pieces; 0 where rows are not centred) and factor of a row.  Sums of 16-bit elements and of their squares lose nothing in 64 bits
  // where the elements are of one size, and K^2 times the variance is K times the second less the square of the first; elements of 32 bits are squared without the mean.
  auto row_stats = [&](const Vec8<DT>(&v)[NV], float &m1, float &m2, float &r) {
    double s = 0.0, q = 0.0, mean = 0.0, var;
    if (a.centred) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const double d = (double)vec8_get(v[j], i);
          s += d;
          q = __builtin_fma(d, d, q);
        }
    } else {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const double d = (double)vec8_get(v[j], i);
          q = __builtin_fma(d, d, q);
        }
    }
    row_sums(s, q);
    var = q * a.inverse_K;
    if (a.centred) {
      mean = s / (double)a.K;  // (exact for rows of one value)
      if constexpr (DT == AC4K_DTYPE_FP32) {
        q = 0.0;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const int k = (j * LPR + sub) * 8;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const double d = (MODE == NORM_BLOCK ? k : k + i) < Ks ? (double)vec8_get(v[j], i) - mean : 0.0;
            q = __builtin_fma(d, d, q);
          }
        }
        row_sums(s, q);
        var = q * a.inverse_K;
      } else {
        var = __builtin_fma(-s, s, (double)a.K * q);
        var = var < 0.0 ? 0.0 : var * (a.inverse_K * a.inverse_K);  // (NaN stays)
      }
    }
    m1 = (float)mean;
    m2 = (float)(mean - (double)m1);
    r = norm_factor(var + a.eps);
  };
  uint32_t block_m = 0;
  const int64_t row0 = (int64_t)blockIdx.x * rows_per_block;
  for (int it = 0; it * GROUPS < rows_per_block; ++it) {
    const int64_t row = row0 + it * GROUPS + group;
    const bool valid = row < a.rows;
    if (WPR <= 1 && OUT != NORM_NVFP4_ONE && !(OUT == NORM_NVFP4_SECOND && it == 0) && !valid && !(NVFP4 && row < a.Rp)) break;  // (rows of several waves meet at barriers)
    Vec8<DT> h[NV];
    float r = 0.0f, m1 = 0.0f, m2 = 0.0f;
    // BLOCK: a vector of this row.  (A row behind the last one is that one again; nothing is kept of it.)
    using W = typename Elem<WT>::T;
    const int64_t row_in = BLOCK && !valid ? a.rows - 1 : row;
    auto vector_of = [&](const NormVector &p) {
      const uint32_t at = p.rows == 0 ? 0 : p.rows == 1 ? (uint32_t)row_in : (uint32_t)row_in / p.rows;
      return static_cast<const W *>(p.p) + at * p.stride;
    };
    const T *xp = static_cast<const T *>(a.x) + row_in * a.x_stride;
    if constexpr (BLOCK) {
#pragma unroll
      for (int j = 0; j < NV; ++j) row_piece(h[j], xp, (j * LPR + sub) * 8, true);
    } else {
      Vec8<DT> x_cut;
      cut_load(x_cut, xp, k_cut, cut_mine && valid, cut);
#pragma unroll
      for (int j = 0; j < NV; ++j) row_vector(h[j], xp, (j * LPR + sub) * 8, valid ? a.K : 0, x_cut);
    }
    if constexpr (BLOCK) {
      if (SUMS && a.residual) {
        const T *rp = static_cast<const T *>(a.residual) + row_in * a.residual_stride;
        T *sp = static_cast<T *>(a.sum) + row * a.sum_stride;
        Vec8<DT> q[NV], q_cut;
#pragma unroll
        for (int j = 0; j < NV; ++j) row_piece(q[j], rp, (j * LPR + sub) * 8, false);
        const bool gated = a.gate.p != nullptr, post = a.post != nullptr;
        const W *gp = vector_of(a.gate), *pp = static_cast<const W *>(a.post);
        float pr = 1.0f;
        if (post) row_stats(h, m1, m2, pr);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const int k = (j * LPR + sub) * 8;
          float f[8];
          Vec8<WT> v;
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = vec8_get(h[j], i);
          if (post) {
            row_piece(v, pp, k, false);
            if (a.centred) {
#pragma unroll
              for (int i = 0; i < 8; ++i) f[i] = (f[i] - m1) - m2;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = f[i] * pr * vec8_get(v, i);
          }
          if (gated) {
            row_piece(v, gp, k, false);
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = __builtin_fmaf(f[i], vec8_get(v, i), vec8_get(q[j], i) * a.alpha);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = vec8_get(q[j], i) * a.alpha + f[i];
          }
          // behind the row h is 0: all that is loaded there is (NORM_BLOCK_CUT: a row with a mean that is not finite is NaN anyway)
          vec8_set(h[j], f);
          if constexpr (MODE == NORM_BLOCK) {
#pragma unroll
            for (uint32_t &w : h[j].w) w = k < Ks ? w : 0u;
            if (valid && k < Ks) vec8_store_all(sp + k, h[j]);
          } else {
            if (valid && k + 8 <= Ks) vec8_store_all(sp + k, h[j]);
            else if (k < Ks) q_cut = h[j];
          }
        }
        if (MODE == NORM_BLOCK_CUT && cut_mine && valid) vec8_store_some(sp + k_cut, q_cut, cut);
      }
      if constexpr (SUMS) {
        row_stats(h, m1, m2, r);
      } else if (a.centred) {
        m1 = a.means[2 * row_in];
        m2 = a.means[2 * row_in + 1];
      }
    } else if constexpr (SUMS) {
      if (a.residual && valid) {
        const T *rp = static_cast<const T *>(a.residual) + row * a.residual_stride;
        Vec8<DT> q[HELD ? NV : 1], r_cut;
        cut_load(r_cut, rp, k_cut, cut_mine, cut);
#pragma unroll
        for (int j = 0; j < (HELD ? NV : 0); ++j) row_vector(q[j], rp, (j * LPR + sub) * 8, a.K, r_cut);
        T *sp = static_cast<T *>(a.sum) + row * a.sum_stride;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const int k = (j * LPR + sub) * 8;
          Vec8<DT> &v = q[HELD ? j : 0];
          if constexpr (!HELD) row_vector(v, rp, k, a.K, r_cut);
          float f[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = vec8_get(h[j], i) + vec8_get(v, i);
          vec8_set(h[j], f);
          if (k + 8 <= a.K) vec8_store_all(sp + k, h[j]);
          else if (k < a.K) r_cut = h[j];
        }
        if (cut_mine) vec8_store_some(sp + k_cut, r_cut, cut);
      }
      double s = 0.0;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const double v = vec8_get(h[j], i);
          s = __builtin_fma(v, v, s);
        }
      s = group_sum<IN_WAVE>(s);
      if constexpr (WPR > 1) {
        if (it) __syncthreads();  // the parts of the row before have been read
        if ((tid & 63) == 0) part[0][wave] = s;
        __syncthreads();
        s = 0.0;
#pragma unroll
        for (int i = 0; i < WPR; ++i) s += part[0][group * WPR + i];
      }
      r = norm_factor(s * a.inverse_K + a.eps);
    }
    if constexpr (!SUMS) {
      r = valid ? a.factors[row] : 0.0f;
      if (it == 0) {  // (the loads of the first row are under way)
        uint32_t m = 0;
        if constexpr (BLOCK) {
          for (int i = tid * 4; i < a.maxima_count; i += 64 * BW * 4) {
            if (i + 4 <= a.maxima_count) {
              const u32x4 v = *reinterpret_cast<const u32x4_elem *>(a.maxima + i);
              m = umax32(umax32(umax32(m, v.x), umax32(v.y, v.z)), v.w);
            } else {
              for (int j = i; j < a.maxima_count; ++j) m = umax32(m, __float_as_uint(a.maxima[j]));
            }
          }
        } else {
          for (int i = tid; i < a.maxima_count; i += 64 * BW) m = umax32(m, __float_as_uint(a.maxima[i]));
        }
        global_scale(block_max(group_umax<64>(m)));
      }
    }
    const W *const scp = BLOCK ? vector_of(a.scale) : nullptr, *const shp = BLOCK ? vector_of(a.shift) : nullptr;
    // y of vector j
    auto values = [&](int j, float (&y)[8]) {
      const int k = (j * LPR + sub) * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = vec8_get(h[j], i);
      if (BLOCK && a.centred) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = (y[i] - m1) - m2;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = y[i] * r;
      if (weighted) {
        Vec8<WT> &v = w[HELD ? j : 0];
        if constexpr (BLOCK) row_piece(v, static_cast<const W *>(a.weight), k, false);
        else if constexpr (!HELD) vec8_load(v, a.weight, k, a.K);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = y[i] * vec8_get(v, i);
      }
      if constexpr (BLOCK) {
        Vec8<WT> v, u;
        if (a.scale.p && a.shift.p) {
          row_piece(v, scp, k, false);
          row_piece(u, shp, k, false);
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = __builtin_fmaf(y[i], 1.0f + vec8_get(v, i), vec8_get(u, i));
        } else if (a.scale.p) {
          row_piece(v, scp, k, false);
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = y[i] * (1.0f + vec8_get(v, i));
        } else if (a.shift.p) {
          row_piece(v, shp, k, false);
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = y[i] + vec8_get(v, i);
        }
      }
      // behind the row the product 0 * r * 0 is not 0 where r is not finite, and a centred row is not 0
      if constexpr (BLOCK) {
        if constexpr (MODE == NORM_BLOCK_CUT && OUT != NORM_PLAIN) {
          int left = Ks - k;
          asm("" : "+v"(left));
          if (left < 8) {
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = i < left ? y[i] : 0.0f;
          }
        }
      } else if (k + 8 > a.K) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = k + i < a.K ? y[i] : 0.0f;
      }
    };
    auto max8 = [](const float (&y)[8]) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = umax32(m, __float_as_uint(y[i]) & 0x7fffffffu);
      return m;
    };
    if constexpr (OUT == NORM_PLAIN) {
      if (valid) {
        T *op = static_cast<T *>(a.out) + row * a.out_stride;
        Vec8<DT> o, o_cut;
        vec8_zero(o_cut);
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const int k = (j * LPR + sub) * 8;
          if (k >= a.K) continue;
          float y[8];
          values(j, y);
          vec8_set(o, y);
          if (MODE == NORM_BLOCK || k + 8 <= a.K) vec8_store_all(op + k, o);
          else o_cut = o;
        }
        if (cut_mine) vec8_store_some(op + k_cut, o_cut, cut);
      }
    } else if constexpr (OUT == NORM_FP8 || OUT == NORM_INT8 || OUT == NORM_STATS || OUT == NORM_NVFP4_ONE) {
      uint32_t m = 0;
      constexpr bool KEEP = (OUT == NORM_FP8 || OUT == NORM_INT8) && NV <= 4;  // y stays in registers for the conversion
      float kept[KEEP ? NV : 1][8];
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if constexpr (KEEP) {
          float y[8] = {};
          if ((j * LPR + sub) * 8 < a.K) values(j, y);
#pragma unroll
          for (int i = 0; i < 8; ++i) kept[j][i] = y[i];
          m = umax32(m, max8(y));
        } else {
          if ((j * LPR + sub) * 8 >= a.K) continue;
          float y[8];
          values(j, y);
          m = umax32(m, max8(y));
        }
      }
      if constexpr (OUT == NORM_STATS) {
        if (valid) {
          block_m = umax32(block_m, m);
          if (sub == 0) {
            a.factors[row] = r;
            if (BLOCK && a.centred) a.means[2 * row] = m1, a.means[2 * row + 1] = m2;
          }
        }
        continue;
      }
      m = group_umax<OUT == NORM_NVFP4_ONE ? 64 : IN_WAVE>(valid ? m : 0);
      if constexpr (OUT == NORM_NVFP4_ONE) {  // one workgroup, one pass of its loop
        global_scale(block_max(m));
      } else {
        if constexpr (WPR > 1) {
          if ((tid & 63) == 0) part_max[wave] = m;
          __syncthreads();
#pragma unroll
          for (int i = 0; i < WPR; ++i) m = umax32(m, part_max[group * WPR + i]);
        }
        if (!valid) continue;
        float amax = __uint_as_float(m);
        if (amax < NORM_LEAST) amax = 0.0f;
        const float most = OUT == NORM_FP8 ? 448.0f : 127.0f;
        if (sub == 0) static_cast<float *>(a.sf)[row] = amax * (1.0f / most);
        const float factor = amax == 0.0f ? 0.0f : 1.0f / amax * most;  // one division a row; with the scale's product two roundings each
        uint8_t *op = static_cast<uint8_t *>(a.out) + row * a.Kp;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const int k = (j * LPR + sub) * 8;
          if (k >= a.Kp) continue;
          float y[8];
          if constexpr (KEEP) {
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = kept[j][i];
          } else {
            values(j, y);
          }
          // |y * factor| is at most `most` and three roundings, which the conversion rounds back to it: nothing to clamp
          uint32_t lo, hi;
          if constexpr (OUT == NORM_FP8) {
            lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0] * factor, y[1] * factor, 0, false);
            lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[2] * factor, y[3] * factor, lo, true);
            hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[4] * factor, y[5] * factor, 0, false);
            hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[6] * factor, y[7] * factor, hi, true);
            if (factor != factor) lo = hi = 0x7f7f7f7fu;
          } else {
            // added to 1.5 * 2^23, a value is rounded to the nearest whole number (ties to even), whose low byte is that of the sum
            uint32_t b[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) b[i] = __float_as_uint(y[i] * factor + 12582912.0f);
            auto bytes4 = [](uint32_t p, uint32_t q, uint32_t r, uint32_t t) {
              return __builtin_amdgcn_perm(__builtin_amdgcn_perm(t, r, 0x0c0c0400u), __builtin_amdgcn_perm(q, p, 0x0c0c0400u), 0x05040100u);
            };
            lo = bytes4(b[0], b[1], b[2], b[3]);
            hi = bytes4(b[4], b[5], b[6], b[7]);
            if (factor != factor) lo = hi = 0;
          }
          st_elem_u2(op + k, make_uint2(lo, hi));
        }
      }
    }
    if constexpr (NVFP4) {
      // (lanes of a block of 16 are neighbours; all 64 take part in the exchanges)
      uint8_t *op = static_cast<uint8_t *>(a.out) + (valid ? row : 0) * (a.Kp / 2);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int k = (j * LPR + sub) * 8;
        if ((j * LPR + (sub & ~63)) * 8 >= a.Kp) continue;  // a whole wave
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = 0.0f;
        if (valid && k < a.K) values(j, y);
        uint32_t m = max8(y);
        m = umax32(m, dpp_u32<DPP_QUAD_XOR1>(m));
        uint32_t code;
        const float o = nvfp4_block_scale(__uint_as_float(m), alpha, lut, code);
        if (!valid) code = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] *= o;
        const uint32_t packed = o != o ? 0x77777777u : f32x8_to_e2m1x8(y);
        const uint32_t sfw = code | (dpp_u32<DPP_ROW_SHL(2)>(code) << 8) | (dpp_u32<DPP_ROW_SHL(4)>(code) << 16) |
                             (dpp_u32<DPP_ROW_SHL(6)>(code) << 24);
        if (k < a.Kp) {
          if (valid) *reinterpret_cast<uint32_t *>(op + k / 2) = packed;
          if ((sub & 7) == 0 && row < a.Rp) static_cast<uint32_t *>(a.sf)[k / 64 * a.Rp + row] = sfw;
        }
      }
    }
  }
  if constexpr (OUT == NORM_STATS) {
    const uint32_t m = block_max(group_umax<64>(block_m));
    if (tid == 0) a.maxima[blockIdx.x] = __uint_as_float(m);
  }
  if constexpr (OUT == NORM_NVFP4_ONE) {  // scales of the rows behind the last group
    const int first = rows_per_block, pad = (int)a.Rp - first, n = (int)(a.Kp / 64) * pad;
    for (int i = tid; i < n; i += 64 * BW) static_cast<uint32_t *>(a.sf)[(int64_t)(i / pad) * a.Rp + first + i % pad] = 0u;
  }
  if constexpr (OUT == NORM_FP8 || OUT == NORM_INT8) {  // scales of the rows behind the last one
    if (blockIdx.x == gridDim.x - 1 && a.rows + tid < a.Rp) static_cast<float *>(a.sf)[a.rows + tid] = 0.0f;
  }
}

// Shape of a launch: so many waves a row that a lane holds two or three vectors of it (weights and residual beside them stay under 80 registers,
// and six to eight waves on a SIMD hide each other's loads and reductions), more only behind sixteen waves.
struct NormPlan {
  int bw, lpr, nv, rows_per_block;
};
static NormPlan norm_plan(int64_t rows, int64_t K, bool nvfp4) {
  const int64_t vecs = ceil_div(K, 512);  // of a wave
  NormPlan p;
  p.lpr = K <= 128 ? 16 : K <= 256 ? 32 : 64 * (vecs <= 2 ? 1 : vecs <= 4 ? 2 : vecs <= 12 ? 4 : vecs <= 16 ? 8 : 16);
  const int64_t need = ceil_div(K, 8 * p.lpr);
  p.nv = need <= 1 && p.lpr <= 64 ? 1 : need <= 2 ? 2 : need <= 3 && p.lpr == 256 ? 3 : need <= 4 ? 4 : 8;
  p.bw = p.lpr < 256 ? 4 : p.lpr / 64;
  // A workgroup takes some rows one after the other where there are workgroups enough: they share the weights, and nvfp4 scales of
  // neighbouring rows leave for one line.  Second launch of nvfp4, 8192 x 4096, rows a workgroup / us: 1 48, 4 27, 8 23, 16 28;
  // 75600 x 5120 to bf16: 1 279, 2 264, 4 281, 16 310.
  const int groups = 64 * p.bw / p.lpr;
  const int64_t sets = ceil_div(rows, groups);
  int64_t turns = nvfp4 ? (sets >= 8192 ? 8 : sets >= 2048 ? 4 : sets >= 1024 ? 2 : 1) : sets >= 2048 ? 2 : 1;
  if (turns < sets >> 20) turns = (sets >> 20) + 1;  // 2^32 threads a launch
  p.rows_per_block = (int)(turns * groups);
  return p;
}

// vectors of a lane in the kernel that takes a tensor in one workgroup (128 registers)
constexpr int norm_one_vectors(int dtype) { return dtype == AC4K_DTYPE_FP32 ? 2 : 4; }

template <int MODE, int DT, int WT, int OUT>
static int launch_norm(const NormArgs &a, const NormPlan &p, hipStream_t st) {
  const int64_t rows = OUT == NORM_NVFP4 || OUT == NORM_NVFP4_SECOND ? a.Rp : a.rows;
  const int64_t blocks = ceil_div(rows, p.rows_per_block);
  auto go = [&](auto kernel, int bw) { hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(64 * bw), 0, st, a, p.rows_per_block); };
#define AC4K_NORM(BW, LPR, NV) \
  if (p.bw == BW && p.lpr == LPR && p.nv == NV) return go(norm_rows_kernel<MODE, DT, WT, OUT, BW, LPR, NV>, BW), 0
  constexpr int NV1 = norm_one_vectors(DT);
  if constexpr (OUT == NORM_NVFP4_ONE) {
    AC4K_NORM(8, 512, 2);
    AC4K_NORM(16, 64, NV1);
    AC4K_NORM(16, 128, NV1);
    AC4K_NORM(16, 256, NV1);
    AC4K_NORM(16, 512, NV1);
    AC4K_NORM(16, 1024, NV1);
  } else {
    AC4K_NORM(4, 16, 1);
    AC4K_NORM(4, 32, 1);
    AC4K_NORM(4, 64, 1);
    AC4K_NORM(4, 64, 2);
    AC4K_NORM(4, 128, 2);
    AC4K_NORM(4, 256, 2);
    AC4K_NORM(4, 256, 3);
    AC4K_NORM(8, 512, 2);
    AC4K_NORM(16, 1024, 2);
    AC4K_NORM(16, 1024, 4);
    if constexpr (MODE == NORM_ROWS) AC4K_NORM(16, 1024, 8);
  }
#undef AC4K_NORM
  return set_error("norm of rows: no kernel for %d lanes a row and %d vectors a lane", p.lpr, p.nv);
}

// Tensors of up to 32768 elements (fp32: half) in 16 rows at the most: one workgroup holds all of them and finds the global scale by itself.
static bool norm_one(int64_t rows, int64_t K, int dtype, NormPlan &p) {
  if (rows == 1 && K <= 8192) {
    p = {8, 512, 2, 1};
    return true;
  }
  int wpr = 16;
  while (wpr > 1 && 16 / wpr < rows) wpr /= 2;
  if (16 / wpr < rows || ceil_div(K, 512 * wpr) > norm_one_vectors(dtype)) return false;
  p = {16, 64 * wpr, norm_one_vectors(dtype), 16 / wpr};
  return true;
}
// Its first launch: few enough workgroups that each of the second can read the maxima of all (rows of a block, 8192 x 4096: at most 2048 of them 53.4 + 25.3 us, 4096
// 49.5 + 27.6, with the maxima read four at a time)
static NormPlan norm_stats_plan(int64_t rows, int64_t K, int mode) {
  NormPlan p = norm_plan(rows, K, false);
  const int64_t least = ceil_div(rows, mode == NORM_ROWS ? 2048 : 4096);
  if (p.rows_per_block < least) p.rows_per_block = (int)align_up(least, 64 * p.bw / p.lpr);
  return p;
}
static int64_t norm_workspace(int64_t rows, int64_t K, int dtype, int mode) {
  NormPlan p;
  if (norm_one(rows, K, dtype, p)) return 0;
  return 4 * (align_up(rows, 64) + ceil_div(rows, norm_stats_plan(rows, K, mode).rows_per_block));
}

template <int MODE, int DT, int WT>
static int norm_dtype(NormArgs a, int precision, bool find_scale, float *workspace, int dtype, hipStream_t st) {
  if (precision == AC4K_PRECISION_NVFP4 && find_scale) {
    NormPlan p;
    if (norm_one(a.rows, a.K, dtype, p)) return launch_norm<MODE, DT, WT, NORM_NVFP4_ONE>(a, p, st);
    p = norm_stats_plan(a.rows, a.K, MODE);
    a.factors = workspace;
    a.maxima = workspace + align_up(a.rows, 64);
    a.maxima_count = (int)ceil_div(a.rows, p.rows_per_block);
    a.means = a.maxima + a.maxima_count;
    if (int rc = launch_norm<MODE, DT, WT, NORM_STATS>(a, p, st)) return rc;
    if (a.residual) a.x = a.sum, a.x_stride = a.sum_stride;
    return launch_norm<MODE, DT, WT, NORM_NVFP4_SECOND>(a, norm_plan(a.rows, a.K, true), st);
  }
  NormPlan p = norm_plan(a.rows, a.K, precision == AC4K_PRECISION_NVFP4);
  // five workgroups a CU: with two rows each, 4002 rows are a round and a half (to int8 54.3 us, one row each 50.5)
  const int groups = 64 * p.bw / p.lpr;
  if (MODE != NORM_ROWS && precision != AC4K_PRECISION_NVFP4 && ceil_div(a.rows, groups) < 8192) p.rows_per_block = groups;
  switch (precision) {
    case AC4K_PRECISION_NONE: return launch_norm<MODE, DT, WT, NORM_PLAIN>(a, p, st);
    case AC4K_PRECISION_FP8: return launch_norm<MODE, DT, WT, NORM_FP8>(a, p, st);
    case AC4K_PRECISION_INT8: return launch_norm<MODE, DT, WT, NORM_INT8>(a, p, st);
    default: return launch_norm<MODE, DT, WT, NORM_NVFP4>(a, p, st);
  }
}

}  // namespace ac4k

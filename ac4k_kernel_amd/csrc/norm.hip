// Root-mean-square norm of rows, with a residual's addition in front and a quantizer behind, and the inverse of the quantizers.
//
//   h = round(x + residual)           (x's type; x itself without a residual)
//   r = fp32(1 / sqrt(mean(h^2) + eps))
//   y = (h * r) * weight              (fp32, two products)
// and y leaves in x's type, or as one of the formats of the quantizers: rows of e4m3 or int8 with one scale a row, or nvfp4 with e4m3
// scales of 16 and one fp32 scale max|y| / 2688, from the values in 32 bits: there is no rounding to 16 bits in between.
//
// The sum of squares is held in 64 bits.  A code next to a border of its format goes by the last place of r, and with 64 bits r is the
// correctly rounded factor for every order of the sum, but for about one row in ten million (see norm_factor): splits of a row over 1, 4
// or 16 waves give the same codes, but for these.
//
// Rows that are all zero (or whose largest |y| is under 2^-100, where the scale would leave the normal fp32 numbers) quantize to zero
// codes and a zero scale.
//
// Bound by memory: a row is read once and stays in registers between the sum, the maximum and the conversion; the counters show every byte
// read and written once.  75600 x 5120 bf16 262 us, 5.9 TB/s (the vector port is busy for 60 % of that); 1000000 x 128 90 us, 5.7 TB/s; one row of 8192
// 3.7 us, a chain of load, sum, maximum and store.  4001 x 5003 to int8 with fp32 weights, 20-21 us where its bytes need 13, is bound by vector
// instructions: 144 for eight elements, the port busy for 80 %.
// nvfp4 without a given global scale takes a second launch, which reads h again (from the memory-side cache where it fits) with r at
// hand: 8192 x 4096 with a residual 38 + 23 us under the profiler, 59 a call of many, for 46 of bytes; with the scale given 47 and 44.5; up to 32768 elements
// one workgroup does all: 1 x 8192 4.6 us.  Long rows have fewer waves to hide a row's chain: 8192 x 16384 bf16 106 us (5.1 TB/s), to e4m3 114 (3.5).
// Rows of more than 32768 elements (fp32 to nvfp4 with a given scale: 16384) spill 40 to 90 registers: 2048 x 65536 162 (3.3), to e4m3 186 (2.2).
#include "elements.h"

namespace ac4k {

enum NormOut { NORM_PLAIN = 0, NORM_FP8 = 1, NORM_INT8 = 2, NORM_NVFP4 = 3, NORM_STATS = 4, NORM_NVFP4_SECOND = 5, NORM_NVFP4_ONE = 6 };

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
template <int DT, int WT, int OUT, int BW, int LPR, int NV>
__global__ __launch_bounds__(64 * BW) void rms_norm_kernel(NormArgs a, int rows_per_block) {
  using T = typename Elem<DT>::T;
  constexpr int GROUPS = 64 * BW / LPR, WPR = LPR / 64;  // WPR: waves a row, 0 where a wave has several
  constexpr int IN_WAVE = LPR < 64 ? LPR : 64;
  constexpr bool NVFP4 = OUT == NORM_NVFP4 || OUT == NORM_NVFP4_SECOND || OUT == NORM_NVFP4_ONE;
  constexpr bool SUMS = OUT != NORM_NVFP4_SECOND;  // x is normalized here, not by an earlier launch
  __shared__ double part[WPR > 1 ? BW : 1];
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
  const int cut = (int)(a.K & 7);
  const int64_t k_cut = a.K - cut;
  const bool cut_mine = cut != 0 && (int)(k_cut / 8 % LPR) == sub;
  // the weights, once for all rows of the workgroup, and under way before the first row's sum is known; rows of eight vectors leave no
  // registers for them, and read them where they are used
  constexpr bool HELD = NV <= 4;
  Vec8<WT> w[HELD ? NV : 1];
  const bool weighted = a.weight != nullptr;
  if (HELD && weighted) {
    Vec8<WT> w_cut;
    cut_load(w_cut, a.weight, k_cut, cut_mine, cut);
#pragma unroll
    for (int j = 0; j < (HELD ? NV : 0); ++j) row_vector(w[j], a.weight, (j * LPR + sub) * 8, a.K, w_cut);
  }
  uint32_t block_m = 0;
  const int64_t row0 = (int64_t)blockIdx.x * rows_per_block;
  for (int it = 0; it * GROUPS < rows_per_block; ++it) {
    const int64_t row = row0 + it * GROUPS + group;
    const bool valid = row < a.rows;
    if (WPR <= 1 && OUT != NORM_NVFP4_ONE && !(OUT == NORM_NVFP4_SECOND && it == 0) && !valid && !(NVFP4 && row < a.Rp)) break;  // (rows of several waves meet at barriers)
    Vec8<DT> h[NV];
    float r = 0.0f;
    {
      const T *xp = static_cast<const T *>(a.x) + row * a.x_stride;
      Vec8<DT> x_cut;
      cut_load(x_cut, xp, k_cut, cut_mine && valid, cut);
#pragma unroll
      for (int j = 0; j < NV; ++j) row_vector(h[j], xp, (j * LPR + sub) * 8, valid ? a.K : 0, x_cut);
    }
    if constexpr (SUMS) {
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
        if ((tid & 63) == 0) part[wave] = s;
        __syncthreads();
        s = 0.0;
#pragma unroll
        for (int i = 0; i < WPR; ++i) s += part[group * WPR + i];
      }
      r = norm_factor(s * a.inverse_K + a.eps);
    } else {
      r = valid ? a.factors[row] : 0.0f;
      if (it == 0) {  // (the loads of the first row are under way)
        uint32_t m = 0;
        for (int i = tid; i < a.maxima_count; i += 64 * BW) m = umax32(m, __float_as_uint(a.maxima[i]));
        global_scale(block_max(group_umax<64>(m)));
      }
    }
    // y of vector j
    auto values = [&](int j, float (&y)[8]) {
      const int k = (j * LPR + sub) * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = vec8_get(h[j], i) * r;
      if (weighted) {
        Vec8<WT> &v = w[HELD ? j : 0];
        if constexpr (!HELD) vec8_load(v, a.weight, k, a.K);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = y[i] * vec8_get(v, i);
      }
      // behind the row the product 0 * r * 0 is not 0 where r is not finite
      if (k + 8 > a.K) {
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
          if (k + 8 <= a.K) vec8_store_all(op + k, o);
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
          if (sub == 0) a.factors[row] = r;
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

template <int DT, int WT, int OUT>
static int launch_norm(const NormArgs &a, const NormPlan &p, hipStream_t st) {
  const int64_t rows = OUT == NORM_NVFP4 || OUT == NORM_NVFP4_SECOND ? a.Rp : a.rows;
  const int64_t blocks = ceil_div(rows, p.rows_per_block);
  auto go = [&](auto kernel, int bw) { hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(64 * bw), 0, st, a, p.rows_per_block); };
#define AC4K_NORM(BW, LPR, NV) \
  if (p.bw == BW && p.lpr == LPR && p.nv == NV) return go(rms_norm_kernel<DT, WT, OUT, BW, LPR, NV>, BW), 0
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
    AC4K_NORM(16, 1024, 8);
  }
#undef AC4K_NORM
  return set_error("rms_norm: no kernel for %d lanes a row and %d vectors a lane", p.lpr, p.nv);
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
// Its first launch: few enough workgroups that each of the second can read the maxima of all
static NormPlan norm_stats_plan(int64_t rows, int64_t K) {
  NormPlan p = norm_plan(rows, K, false);
  const int64_t least = ceil_div(rows, 2048);
  if (p.rows_per_block < least) p.rows_per_block = (int)align_up(least, 64 * p.bw / p.lpr);
  return p;
}
static int64_t norm_workspace(int64_t rows, int64_t K, int dtype) {
  NormPlan p;
  if (norm_one(rows, K, dtype, p)) return 0;
  return 4 * (align_up(rows, 64) + ceil_div(rows, norm_stats_plan(rows, K).rows_per_block));
}

template <int DT, int WT>
static int norm_dtype(NormArgs a, int precision, bool find_scale, float *workspace, int dtype, hipStream_t st) {
  if (precision == AC4K_PRECISION_NVFP4 && find_scale) {
    NormPlan p;
    if (norm_one(a.rows, a.K, dtype, p)) return launch_norm<DT, WT, NORM_NVFP4_ONE>(a, p, st);
    p = norm_stats_plan(a.rows, a.K);
    a.factors = workspace;
    a.maxima = workspace + align_up(a.rows, 64);
    a.maxima_count = (int)ceil_div(a.rows, p.rows_per_block);
    if (int rc = launch_norm<DT, WT, NORM_STATS>(a, p, st)) return rc;
    if (a.residual) a.x = a.sum, a.x_stride = a.sum_stride;
    return launch_norm<DT, WT, NORM_NVFP4_SECOND>(a, norm_plan(a.rows, a.K, true), st);
  }
  const NormPlan p = norm_plan(a.rows, a.K, precision == AC4K_PRECISION_NVFP4);
  switch (precision) {
    case AC4K_PRECISION_NONE: return launch_norm<DT, WT, NORM_PLAIN>(a, p, st);
    case AC4K_PRECISION_FP8: return launch_norm<DT, WT, NORM_FP8>(a, p, st);
    case AC4K_PRECISION_INT8: return launch_norm<DT, WT, NORM_INT8>(a, p, st);
    default: return launch_norm<DT, WT, NORM_NVFP4>(a, p, st);
  }
}

// ---------------------------------------------------------------------------
// the inverse of the quantizers
// ---------------------------------------------------------------------------
struct DequantArgs {
  void *out;
  const uint8_t *q;
  const void *sf;
  const float *gs;
  int64_t lead, R, W, Rp, cols;  // W: elements of a quantized row
  int64_t gs_stride;             // 0: one scale for all leading planes
};

// A wave takes 512 columns of four rows, a workgroup 16 rows, whose nvfp4 scales are whole 64-byte runs.  A lane takes eight elements of a row,
// as one vector of 16 bytes of the output or two, so that a wave's stores are whole runs of a kilobyte.
// 8192 x 4096 nvfp4 to bf16 14.4 us, 6.1 TB/s; 300000 x 128, a quarter of the lanes at work, 26 us, 3.7 TB/s.
template <int DT, int PRECISION>
__global__ __launch_bounds__(256) void dequantize_kernel(DequantArgs a) {
  using T = typename Elem<DT>::T;
  constexpr int V = 16 / sizeof(T), PIECES = 8 / V;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t spans = (uint32_t)ceil_div(a.W, 512), bands = (uint32_t)ceil_div(a.R, 16);
  const uint32_t rest = blockIdx.x / spans, span = blockIdx.x - rest * spans;
  const uint32_t lead = rest / bands, band = rest - lead * bands;
  const int64_t k0 = span * 512ll + lane * V;
  if (k0 >= a.cols) return;
  const float gs = PRECISION == AC4K_PRECISION_NVFP4 ? a.gs[lead * a.gs_stride] : 1.0f;
  uint32_t v[4][2];  // eight elements: nibbles in the first word (two pieces: half of it each), bytes in both
  float s[4][PIECES];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t row = band * 16ll + wave * 4 + i;
    if (row >= a.R) break;
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      const int64_t k = k0 + p * 64 * V;
      if (k >= a.cols) break;
      if constexpr (PRECISION == AC4K_PRECISION_NVFP4) {
        const uint8_t *q = a.q + (lead * a.R + row) * (a.W / 2) + k / 2;
        v[i][p] = V == 8 ? *reinterpret_cast<const uint32_t *>(q) : *reinterpret_cast<const uint16_t *>(q);
        s[i][p] = e4m3_to_f32(static_cast<const uint8_t *>(a.sf)[((lead * (a.W / 64) + k / 64) * a.Rp + row) * 4 + k % 64 / 16]);
      } else {
        const uint8_t *q = a.q + (lead * a.R + row) * a.W + k;
        if constexpr (V == 8) {
          const u32x2 w = *reinterpret_cast<const u32x2_elem *>(q);
          v[i][0] = w.x, v[i][1] = w.y;
        } else {
          typedef uint32_t u32_byte __attribute__((aligned(1)));
          v[i][p] = *reinterpret_cast<const u32_byte *>(q);
        }
        s[i][p] = static_cast<const float *>(a.sf)[lead * a.Rp + row];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t row = band * 16ll + wave * 4 + i;
    if (row >= a.R) break;
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      const int64_t k = k0 + p * 64 * V;
      if (k >= a.cols) break;
      float f[V];
#pragma unroll
      for (int e = 0; e < V; e += 2) {
        if constexpr (PRECISION == AC4K_PRECISION_NVFP4) {
          // e2m1 times the scale of 16 is exact; the product with the global scale is the one rounding in 32 bits
          const f32x2 d = e == 0   ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(v[i][p], 1.0f, 0)
                          : e == 2 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(v[i][p], 1.0f, 1)
                          : e == 4 ? __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(v[i][p], 1.0f, 2)
                                   : __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(v[i][p], 1.0f, 3);
          f[e] = d.x * s[i][p] * gs;
          f[e + 1] = d.y * s[i][p] * gs;
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint32_t b = v[i][V == 8 ? e / 4 : p] >> (8 * ((e + h) & 3)) & 0xffu;
            f[e + h] = (PRECISION == AC4K_PRECISION_INT8 ? (float)(int8_t)b : e4m3_to_f32(b)) * s[i][p];
          }
        }
      }
      T *out = static_cast<T *>(a.out) + (lead * a.R + row) * a.cols + k;
      if (k + V <= a.cols) {
        u32x4 w;
        if constexpr (V == 8) w = (u32x4){Elem<DT>::cvt2(f[0], f[1]), Elem<DT>::cvt2(f[2], f[3]), Elem<DT>::cvt2(f[4], f[5]), Elem<DT>::cvt2(f[6], f[7])};
        else w = (u32x4){__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])};
        *reinterpret_cast<u32x4_elem *>(out) = w;
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (k + e < a.cols) out[e] = Elem<DT>::cvt(f[e]);
      }
    }
  }
}

template <int DT>
static void launch_dequantize(const DequantArgs &a, int precision, int64_t blocks, hipStream_t st) {
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), 0, st, a); };
  if (precision == AC4K_PRECISION_NVFP4) go(dequantize_kernel<DT, AC4K_PRECISION_NVFP4>);
  else if (precision == AC4K_PRECISION_FP8) go(dequantize_kernel<DT, AC4K_PRECISION_FP8>);
  else go(dequantize_kernel<DT, AC4K_PRECISION_INT8>);
}

}  // namespace ac4k

using namespace ac4k;

static bool float_tag(int d) { return d == AC4K_DTYPE_BF16 || d == AC4K_DTYPE_FP16 || d == AC4K_DTYPE_FP32; }

extern "C" __attribute__((visibility("default"))) int64_t ac4k_rms_norm_workspace_bytes(int64_t rows, int64_t K, int dtype, int precision,
                                                                                       int given_scale) {
  if (rows < 1 || K < 1 || K > AC4K_NORM_MAX_COLS || !float_tag(dtype) || precision != AC4K_PRECISION_NVFP4 || given_scale) return 0;
  return norm_workspace(rows, K, dtype);
}

extern "C" __attribute__((visibility("default"))) int ac4k_rms_norm(
    void *out, int64_t out_stride, void *sf, float *global_scale, int given_scale, const void *x, int64_t x_stride, const void *residual,
    int64_t residual_stride, void *sum, int64_t sum_stride, const void *weight, int weight_dtype, int64_t rows, int64_t K, int dtype,
    int precision, double eps, void *workspace, int64_t workspace_bytes, ac4k_stream_t stream) {
  AC4K_REQUIRE(out && x, "null pointer argument");
  AC4K_REQUIRE(rows >= 1 && K >= 1, "rows and columns must be positive (rows=%lld K=%lld)", (long long)rows, (long long)K);
  AC4K_REQUIRE(K <= AC4K_NORM_MAX_COLS, "rows of at most %d elements, got %lld", (int)AC4K_NORM_MAX_COLS, (long long)K);
  AC4K_REQUIRE(rows < (1ll << 31) - 16, "too many rows (%lld)", (long long)rows);
  AC4K_REQUIRE(float_tag(dtype), "x must be bfloat16, half or float (dtype tag %d)", dtype);
  AC4K_REQUIRE(!weight || weight_dtype == dtype || weight_dtype == AC4K_DTYPE_FP32, "weight must have the type of x or be float (dtype tag %d)", weight_dtype);
  AC4K_REQUIRE(precision >= AC4K_PRECISION_NONE && precision <= AC4K_PRECISION_NVFP4, "unknown precision %d", precision);
  AC4K_REQUIRE(!residual == !sum, "a residual comes with a place for the sum, and the other way round");
  AC4K_REQUIRE(precision == AC4K_PRECISION_NONE || (sf && ((uintptr_t)sf & 3) == 0 && ((uintptr_t)out & 3) == 0),
               "a quantized output needs scales, both on 4 bytes");
  AC4K_REQUIRE(precision != AC4K_PRECISION_NVFP4 || global_scale, "nvfp4 needs a global scale, given or to be written");
  AC4K_REQUIRE(eps >= 0.0, "eps must not be negative");
  const bool find = precision == AC4K_PRECISION_NVFP4 && !given_scale;
  const int64_t need = ac4k_rms_norm_workspace_bytes(rows, K, dtype, precision, given_scale);
  AC4K_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 3) == 0),
               "workspace of %lld bytes needed, on 4 bytes", (long long)need);
  NormArgs a{};
  a.x = x, a.residual = residual, a.weight = weight, a.sum = sum, a.out = out, a.sf = sf, a.gs = global_scale;
  a.rows = rows, a.K = K, a.Rp = align_up(rows, 16);
  a.Kp = precision == AC4K_PRECISION_NVFP4 ? align_up(K, 64) : align_up(K, 16);
  a.x_stride = x_stride, a.residual_stride = residual_stride, a.sum_stride = sum_stride, a.out_stride = out_stride;
  a.eps = eps;
  a.inverse_K = 1.0 / (double)K;
  hipStream_t st = (hipStream_t)stream;
  int rc;
  auto go = [&](auto kernels) { rc = kernels(a, precision, find, static_cast<float *>(workspace), dtype, st); };
  const bool w32 = weight && weight_dtype == AC4K_DTYPE_FP32;
  if (dtype == AC4K_DTYPE_FP32) go(norm_dtype<AC4K_DTYPE_FP32, AC4K_DTYPE_FP32>);
  else if (dtype == AC4K_DTYPE_BF16) w32 ? go(norm_dtype<AC4K_DTYPE_BF16, AC4K_DTYPE_FP32>) : go(norm_dtype<AC4K_DTYPE_BF16, AC4K_DTYPE_BF16>);
  else w32 ? go(norm_dtype<AC4K_DTYPE_FP16, AC4K_DTYPE_FP32>) : go(norm_dtype<AC4K_DTYPE_FP16, AC4K_DTYPE_FP16>);
  if (rc) return rc;
  return check_launch("ac4k_rms_norm");
}

extern "C" __attribute__((visibility("default"))) int ac4k_dequantize(void *out, int dtype, const void *q, const void *sf, const float *global_scale,
                                                                      int64_t global_scale_stride, int64_t lead, int64_t R, int64_t W,
                                                                      int64_t cols, int precision, ac4k_stream_t stream) {
  AC4K_REQUIRE(out && q && sf, "null pointer argument");
  AC4K_REQUIRE(lead >= 1 && R >= 1 && W >= 1 && cols >= 1, "sizes must be positive");
  AC4K_REQUIRE(cols <= W, "at most the %lld columns of a quantized row, got %lld", (long long)W, (long long)cols);
  AC4K_REQUIRE(float_tag(dtype), "out must be bfloat16, half or float (dtype tag %d)", dtype);
  AC4K_REQUIRE(precision >= AC4K_PRECISION_FP8 && precision <= AC4K_PRECISION_NVFP4, "unknown precision %d", precision);
  AC4K_REQUIRE(precision != AC4K_PRECISION_NVFP4 || (global_scale && W % 64 == 0 && ((uintptr_t)q & 3) == 0),
               "nvfp4 comes in whole chunks of 64, on 4 bytes and with a global scale");
  AC4K_REQUIRE(precision == AC4K_PRECISION_NVFP4 || (W % 16 == 0 && ((uintptr_t)sf & 3) == 0), "8-bit rows come in whole pieces of 16, scales on 4 bytes");
  const int64_t spans = ceil_div(W, 512), bands = ceil_div(R, 16);
  AC4K_REQUIRE(spans < (1ll << 24) && bands < (1ll << 24) && lead < (1ll << 24) && spans * bands < (1ll << 24) && spans * bands * lead < (1ll << 24),
               "tensor too large");  // 2^32 threads a launch
  const DequantArgs a{out, static_cast<const uint8_t *>(q), sf, global_scale, lead, R, W, align_up(R, 16), cols, global_scale_stride};
  hipStream_t st = (hipStream_t)stream;
  if (dtype == AC4K_DTYPE_BF16) launch_dequantize<AC4K_DTYPE_BF16>(a, precision, spans * bands * lead, st);
  else if (dtype == AC4K_DTYPE_FP16) launch_dequantize<AC4K_DTYPE_FP16>(a, precision, spans * bands * lead, st);
  else launch_dequantize<AC4K_DTYPE_FP32>(a, precision, spans * bands * lead, st);
  return check_launch("ac4k_dequantize");
}

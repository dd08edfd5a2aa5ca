// What the linear kernels of linear_kernels.h, linear_fused.hip and linear_grouped.hip share.
#pragma once

#include "ac4k_common.h"

namespace ac4k {

// --- output / bias element types -------------------------------------------
template <int DT>
struct Elem;
template <>
struct Elem<AC4K_DTYPE_BF16> {
  using T = uint16_t;
  static __device__ __forceinline__ float load(const void *p, int64_t i) {
    return bf16_bits_to_f32(static_cast<const uint16_t *>(p)[i]);
  }
  // round to nearest even, NaN stays NaN: v_cvt_pk_bf16_f32
  static __device__ __forceinline__ T cvt(float f) { return __builtin_bit_cast(uint16_t, (__bf16)f); }
  static __device__ __forceinline__ uint32_t cvt2(float lo, float hi) {
    typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
    const f32x2 v = {lo, hi};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2_t));
  }
};
template <>
struct Elem<AC4K_DTYPE_FP16> {
  using T = _Float16;
  static __device__ __forceinline__ float load(const void *p, int64_t i) {
    return (float)static_cast<const _Float16 *>(p)[i];
  }
  static __device__ __forceinline__ T cvt(float f) { return (_Float16)f; }
  static __device__ __forceinline__ uint32_t cvt2(float lo, float hi) {
    const f16x2 v = {(_Float16)lo, (_Float16)hi};
    return __builtin_bit_cast(uint32_t, v);
  }
};
template <>
struct Elem<AC4K_DTYPE_FP32> {
  using T = float;
  static __device__ __forceinline__ float load(const void *p, int64_t i) {
    return static_cast<const float *>(p)[i];
  }
  static __device__ __forceinline__ T cvt(float f) { return f; }
  static __device__ __forceinline__ uint32_t cvt2(float lo, float) { return __float_as_uint(lo); }  // unused: 4-byte outputs are not packed
};
constexpr int BIAS_NONE = 3;
constexpr int BIAS_EPILOGUE = 4;  // all of Epilogue below, told apart while the kernel runs: uniform branches, once an output

// What follows the product with an epilogue: round(act(product + bias) + residual)
struct Epilogue {
  const void *bias = nullptr;      // [N] of bias_dtype, or null
  const void *residual = nullptr;  // [M, N] of D's type, or null
  int64_t residual_stride = 0;     // elements between rows
  int bias_dtype = 0, activation = 0;
};

__device__ __forceinline__ float epilogue_bias(const Epilogue &ep, int64_t n) {
  return ep.bias_dtype == AC4K_DTYPE_BF16   ? Elem<AC4K_DTYPE_BF16>::load(ep.bias, n)
         : ep.bias_dtype == AC4K_DTYPE_FP16 ? Elem<AC4K_DTYPE_FP16>::load(ep.bias, n)
                                            : Elem<AC4K_DTYPE_FP32>::load(ep.bias, n);
}

// x / (1 + e^-g(x)) with g(x) = x (silu) or 2 sqrt(2 / pi) (x + 0.044715 x^3), of which gelu's approximation by tanh is made: tanh(z) = 2 / (1 + e^-2z) - 1.
// k1, k3: coefficients of -g / ln 2.  x^2 is cut off where it would be infinite; the square is as good as that far out.
__device__ __forceinline__ float times_sigmoid(float x, float k1, float k3) {
  const float e = __builtin_amdgcn_exp2f(x * (k1 + k3 * __builtin_fminf(x * x, 1e30f)));
  return x * __builtin_amdgcn_rcpf(1.0f + e);
}
// x Phi(x), the normal distribution's Phi(-a) = e^(-a^2 / 2) R(a) for a = |x|.  R = erfcx(a / sqrt 2) / 2 falls smoothly from 1/2 to 0; in t = 1 / (1 + 0.305 a) a
// polynomial of degree eight without constant, fitted to the least relative error over a = 0 to 14, is 1.0e-7 off at the most (4.1e-7 in 32 bits).
__device__ __forceinline__ float gelu(float x) {
  const float a = __builtin_fabsf(x);
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(a, 0.305f, 1.0f));
  float r = 0.036702316254377365f;
  r = __builtin_fmaf(r, t, -0.15300191938877106f);
  r = __builtin_fmaf(r, t, 0.18574152886867523f);
  r = __builtin_fmaf(r, t, -0.03800073266029358f);
  r = __builtin_fmaf(r, t, 0.12103506177663803f);
  r = __builtin_fmaf(r, t, 0.1034165620803833f);
  r = __builtin_fmaf(r, t, 0.12246755510568619f);
  r = __builtin_fmaf(r, t, 0.121639683842659f);
  const float tail = r * t * __builtin_amdgcn_exp2f(a * a * -0.7213475204444817f);  // Phi(-a)
  const float far = __builtin_fminf(x, 20.0f) * tail;  // (the tail of an infinite x is 0)
  return x < 0.0f ? far : x - far;
}
// F: what is done with a function of one value
template <typename F>
__device__ __forceinline__ void with_activation(int kind, F f) {
  constexpr float LOG2E = 1.4426950408889634f, TANH = -2.0f * 0.7978845608028654f * LOG2E;
  if (kind == AC4K_ACTIVATION_GELU) {
    f([](float x) { return gelu(x); });
  } else if (kind == AC4K_ACTIVATION_SILU || kind == AC4K_ACTIVATION_GELU_TANH) {
    const float k1 = kind == AC4K_ACTIVATION_SILU ? -LOG2E : TANH, k3 = kind == AC4K_ACTIVATION_SILU ? 0.0f : TANH * 0.044715f;
    f([=](float x) { return times_sigmoid(x, k1, k3); });
  } else {
    const float least = kind == AC4K_ACTIVATION_RELU ? 0.0f : -__builtin_inff();
    f([=](float x) { return x < least ? least : x; });  // (a NaN stays)
  }
}
// V outputs of row m from column n on; those from column N on are not used
template <int D_DT, int V>
__device__ __forceinline__ void finish_values(const Epilogue &ep, float (&v)[V], int64_t m, int64_t n, int64_t N) {
  if (ep.bias) {
#pragma unroll
    for (int q = 0; q < V; ++q) v[q] += n + q < N ? epilogue_bias(ep, n + q) : 0.0f;
  }
  with_activation(ep.activation, [&](auto act) {
#pragma unroll
    for (int q = 0; q < V; ++q) v[q] = act(v[q]);
  });
  if (ep.residual) {
#pragma unroll
    for (int q = 0; q < V; ++q) v[q] += n + q < N ? Elem<D_DT>::load(ep.residual, m * ep.residual_stride + n + q) : 0.0f;
  }
}

// dword `w` (8 nibbles) times block scale `sc` (both halves of `sc2` hold candidates, HI picks)
template <bool HI>
__device__ __forceinline__ f16x8 decode_dword(uint32_t w, f16x2 sc2) {
  const f16x2 sc = HI ? (f16x2){sc2.y, sc2.y} : (f16x2){sc2.x, sc2.x};
  f16x2 d0 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 0) * sc;
  f16x2 d1 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 1) * sc;
  f16x2 d2 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 2) * sc;
  f16x2 d3 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 3) * sc;
  return (f16x8){d0.x, d0.y, d1.x, d1.y, d2.x, d2.y, d3.x, d3.y};
}

// --- 16 weight rows per workgroup ------------------------------------------------
constexpr int R16_ROWS = 16, R16_WAVES = 8, R16_STEP = 128;
// A launch carries fewer than 2^32 threads along a grid dim and drops the rest without an error: weights of up to 2^27 - 16 rows.
static inline bool rows16_grid_ok(int64_t N) { return ceil_div(N, R16_ROWS) * (64 * R16_WAVES) < (1ll << 32); }

// End of these kernels: the sums of the eight waves in the order of the waves, scale, bias, store.
template <int D_DT, int BIAS_DT, int MT>
__device__ __forceinline__ void rows16_finish(const f32x4 (&acc)[MT][2], float4 (*part)[MT][64], void *out, const void *bias, float scale,
                                              int64_t M, int64_t N, int64_t n0, const Epilogue *ep = nullptr) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  // lane (r, g): activation row r of tile i, weight rows 4 g .. 4 g + 3
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const f32x4 v = acc[i][0] + acc[i][1];
    part[wave][i][lane] = make_float4(v[0], v[1], v[2], v[3]);
  }
  __syncthreads();
  if (wave >= MT) return;
  float4 v = part[0][wave][lane];
#pragma unroll
  for (int q = 1; q < R16_WAVES; ++q) {
    const float4 o = part[q][wave][lane];
    v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
  }
  const int m = wave * 16 + r;
  const int64_t n = n0 + g * 4;
  if (m >= (int)M || n >= N) return;
  using DE = Elem<D_DT>;
  float o[4] = {v.x * scale, v.y * scale, v.z * scale, v.w * scale};
  if constexpr (BIAS_DT == BIAS_EPILOGUE) {
    finish_values<D_DT, 4>(*ep, o, m, n, N);
  } else if constexpr (BIAS_DT != BIAS_NONE) {
#pragma unroll
    for (int q = 0; q < 4; ++q) o[q] += n + q < N ? Elem<BIAS_DT>::load(bias, n + q) : 0.0f;
  }
  typename DE::T *dst = static_cast<typename DE::T *>(out) + (int64_t)m * N + n;
  if ((N & 3) == 0 && ((uintptr_t)out & 15) == 0) {
    if constexpr (sizeof(typename DE::T) == 2)
      *reinterpret_cast<uint2 *>(dst) = make_uint2(DE::cvt2(o[0], o[1]), DE::cvt2(o[2], o[3]));
    else
      *reinterpret_cast<float4 *>(dst) = make_float4(o[0], o[1], o[2], o[3]);
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (n + q < N) dst[q] = DE::cvt(o[q]);
  }
}

// quantize and linear in one launch (linear_fused.hip); rows16 kernels fit the shape and the operands are on 16 bytes
struct FusedArgs {
  void *D;
  const uint16_t *X;       // [M, K] bf16; null: the activation is in X_q, X_sf and X_gs (M <= 16)
  uint8_t *X_q, *X_sf;     // the quantized activation, for the caller
  float *X_gs;
  const uint8_t *B;
  const uint32_t *B_sf;
  const float *B_gs;
  const void *bias;
  int64_t M, N, K, Mp, Np;
};
constexpr int64_t FUSED_ELEMS = 16384;  // of the activation
int launch_fused_rows16(const FusedArgs &a, int d_dtype, int bias_dtype, hipStream_t st);

}  // namespace ac4k

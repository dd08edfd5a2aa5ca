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
#include "norm_rows.h"

namespace ac4k {

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
  return norm_workspace(rows, K, dtype, NORM_ROWS);
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
  if (dtype == AC4K_DTYPE_FP32) go(norm_dtype<NORM_ROWS, AC4K_DTYPE_FP32, AC4K_DTYPE_FP32>);
  else if (dtype == AC4K_DTYPE_BF16) w32 ? go(norm_dtype<NORM_ROWS, AC4K_DTYPE_BF16, AC4K_DTYPE_FP32>) : go(norm_dtype<NORM_ROWS, AC4K_DTYPE_BF16, AC4K_DTYPE_BF16>);
  else w32 ? go(norm_dtype<NORM_ROWS, AC4K_DTYPE_FP16, AC4K_DTYPE_FP32>) : go(norm_dtype<NORM_ROWS, AC4K_DTYPE_FP16, AC4K_DTYPE_FP16>);
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

// Norms around a block of a transformer: what it returns is normed (post), gated and added to the residual, and the sum is normed and modulated for the next block.
//
//   u = x,  or (x - mean(x)) / sqrt(var(x) + eps) * post              (rows of K; rms: mean 0 and the mean square)
//   h = round(residual_scale * residual + gate * u)                     (x's type; x itself without a residual)
//   y = (h - mean(h)) / sqrt(var(h) + eps) * weight * (1 + scale) + shift
// and y leaves as from rms_norm, with whose kernel it is computed (norm_rows.h): in x's type or in the format of a quantizer, from 32 bits.  Sums, means and
// squares are held in 64 bits; the mean is taken off in two pieces of 32 bits.
//
// Bound by memory where rows have whole vectors: 75600 x 5120 bf16, layer norm with gate, scale and shift of one sequence, 600 us, 5.2 TB/s, the rate of a copy (1477 MiB
// read, 1477 written; the vector port is busy for 50 %).  8192 x 4096 with post norm and gate to nvfp4 49 + 25 us, where one pass over its bytes takes 42: the second launch reads h
// again, and the first one's port is busy for 72 %.  Rows that end inside a vector, 4002 x 5003 layer norm to int8 with vectors in fp32, 48 us where the bytes need 27:
// every row reads its three vectors of 20 KB through the caches, at no alignment.  One row of 8192 with post norm to e4m3 5.4 us (rms_norm 3.7).
// As first built, with all vectors held in registers ahead of their use, 198 to 256 registers left one or two waves on a SIMD: 983, 65 + 25 and 124 us.
#include "norm_rows.h"

using namespace ac4k;

static bool float_tag(int d) { return d == AC4K_DTYPE_BF16 || d == AC4K_DTYPE_FP16 || d == AC4K_DTYPE_FP32; }

extern "C" __attribute__((visibility("default"))) int64_t ac4k_block_norm_workspace_bytes(int64_t rows, int64_t K, int dtype, int precision, int given_scale) {
  if (rows < 1 || K < 1 || K > AC4K_BLOCK_NORM_MAX_COLS || !float_tag(dtype) || precision != AC4K_PRECISION_NVFP4 || given_scale) return 0;
  const int64_t factors = norm_workspace(rows, K, dtype, NORM_BLOCK);
  return factors ? factors + 8 * rows : 0;  // the means behind them
}

extern "C" __attribute__((visibility("default"))) int ac4k_block_norm(
    void *out, int64_t out_stride, void *sf, float *global_scale, int given_scale, const void *x, int64_t x_stride, const void *residual,
    int64_t residual_stride, void *sum, int64_t sum_stride, const void *weight, const void *post_weight, const void *gate, int64_t gate_stride, int64_t gate_rows,
    const void *scale, int64_t scale_stride, int64_t scale_rows, const void *shift, int64_t shift_stride, int64_t shift_rows, int vector_dtype, int64_t rows,
    int64_t K, int dtype, int precision, int kind, double residual_scale, double eps, void *workspace, int64_t workspace_bytes, ac4k_stream_t stream) {
  AC4K_REQUIRE(out && x, "null pointer argument");
  AC4K_REQUIRE(rows >= 1 && K >= 1, "rows and columns must be positive (rows=%lld K=%lld)", (long long)rows, (long long)K);
  AC4K_REQUIRE(K <= AC4K_BLOCK_NORM_MAX_COLS, "rows of at most %d elements, got %lld", (int)AC4K_BLOCK_NORM_MAX_COLS, (long long)K);
  AC4K_REQUIRE(rows < (1ll << 31) - 16, "too many rows (%lld)", (long long)rows);
  AC4K_REQUIRE(float_tag(dtype), "x must be bfloat16, half or float (dtype tag %d)", dtype);
  AC4K_REQUIRE(vector_dtype == dtype || vector_dtype == AC4K_DTYPE_FP32, "vectors must have the type of x or be float (dtype tag %d)", vector_dtype);
  AC4K_REQUIRE(precision >= AC4K_PRECISION_NONE && precision <= AC4K_PRECISION_NVFP4, "unknown precision %d", precision);
  AC4K_REQUIRE(kind == AC4K_NORM_RMS || kind == AC4K_NORM_LAYER, "unknown kind %d", kind);
  AC4K_REQUIRE(!residual == !sum, "a residual comes with a place for the sum, and the other way round");
  AC4K_REQUIRE(residual || (!gate && !post_weight), "a gate or a post weight comes with a residual");
  AC4K_REQUIRE(precision == AC4K_PRECISION_NONE || (sf && ((uintptr_t)sf & 3) == 0 && ((uintptr_t)out & 3) == 0),
               "a quantized output needs scales, both on 4 bytes");
  AC4K_REQUIRE(precision != AC4K_PRECISION_NVFP4 || global_scale, "nvfp4 needs a global scale, given or to be written");
  AC4K_REQUIRE(eps >= 0.0, "eps must not be negative");
  for (int64_t n : {gate_rows, scale_rows, shift_rows}) AC4K_REQUIRE(n >= 0 && n < (1ll << 31), "rows of a vector must be 0 (all) or positive, got %lld", (long long)n);
  const bool find = precision == AC4K_PRECISION_NVFP4 && !given_scale;
  const int64_t need = ac4k_block_norm_workspace_bytes(rows, K, dtype, precision, given_scale);
  AC4K_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 3) == 0),
               "workspace of %lld bytes needed, on 4 bytes", (long long)need);
  NormArgs a{};
  a.x = x, a.residual = residual, a.weight = weight, a.sum = sum, a.out = out, a.sf = sf, a.gs = global_scale;
  a.rows = rows, a.K = K, a.Rp = align_up(rows, 16);
  a.Kp = precision == AC4K_PRECISION_NVFP4 ? align_up(K, 64) : align_up(K, 16);
  a.x_stride = x_stride, a.residual_stride = residual_stride, a.sum_stride = sum_stride, a.out_stride = out_stride;
  a.eps = eps;
  a.inverse_K = 1.0 / (double)K;
  a.gate = {gate, gate_stride, (uint32_t)gate_rows}, a.scale = {scale, scale_stride, (uint32_t)scale_rows}, a.shift = {shift, shift_stride, (uint32_t)shift_rows};
  a.post = post_weight;
  a.alpha = (float)residual_scale;
  a.centred = kind == AC4K_NORM_LAYER;
  hipStream_t st = (hipStream_t)stream;
  auto go = [&](auto whole, auto cut) { return (K % 8 == 0 ? whole : cut)(a, precision, find, static_cast<float *>(workspace), dtype, st); };
#define AC4K_BLOCK(DT, VT) go(norm_dtype<NORM_BLOCK, AC4K_DTYPE_##DT, AC4K_DTYPE_##VT>, norm_dtype<NORM_BLOCK_CUT, AC4K_DTYPE_##DT, AC4K_DTYPE_##VT>)
  const bool v32 = vector_dtype == AC4K_DTYPE_FP32;
  int rc;
  if (dtype == AC4K_DTYPE_FP32) rc = AC4K_BLOCK(FP32, FP32);
  else if (dtype == AC4K_DTYPE_BF16) rc = v32 ? AC4K_BLOCK(BF16, FP32) : AC4K_BLOCK(BF16, BF16);
  else rc = v32 ? AC4K_BLOCK(FP16, FP32) : AC4K_BLOCK(FP16, FP16);
#undef AC4K_BLOCK
  if (rc) return rc;
  return check_launch("ac4k_block_norm");
}

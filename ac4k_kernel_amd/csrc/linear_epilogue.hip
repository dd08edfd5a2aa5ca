// The linear with an activation and a residual in its epilogue:  D = round(act((A . B^T) * (gsA*gsB) + bias) + residual).  The kernels, plans and scratch are those of
// the plain linear (linear_kernels.h); bias, activation and residual follow the sums in 32 bits, and there is one rounding, to D's type.
//
// What it costs over the plain linear on the same card, us (plain / relu / silu / gelu / residual / gelu and residual): 8192 x 14336 x 4096 bf16 654 / 677 / 696 / 727 / 703 /
// 754 - gelu is 24 instructions' time an output, which nothing hides with one wave on a SIMD, the residual 235 MB -; 1001 x 5003 x 2880 fp32 35.9 / 36.8 / 38.1 / 39.3 / 40.4 /
// 43.4.  1 x 14336 x 4096 10.7 alone, as the plain one.  Activations on the sums where they are, in the accumulation registers, spilled them: 1050 to 1150 us.
#include "linear_kernels.h"

namespace ac4k {

template <int D_DT>
static int run(const LinearArgs &a, void *workspace, int64_t need, hipStream_t st) {
  if (need == 0) return launch_linear<D_DT, BIAS_EPILOGUE>(a, st);
  SkinnyPlan p;
  if (skinny_plan(a.M, a.N, a.K, p)) {
    const SkinnyArgs sa{a.D, a.A, reinterpret_cast<const uint8_t *>(a.A_sf), a.Mp, a.B, a.B_sf, a.A_gs, a.B_gs, nullptr, static_cast<float *>(workspace),
                        a.M, a.N, a.K, a.Np, p.ks_len, p.split_k, 0, a.ep};
    return launch_skinny<D_DT, BIAS_EPILOGUE>(sa, p, st);
  }
  MidPlan mp;
  AC4K_REQUIRE(mid_plan(a.M, a.N, a.K, mp), "no plan for a shape with scratch");
  return launch_mid<D_DT, BIAS_EPILOGUE>(a, mp, static_cast<float *>(workspace), need, st);
}

}  // namespace ac4k

using namespace ac4k;

extern "C" __attribute__((visibility("default"))) int ac4k_linear_nvfp4_epilogue(
    void *D, int d_dtype, const void *A, const void *A_sf, const float *A_gs, const void *B, const void *B_sf, const float *B_gs, const void *bias, int bias_dtype,
    int activation, const void *residual, int64_t residual_stride, int64_t M, int64_t N, int64_t K, void *workspace, int64_t workspace_bytes, ac4k_stream_t stream) {
  AC4K_REQUIRE(D && A && A_sf && A_gs && B && B_sf && B_gs, "null pointer argument");
  AC4K_REQUIRE(M >= 1 && N >= 1 && K >= 1, "M, N, K must be positive (M=%lld N=%lld K=%lld)", (long long)M, (long long)N, (long long)K);
  AC4K_REQUIRE(K % 16 == 0, "A size(1)*2 must be multiple of 16 but see %lld", (long long)K);
  AC4K_REQUIRE(((uintptr_t)A & 7) == 0 && ((uintptr_t)B & 7) == 0 && ((uintptr_t)A_sf & 3) == 0 && ((uintptr_t)B_sf & 3) == 0,
               "A/B must be 8-byte aligned and the scale tensors 4-byte aligned");
  AC4K_REQUIRE(!bias || bias_dtype == AC4K_DTYPE_BF16 || bias_dtype == AC4K_DTYPE_FP16 || bias_dtype == AC4K_DTYPE_FP32,
               "bias must be bfloat16, half or float (dtype tag %d)", bias_dtype);
  AC4K_REQUIRE(activation >= AC4K_ACTIVATION_NONE && activation <= AC4K_ACTIVATION_SILU, "unknown activation %d", activation);
  AC4K_REQUIRE(ceil_div(M, T_BM) * ceil_div(N, T_BN) < (1ll << 24), "problem too large");  // 2^32 threads a launch
  const bool aligned = (((uintptr_t)A | (uintptr_t)B) & 15) == 0;
  const int64_t need = aligned ? ac4k_linear_nvfp4_scratch_bytes(M, N, K) : 0;
  if (need > 0) {
    AC4K_REQUIRE(workspace && ((uintptr_t)workspace & 255) == 0, "workspace must be 256-byte aligned");
    AC4K_REQUIRE(workspace_bytes >= need, "workspace too small: %lld bytes needed", (long long)need);
  }
  LinearArgs a{D, static_cast<const uint8_t *>(A), static_cast<const uint8_t *>(B), static_cast<const uint32_t *>(A_sf), static_cast<const uint32_t *>(B_sf),
               A_gs, B_gs, nullptr, M, N, K, align_up(M, 16), align_up(N, 16)};
  a.ep = Epilogue{bias, residual, residual_stride, bias_dtype, activation};
  hipStream_t st = (hipStream_t)stream;
  int rc;
  switch (d_dtype) {
    case AC4K_DTYPE_BF16: rc = run<AC4K_DTYPE_BF16>(a, workspace, need, st); break;
    case AC4K_DTYPE_FP16: rc = run<AC4K_DTYPE_FP16>(a, workspace, need, st); break;
    case AC4K_DTYPE_FP32: rc = run<AC4K_DTYPE_FP32>(a, workspace, need, st); break;
    default: return set_error("d must be bfloat16, half or float (dtype tag %d)", d_dtype);
  }
  if (rc) return rc;
  return check_launch("ac4k_linear_nvfp4_epilogue");
}

// Linears grouped by expert on NVFP4 operands: row i of the output is row rows[i] of x (row i without `rows`) times the weight of the expert
// whose range of offsets holds i,
//
//   D[i] = (x[rows[i]] . W[e]^T) * (gs_x * gs_W[e]) + bias[e],   offsets[e] <= i < offsets[e + 1].
//
// The sizes of the groups are on the GPU and nothing waits for them: launches are made for the largest number of tiles that the row and
// expert counts allow, and workgroups without a tile end at once.  Offsets are taken as clamped to [0, rows] and rising, row indexes as
// clamped to x: a wrong table gives wrong rows, not an access outside of the operands.  Output rows that no group holds stay as they are.
#include "linear_common.h"

namespace ac4k {

struct GroupedArgs {
  void *D;
  const uint8_t *A;
  const uint32_t *A_sf;
  const float *A_gs;
  const int32_t *rows;     // or null
  const uint8_t *B;
  const uint32_t *B_sf;
  const float *B_gs;
  int64_t B_gs_stride;
  const void *bias;        // [E, N]
  const int32_t *offsets;  // [E + 1]
  int64_t T, Tp, M, N, Np, K, E;
};

struct Group {
  int first, count;
};
__device__ __forceinline__ Group group_of(const int32_t *offsets, int64_t e, int64_t M) {
  const int lo = offsets[e], hi = offsets[e + 1];
  const int first = lo < 0 ? 0 : lo > (int)M ? (int)M : lo;
  const int end = hi > (int)M ? (int)M : hi;
  return {first, end > first ? end - first : 0};
}

// ===========================================================================
// 16 weight rows of an expert and all of K in a workgroup, the expert's rows 16 * MT at a time: groups of few rows, where the weights
// are read once, and every shape that the tiles do not take.  The eight waves take the 128-k steps in turn; see linear_nvfp4_rows16_kernel for
// the layout of a step (lane (row r, quarter g): 16 bytes of its weight row and of its activation row, the operands of four MFMAs of 16 x 16 x 32).
// A step's second half that K does not have is read from its first one, with weight scales so small that they round to zero.
// ===========================================================================
constexpr int G16_DEPTH = 3;

template <int D_DT, int BIAS_DT, int MT>
__global__ __launch_bounds__(64 * R16_WAVES, 2) void linear_grouped_rows16_kernel(GroupedArgs a) {
  __shared__ float4 part[R16_WAVES][MT][64];
  const Group grp = group_of(a.offsets, blockIdx.y, a.M);
  if (grp.count == 0) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int64_t e = blockIdx.y, n0 = (int64_t)blockIdx.x * R16_ROWS, kb = a.K >> 1;
  const int nst = (int)ceil_div(a.K, R16_STEP);
  const int cnt = (nst - wave + R16_WAVES - 1) / R16_WAVES;  // steps of this wave; none where K is short
  const bool tail = a.K % R16_STEP != 0;
  const int wr = n0 + r < a.N ? r : (int)(a.N - 1 - n0);  // rows past N read the last row; their outputs are never stored
  const uint8_t *const w_row = a.B + (e * a.N + n0 + wr) * kb;
  const uint8_t *const ws_row = reinterpret_cast<const uint8_t *>(a.B_sf) + (e * (a.K >> 6) * a.Np + n0 + wr) * 4;
  const float scale = *a.A_gs * a.B_gs[e * a.B_gs_stride];
  for (int m0 = 0; m0 < grp.count; m0 += 16 * MT) {
    const uint8_t *x_row[MT], *xs_row[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int m = m0 + i * 16 + r < grp.count ? m0 + i * 16 + r : grp.count - 1;  // rows past the group likewise
      int64_t src = grp.first + m;
      if (a.rows) {
        src = a.rows[src];
        src = src < 0 ? 0 : src < a.T ? src : a.T - 1;
      }
      x_row[i] = a.A + src * kb;
      xs_row[i] = reinterpret_cast<const uint8_t *>(a.A_sf) + src * 4;
    }
    struct Step {
      uint4 w, x[MT];
      uint32_t ws, xs[MT];
    };
    auto load = [&](Step &st, int t) {
      const int s = wave + t * R16_WAVES;
      const int gg = tail && s == nst - 1 ? g & 1 : g;
      const int64_t at = (int64_t)s * (R16_STEP / 2) + gg * 16;
      const int64_t chunk = 2 * s + (gg >> 1);
      st.w = *reinterpret_cast<const uint4 *>(w_row + at);
      st.ws = *reinterpret_cast<const uint16_t *>(ws_row + chunk * a.Np * 4 + (gg & 1) * 2);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        st.x[i] = *reinterpret_cast<const uint4 *>(x_row[i] + at);
        st.xs[i] = *reinterpret_cast<const uint16_t *>(xs_row[i] + chunk * a.Tp * 4 + (gg & 1) * 2);
      }
    };
    f32x4 acc[MT][2];  // two independent accumulation chains
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[i][0] = acc[i][1] = (f32x4)(0.0f);
    auto multiply = [&](const Step &st, int t) {
      const float fac = tail && wave + t * R16_WAVES == nst - 1 && g >= 2 ? 0x1p-60f : 1.0f;
      const f16x2 wsc = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(st.ws, fac, false);
      const f16x8 w0 = decode_dword<false>(st.w.x, wsc), w1 = decode_dword<false>(st.w.y, wsc);
      const f16x8 w2 = decode_dword<true>(st.w.z, wsc), w3 = decode_dword<true>(st.w.w, wsc);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const f16x2 xsc = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(st.xs[i], 1.0f, false);
        acc[i][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w0, decode_dword<false>(st.x[i].x, xsc), acc[i][0], 0, 0, 0);
        acc[i][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w1, decode_dword<false>(st.x[i].y, xsc), acc[i][1], 0, 0, 0);
        acc[i][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w2, decode_dword<true>(st.x[i].z, xsc), acc[i][0], 0, 0, 0);
        acc[i][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w3, decode_dword<true>(st.x[i].w, xsc), acc[i][1], 0, 0, 0);
      }
    };
    Step ring[G16_DEPTH];
#pragma unroll
    for (int d = 0; d < G16_DEPTH; ++d)
      if (d < cnt) load(ring[d], d);
    int t = 0;
    for (; t + G16_DEPTH < cnt; t += G16_DEPTH) {
#pragma unroll
      for (int d = 0; d < G16_DEPTH; ++d) {
        multiply(ring[d], t + d);
        if (t + d + G16_DEPTH < cnt) load(ring[d], t + d + G16_DEPTH);
      }
    }
#pragma unroll
    for (int d = 0; d < G16_DEPTH; ++d)
      if (t + d < cnt) multiply(ring[d], t + d);

    using T = typename Elem<D_DT>::T;
    if (m0) __syncthreads();  // the sums of the rows before have been read
    const char *bias = static_cast<const char *>(a.bias);
    if constexpr (BIAS_DT != BIAS_NONE) bias += e * a.N * (int64_t)sizeof(typename Elem<BIAS_DT>::T);
    rows16_finish<D_DT, BIAS_DT, MT>(acc, part, static_cast<T *>(a.D) + (int64_t)(grp.first + m0) * a.N, bias, scale, grp.count - m0, a.N, n0);
  }
}

template <int D_DT, int BIAS_DT>
static int launch_grouped(const GroupedArgs &a, hipStream_t st) {
  const dim3 grid((unsigned)ceil_div(a.N, R16_ROWS), (unsigned)a.E);
  if (a.M <= 16 * a.E) hipLaunchKernelGGL((linear_grouped_rows16_kernel<D_DT, BIAS_DT, 1>), grid, dim3(64 * R16_WAVES), 0, st, a);
  else hipLaunchKernelGGL((linear_grouped_rows16_kernel<D_DT, BIAS_DT, 2>), grid, dim3(64 * R16_WAVES), 0, st, a);
  return 0;
}

template <int D_DT>
static int grouped_bias(const GroupedArgs &a, int bias_dtype, hipStream_t st) {
  if (!a.bias) return launch_grouped<D_DT, BIAS_NONE>(a, st);
  switch (bias_dtype) {
    case AC4K_DTYPE_BF16: return launch_grouped<D_DT, AC4K_DTYPE_BF16>(a, st);
    case AC4K_DTYPE_FP16: return launch_grouped<D_DT, AC4K_DTYPE_FP16>(a, st);
    case AC4K_DTYPE_FP32: return launch_grouped<D_DT, AC4K_DTYPE_FP32>(a, st);
  }
  return set_error("bias must be bfloat16, half or float (dtype tag %d)", bias_dtype);
}

}  // namespace ac4k

using namespace ac4k;

extern "C" __attribute__((visibility("default"))) int64_t ac4k_linear_grouped_nvfp4_workspace_bytes(int64_t M, int64_t N, int64_t K, int64_t E, int has_rows) {
  return 0;
}

extern "C" __attribute__((visibility("default"))) int ac4k_linear_grouped_nvfp4(
    void *D, int d_dtype, const void *A, const void *A_sf, const float *A_gs, int64_t T, const int32_t *rows, const void *B, const void *B_sf,
    const float *B_gs, int64_t B_gs_stride, const void *bias, int bias_dtype, const int32_t *offsets, int64_t M, int64_t N, int64_t K, int64_t E,
    void *workspace, int64_t workspace_bytes, ac4k_stream_t stream) {
  AC4K_REQUIRE(D && A && A_sf && A_gs && B && B_sf && B_gs && offsets, "null pointer argument");
  AC4K_REQUIRE(M >= 1 && N >= 1 && K >= 1 && E >= 1 && T >= 1, "sizes must be positive (M=%lld N=%lld K=%lld E=%lld T=%lld)", (long long)M,
               (long long)N, (long long)K, (long long)E, (long long)T);
  AC4K_REQUIRE(K % 64 == 0, "K must be a multiple of 64 but see %lld", (long long)K);
  AC4K_REQUIRE(rows || T == M, "without rows, x has one row for each of the output (%lld, not %lld)", (long long)M, (long long)T);
  AC4K_REQUIRE((((uintptr_t)A | (uintptr_t)B) & 15) == 0 && (((uintptr_t)A_sf | (uintptr_t)B_sf) & 3) == 0,
               "A/B must be 16-byte aligned and the scale tensors 4-byte aligned");
  AC4K_REQUIRE(M < (1ll << 27) && N < (1ll << 27) && T < (1ll << 31) - 16 && K < (1ll << 22) && E <= 65535, "problem too large");
  AC4K_REQUIRE(ceil_div(N, R16_ROWS) * (64 * R16_WAVES) < (1ll << 32), "problem too large");
  GroupedArgs a{D, static_cast<const uint8_t *>(A), static_cast<const uint32_t *>(A_sf), A_gs, rows, static_cast<const uint8_t *>(B),
                static_cast<const uint32_t *>(B_sf), B_gs, B_gs_stride, bias, offsets, T, align_up(T, 16), M, N, align_up(N, 16), K, E};
  hipStream_t st = (hipStream_t)stream;
  int rc;
  switch (d_dtype) {
    case AC4K_DTYPE_BF16: rc = grouped_bias<AC4K_DTYPE_BF16>(a, bias_dtype, st); break;
    case AC4K_DTYPE_FP16: rc = grouped_bias<AC4K_DTYPE_FP16>(a, bias_dtype, st); break;
    case AC4K_DTYPE_FP32: rc = grouped_bias<AC4K_DTYPE_FP32>(a, bias_dtype, st); break;
    default: return set_error("d must be bfloat16, half or float (dtype tag %d)", d_dtype);
  }
  if (rc) return rc;
  return check_launch("ac4k_linear_grouped_nvfp4");
}

// NVFP4 dot-scale linear for gfx950:  D = (A . B^T) * (gsA*gsB) + bias  (lib/cuda/sm120/linear_nvfp4.cu:337-751).  The kernels and their plans are in
// linear_kernels.h; here are the entry points of the C ABI and the instantiations for each type of output and bias.
#include "linear_kernels.h"

namespace ac4k {

template <int D_DT>
static int dispatch_skinny_bias(const SkinnyArgs &a, const SkinnyPlan &p, int bias_dtype, hipStream_t st) {
  if (!a.bias) return launch_skinny<D_DT, BIAS_NONE>(a, p, st);
  switch (bias_dtype) {
    case AC4K_DTYPE_BF16: return launch_skinny<D_DT, AC4K_DTYPE_BF16>(a, p, st);
    case AC4K_DTYPE_FP16: return launch_skinny<D_DT, AC4K_DTYPE_FP16>(a, p, st);
    case AC4K_DTYPE_FP32: return launch_skinny<D_DT, AC4K_DTYPE_FP32>(a, p, st);
  }
  return set_error("bias must be bfloat16, half or float (dtype tag %d)", bias_dtype);
}

static int dispatch_skinny(const SkinnyArgs &a, const SkinnyPlan &p, int d_dtype, int bias_dtype, hipStream_t st) {
  switch (d_dtype) {
    case AC4K_DTYPE_BF16: return dispatch_skinny_bias<AC4K_DTYPE_BF16>(a, p, bias_dtype, st);
    case AC4K_DTYPE_FP16: return dispatch_skinny_bias<AC4K_DTYPE_FP16>(a, p, bias_dtype, st);
    case AC4K_DTYPE_FP32: return dispatch_skinny_bias<AC4K_DTYPE_FP32>(a, p, bias_dtype, st);
  }
  return set_error("d must be bfloat16, half or float (dtype tag %d)", d_dtype);
}

template <int D_DT>
static int dispatch_bias(const LinearArgs &a, int bias_dtype, hipStream_t st) {
  if (!a.bias) return launch_linear<D_DT, BIAS_NONE>(a, st);
  switch (bias_dtype) {
    case AC4K_DTYPE_BF16: return launch_linear<D_DT, AC4K_DTYPE_BF16>(a, st);
    case AC4K_DTYPE_FP16: return launch_linear<D_DT, AC4K_DTYPE_FP16>(a, st);
    case AC4K_DTYPE_FP32: return launch_linear<D_DT, AC4K_DTYPE_FP32>(a, st);
  }
  return set_error("bias must be bfloat16, half or float (dtype tag %d)", bias_dtype);
}

}  // namespace ac4k

using namespace ac4k;

extern "C" __attribute__((visibility("default"))) int ac4k_linear_nvfp4(void *D, int d_dtype, const void *A, const void *A_sf, const float *A_gs,
                                 const void *B, const void *B_sf, const float *B_gs, const void *bias,
                                 int bias_dtype, int64_t M, int64_t N, int64_t K, ac4k_stream_t stream) {
  AC4K_REQUIRE(D && A && A_sf && A_gs && B && B_sf && B_gs, "null pointer argument");
  AC4K_REQUIRE(M >= 1 && N >= 1 && K >= 1, "M, N, K must be positive (M=%lld N=%lld K=%lld)", (long long)M,
               (long long)N, (long long)K);
  AC4K_REQUIRE(K % 16 == 0, "A size(1)*2 must be multiple of 16 but see %lld", (long long)K);
  AC4K_REQUIRE(((uintptr_t)A & 7) == 0 && ((uintptr_t)B & 7) == 0 && ((uintptr_t)A_sf & 3) == 0 &&
                   ((uintptr_t)B_sf & 3) == 0,
               "A/B must be 8-byte aligned and the scale tensors 4-byte aligned");
  AC4K_REQUIRE(ceil_div(M, T_BM) * ceil_div(N, T_BN) < (1ll << 31), "problem too large");
  LinearArgs a{D,
               static_cast<const uint8_t *>(A),
               static_cast<const uint8_t *>(B),
               static_cast<const uint32_t *>(A_sf),
               static_cast<const uint32_t *>(B_sf),
               A_gs,
               B_gs,
               bias,
               M,
               N,
               K,
               align_up(M, 16),
               align_up(N, 16)};
  hipStream_t st = (hipStream_t)stream;
  int rc;
  switch (d_dtype) {
    case AC4K_DTYPE_BF16: rc = dispatch_bias<AC4K_DTYPE_BF16>(a, bias_dtype, st); break;
    case AC4K_DTYPE_FP16: rc = dispatch_bias<AC4K_DTYPE_FP16>(a, bias_dtype, st); break;
    case AC4K_DTYPE_FP32: rc = dispatch_bias<AC4K_DTYPE_FP32>(a, bias_dtype, st); break;
    default: return set_error("d must be bfloat16, half or float (dtype tag %d)", d_dtype);
  }
  if (rc) return rc;
  return check_launch("ac4k_linear_nvfp4");
}

namespace ac4k {

template <int D_DT>
static int dispatch_mid_bias(const LinearArgs &a, const MidPlan &p, float *partial, int64_t partial_bytes, int bias_dtype,
                             hipStream_t st) {
  if (!a.bias) return launch_mid<D_DT, BIAS_NONE>(a, p, partial, partial_bytes, st);
  switch (bias_dtype) {
    case AC4K_DTYPE_BF16: return launch_mid<D_DT, AC4K_DTYPE_BF16>(a, p, partial, partial_bytes, st);
    case AC4K_DTYPE_FP16: return launch_mid<D_DT, AC4K_DTYPE_FP16>(a, p, partial, partial_bytes, st);
    case AC4K_DTYPE_FP32: return launch_mid<D_DT, AC4K_DTYPE_FP32>(a, p, partial, partial_bytes, st);
  }
  return set_error("bias must be bfloat16, half or float (dtype tag %d)", bias_dtype);
}

static int dispatch_mid(const LinearArgs &a, const MidPlan &p, float *partial, int64_t partial_bytes, int d_dtype,
                        int bias_dtype, hipStream_t st) {
  switch (d_dtype) {
    case AC4K_DTYPE_BF16: return dispatch_mid_bias<AC4K_DTYPE_BF16>(a, p, partial, partial_bytes, bias_dtype, st);
    case AC4K_DTYPE_FP16: return dispatch_mid_bias<AC4K_DTYPE_FP16>(a, p, partial, partial_bytes, bias_dtype, st);
    case AC4K_DTYPE_FP32: return dispatch_mid_bias<AC4K_DTYPE_FP32>(a, p, partial, partial_bytes, bias_dtype, st);
  }
  return set_error("d must be bfloat16, half or float (dtype tag %d)", d_dtype);
}

// one K range of the tile kernel with a given plan (the entry point of the weight image)
template <int D_DT>
static int dispatch_prepacked_bias(const LinearArgs &a, const TilePlan &p, int bias_dtype, hipStream_t st) {
  const SplitK one{nullptr, 1};
  if (!a.bias) return launch_tile_plan<D_DT, BIAS_NONE>(a, p, one, st);
  switch (bias_dtype) {
    case AC4K_DTYPE_BF16: return launch_tile_plan<D_DT, AC4K_DTYPE_BF16>(a, p, one, st);
    case AC4K_DTYPE_FP16: return launch_tile_plan<D_DT, AC4K_DTYPE_FP16>(a, p, one, st);
    case AC4K_DTYPE_FP32: return launch_tile_plan<D_DT, AC4K_DTYPE_FP32>(a, p, one, st);
  }
  return set_error("bias must be bfloat16, half or float (dtype tag %d)", bias_dtype);
}

// shared tail of the two decode-sized entry points: packed activation in, partial sums in the workspace
static int run_skinny(void *D, int d_dtype, const void *Aq, const void *A_sf, const float *A_gs, const void *B,
                      const void *B_sf, const float *B_gs, const void *bias, int bias_dtype, int64_t M, int64_t N,
                      int64_t K, const SkinnyPlan &p, void *workspace, hipStream_t st) {
  SkinnyArgs a{D,
               static_cast<const uint8_t *>(Aq),
               static_cast<const uint8_t *>(A_sf),
               align_up(M, 16),
               static_cast<const uint8_t *>(B),
               static_cast<const uint32_t *>(B_sf),
               A_gs,
               B_gs,
               bias,
               static_cast<float *>(workspace),
               M,
               N,
               K,
               align_up(N, 16),
               p.ks_len,
               p.split_k};
  return dispatch_skinny(a, p, d_dtype, bias_dtype, st);
}

static int check_skinny(const SkinnyPlan &p, bool ok, const void *B, void *workspace, int64_t workspace_bytes) {
  AC4K_REQUIRE(ok, "no workspace-assisted path for this shape: decode-sized shapes need 1 <= M <= 32 and K a multiple of 256");
  AC4K_REQUIRE(((uintptr_t)B & 15) == 0, "weights must be 16-byte aligned");
  if (p.partial_bytes > 0) {  // one K range per tile needs no scratch
    AC4K_REQUIRE(workspace && ((uintptr_t)workspace & 255) == 0, "workspace must be 256-byte aligned");
    AC4K_REQUIRE(workspace_bytes >= p.partial_bytes, "workspace too small: %lld bytes needed", (long long)p.partial_bytes);
  }
  return 0;
}

}  // namespace ac4k

extern "C" __attribute__((visibility("default"))) int64_t ac4k_linear_nvfp4_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  SkinnyPlan p;
  if (skinny_plan(M, N, K, p)) return p.partial_bytes;
  MidPlan mp;
  if (mid_plan(M, N, K, mp)) return mp.bytes;
  return 0;
}

extern "C" __attribute__((visibility("default"))) int64_t ac4k_linear_nvfp4_scratch_bytes(int64_t M, int64_t N, int64_t K) {
  SkinnyPlan p;
  if (skinny_plan(M, N, K, p)) return p.rows16 ? 0 : p.partial_bytes;
  MidPlan mp;
  if (mid_plan(M, N, K, mp)) return mp.has_ksplit || mp.tp.splits > 1 ? mp.bytes : 0;
  return 0;
}

namespace ac4k {

// K that the `skinny` entry points take: whole stages of the kernels they began with
static bool skinny_entry_k(int64_t M, int64_t K) { return K % (M > 32 ? P_BK : SK_STEP) == 0; }

}  // namespace ac4k

extern "C" __attribute__((visibility("default"))) int ac4k_debug_linear_decode_kernel(int64_t M, int64_t N, int64_t K, int *fused_launches) {
  SkinnyPlan p;
  const bool ok = skinny_plan(M, N, K, p);
  if (fused_launches) *fused_launches = !ok || !skinny_entry_k(M, K) ? 0 : p.fused ? 1 : p.rows16 || p.split_k == 1 ? 2 : 3;
  return !ok ? 0 : p.lds_x ? DECODE_ROWS16_LDS : p.rows16 ? DECODE_ROWS16 : p.kind;
}

extern "C" __attribute__((visibility("default"))) int64_t ac4k_linear_nvfp4_skinny_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  return skinny_entry_k(M, K) ? ac4k_linear_nvfp4_workspace_bytes(M, N, K) : 0;
}

namespace ac4k {

// body of the two workspace-assisted entry points (caller's workspace / the library's static array)
static int linear_skinny_impl(void *D, int d_dtype, const void *A, const void *A_sf, const float *A_gs, const void *B,
                              const void *B_sf, const float *B_gs, const void *bias, int bias_dtype, int64_t M,
                              int64_t N, int64_t K, void *workspace, int64_t workspace_bytes, hipStream_t st,
                              const char *what) {
  AC4K_REQUIRE(D && A && A_sf && A_gs && B && B_sf && B_gs, "null pointer argument");
  AC4K_REQUIRE(M >= 1 && N >= 1 && K >= 1, "M, N, K must be positive (M=%lld N=%lld K=%lld)", (long long)M,
               (long long)N, (long long)K);
  MidPlan mp;
  if (M > 32 && skinny_entry_k(M, K) && mid_plan(M, N, K, mp)) {  // few tiles, long K: split-K
    AC4K_REQUIRE((((uintptr_t)A | (uintptr_t)B) & 15) == 0 && (((uintptr_t)A_sf | (uintptr_t)B_sf) & 3) == 0,
                 "A and B must be 16-byte aligned and the scale tensors 4-byte aligned");
    if (mp.bytes > 0) {  // one K range per tile needs no scratch
      AC4K_REQUIRE(workspace && ((uintptr_t)workspace & 255) == 0, "workspace must be 256-byte aligned");
      AC4K_REQUIRE(workspace_bytes >= mp.bytes, "workspace too small: %lld bytes needed", (long long)mp.bytes);
    }
    LinearArgs la{D, static_cast<const uint8_t *>(A), static_cast<const uint8_t *>(B),
                  static_cast<const uint32_t *>(A_sf), static_cast<const uint32_t *>(B_sf), A_gs, B_gs, bias,
                  M, N, K, align_up(M, 16), align_up(N, 16)};
    if (int rc = dispatch_mid(la, mp, static_cast<float *>(workspace), workspace ? workspace_bytes : 0, d_dtype, bias_dtype, st))
      return rc;
    return check_launch(what);
  }
  SkinnyPlan p;
  const bool ok = skinny_entry_k(M, K) && skinny_plan(M, N, K, p);
  if (int rc = check_skinny(p, ok, B, workspace, workspace_bytes)) return rc;
  AC4K_REQUIRE(((uintptr_t)A & 15) == 0, "A must be 16-byte aligned");
  if (int rc = run_skinny(D, d_dtype, A, A_sf, A_gs, B, B_sf, B_gs, bias, bias_dtype, M, N, K, p, workspace, st))
    return rc;
  return check_launch(what);
}

// ---------------------------------------------------------------------------
// Scratch of the entry point that allocates nothing: one array per GPU, held until the process ends.
// In host code the array's name is only a handle: its device address comes from hipGetSymbolAddress,
// once per device with that device current, and that pointer is what the kernels are given.
// ---------------------------------------------------------------------------
constexpr int64_t STATIC_SCRATCH_BYTES = AC4K_STATIC_SCRATCH_BYTES;
static __device__ __align__(256) unsigned char scratch[STATIC_SCRATCH_BYTES];

static int static_scratch(void **ptr_out) {
  constexpr int MAX_DEV = 64;
  static void *ptrs[MAX_DEV] = {};
  static std::mutex mu;
  int dev = -1;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return set_error("hipGetDevice: %s", hipGetErrorString(e));
  AC4K_REQUIRE(dev >= 0 && dev < MAX_DEV, "device index %d out of range", dev);
  std::lock_guard<std::mutex> lock(mu);
  if (!ptrs[dev]) {
    void *p = nullptr;
    e = hipGetSymbolAddress(&p, HIP_SYMBOL(scratch));
    if (e != hipSuccess || !p) return set_error("hipGetSymbolAddress(scratch): %s", hipGetErrorString(e));
    ptrs[dev] = p;
  }
  *ptr_out = ptrs[dev];
  return 0;
}

}  // namespace ac4k

extern "C" __attribute__((visibility("default"))) int ac4k_linear_nvfp4_skinny(void *D, int d_dtype, const void *A, const void *A_sf, const float *A_gs,
                                        const void *B, const void *B_sf, const float *B_gs, const void *bias,
                                        int bias_dtype, int64_t M, int64_t N, int64_t K, void *workspace,
                                        int64_t workspace_bytes, ac4k_stream_t stream) {
  return linear_skinny_impl(D, d_dtype, A, A_sf, A_gs, B, B_sf, B_gs, bias, bias_dtype, M, N, K, workspace,
                            workspace_bytes, (hipStream_t)stream, "ac4k_linear_nvfp4_skinny");
}

extern "C" __attribute__((visibility("default"))) int ac4k_linear_nvfp4_workspace(void *D, int d_dtype, const void *A, const void *A_sf, const float *A_gs,
                                        const void *B, const void *B_sf, const float *B_gs, const void *bias,
                                        int bias_dtype, int64_t M, int64_t N, int64_t K, void *workspace,
                                        int64_t workspace_bytes, ac4k_stream_t stream) {
  // what the kernels that split K do not take runs without scratch, for every K alike: shapes that need none, operands that
  // are not aligned for them, and everything that ac4k_linear_nvfp4 refuses with its own message
  SkinnyPlan p;
  MidPlan mp;
  const bool aligned = D && A && A_sf && A_gs && B && B_sf && B_gs && (((uintptr_t)A | (uintptr_t)B) & 15) == 0 &&
                       (((uintptr_t)A_sf | (uintptr_t)B_sf) & 3) == 0;
  const bool skinny = aligned && skinny_plan(M, N, K, p);
  const bool mid = aligned && !skinny && mid_plan(M, N, K, mp);
  const int64_t need = skinny ? p.partial_bytes : mid ? mp.bytes : 0;
  if (need == 0) return ac4k_linear_nvfp4(D, d_dtype, A, A_sf, A_gs, B, B_sf, B_gs, bias, bias_dtype, M, N, K, stream);
  AC4K_REQUIRE(workspace && ((uintptr_t)workspace & 255) == 0, "workspace must be 256-byte aligned");
  AC4K_REQUIRE(workspace_bytes >= need, "workspace too small: %lld bytes needed", (long long)need);
  int rc;
  if (skinny) {
    rc = run_skinny(D, d_dtype, A, A_sf, A_gs, B, B_sf, B_gs, bias, bias_dtype, M, N, K, p, workspace, (hipStream_t)stream);
  } else {
    LinearArgs la{D, static_cast<const uint8_t *>(A), static_cast<const uint8_t *>(B),
                  static_cast<const uint32_t *>(A_sf), static_cast<const uint32_t *>(B_sf), A_gs, B_gs, bias,
                  M, N, K, align_up(M, 16), align_up(N, 16)};
    rc = dispatch_mid(la, mp, static_cast<float *>(workspace), workspace_bytes, d_dtype, bias_dtype, (hipStream_t)stream);
  }
  if (rc) return rc;
  return check_launch("ac4k_linear_nvfp4_workspace");
}

extern "C" __attribute__((visibility("default"))) int ac4k_linear_nvfp4_skinny_static(void *D, int d_dtype, const void *A, const void *A_sf,
                                               const float *A_gs, const void *B, const void *B_sf,
                                               const float *B_gs, const void *bias, int bias_dtype, int64_t M,
                                               int64_t N, int64_t K, ac4k_stream_t stream) {
  AC4K_REQUIRE(M >= 1 && N >= 1 && K >= 1, "M, N, K must be positive (M=%lld N=%lld K=%lld)", (long long)M,
               (long long)N, (long long)K);
  const int64_t need = ac4k_linear_nvfp4_skinny_workspace_bytes(M, N, K);
  AC4K_REQUIRE(need <= STATIC_SCRATCH_BYTES,
               "shape needs %lld bytes of scratch, the static scratch holds %lld: use ac4k_linear_nvfp4_skinny with a "
               "workspace of the caller",
               (long long)need, (long long)STATIC_SCRATCH_BYTES);
  void *ws = nullptr;
  if (int rc = static_scratch(&ws)) return rc;
  // the partial sums are written before they are read: nothing in the array has to start at zero
  return linear_skinny_impl(D, d_dtype, A, A_sf, A_gs, B, B_sf, B_gs, bias, bias_dtype, M, N, K, ws,
                            STATIC_SCRATCH_BYTES, (hipStream_t)stream, "ac4k_linear_nvfp4_skinny_static");
}

namespace ac4k {

// One workgroup writes one block of the weight image: 128 rows x 64 packed bytes (rows past N zero),
// piece p of row r at position p ^ ((r >> 1) & 3), then the scale dwords [2 chunks][128 rows].
__global__ __launch_bounds__(256) void prepack_weight_kernel(uint8_t *image, const uint8_t *B, const uint32_t *B_sf,
                                                             int64_t N, int64_t K, int64_t Np) {
  const int64_t kt = blockIdx.x, band = blockIdx.y;
  uint8_t *blk = image + (band * gridDim.x + kt) * W_BLOCK_BYTES;
  const int t = threadIdx.x;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = (t + i * 256) >> 2, pc = t & 3;
    const int64_t row = band * W_BLOCK_ROWS + r;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (row < N) v = *reinterpret_cast<const uint4 *>(B + row * (K >> 1) + kt * (W_BLOCK_K / 2) + pc * 16);
    *reinterpret_cast<uint4 *>(blk + r * (W_BLOCK_K / 2) + ((pc ^ ((r >> 1) & 3)) * 16)) = v;
  }
  const int c = t >> 7, r = t & 127;
  const int64_t row = band * W_BLOCK_ROWS + r;
  reinterpret_cast<uint32_t *>(blk + W_BLOCK_DATA)[c * W_BLOCK_ROWS + r] = row < N ? B_sf[(kt * 2 + c) * Np + row] : 0u;
}

static int64_t weight_image_bytes(int64_t N, int64_t K) {
  if (N < 1 || K < W_BLOCK_K || K % W_BLOCK_K != 0) return 0;
  return ceil_div(N, W_BLOCK_ROWS) * (K / W_BLOCK_K) * W_BLOCK_BYTES;
}

// How a linear on a weight image runs: the LDS-ring kernel or 16-row workgroups for decode-sized M (K >= 256), the K-split-waves
// kernel for 32 < M <= 128, the tile kernel otherwise, split along K when the workspace entry point of the plain
// layout would split too.
struct PrepackedPlan {
  bool ring, mid;
  SkinnyPlan sp;
  KsplitPlan kp;
  TilePlan tp;
  int64_t partial_bytes;
};
// 16-row workgroups on an image, where a step of a wave's rows is one run of a kilobyte, against its ring kernel, by these estimates (us,
// weights from HBM, fitted to 160 shapes of N = 256 to 28672, K = 256 to 16384 and M = 1 to 32).  Ring / 16 rows as measured:
// M = 1, 4096 x 4096 10.5 / 4.3, 28672 x 8192 32.3 / 28.1; M = 8, 28672 x 8192 32.5 / 31.2; M = 16, 4096 x 14336 18.1 / 10.1, 14336 x 4096 16.1 / 10.9,
// 28672 x 8192 33.0 / 35.0, 27264 x 256 5.3 / 4.7; M = 20, 12288 x 12288 39.5 / 30.6, 27264 x 256 5.4 / 6.9, 28672 x 4096 21.0 / 24.1; M = 32,
// 4096 x 14336 17.8 / 14.8, 2688 x 14208 14.8 / 11.8, 14336 x 14336 33.5 / 47.6, 256 x 14336 10.4 / 12.4.
// Two tiles of activation rows (M > 16): two workgroups on a CU have their steps nearly one after the other (24 x 4096 x 8192 8.8 us, 4112 rows 13.3), and
// the estimates have to differ by more than they err: of 423 shapes of M = 17 to 32 383 take 16 rows, four of these 3 to
// 5 % slower than the ring (394 and 13 by 2 to 18 % without the two: 31 x 320 x 14080 10.7 / 12.7, 29 x 22656 x 512 6.7 / 7.7).
static bool rows16_faster_image(int64_t M, int64_t N, int64_t K, const SkinnyPlan &p) {
  const double m = (double)M, cus = (double)decode_cu_count(), million = 1e-6 * (double)N * (double)K;
  const double steps = (double)ceil_div(ceil_div(K, R16_STEP), R16_WAVES), wgs = (double)ceil_div(N, R16_ROWS) / (2.0 * cus);
  const double last = wgs > 1.0 && wgs < 2.0 ? sqrt(2.0 / wgs) : 1.0;  // a second round that is not full
  const double rows16 = M <= 16 ? fmax(0.35 * wgs + (0.10 + 0.0022 * m) * million, (0.37 + 0.003 * m) * steps)
                                : fmax(last * (wgs + (0.126 + 0.0016 * m) * million), (wgs > 0.5 ? 1.8 : 1.0) * (0.5 + 0.006 * m) * steps);
  const double rounds = ceil((double)(p.groups * p.split_k) / cus), stages = (double)ceil_div(ceil_div(K, ST_BK), p.split_k);
  const double ring = 4.2 + 0.03 * m + 0.8 * stages + 0.3 * fmin(stages, 8.0);
  return (M <= 16 ? 1.0 : 1.1) * (2.5 + rows16) < rounds * ring + (p.split_k > 1 ? 4.0 : 0.0);
}

static bool prepacked_plan(int64_t M, int64_t N, int64_t K, PrepackedPlan &p) {
  const int64_t bytes = weight_image_bytes(N, K);
  if (M < 1 || bytes == 0 || bytes >= (1ll << 32) || (K >> 1) * 256 >= (1ll << 31) || N >= (1ll << 27)) return false;
  p.ring = M <= 32 && K >= ST_BK;
  p.mid = !p.ring && ksplit_shape(M, N, K);
  if (p.ring) {
    plan_lds_ring(M, N, K, p.sp);
    p.sp.rows16 = !forced_decode_kernel() && rows16_faster_image(M, N, K, p.sp);
    p.sp.fused = p.sp.lds_x = false;
    p.partial_bytes = p.sp.rows16 ? 0 : p.sp.partial_bytes;
  } else if (p.mid) {
    p.kp = ksplit_plan(M, N, K, true);
    p.partial_bytes = p.kp.partial_bytes;
  } else {
    p.partial_bytes = tile_scratch_bytes(M, N, K);
    p.tp = tile_plan(M, N, K, p.partial_bytes);
  }
  return true;
}

}  // namespace ac4k

extern "C" __attribute__((visibility("default"))) int64_t ac4k_prepack_weight_nvfp4_bytes(int64_t N, int64_t K) {
  const int64_t bytes = weight_image_bytes(N, K);
  return bytes < (1ll << 32) ? bytes : 0;
}

extern "C" __attribute__((visibility("default"))) int ac4k_prepack_weight_nvfp4(void *image, const void *B, const void *B_sf, int64_t N, int64_t K,
                                                                                ac4k_stream_t stream) {
  AC4K_REQUIRE(image && B && B_sf, "null pointer argument");
  const int64_t bytes = ac4k_prepack_weight_nvfp4_bytes(N, K);
  AC4K_REQUIRE(bytes > 0, "no weight image for N = %lld, K = %lld: K must be a multiple of 128 and the image smaller than 4 GiB",
               (long long)N, (long long)K);
  AC4K_REQUIRE((((uintptr_t)image | (uintptr_t)B) & 15) == 0 && ((uintptr_t)B_sf & 3) == 0,
               "image and B must be 16-byte aligned, B_sf 4-byte aligned");
  hipLaunchKernelGGL(prepack_weight_kernel, dim3((unsigned)(K / W_BLOCK_K), (unsigned)ceil_div(N, W_BLOCK_ROWS)), dim3(256), 0,
                     (hipStream_t)stream, static_cast<uint8_t *>(image), static_cast<const uint8_t *>(B),
                     static_cast<const uint32_t *>(B_sf), N, K, align_up(N, 16));
  return check_launch("ac4k_prepack_weight_nvfp4");
}

extern "C" __attribute__((visibility("default"))) int64_t ac4k_linear_nvfp4_prepacked_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  PrepackedPlan p;
  return prepacked_plan(M, N, K, p) ? p.partial_bytes : 0;
}

extern "C" __attribute__((visibility("default"))) int ac4k_debug_linear_prepacked_decode_kernel(int64_t M, int64_t N, int64_t K) {
  PrepackedPlan p;
  if (!prepacked_plan(M, N, K, p) || !p.ring) return 0;
  return p.sp.rows16 ? DECODE_ROWS16 : DECODE_LDS_RING;
}

extern "C" __attribute__((visibility("default"))) int ac4k_linear_nvfp4_prepacked(void *D, int d_dtype, const void *A, const void *A_sf, const float *A_gs,
                                                                                  const void *W_image, const float *B_gs, const void *bias,
                                                                                  int bias_dtype, int64_t M, int64_t N, int64_t K, void *workspace,
                                                                                  int64_t workspace_bytes, ac4k_stream_t stream) {
  AC4K_REQUIRE(D && A && A_sf && A_gs && W_image && B_gs, "null pointer argument");
  AC4K_REQUIRE(M >= 1 && N >= 1, "M and N must be positive (M = %lld, N = %lld)", (long long)M, (long long)N);
  PrepackedPlan p;
  AC4K_REQUIRE(prepacked_plan(M, N, K, p), "no weight image for N = %lld, K = %lld (ac4k_prepack_weight_nvfp4_bytes returns 0)",
               (long long)N, (long long)K);
  AC4K_REQUIRE((((uintptr_t)A | (uintptr_t)W_image) & 15) == 0 && ((uintptr_t)A_sf & 3) == 0,
               "A and the weight image must be 16-byte aligned, A_sf 4-byte aligned");
  AC4K_REQUIRE(ceil_div(M, 128) * ceil_div(N, 64) < (1ll << 31), "problem too large");
  if (p.partial_bytes > 0) {
    AC4K_REQUIRE(workspace && ((uintptr_t)workspace & 255) == 0, "workspace must be 256-byte aligned");
    AC4K_REQUIRE(workspace_bytes >= p.partial_bytes, "workspace too small: %lld bytes needed", (long long)p.partial_bytes);
  }
  hipStream_t st = (hipStream_t)stream;
  if (p.ring) {
    SkinnyArgs a{D, static_cast<const uint8_t *>(A), static_cast<const uint8_t *>(A_sf), align_up(M, 16),
                 static_cast<const uint8_t *>(W_image), nullptr, A_gs, B_gs, bias, static_cast<float *>(workspace),
                 M, N, K, align_up(N, 16), 0, p.sp.split_k, 1};
    if (int rc = dispatch_skinny(a, p.sp, d_dtype, bias_dtype, st)) return rc;
    return check_launch("ac4k_linear_nvfp4_prepacked");
  }
  LinearArgs la{D, static_cast<const uint8_t *>(A), static_cast<const uint8_t *>(W_image),
                static_cast<const uint32_t *>(A_sf), nullptr, A_gs, B_gs, bias,
                M, N, K, align_up(M, 16), align_up(N, 16), 1};
  int rc;
  if (p.mid || p.tp.splits > 1) {
    rc = dispatch_mid(la, MidPlan{p.mid, p.mid ? p.kp : KsplitPlan{0, 0, 1, 0}, p.tp, p.partial_bytes},
                      static_cast<float *>(workspace), workspace_bytes, d_dtype, bias_dtype, st);
  } else {
    switch (d_dtype) {
      case AC4K_DTYPE_BF16: rc = dispatch_prepacked_bias<AC4K_DTYPE_BF16>(la, p.tp, bias_dtype, st); break;
      case AC4K_DTYPE_FP16: rc = dispatch_prepacked_bias<AC4K_DTYPE_FP16>(la, p.tp, bias_dtype, st); break;
      case AC4K_DTYPE_FP32: rc = dispatch_prepacked_bias<AC4K_DTYPE_FP32>(la, p.tp, bias_dtype, st); break;
      default: return set_error("d must be bfloat16, half or float (dtype tag %d)", d_dtype);
    }
  }
  if (rc) return rc;
  return check_launch("ac4k_linear_nvfp4_prepacked");
}

namespace ac4k {

static bool overlap(const void *a, int64_t a_bytes, const void *b, int64_t b_bytes) {
  return (uintptr_t)a < (uintptr_t)b + (uintptr_t)b_bytes && (uintptr_t)b < (uintptr_t)a + (uintptr_t)a_bytes;
}

}  // namespace ac4k

extern "C" __attribute__((visibility("default"))) int ac4k_linear_nvfp4_fused_bf16(void *D, int d_dtype, const void *X, void *X_q, void *X_sf,
                                            float *X_gs, const void *B, const void *B_sf, const float *B_gs,
                                            const void *bias, int bias_dtype, int64_t M, int64_t N, int64_t K,
                                            void *workspace, int64_t workspace_bytes, ac4k_stream_t stream) {
  AC4K_REQUIRE(D && X && X_q && X_sf && X_gs && B && B_sf && B_gs, "null pointer argument");
  AC4K_REQUIRE(M >= 1 && M <= 32, "the fused skinny linear takes 1 <= M <= 32 (got %lld)", (long long)M);
  AC4K_REQUIRE(N >= 1 && K >= 1, "N and K must be positive (N=%lld K=%lld)", (long long)N, (long long)K);
  SkinnyPlan p;
  const bool ok = skinny_entry_k(M, K) && skinny_plan(M, N, K, p);
  if (int rc = check_skinny(p, ok, B, workspace, workspace_bytes)) return rc;
  hipStream_t st = (hipStream_t)stream;
  AC4K_REQUIRE(((uintptr_t)X & 15) == 0, "activation must be 16-byte aligned");
  // (one launch reads X to its end while it stores: outputs over X, as in a linear in place, need the order of two)
  if (p.fused && (((uintptr_t)X_q | (uintptr_t)B) & 15) == 0 && (((uintptr_t)X_sf | (uintptr_t)B_sf) & 3) == 0 &&
      !overlap(X, M * K * 2, D, M * N * (d_dtype == AC4K_DTYPE_FP32 ? 4 : 2)) && !overlap(X, M * K * 2, X_q, M * K / 2) &&
      !overlap(X, M * K * 2, X_sf, K / 64 * align_up(M, 16) * 4) && !overlap(X, M * K * 2, X_gs, 4)) {
    const FusedArgs a{D, static_cast<const uint16_t *>(X), static_cast<uint8_t *>(X_q), static_cast<uint8_t *>(X_sf), X_gs,
                      static_cast<const uint8_t *>(B), static_cast<const uint32_t *>(B_sf), B_gs, bias, M, N, K, align_up(M, 16), align_up(N, 16)};
    if (int rc = launch_fused_rows16(a, d_dtype, bias_dtype, st)) return rc;
    return check_launch("ac4k_linear_nvfp4_fused_bf16");
  }
  if (int rc = ac4k_quantize_nvfp4_bf16(X_q, X_sf, X_gs, X, 1, 1, M, K, 0, 0, K, 1, 0, 2688.0f, stream)) return rc;
  if (int rc = run_skinny(D, d_dtype, X_q, X_sf, X_gs, B, B_sf, B_gs, bias, bias_dtype, M, N, K, p, workspace,
                          st))
    return rc;
  return check_launch("ac4k_linear_nvfp4_fused_bf16");
}

extern "C" __attribute__((visibility("default"))) int ac4k_set_linear_tuning(int mi, int nj, int splits, int skinny_ks,
                                                                          int decode_kernel) {
  // every argument is checked before any is stored: a rejected call changes nothing
  AC4K_REQUIRE(decode_kernel >= 0 && decode_kernel <= 3,
               "decode_kernel must be 0 (by shape), 1 (register kernel), 2 (LDS-ring kernel) or 3 (LDS-ring kernel with "
               "64-row tiles) (got %d)", decode_kernel);
  const bool no_plan = mi == 0 && nj == 0 && splits == 0;
  AC4K_REQUIRE(no_plan || (mi >= 2 && mi <= 4 && (nj == 1 || nj == 2 || nj == 4) && !(mi != 2 && nj == 1) && splits >= 1 &&
                           splits <= 0xffff),
               "tile plan must be mi in {2,3,4}, nj in {1,2,4} (1 with mi = 2), 1 <= splits (got %d,%d,%d)", mi, nj, splits);
  AC4K_REQUIRE(skinny_ks >= 0 && skinny_ks % 256 == 0, "skinny_ks must be 0 (automatic) or a multiple of 256 (got %d)",
               skinny_ks);
  ac4k::g_forced_decode_kernel.store(decode_kernel);
  ac4k::g_forced_tile_plan.store(no_plan ? 0u : (uint32_t)mi | ((uint32_t)nj << 8) | ((uint32_t)splits << 16));
  ac4k::g_forced_skinny_ks.store(skinny_ks);
  return 0;
}

#ifdef AC4K_LINEAR_TIMELINE
// Timeline build only: copies the per-workgroup stamps of the last tile / K-split-waves launch to host
// memory ([8192][6]: 100 MHz ticks at kernel entry, loop entry, loop exit, kernel exit; shader cycles in
// the loop; XCC and hardware id for the tile kernel).  Synchronises the device.
extern "C" __attribute__((visibility("default"))) int ac4k_debug_linear_timeline(uint64_t *host_out) {
  hipError_t e = hipDeviceSynchronize();
  if (e == hipSuccess) e = hipMemcpyFromSymbol(host_out, HIP_SYMBOL(ac4k::g_linear_timeline), sizeof(uint64_t) * 8192 * 6);
  return e == hipSuccess ? 0 : ac4k::set_error("ac4k_debug_linear_timeline: %s", hipGetErrorString(e));
}
#endif

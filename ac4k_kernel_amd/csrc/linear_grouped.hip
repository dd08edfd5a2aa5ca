// Linears grouped by expert on NVFP4 operands: row i of the output is row rows[i] of x (row i without `rows`) times the weight of the expert
// whose range of offsets holds i,
//
//   D[i] = (x[rows[i]] . W[e]^T) * (gs_x * gs_W[e]) + bias[e],   offsets[e] <= i < offsets[e + 1].
//
// The sizes of the groups are on the GPU and nothing waits for them: launches are made for the largest number of tiles that the row and
// expert counts allow, and workgroups without a tile end at once.  Offsets are taken as clamped to [0, rows] and rising, row indexes as
// clamped to x: a wrong table gives wrong rows, not an access outside of the operands.  Output rows that no group holds stay as they are, or
// become zero where the caller's output is new memory.
//
// Few rows an expert are bound by the weights' bytes, many by the matrix cores.  128 rows on 64 experts of 2048 x 4096 61-68 us (55 of bytes at the rate of a
// copy; 440 tiles on 256 CUs leave some a tile less), 16384 rows on 8 experts of 14336 x 4096 1399-1540 us by the card, 1.25-1.38 PFLOP/s, matrix cores busy for
// 82 % of the time, 4004 rows in uneven groups on 32 experts of 1003 x 2880 42-44 us (45-46 under the profiler) where the products need 19: half-filled tiles and
// prologues, matrix cores busy for 39 %.
#include <math.h>

#include "linear_tile.h"

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
  bool whole;              // rows of D in front of the first range and behind the last one become zero
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

// The rows of D that no range holds, in front of `first` and from `last` on, by the workgroups of the launch along x in equal shares, before their own work.  (A clearing launch in front would write all of D a second time: half a gigabyte of the 1.4 ms of 16384 x 14336.)
template <int D_DT>
__device__ __forceinline__ void zero_other_rows(const GroupedArgs &a, int64_t first, int64_t last) {
  using T = typename Elem<D_DT>::T;
  constexpr int V = 16 / sizeof(T);
  if (last < first) last = first;
  if (first == 0 && last == a.M) return;
  const int64_t at = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, step = (int64_t)gridDim.x * blockDim.x;
  auto zero = [&](int64_t row, int64_t rows) {
    T *p = static_cast<T *>(a.D) + row * a.N;
    const int64_t n = rows * a.N;
    for (int64_t i = at * V; i < n; i += step * V) {
      if (i + V <= n) {
        *reinterpret_cast<u32x4_elem *>(p + i) = (u32x4){0, 0, 0, 0};
      } else {
        for (int64_t k = i; k < n; ++k) p[k] = T(0);
      }
    }
  };
  zero(0, first);
  zero(last, a.M - last);
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
  if (a.whole && blockIdx.y == gridDim.y - 1) zero_other_rows<D_DT>(a, group_of(a.offsets, 0, a.M).first, grp.first + grp.count);
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

// ===========================================================================
// The tile kernel of the linears on the tiles of all groups.  A group's tiles start at a multiple of four rows, at or in front of its first one (a
// transfer of scales is four rows), and go up to its end; the tiles of all groups are one sequence, dealt to the XCDs and walked in bands as
// those of one matrix are.  Every workgroup finds its tile by itself: the tile counts of 64 experts a step, one a lane, summed over the wave.
// ===========================================================================
template <int BM>
__device__ __forceinline__ int group_tiles(const Group &g) {
  return g.count == 0 ? 0 : ((g.first & 3) + g.count + BM - 1) / BM;
}
__device__ __forceinline__ int wave_prefix(int v) {  // inclusive: inside rows of 16 lanes, then the last lane of a row to those behind it
  v += (int)dpp_u32<DPP_ROW_SHR(1)>((uint32_t)v);
  v += (int)dpp_u32<DPP_ROW_SHR(2)>((uint32_t)v);
  v += (int)dpp_u32<DPP_ROW_SHR(4)>((uint32_t)v);
  v += (int)dpp_u32<DPP_ROW_SHR(8)>((uint32_t)v);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast:15 to rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast:31 to rows 2 and 3
  return v;
}

struct GroupTile {
  int e, first, count, tile, tn;  // tile: index inside the group; e < 0: none
  int rows_first, rows_last;      // of all groups: first row of the first one, end of the last one
};
template <int BM, int BN>
__device__ __forceinline__ GroupTile tile_of_groups(const GroupedArgs &a) {
  const int lane = threadIdx.x & 63, E = (int)a.E;
  const uint32_t tiles_n = (uint32_t)ceil_div(a.N, BN);
  int64_t sum = 0;
  Group grp{0, 0};
  int incl = 0, rows_first = 0;
  for (int base = 0; base < E; base += 64) {
    grp = base + lane < E ? group_of(a.offsets, base + lane, a.M) : Group{0, 0};
    incl = wave_prefix(group_tiles<BM>(grp));
    sum += __builtin_amdgcn_readlane(incl, 63);
    if (base == 0) rows_first = __builtin_amdgcn_readlane(grp.first, 0);
  }
  const int rows_last = __builtin_amdgcn_readlane(grp.first + grp.count, (E - 1) & 63);
  // (offsets that overlap could name more tiles than the launch has)
  const uint32_t most = gridDim.x / tiles_n;
  const uint32_t total = (uint32_t)__builtin_amdgcn_readfirstlane((int)(sum < most ? sum : most));
  if (blockIdx.x >= total * tiles_n) return {-1, 0, 0, 0, 0, rows_first, rows_last};
  const TileCoord tc = tile_of_workgroup<4>(blockIdx.x, total, tiles_n);
  const int tm = __builtin_amdgcn_readfirstlane((int)tc.m);
  int before = 0, base = 0;
  if (E > 64) {
    for (; base < E; base += 64) {
      grp = base + lane < E ? group_of(a.offsets, base + lane, a.M) : Group{0, 0};
      incl = wave_prefix(group_tiles<BM>(grp));
      const int here = __builtin_amdgcn_readlane(incl, 63);
      if (tm < before + here) break;  // (some step has it: tm < total)
      before += here;
    }
  }
  const int l = __builtin_ctzll(__ballot(before + incl > tm));
  const int tiles = __builtin_amdgcn_readlane(group_tiles<BM>(grp), l);
  return {base + l, __builtin_amdgcn_readlane(grp.first, l), __builtin_amdgcn_readlane(grp.count, l), tm - (before + __builtin_amdgcn_readlane(incl, l) - tiles),
          __builtin_amdgcn_readfirstlane((int)tc.n), rows_first, rows_last};
}

template <int D_DT, int BIAS_DT, int MI, int NJ, int PS, int KW, bool EARLY, int PER_CU>
__global__ __launch_bounds__(256, PER_CU) void linear_grouped_tile_kernel(GroupedArgs a) {
  extern __shared__ __attribute__((aligned(16))) char plds[];
  constexpr int BM = 64 * MI, BN = 64 * NJ;
  const GroupTile t = tile_of_groups<BM, BN>(a);
  if (a.whole) zero_other_rows<D_DT>(a, t.rows_first, t.rows_last);
  if (t.e < 0) return;
  const int64_t kb = a.K >> 1, e = t.e;
  LinearArgs la{a.D, a.A, a.B + e * a.N * kb, a.A_sf, a.B_sf + e * (a.K >> 6) * a.Np, a.A_gs, a.B_gs + e * a.B_gs_stride, nullptr,
                t.first + t.count, a.N, a.K, a.Tp, a.Np};
  if constexpr (BIAS_DT != BIAS_NONE) la.bias = static_cast<const typename Elem<BIAS_DT>::T *>(a.bias) + e * a.N;
  tile256p<D_DT, BIAS_DT, MI, NJ, PS, KW, EARLY, true>(la, SplitK{nullptr, 1}, plds, TileRows{(t.first & ~3) + (int64_t)t.tile * BM, t.first, a.rows, a.T}, t.tn);
}

// Scales of gathered rows, a column for each row of the output: tiles of more than 64 rows fetch those of four neighbours at once.  (In front of tiles of 64
// rows, which gather by themselves, this launch took 5 of 73 us.)
__global__ __launch_bounds__(256) void gather_scales_kernel(uint32_t *out, const uint32_t *sf, const int32_t *rows, int64_t M, int64_t Mp, int64_t T,
                                                            int64_t Tp) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, chunk = blockIdx.y;
  if (i >= Mp) return;
  int64_t row = i < M ? rows[i] : 0;
  row = row < 0 ? 0 : row < T ? row : T - 1;
  out[chunk * Mp + i] = i < M ? sf[chunk * Tp + row] : 0u;
}

enum GroupedKind { GROUPED_NONE = 0, GROUPED_ROWS16 = 1, GROUPED_64_128 = 2, GROUPED_64_256 = 3, GROUPED_256_256 = 4 };
// which kernel the last call of this host thread launched (introspection for tests)
static thread_local int g_last_grouped_kernel = GROUPED_NONE;

// (the tile kernel's 32-bit lane offsets: whole of x where rows are gathered, the rows of a tile and of a band otherwise)
static bool grouped_tiles_fit(int64_t T, int64_t N, int64_t K, bool gather) {
  return K >= P_BK && (K >> 1) * 260 < (1ll << 31) && (!gather || T * (K >> 1) < (1ll << 32) - 64) && N < (1ll << 27);
}
// Which kernel, by the time that each is expected to take (us), fitted to 100 shapes of 8 to 128 experts, N of 1003 to 14336, K of 2048 to 14336 and 1 to
// 2048 rows an expert.  What is known on the host are the counts; the groups are taken for those of rows dealt out evenly at random.  A tile of a
// shape takes so long for each 4096 of K, and so long besides, with its CU full of them; tiles go to the CUs in whole rounds while these
// are few.  64 x 256 and 64 x 128 tiles are two to a CU: memory latency and the exchange at the end of one lie under the other's work.
// Measured, us (256 x 256 / 64 x 256 / 64 x 128 / 16 rows):  8 experts of 14336 x 4096, 2 rows each 162 / 57 / 66 / 80, 128 157 / 137 / 147 / 570,
// 2048 1291 / 1498 / 1795; 8 of 4096 x 14336, 8 rows 236 / 92 / 69 / 73; 16 of 4096 x 4096, 512 rows 237 / 235 / 274; 8 of 64 x 4096, 16 rows 69 / 33 / 23 / 12,
// 512 69 / 35 / 24; 128 x 128 tiles, one or two to a CU,
// were nowhere more than 6 % ahead of the best of these.
static GroupedKind grouped_kind(int64_t T, int64_t M, int64_t N, int64_t K, int64_t E, bool gather) {
  if (!grouped_tiles_fit(T, N, K, gather)) return GROUPED_ROWS16;
  const int cu = device_cu_count();
  const double cus = cu > 0 ? cu : 256, k = (double)K / 4096;
  const double groups = (double)E * -expm1((double)M * log1p(-1.0 / ((double)E + 1e-9)));  // that have rows
  auto tiles = [&](int bm, int bn) {  // a CU
    const double m = (double)M / bm + groups / 2;
    return (m > groups ? m : groups) * (double)ceil_div(N, bn) / cus;
  };
  auto rounds = [](double x) { return x <= 3 ? ceil(x) : x + 0.25; };
  const double launch = 6, t256 = launch + rounds(tiles(256, 256)) * (76 * k + 10.5), t64 = launch + rounds(tiles(64, 256)) * (24.3 * k + 2.5);
  const double x = tiles(64, 128), t128 = launch + (x <= 1 ? 19 * k + 1 : rounds(x) * (14 * k + 1.7));
  GroupedKind kind = t256 < t64 ? GROUPED_256_256 : GROUPED_64_256;
  double best = t256 < t64 ? t256 : t64;
  if (t128 < best) kind = GROUPED_64_128, best = t128;
  // 16 weight rows a workgroup: the weights' bytes, and what a second set of 16 activation rows adds
  const double read = groups * (double)N * (double)K * 0.5625 / 3.5e6;
  if ((double)M <= 32 * groups && 8 + read * ((double)M <= 16 * groups ? 1.0 : 2.3) < best) kind = GROUPED_ROWS16;
  return kind;
}

// Workgroups of a tile launch: rows in tiles, and at most one tile more for each group that has rows
static int64_t grouped_tiles(int64_t M, int64_t N, int64_t E, GroupedKind kind) {
  const int bm = kind == GROUPED_256_256 ? 256 : 64, bn = kind == GROUPED_64_128 ? 128 : 256;
  const int64_t groups = E < M ? E : M;
  return (M + groups * (bm + 2)) / bm * ceil_div(N, bn);
}

template <int D_DT, int BIAS_DT, int MI, int NJ, int KW, int PS, int PER_CU>
static int launch_grouped_tile(GroupedArgs a, GroupedKind kind, uint32_t *scales, hipStream_t st) {
  const bool early = a.K % P_BK != 0;
  auto *kern = early ? linear_grouped_tile_kernel<D_DT, BIAS_DT, MI, NJ, PS, KW, true, PER_CU> : linear_grouped_tile_kernel<D_DT, BIAS_DT, MI, NJ, PS, KW, false, PER_CU>;
  using PL = PLayout<64 * MI, 64 * NJ, PS>;
  static std::atomic<uint32_t> lds_ok[2];
  if (int rc = allow_dynamic_lds(kern, lds_ok[early], PL::LDS_BYTES)) return rc;
  if (MI > 1 && a.rows) {
    const int64_t Mp = align_up(a.M, 16);
    hipLaunchKernelGGL(gather_scales_kernel, dim3((unsigned)ceil_div(Mp, 256), (unsigned)(a.K / 64)), dim3(256), 0, st, scales, a.A_sf, a.rows, a.M, Mp, a.T, a.Tp);
    a.A_sf = scales;
    a.Tp = Mp;
  }
  hipLaunchKernelGGL(kern, dim3((unsigned)grouped_tiles(a.M, a.N, a.E, kind)), dim3(256), PL::LDS_BYTES, st, a);
  return 0;
}

template <int D_DT, int BIAS_DT>
static int launch_grouped(const GroupedArgs &a, GroupedKind kind, uint32_t *scales, hipStream_t st) {
  switch (kind) {
    case GROUPED_256_256: return launch_grouped_tile<D_DT, BIAS_DT, 4, 4, 1, 3, 1>(a, kind, scales, st);
    case GROUPED_64_256: return launch_grouped_tile<D_DT, BIAS_DT, 1, 4, 2, 3, 2>(a, kind, scales, st);
    case GROUPED_64_128: return launch_grouped_tile<D_DT, BIAS_DT, 1, 2, 2, 5, 2>(a, kind, scales, st);
    default: break;  // GROUPED_ROWS16
  }
  const dim3 grid((unsigned)ceil_div(a.N, R16_ROWS), (unsigned)a.E);
  if (a.M <= 16 * a.E) hipLaunchKernelGGL((linear_grouped_rows16_kernel<D_DT, BIAS_DT, 1>), grid, dim3(64 * R16_WAVES), 0, st, a);
  else hipLaunchKernelGGL((linear_grouped_rows16_kernel<D_DT, BIAS_DT, 2>), grid, dim3(64 * R16_WAVES), 0, st, a);
  return 0;
}

template <int D_DT>
static int grouped_bias(const GroupedArgs &a, int bias_dtype, GroupedKind kind, uint32_t *scales, hipStream_t st) {
  if (!a.bias) return launch_grouped<D_DT, BIAS_NONE>(a, kind, scales, st);
  switch (bias_dtype) {
    case AC4K_DTYPE_BF16: return launch_grouped<D_DT, AC4K_DTYPE_BF16>(a, kind, scales, st);
    case AC4K_DTYPE_FP16: return launch_grouped<D_DT, AC4K_DTYPE_FP16>(a, kind, scales, st);
    case AC4K_DTYPE_FP32: return launch_grouped<D_DT, AC4K_DTYPE_FP32>(a, kind, scales, st);
  }
  return set_error("bias must be bfloat16, half or float (dtype tag %d)", bias_dtype);
}

}  // namespace ac4k

using namespace ac4k;

extern "C" __attribute__((visibility("default"))) int64_t ac4k_linear_grouped_nvfp4_workspace_bytes(int64_t T, int64_t M, int64_t N, int64_t K, int64_t E,
                                                                                                   int has_rows) {
  if (T < 1 || M < 1 || N < 1 || K < 64 || K % 64 != 0 || E < 1 || !has_rows || grouped_kind(T, M, N, K, E, true) != GROUPED_256_256) return 0;
  return K / 64 * align_up(M, 16) * 4;
}

static int grouped_linear(
    bool whole, void *D, int d_dtype, const void *A, const void *A_sf, const float *A_gs, int64_t T, const int32_t *rows, const void *B, const void *B_sf,
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
                static_cast<const uint32_t *>(B_sf), B_gs, B_gs_stride, bias, offsets, T, align_up(T, 16), M, N, align_up(N, 16), K, E, whole};
  hipStream_t st = (hipStream_t)stream;
  const GroupedKind kind = grouped_kind(T, M, N, K, E, rows != nullptr);
  const int64_t need = ac4k_linear_grouped_nvfp4_workspace_bytes(T, M, N, K, E, rows != nullptr);
  AC4K_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0), "workspace of %lld bytes needed, on 16 bytes",
               (long long)need);
  AC4K_REQUIRE(d_dtype == AC4K_DTYPE_BF16 || d_dtype == AC4K_DTYPE_FP16 || d_dtype == AC4K_DTYPE_FP32, "d must be bfloat16, half or float (dtype tag %d)", d_dtype);
  AC4K_REQUIRE(!bias || bias_dtype == AC4K_DTYPE_BF16 || bias_dtype == AC4K_DTYPE_FP16 || bias_dtype == AC4K_DTYPE_FP32,
               "bias must be bfloat16, half or float (dtype tag %d)", bias_dtype);
  AC4K_REQUIRE(kind == GROUPED_ROWS16 || grouped_tiles(M, N, E, kind) < (1ll << 24), "problem too large");  // 2^32 threads a launch
  int rc;
  switch (d_dtype) {
    case AC4K_DTYPE_BF16: rc = grouped_bias<AC4K_DTYPE_BF16>(a, bias_dtype, kind, static_cast<uint32_t *>(workspace), st); break;
    case AC4K_DTYPE_FP16: rc = grouped_bias<AC4K_DTYPE_FP16>(a, bias_dtype, kind, static_cast<uint32_t *>(workspace), st); break;
    case AC4K_DTYPE_FP32: rc = grouped_bias<AC4K_DTYPE_FP32>(a, bias_dtype, kind, static_cast<uint32_t *>(workspace), st); break;
    default: return set_error("d must be bfloat16, half or float (dtype tag %d)", d_dtype);
  }
  if (rc) return rc;
  g_last_grouped_kernel = kind;
  return check_launch("ac4k_linear_grouped_nvfp4");
}

extern "C" __attribute__((visibility("default"))) int ac4k_linear_grouped_nvfp4(
    void *D, int d_dtype, const void *A, const void *A_sf, const float *A_gs, int64_t T, const int32_t *rows, const void *B, const void *B_sf,
    const float *B_gs, int64_t B_gs_stride, const void *bias, int bias_dtype, const int32_t *offsets, int64_t M, int64_t N, int64_t K, int64_t E,
    void *workspace, int64_t workspace_bytes, ac4k_stream_t stream) {
  return grouped_linear(false, D, d_dtype, A, A_sf, A_gs, T, rows, B, B_sf, B_gs, B_gs_stride, bias, bias_dtype, offsets, M, N, K, E, workspace,
                        workspace_bytes, stream);
}

extern "C" __attribute__((visibility("default"))) int ac4k_linear_grouped_nvfp4_whole(
    void *D, int d_dtype, const void *A, const void *A_sf, const float *A_gs, int64_t T, const int32_t *rows, const void *B, const void *B_sf,
    const float *B_gs, int64_t B_gs_stride, const void *bias, int bias_dtype, const int32_t *offsets, int64_t M, int64_t N, int64_t K, int64_t E,
    void *workspace, int64_t workspace_bytes, ac4k_stream_t stream) {
  return grouped_linear(true, D, d_dtype, A, A_sf, A_gs, T, rows, B, B_sf, B_gs, B_gs_stride, bias, bias_dtype, offsets, M, N, K, E, workspace,
                        workspace_bytes, stream);
}

extern "C" __attribute__((visibility("default"))) int ac4k_debug_last_grouped_kernel(void) { return ac4k::g_last_grouped_kernel; }

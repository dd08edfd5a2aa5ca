// The tile kernel of the NVFP4 linears, as a function of a workgroup: linear_kernels.h runs it on the tiles of one matrix, linear_grouped.hip on those of
// the experts' ones.
#pragma once

#include <atomic>
#include <type_traits>

#include "linear_common.h"

namespace ac4k {

struct LinearArgs {
  void *D;
  const uint8_t *A, *B;
  const uint32_t *A_sf, *B_sf;  // one dword per (64-chunk, row): sf_u32[chunk * rows_padded + row]
  const float *A_gs, *B_gs;
  const void *bias;
  int64_t M, N, K, Mp, Np;
  int prepacked = 0;  // B points at a weight image (W_BLOCK_BYTES blocks, see below) and B_sf is unused
  Epilogue ep = {};
};

// --- pre-packed weight image -----------------------------------------------------
// Static weights can be re-laid once into the order the kernels fetch them: one block per
// (128 rows, 128 k), blocks of a 128-row band consecutive along k, bands consecutive along n (N is
// padded with zero rows to a whole band).  A block is the LDS stage picture of those rows: 128 rows x
// 64 packed bytes with the 16-byte piece p of row r at position p ^ ((r >> 1) & 3), followed by the
// scale dwords [2 chunks][128 rows].  Every LDS-DMA transfer of a stage then reads one contiguous
// kilobyte, and a stage of the decode-sized kernel (256 k) is one contiguous run of two blocks.
constexpr int W_BLOCK_ROWS = 128, W_BLOCK_K = 128;
constexpr int W_BLOCK_DATA = W_BLOCK_ROWS * W_BLOCK_K / 2;            // 8192
constexpr int W_BLOCK_BYTES = W_BLOCK_DATA + 2 * W_BLOCK_ROWS * 4;    // 9216

// --- workgroup -> output tile ---------------------------------------------------
// Workgroups are dealt round-robin to the 8 XCDs, each with its own L2.  Workgroup `pid` is first
// renumbered so that every XCD owns one contiguous run of the tile sequence, and the sequence walks
// the tiles in bands of GROUP_M tile-rows, column by column inside a band: the workgroups resident
// on one XCD at a time then cover a compact GROUP_M x (CUs / GROUP_M) patch and share its operand
// panels through that L2.
// (32 bits: a grid has fewer than 2^32 workgroups.  The quotients of 64 bits that were here, and of the range below where there is only one, took every
// workgroup a third of a microsecond: 300 x 1024 x 256 5.23 -> 4.83 us, 2898 x 600 x 256 5.83 -> 5.46.)
struct TileCoord {
  uint32_t m, n;
};
template <int GROUP_M>
__device__ __forceinline__ TileCoord tile_of_workgroup(uint32_t pid, uint32_t tiles_m, uint32_t tiles_n) {
  const uint32_t ntiles = tiles_m * tiles_n;
  const uint32_t per = ntiles / 8, rem = ntiles % 8;
  const uint32_t xcd = pid % 8, idx = pid / 8;
  pid = xcd * per + (xcd < rem ? xcd : rem) + idx;
  const uint32_t band = pid / (GROUP_M * tiles_n), in_band = pid - band * (GROUP_M * tiles_n);
  const uint32_t first_m = band * GROUP_M;
  const uint32_t rows = (tiles_m - first_m) < GROUP_M ? (tiles_m - first_m) : GROUP_M;
  const uint32_t col = in_band / rows;
  return {first_m + in_band - col * rows, col};
}
// stages [first, first + count) of K range `range` of `ranges`; in scalar registers, said plainly: the compiler otherwise takes the
// quotients, and with them the loop and the addresses, to the lanes
struct StageRange {
  int first, count;
};
__device__ __forceinline__ StageRange stage_range(int stages, uint32_t range, int ranges) {
  if (ranges == 1) return {0, stages};
  const int first = __builtin_amdgcn_readfirstlane((int)((int64_t)stages * range / ranges));
  return {first, __builtin_amdgcn_readfirstlane((int)((int64_t)stages * (range + 1) / ranges)) - first};
}

// ===========================================================================
// (64 MI) x (64 NJ) tile, packed operands in LDS, decode after the fragment load.
//
// The packed A/B slices and their scale dwords go from global memory straight into LDS with
// LDS-DMA loads (global_load_lds: no VGPR staging, no LDS store instruction), PS stages of
// 128 k each.  A wave (4 waves, 2x2, (32 MI) x (32 NJ) each) reads for every 32-row fragment ONE
// 16-byte word per lane per 64-chunk: lane (row r, half h) owns elements [32h, 32h+32) of the
// chunk; dword s of that word feeds MFMA sub-step s.  The same k-slot assignment is used for A
// and B, so the permutation of k inside a chunk cancels in the dot product.  Decode per dword:
// 4 x v_cvt_scalef32_pk_f16_fp4 + 4 x v_pk_mul_f16 by the block scale (E4M3 -> fp16 with
// v_cvt_scalef32_pk_f16_fp8, splat through op_sel); the decode of a sub-step is interleaved with
// the MFMAs of the previous one (TileWave below).
// KW == 1: the waves multiply a quarter of the tile each, over all of a stage, with one workgroup barrier per 128 k, placed in the
// middle of the step so that the next stage is readable before the current one ends.  KW == 2, for the tiles of up to 256 x 128: two waves
// multiply one half of the tile each over one 64-chunk of a stage and two over the other, and meet at the end through LDS: 4 decode
// instructions per MFMA instead of 6 for 256 x 128 and 128 x 256, 4.7 instead of 6.7 for 192 x 128, 6 instead of 8 for 128 x 128.
// Bound by instruction issue of a single wave per SIMD and, where the whole GPU is busy for long, by power.  Cycles per MFMA and wave, with
// KW == 1, the decoding pinned between the MFMAs and the scales fetched a dword per lane / now: 256 x 256 41.2 / 35.2, 256 x 128 51 / 39,
// 192 x 128 58 / 44, 128 x 128 70 / 51.  Back to back, us: 1024 x 4096 x 4096 38.3 / 32.8, 1001 x 5003 x 2880 35.7 / 33.6, 2048 x 4096 x 4096
// 58.2 / 53.8, 2048 x 14336 x 4096 183.8 / 175.5, 75600 x 5120 x 5120 2776 / 2673 (the clock comes down by half of what the loop gains).  256 x 128
// and 128 x 256 tiles run KW == 2 on long ranges only (PAIR_STAGES), for the exchange.
// Split-K: blockIdx.y selects a contiguous range of stages; with more than one range the
// accumulators go to an fp32 partial buffer and a second kernel adds the ranges.
// Requires K % 64 == 0, K >= 128 and 16-byte aligned operands.  EARLY: K % 128 == 64.  The stages start one
// chunk early, at k = -64, so that only stage 0 is special and the loop is not: the prologue fetches k-chunk 0
// into both halves of it and clears the scales of the first half.  (1001 x 5003 x 2880, fp32 out: 75 -> 45 us, the
// 128x128 kernel against this one; 300 x 4096 x 4160: 93 -> 28.)  A variant of its own: decided at run time, the longer
// prologue cost the 128 x 128 tiles of every other K 0.2 to 0.4 us (kernel alone, 160 x 2000 x 8192 in eight K ranges:
// 18.1 us, 17.3 without; 256 x 4096 x 4096 in four 20.7 and 19.8).
// ===========================================================================
constexpr int P_BK = 128;     // k per stage (two 64-chunks)
constexpr int P_ROW = 64;     // packed bytes per row per stage: [chunk][half] x 16 B

template <int BM, int BN, int PS>
struct PLayout {               // byte offsets inside one LDS stage; PS stages
  static constexpr int OFF_B = BM * P_ROW;                 // B rows follow the A rows
  static constexpr int OFF_SFA = OFF_B + BN * P_ROW;       // scale dwords: [chunk][BM rows]
  static constexpr int NSA = (BM + 127) / 128, NSB = (BN + 127) / 128;  // kilobytes, and transfers, of scales
  static constexpr int OFF_SFB = OFF_SFA + NSA * 1024;     // [chunk][BN rows]
  static constexpr int STAGE_BYTES = OFF_SFB + NSB * 1024;
  static_assert(NSA + NSB <= 4, "a scale transfer per wave");
  static constexpr int LDS_BYTES = PS * STAGE_BYTES;
  static_assert(LDS_BYTES <= 160 * 1024, "stages must fit in the CU's LDS");
};

// two of the eight values of a dword of nibbles, without their scale; q (0..3) is a constant after unrolling
__device__ __forceinline__ f16x2 decode_pair(uint32_t w, int q) {
  if (q == 0) return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 0);
  if (q == 1) return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 1);
  if (q == 2) return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 3);
}

// f(i) for the share of COUNT things that belongs behind the m-th of OF instructions (a loop of a known length, so that it unrolls
// before the one over m does)
template <int COUNT, int OF, typename F>
__device__ __forceinline__ void deal(int m, F &&f) {
#pragma unroll
  for (int x = 0; x < (COUNT + OF - 1) / OF; ++x) {
    const int i = COUNT * m / OF + x;
    if (i < COUNT * (m + 1) / OF) f(i);
  }
}

// What a wave of the tile kernels holds: packed fragments of a 64-chunk, 32 rows each, WI of A first, then WJ of B, in two sets (one
// multiplied while the other arrives), and the sums of WI x WJ blocks.  Lane (row r, half h) of a fragment has elements
// [32 h, 32 h + 32) of the chunk; dword s of them belongs to sub-step s, 16 k.
//
// The loop bodies are written out in the order in which they issue.  A wave is alone on its SIMD and issues an instruction of any kind
// every 5 cycles; an MFMA takes 8.6 of these and keeps the matrix core busy for 32.  Up to four or five instructions behind every
// MFMA are free, and what stands in a clump leaves the matrix core idle, so everything is dealt out evenly: the decoding,
// the LDS reads and the transfers.  (Left to the compiler, with only the decoding pinned between the MFMAs: 41.2 cycles an MFMA in
// 256 x 256 tiles, 36.4 so, 35.2 with the scales in 16-byte transfers.)
template <int WI, int WJ>
struct TileWave {
  static constexpr int NF = WI + WJ, NM = WI * WJ;
  uint4 packed[2][NF];
  uint32_t sf[2][NF];    // the scale bytes of the lane's two blocks
  f16x2 scale[2][NF];    // the same as fp16
  u32x4 decoded[2][NF];  // operands of a sub-step, double buffered
  f32x16 acc[WI][WJ];

  // item i of decoding sub-step s of set `set` into buffer d: two values of fragment i / 4.  wfac: power of two on the scales of B
  __device__ __forceinline__ void decode_item(int d, int set, int s, int i, float wfac = 1.0f) {
    const int f = i >> 2, q = i & 3;
    if (s == 0 && q == 0) scale[set][f] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(sf[set][f], f < WI ? 1.0f : wfac, false);
    const f16x2 sc = s < 2 ? (f16x2){scale[set][f].x, scale[set][f].x} : (f16x2){scale[set][f].y, scale[set][f].y};
    const uint4 &v = packed[set][f];
    decoded[d][f][q] = __builtin_bit_cast(uint32_t, decode_pair(s == 0 ? v.x : s == 1 ? v.y : s == 2 ? v.z : v.w, q) * sc);
  }
  // One sub-step: the MFMAs on buffer d, under them the decoding of sub-step s of set `set` into the other buffer, and extra(m) behind MFMA m
  template <typename F>
  __device__ __forceinline__ void substep(int d, int set, int s, F &&extra, float wfac = 1.0f) {
#pragma unroll
    for (int m = 0; m < NM; ++m) {
      // boustrophedon order: every MFMA shares one operand with the one before it (measured 0.6 %
      // faster than row by row on the power-limited 8192^3 problem: less operand switching)
      const int i = m / WJ, j = (i & 1) ? WJ - 1 - m % WJ : m % WJ;
      acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, decoded[d][WI + j]), __builtin_bit_cast(f16x8, decoded[d][i]),
                                                         acc[i][j], 0, 0, 0);  // D^T block
      deal<4 * NF, NM>(m, [&](int e) { decode_item(1 - d, set, s, e, wfac); });
      extra(m);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < WI; ++i)
#pragma unroll
      for (int j = 0; j < WJ; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
  }
};

// Build with -DAC4K_LINEAR_TIMELINE (`build.py --timeline`) to record per workgroup the 100 MHz clock at
// kernel entry, loop entry, loop exit and kernel exit plus the shader cycles spent in the loop of the
// tile kernel and of the K-split-waves kernel; ac4k_debug_linear_timeline copies the stamps out
// (a profiling aid; not compiled into the library).
#ifdef AC4K_LINEAR_TIMELINE
static __device__ uint64_t g_linear_timeline[8192][6];
#define AC4K_LTL(i, v)                                                     \
  do {                                                                     \
    if (threadIdx.x == 0 && blockIdx.x + gridDim.x * blockIdx.y < 8192)      \
      g_linear_timeline[blockIdx.x + gridDim.x * blockIdx.y][i] = (v);        \
  } while (0)
#else
#define AC4K_LTL(i, v)
#endif

struct SplitK {
  float *partial;  // [splits][M][N] fp32, or null: convert and store to D
  int splits;
};

// the first `cols` elements of S bytes (at least one) of a 16-byte piece, to any element
template <int S>
__device__ __forceinline__ void store_piece(char *dst, const u32x4 &v, int cols) {
  if (cols >= 16 / S) {
    *reinterpret_cast<u32x4_elem *>(dst) = v;
    return;
  }
  const int dwords = cols * S / 4;  // whole ones
  if (dwords & 2) *reinterpret_cast<u32x2_elem *>(dst) = (u32x2){v.x, v.y};
  if (dwords & 1) *reinterpret_cast<u32_elem *>(dst + (dwords & 2) * 4) = dwords & 2 ? v.z : v.x;
  if constexpr (S == 2)
    if (cols & 1) *reinterpret_cast<uint16_t *>(dst + dwords * 4) = (uint16_t)(dwords & 2 ? dwords & 1 ? v.w : v.z : dwords & 1 ? v.y : v.x);
}

// Epilogue of the packed-LDS tile kernel: the accumulators of one wave, (32*MI) x (32*NJ) outputs, to
// `out` (row stride N).  acc[i][j] holds the TRANSPOSED 32x32 block (the MFMAs are issued with the
// operands swapped): lane l, element e <-> n = j*32 + (e>>2)*8 + (l>>5)*4 + (e&3), m = i*32 + (l&31),
// i.e. four consecutive n per lane.  RAW stores the fp32 sums as they are (split-K partials);
// otherwise out = cvt(acc * scale + bias).  Outputs are staged through LDS (`lds`, free at this
// point), one wave-private block of RP rows at a time, so that every lane stores 16 bytes and a
// wave store covers whole row segments; the bias of the tile's columns sits behind the staging
// blocks as fp32.  Callers have passed a workgroup barrier after their last read of `lds`.
// LOWER: rows in front of m_lo are left out, too.
template <int OUT_DT, int BIAS_DT, bool RAW, int MI, int NJ, int LDS_BYTES, bool LOWER>
__device__ __forceinline__ void store_tile(const f32x16 (&acc)[MI][NJ], char *lds, void *out, const void *bias,
                                           float scale, int64_t M, int64_t N, int64_t m0, int64_t n0,
                                           int64_t tile_n0, int64_t m_lo) {
  using DE = Elem<OUT_DT>;
  using DT = typename DE::T;
  DT *Dp = static_cast<DT *>(out);
  constexpr int S = sizeof(DT);
  constexpr int WN = 32 * NJ;               // columns per wave
  constexpr int RP = S == 2 && MI % 2 == 0 ? 64 : 32;  // rows per staging pass
  constexpr int PITCH = WN * S + 16;        // bytes per staged row, 16 bytes of padding
  constexpr int STG_BYTES = 4 * RP * PITCH;
  static_assert(STG_BYTES + 2 * WN * 4 <= LDS_BYTES, "epilogue staging and bias must fit in LDS");
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5, wn = wave & 1;
  const float *bias_s = reinterpret_cast<const float *>(lds + STG_BYTES) + wn * WN + half * 4;
  if constexpr (BIAS_DT != BIAS_NONE) {
    if (tid < 2 * WN) {
      const int64_t n = tile_n0 + tid;
      reinterpret_cast<float *>(lds + STG_BYTES)[tid] = n < N ? Elem<BIAS_DT>::load(bias, n) : 0.0f;
    }
    __syncthreads();
  }
  // the four outputs acc[i][j][4g .. 4g+3] of a lane, scaled, plus their bias b
  // The 256x256 tile keeps its 256 sums per lane in accumulation registers.  Left alone, the compiler
  // moves all of them to ordinary registers at the top of the epilogue and spills what does not fit;
  // reading them with a volatile move keeps each read inside the pass that stages the value.
  auto sum_of = [&](int i, int j, int e) {
    if constexpr (MI * NJ == 16) {
      float v;
      asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v) : "a"(acc[i][j][e]));
      return v;
    } else {
      return acc[i][j][e];
    }
  };
  auto value4 = [&](int i, int j, int g, const float4 &b) {
    float4 v = make_float4(sum_of(i, j, 4 * g), sum_of(i, j, 4 * g + 1), sum_of(i, j, 4 * g + 2), sum_of(i, j, 4 * g + 3));
    if constexpr (!RAW) {
      v.x *= scale; v.y *= scale; v.z *= scale; v.w *= scale;
    }
    if constexpr (BIAS_DT != BIAS_NONE) {
      v.x += b.x; v.y += b.y; v.z += b.z; v.w += b.w;
    }
    return v;
  };
  // bias of column block j: four 16-byte LDS reads in one go (one wait), kept for the rows of a pass
  auto bias_of = [&](int j, float4 (&b)[4]) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      b[g] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if constexpr (BIAS_DT != BIAS_NONE) b[g] = *reinterpret_cast<const float4 *>(bias_s + j * 32 + g * 8);
    }
  };
  // Rows that start on any element leave in 16-byte stores like aligned ones; the last, partial piece of a row in up to three
  // smaller ones (element by element before, in a loop: fp32 1001 x 5003 x 2880 46.4 -> 40.9 us, bf16 4000 x 5003 x 2880 144 -> 133,
  // N = 5008 129)
  char *stg = lds + wave * (RP * PITCH);
  constexpr int CPR = WN * S / 16;   // 16-byte pieces per staged row
  constexpr int RS = 64 / CPR;       // rows covered by one wave store
  const int lrow = lane / CPR, lq = lane % CPR;
  const int64_t row_bytes = N * S;
  const uint32_t lane_off = (uint32_t)(lrow * row_bytes) + lq * 16;
  char *out0 = reinterpret_cast<char *>(Dp) + (m0 * N + n0) * S;  // wave-uniform
  const bool interior = m0 + 32 * MI <= M && n0 + WN <= N && (!LOWER || m0 >= m_lo);
  const bool whole = N % (16 / S) == 0 || n0 + WN <= N;  // no piece is cut: rows past M and pieces past N are left out
  const int64_t cl = N - n0 - lq * (16 / S);
  const int cols_left = cl > 16 / S ? 16 / S : (int)cl;  // columns of this lane's piece inside the matrix
  const int64_t rl = M - m0 - lrow;
  const int rows_left = rl > 32 * MI ? 32 * MI : (int)rl;  // rows of the block below this lane's first one
  const int rows_skip = LOWER && m_lo > m0 + lrow ? (int)(m_lo - m0 - lrow) : 0;  // of them, in front of m_lo
  auto row_in = [&](int row) { return row < rows_left && (!LOWER || row >= rows_skip); };
#pragma unroll
  for (int p = 0; p < 32 * MI / RP; ++p) {
    asm volatile("" ::: "memory");  // keeps the bias reads of one pass from being merged with the next one's
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      float4 b[4];
      bias_of(j, b);
#pragma unroll
      for (int ii = 0; ii < RP / 32; ++ii) {
        const int i = p * (RP / 32) + ii;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float4 v = value4(i, j, g, b[g]);
          char *dst = stg + (ii * 32 + (lane & 31)) * PITCH + (j * 32 + g * 8 + half * 4) * S;
          if constexpr (S == 2) *reinterpret_cast<uint2 *>(dst) = make_uint2(DE::cvt2(v.x, v.y), DE::cvt2(v.z, v.w));
          else *reinterpret_cast<float4 *>(dst) = v;
        }
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the staging block is private to the wave
    // pass `it` stores rows it*RS .. it*RS+RS-1 of the block: a wave-uniform base that advances by
    // RS rows, plus a fixed 32-bit lane offset; the bounds checks are per lane only on edge tiles
    const char *src = stg + lrow * PITCH + lq * 16;
    char *rowp = out0 + (int64_t)p * RP * row_bytes;
    if (interior) {
#pragma unroll
      for (int it = 0; it < RP / RS; ++it)
        *reinterpret_cast<u32x4_elem *>(rowp + it * RS * row_bytes + lane_off) = *reinterpret_cast<const u32x4 *>(src + it * RS * PITCH);
    } else if (whole) {
#pragma unroll
      for (int it = 0; it < RP / RS; ++it) {
        const u32x4 v = *reinterpret_cast<const u32x4 *>(src + it * RS * PITCH);
        if (cols_left > 0 && row_in(p * RP + it * RS)) *reinterpret_cast<u32x4_elem *>(rowp + it * RS * row_bytes + lane_off) = v;
      }
    } else {
      // (unrolled by four for the small tiles: with all of it 128 x 128 tiles ran 2 % longer, also where no piece is cut - 256 x 4096 x 4096
      // 34.7 -> 33.7 us, 34.3 before there were pieces -; the larger ones lose 0.5 % by it)
      constexpr int CUT = MI * NJ <= 4 ? 4 : RP / RS;
#pragma unroll CUT
      for (int it = 0; it < RP / RS; ++it) {
        const u32x4 v = *reinterpret_cast<const u32x4 *>(src + it * RS * PITCH);
        if (cols_left > 0 && row_in(p * RP + it * RS)) store_piece<S>(rowp + it * RS * row_bytes + lane_off, v, cols_left);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

// The same with what BIAS_EPILOGUE adds.  The sums are staged in 32 bits, 32 rows of the wave at a time, and everything else happens where the rows leave: a
// lane has the same columns in all rows, so that its bias stays in registers, and it reads the residual in the 16 bytes that it stores, one pass ahead.  The passes are
// a loop, in which only the staging is written out for each: what follows, three times for the activations, is most of the code.
template <int OUT_DT, int MI, int NJ, int LDS_BYTES>
__device__ __forceinline__ void store_tile_epilogue(const f32x16 (&acc)[MI][NJ], char *lds, const LinearArgs &a, float scale, int64_t m0, int64_t n0) {
  using DE = Elem<OUT_DT>;
  using DT = typename DE::T;
  constexpr int S = sizeof(DT), V = 16 / S, WN = 32 * NJ, RP = 32;
  constexpr int PITCH = WN * 4 + 16;
  static_assert(4 * RP * PITCH <= LDS_BYTES, "epilogue staging must fit in LDS");
  constexpr int CPR = WN / V, RS = 64 / CPR, IT = RP / RS;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  const int lrow = lane / CPR, lq = lane % CPR;
  char *stg = lds + wave * (RP * PITCH);
  const int64_t n = n0 + lq * V;
  const int64_t cl = a.N - n;
  const int cols = cl > V ? V : (int)cl;  // columns of this lane's piece inside the matrix
  const int64_t rl = a.M - m0 - lrow;
  const int rows_left = cols <= 0 ? 0 : rl > 32 * MI ? 32 * MI : (int)rl;  // rows of the block below this lane's first one
  const bool interior = m0 + 32 * MI <= a.M && n0 + WN <= a.N;
  float bias[V];
#pragma unroll
  for (int q = 0; q < V; ++q) bias[q] = a.ep.bias && q < cols ? epilogue_bias(a.ep, n + q) : 0.0f;
  const char *res = static_cast<const char *>(a.ep.residual) + ((m0 + lrow) * a.ep.residual_stride + n) * S;
  const int64_t res_step = RS * a.ep.residual_stride * S, out_step = RS * a.N * S;
  char *out = static_cast<char *>(a.D) + ((m0 + lrow) * a.N + n) * S;
  u32x4 ahead[IT];
  auto fetch = [&](int row0) {  // the residual of the pass from row0 on
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      const char *p = res + it * res_step;
      if (interior || (row0 + it * RS < rows_left && cols == V)) {
        ahead[it] = *reinterpret_cast<const u32x4_elem *>(p);
      } else if (row0 + it * RS < rows_left) {
        ahead[it] = (u32x4){0, 0, 0, 0};
#pragma unroll
        for (int q = 0; q < V; ++q)
          if (q < cols) {
            if constexpr (S == 4) ahead[it][q] = reinterpret_cast<const uint32_t *>(p)[q];
            else ahead[it][q / 2] |= (uint32_t)reinterpret_cast<const uint16_t *>(p)[q] << (16 * (q & 1));
          }
      }
    }
    res += IT * res_step;
  };
  if (a.ep.residual) fetch(0);
  auto stage = [&](auto index) {
    constexpr int i = decltype(index)::value;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if constexpr (MI * NJ == 16) asm volatile("v_accvgpr_read_b32 %0, %1" : "=v"(v[q]) : "a"(acc[i][j][4 * g + q]));  // (see store_tile)
          else v[q] = acc[i][j][4 * g + q];
        }
        *reinterpret_cast<float4 *>(stg + (lane & 31) * PITCH + (j * 32 + g * 8 + half * 4) * 4) = make_float4(v[0] * scale, v[1] * scale, v[2] * scale, v[3] * scale);
      }
  };
  const float4 *src = reinterpret_cast<const float4 *>(stg + lrow * PITCH + lq * V * 4);
  constexpr int UNROLL = MI * NJ == 16 ? 1 : MI;
#pragma unroll UNROLL
  for (int pass = 0; pass < MI; ++pass) {
    if (pass == 0) stage(std::integral_constant<int, 0>{});
    else if (pass == 1) stage(std::integral_constant<int, 1 % MI>{});
    else if (pass == 2) stage(std::integral_constant<int, 2 % MI>{});
    else stage(std::integral_constant<int, 3 % MI>{});
    u32x4 now[IT];
    if (a.ep.residual) {
#pragma unroll
      for (int it = 0; it < IT; ++it) now[it] = ahead[it];
      if (pass + 1 < MI) fetch((pass + 1) * RP);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the staging block is private to the wave
    with_activation(a.ep.activation, [&](auto act) {
#pragma unroll
      for (int it = 0; it < IT; ++it) {
        float v[V];
#pragma unroll
        for (int q = 0; q < V; q += 4) {
          const float4 f = src[(it * RS * PITCH) / 16 + q / 4];
          v[q] = f.x, v[q + 1] = f.y, v[q + 2] = f.z, v[q + 3] = f.w;
        }
#pragma unroll
        for (int q = 0; q < V; ++q) v[q] = act(v[q] + bias[q]);
        if (a.ep.residual) {
          DT r[V];
          __builtin_memcpy(r, &now[it], 16);
#pragma unroll
          for (int q = 0; q < V; ++q) v[q] += DE::load(r, q);
        }
        u32x4 o;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if constexpr (S == 2) o[q] = DE::cvt2(v[2 * q], v[2 * q + 1]);
          else o[q] = __float_as_uint(v[q]);
        }
        if (interior) *reinterpret_cast<u32x4_elem *>(out + it * out_step) = o;
        else if (pass * RP + it * RS < rows_left) store_piece<S>(out + it * out_step, o, cols);
      }
    });
    out += IT * out_step;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
}

// MI = 32-row fragments that a wave stores along M: 4 (BM = 256), 3 (BM = 192) or 2 (BM = 128);
// NJ = 32-column fragments that a wave stores along N: 4 (BN = 256), 2 (BN = 128) or 1 (BN = 64);
// KW = waves that share the K of a stage; with two of them a wave multiplies twice as many fragments along one side (WI x WJ);
// PS = LDS stages: PS - 1 k-steps (KW == 2: PS) are in flight ahead of the one being multiplied, which a small
// tile needs because its k-step is much shorter than the memory latency.
// Where the rows of a tile are.  In one matrix: first = the tile's index times its height.  GROUPED: first is a multiple of four (the scales of four
// rows are one transfer), and rows in front of `lo` are another group's; with `rows`, row i of the tile's matrix is row rows[i] of a.A,
// clamped to its a_rows rows; a.A_sf is that of a.A in tiles of 64 rows, and has a column for each i already in larger ones.
struct TileRows {
  int64_t first, lo;
  const int32_t *rows;
  int64_t a_rows;
};
template <int D_DT, int BIAS_DT, int MI, int NJ, int PS, int KW, bool EARLY, bool GROUPED>
__device__ __forceinline__ void tile256p(const LinearArgs &a, const SplitK &sk, char *plds, const TileRows &tr, int64_t tn) {
  constexpr int BM = 64 * MI, BN = 64 * NJ;  // two waves along M, two along N
  using PL = PLayout<BM, BN, PS>;
  constexpr int NDA = BM / 4 / 16;         // 16-row A transfers per wave per stage
  constexpr int NDB = BN / 4 / 16;         // 16-row B transfers per wave per stage
  constexpr int NPIECES = NDA + NDB + 1;   // and one of scales
  const int64_t m_first = tr.first;

  // KW == 2: the pair of waves (WI > MI: 0 and 2, 1 and 3; WJ > NJ: 0 and 1, 2 and 3) multiplies the blocks of both
  constexpr bool PAIR_M = KW == 2 && MI < NJ, PAIR_N = KW == 2 && !PAIR_M;
  constexpr int WI = PAIR_M ? 2 * MI : MI, WJ = PAIR_N ? 2 * NJ : NJ;  // fragments that a wave multiplies
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wm = PAIR_M ? 0 : wave >> 1, wn = PAIR_N ? 0 : wave & 1;
  const int half = lane >> 5;
  // this workgroup's range of 128-k stages; `early`: bytes by which they start in front of the row
  const int nkt_all = (int)(EARLY ? ceil_div(a.K, P_BK) : a.K / P_BK);
  constexpr int early = EARLY ? 32 : 0;
  const StageRange range = stage_range(nkt_all, blockIdx.y, sk.splits);
  const int kt0 = range.first, nkt = range.count;

  // LDS-DMA.  One transfer moves 16 rows x 64 B: the four lanes 4r .. 4r+3 read the four 16-byte
  // pieces of row r (one 64-byte sector) and land at LDS base + 16*l, i.e. row-major 64-byte rows.
  // Piece p of row r sits at position p ^ ((r >> 1) & 3) of its row: a fragment read takes one piece
  // of each of 32 rows, and unswizzled those addresses fall on a quarter of the LDS banks (an
  // eight-way conflict on every ds_read_b128).  The 32-bit lane offset is loop invariant and the
  // 64-bit part is a scalar base that advances by 64 bytes per stage.
  const int dma_piece = (lane & 3) ^ ((lane >> 3) & 3);  // tile rows of a transfer start at a multiple of 16
  const int swave = __builtin_amdgcn_readfirstlane(wave);
  const int64_t kb = a.K >> 1;
  uint32_t offA[NDA], offB[NDB];
#pragma unroll
  for (int q = 0; q < NDA; ++q) {
    int64_t ra = (swave * NDA + q) * 16 + (lane >> 2);
    ra = m_first + ra < a.M ? ra : a.M - 1 - m_first;  // rows past the matrix read the last valid row
    if (GROUPED && tr.rows) {
      const int64_t row = tr.rows[m_first + ra];
      ra = row < 0 ? 0 : row < tr.a_rows ? row : tr.a_rows - 1;
    }
    offA[q] = (uint32_t)(ra * kb + dma_piece * 16);
  }
  // weight image: a transfer's 16 rows are one contiguous kilobyte of a block (the swizzle is part of
  // the image); bands past the last one read the last band, whose outputs are never stored
  const int64_t w_band_bytes = (int64_t)nkt_all * W_BLOCK_BYTES, w_last_band = (a.N - 1) / W_BLOCK_ROWS;
  auto w_band_of = [&](int64_t row, int64_t &within) {
    int64_t band = row / W_BLOCK_ROWS;
    within = row % W_BLOCK_ROWS;
    return band < w_last_band ? band : w_last_band;
  };
#pragma unroll
  for (int q = 0; q < NDB; ++q) {
    if (a.prepacked) {
      int64_t within;
      const int64_t band = w_band_of(tn * BN + (swave * NDB + q) * 16, within);
      offB[q] = (uint32_t)(band * w_band_bytes + within * P_ROW + lane * 16);
    } else {
      int64_t rb = (swave * NDB + q) * 16 + (lane >> 2);
      rb = tn * BN + rb < a.N ? rb : a.N - 1 - tn * BN;
      offB[q] = (uint32_t)(rb * kb + dma_piece * 16);
    }
  }
  const int64_t strideB = a.prepacked ? W_BLOCK_BYTES : P_ROW;  // bytes per stage along k
  const uint8_t *baseA = uniform_ptr(a.A + (GROUPED && tr.rows ? 0 : m_first * kb) + (int64_t)kt0 * P_ROW - early);
  const uint8_t *baseB = uniform_ptr(a.prepacked ? a.B + (int64_t)kt0 * W_BLOCK_BYTES : a.B + tn * BN * kb + (int64_t)kt0 * P_ROW - early);
  // scales: a transfer is 256 dwords of the [chunk][row] picture of an operand, a lane four rows of a chunk (16 bytes; the address is on
  // four).  Waves 0 .. NSA - 1 move those of A, the others those of B; a wave past the last transfer repeats the last one, and so do
  // lanes past the picture's end with rows of its last chunk, into the rest of the kilobyte.  (A dword per lane, up to four transfers a wave, cost
  // the loop of 192 x 128 tiles 377 of its 2420 cycles a stage.)
  uint32_t offS, ldsS;
  const uint8_t *baseS;
  int64_t strideS;
  bool firstS;  // this lane's rows belong to the first chunk of a stage
  // Gathered rows of a tile of 64: their scales are not neighbours, and come a dword per lane, the two chunks by waves 0 and 1; those of B by the
  // waves behind them, so that it stays one transfer a wave.
  constexpr bool OWN_SCALES = GROUPED && MI == 1;
  bool dword_scales = false;
  if (OWN_SCALES && tr.rows) {
    static_assert(!OWN_SCALES || 2 + PL::NSB <= 4, "a scale transfer per wave");
    const int t = swave < 2 + PL::NSB ? swave : 1 + PL::NSB;
    dword_scales = t < 2;
    int64_t row;
    int c;
    if (dword_scales) {
      c = t;
      int64_t i = m_first + lane;
      i = tr.rows[i < a.M ? i : a.M - 1];
      row = i < 0 ? 0 : i < tr.a_rows ? i : tr.a_rows - 1;
    } else {
      const int at = (t - 2) * 256 + lane * 4;
      c = at >= BN ? 1 : 0;
      const int loc = at < 2 * BN ? at - c * BN : 0;
      row = tn * BN + loc + 4 <= a.Np ? tn * BN + loc : a.Np - 4;
    }
    const int64_t rows = dword_scales ? a.Mp : a.Np;
    firstS = c == 0;
    offS = (uint32_t)((c * rows + row) * 4);
    strideS = (int64_t)uniform_ptr((const void *)(2 * rows * 4));
    baseS = uniform_ptr(reinterpret_cast<const uint8_t *>(dword_scales ? a.A_sf : a.B_sf) - (EARLY ? rows : 0) * 4 + kt0 * strideS);
    ldsS = (uint32_t)__builtin_amdgcn_readfirstlane(dword_scales ? PL::OFF_SFA + t * (BM * 4) : PL::OFF_SFB + (t - 2) * 1024);
  } else {
    const int t = swave < PL::NSA + PL::NSB ? swave : PL::NSA + PL::NSB - 1;
    const bool isB = t >= PL::NSA;
    const int tt = isB ? t - PL::NSA : t, rows_t = isB ? BN : BM;
    const int at = tt * 256 + lane * 4, c = at >= rows_t ? 1 : 0;
    const int loc = at < 2 * rows_t ? at - c * rows_t : 0;
    const int64_t rows = isB ? a.Np : a.Mp, first = isB ? tn * BN : m_first;
    firstS = c == 0;
    if (isB && a.prepacked) {  // the scale dwords follow the packed rows of the block
      int64_t within;
      const int64_t band = w_band_of(first + loc, within);
      offS = (uint32_t)(band * w_band_bytes + W_BLOCK_DATA + c * (W_BLOCK_ROWS * 4) + within * 4);
      strideS = W_BLOCK_BYTES;
      baseS = uniform_ptr(a.B + (int64_t)kt0 * W_BLOCK_BYTES);
    } else {
      const int64_t row = first + loc + 4 <= rows ? loc : rows - 4 - first;  // (rows are padded to 16)
      offS = (uint32_t)((c * rows + row) * 4);
      strideS = 2 * rows * 4;  // two planes (chunks) per stage
      baseS = uniform_ptr(reinterpret_cast<const uint8_t *>(isB ? a.B_sf : a.A_sf) + (first - (EARLY ? rows : 0)) * 4 + kt0 * strideS);
    }
    strideS = (int64_t)uniform_ptr((const void *)strideS);
    ldsS = (uint32_t)__builtin_amdgcn_readfirstlane((isB ? PL::OFF_SFB : PL::OFF_SFA) + tt * 1024);
  }
  const uint32_t lds_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)plds;
  // LDS destinations of this wave's transfers inside a stage (wave-uniform, loop invariant)
  uint32_t ldsA[NDA], ldsB[NDB];
#pragma unroll
  for (int q = 0; q < NDA; ++q) ldsA[q] = (uint32_t)__builtin_amdgcn_readfirstlane((swave * NDA + q) * 1024);
#pragma unroll
  for (int q = 0; q < NDB; ++q) ldsB[q] = (uint32_t)__builtin_amdgcn_readfirstlane(PL::OFF_B + (swave * NDB + q) * 1024);
  // Source pointers of the k-step being fetched.  They advance by one step per iteration and stop
  // at the last step of the range: fetches past the end re-read the last slice into a stage buffer
  // nobody reads again, which keeps the main loop free of branches.
  struct Src {
    const uint8_t *a, *b, *s;
  };
  auto src_at = [&](int kt) {
    Src p;
    p.a = baseA + (int64_t)kt * P_ROW;
    p.b = baseB + (int64_t)kt * strideB;
    p.s = baseS + kt * strideS;
    return p;
  };
  auto issue_scales = [&](uint32_t stage_lds, const uint8_t *src, uint32_t off) {
    if (OWN_SCALES && dword_scales) dma4(src, off, stage_lds, ldsS);
    else dma16(src, off, stage_lds, ldsS);
  };
  auto issue_piece = [&](uint32_t stage_lds, const Src &p, int q) {
    if (q < NDA) {
      dma16(p.a, offA[q], stage_lds, ldsA[q]);
    } else if (q < NDA + NDB) {
      dma16(p.b, offB[q - NDA], stage_lds, ldsB[q - NDA]);
    } else {
      issue_scales(stage_lds, p.s, offS);
    }
  };
  auto issue_stage = [&](uint32_t stage_lds, const Src &p) {
#pragma unroll
    for (int q = 0; q < NPIECES; ++q) issue_piece(stage_lds, p, q);
  };
  TileWave<WI, WJ> w;
  w.clear();

  // fragment addresses inside a stage (bytes)
  // (a lane's rows differ by multiples of 32, so the swizzle term of its row is (lane >> 1) & 3 for all of them)
  const int fa_off = (wm * (32 * MI) + (lane & 31)) * P_ROW;
  const int fb_off = PL::OFF_B + (wn * (32 * NJ) + (lane & 31)) * P_ROW;
  const int piece_off[2] = {((0 + half) ^ ((lane >> 1) & 3)) * 16, ((2 + half) ^ ((lane >> 1) & 3)) * 16};  // chunk 0, chunk 1
  // KW == 2: the chunk of every stage that this wave multiplies; its first MI x NJ fragments are the ones that it will keep, behind
  // them those of the other wave of the pair, so that no register is chosen at run time
  const int kw = PAIR_M ? swave >> 1 : swave & 1;
  auto row_a = [&](int i) { return 32 * (PAIR_M ? (i < MI ? kw * MI : (1 - kw) * MI) + i % MI : i); };
  auto row_b = [&](int j) { return 32 * (PAIR_N ? (j < NJ ? kw * NJ : (1 - kw) * NJ) + j % NJ : j); };
  // a lane needs the two scale bytes of its half of the chunk: blocks 2*half, 2*half+1
  const int sa_off = PL::OFF_SFA + (wm * (32 * MI) + (lane & 31)) * 4 + half * 2;
  const int sb_off = PL::OFF_SFB + (wn * (32 * NJ) + (lane & 31)) * 4 + half * 2;

  // read r of a chunk into set `set` (by chunk parity, KW == 2 by stage parity): the packed fragments, then the scale bytes
  constexpr int NF = WI + WJ, NM = WI * WJ;
  auto load_item = [&](uint32_t stage_off, int c, int set, int r) {
    const char *st = plds + stage_off;
    const int f = r % NF;
    if (r < NF) {
      const int piece = KW == 2 ? (kw ? piece_off[1] : piece_off[0]) : piece_off[c];
      w.packed[set][f] = *reinterpret_cast<const uint4 *>(st + piece + (f < WI ? fa_off + row_a(f) * P_ROW : fb_off + row_b(f - WI) * P_ROW));
    } else {
      w.sf[set][f] = *reinterpret_cast<const uint16_t *>(st + (f < WI ? sa_off + c * (BM * 4) + row_a(f) * 4 : sb_off + c * (BN * 4) + row_b(f - WI) * 4));
    }
  };

  // prologue: stages 0 .. PS-2 (KW == 2: PS-1) in flight (past the last k-step: the last one again), stage 0
  // visible, the wave's first fragments and first decode
  constexpr int AHEAD = KW == 2 ? PS : PS - 1;
  static_assert(PS >= 3 && (AHEAD - 1) * NPIECES <= 63, "the wait counts below must fit the 6-bit counter");
  const int last = nkt - 1;
  // the stage that fetches past the end repeat: never the short one, whose first half lies in front of the rows
  // (a range of one stage then repeats the stage behind it, which exists: K >= 192)
  const bool short0 = EARLY && kt0 == 0;
  const int again = short0 && last == 0 ? 1 : last;
  {  // stage 0; a short one takes k-chunk 0 into both halves, by its addresses
    Src p = src_at(0);
    const uint32_t shift = short0 && dma_piece < 2 ? 32u : 0u;
#pragma unroll
    for (int q = 0; q < NDA; ++q) dma16(p.a, offA[q] + shift, lds_base, ldsA[q]);
#pragma unroll
    for (int q = 0; q < NDB; ++q) dma16(p.b, offB[q] + shift, lds_base, ldsB[q]);
    issue_scales(lds_base, p.s, offS + (short0 && firstS ? (uint32_t)(strideS / 2) : 0));
  }
  // A range shorter than the ring is fetched as it is and waited for as a whole: its repeats would be most of a short prologue
  // (10650 x 512 x 384 11.4 -> 10.9 us).
  const bool brief = nkt < AHEAD;
#pragma unroll
  for (int d = 1; d < AHEAD; ++d)
    if (!brief || d < nkt) issue_stage(lds_base + d * PL::STAGE_BYTES, src_at(d < last ? d : again));
  if (brief) wait_vmcnt<0>();
  else wait_vmcnt<(AHEAD - 1) * NPIECES>();  // everything of stage 0 has landed, later stages may be in flight
  __syncthreads();
#pragma unroll
  for (int r = 0; r < 2 * NF; ++r) load_item(0, KW == 2 ? kw : 0, 0, r);
  if (short0 && (KW == 1 || kw == 0)) {
#pragma unroll
    for (int f = 0; f < NF; ++f) w.sf[0][f] = 0;
  }
#pragma unroll
  for (int e = 0; e < 4 * NF; ++e) w.decode_item(0, 0, 0, e);
  if constexpr (KW == 2) {  // stage 1 landed, and everybody's fragments of stage 0 in registers
    wait_vmcnt<(AHEAD - 2) * NPIECES>();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __syncthreads();
  }

  // loop-carried, wave-uniform: LDS offsets of the stages holding k-steps kt, kt+1 and of the one
  // being filled with kt+AHEAD (a ring of PS), and the source pointers of k-step min(kt+AHEAD, last)
  uint32_t st_cur = 0, st_nxt = PL::STAGE_BYTES, st_dma = (PS - 1) * PL::STAGE_BYTES;
  auto ring_next = [](uint32_t o) { return o + PL::STAGE_BYTES == (uint32_t)PL::LDS_BYTES ? 0u : o + PL::STAGE_BYTES; };
  Src src = src_at(last < AHEAD ? again : AHEAD);
  auto advance = [&](int kt) {  // the sources, unless they already sit on the last k-step
    const bool adv = kt + AHEAD < last;
    src.a += adv ? P_ROW : 0;
    src.b += adv ? strideB : 0;
    src.s += adv ? strideS : 0;
  };
#ifdef AC4K_LINEAR_TIMELINE
  const uint64_t tl_c0 = __builtin_readcyclecounter();
#endif
  AC4K_LTL(1, wall_clock64());
  // KW == 2: a step multiplies chunk kw of stage kt out of registers (set kt & 1) while that of stage kt+1, which landed before
  // the last barrier, travels to the other set, and stage kt+PS to the ring slot of stage kt
  auto pair_step = [&](int kt, int cur) {
    const uint32_t dma_lds = lds_base + st_cur;
#pragma unroll
    for (int s = 0; s < 4; ++s)
      w.substep(s & 1, s < 3 ? cur : 1 - cur, (s + 1) & 3, [&](int m) {
        if (s < 3) deal<2 * NF, 3 * NM>(s * NM + m, [&](int r) { load_item(st_nxt, kw, 1 - cur, r); });  // past the end this reads a stale stage; the result is never used
        deal<NPIECES, 4 * NM>(s * NM + m, [&](int q) { issue_piece(dma_lds, src, q); });
      });
    wait_vmcnt<(PS - 2) * NPIECES>();                   // own transfers of stage kt+2 have landed
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // and the fragments of stage kt+1 are in registers
    __syncthreads();
    st_cur = st_nxt;
    st_nxt = ring_next(st_nxt);
    advance(kt);
  };
  if constexpr (KW == 2) {  // (nkt >= 1: splits <= stages)
    int kt = 0;
    do {
      pair_step(kt, 0);
      if (kt + 1 < nkt) pair_step(kt + 1, 1);
      kt += 2;
    } while (kt < nkt);
  }
  for (int kt = 0; KW == 1 && kt < nkt; ++kt) {
    // chunk 0: sub-steps 0..3 (fragments of chunk 1 are fetched meanwhile)
#pragma unroll
    for (int s = 0; s < 4; ++s)
      w.substep(s & 1, s < 3 ? 0 : 1, (s + 1) & 3, [&](int m) {
        if (s < 3) deal<2 * NF, 3 * NM>(s * NM + m, [&](int r) { load_item(st_cur, 1, 1, r); });
      });
    // stage kt+1 must be complete (own DMA done, then everybody's; stages kt+2 .. kt+PS-2 may still
    // be in flight); stage kt-1 is free after this
    wait_vmcnt<(PS - 3) * NPIECES>();
    __syncthreads();
    // chunk 1: sub-steps 4..7 (chunk 0 of the next stage is fetched meanwhile); the DMA of stage
    // kt+PS-1 is spread over these sub-steps
    const uint32_t dma_lds = lds_base + st_dma;
#pragma unroll
    for (int s = 0; s < 4; ++s)
      w.substep(s & 1, s < 3 ? 1 : 0, (s + 1) & 3, [&](int m) {
        if (s < 3) deal<2 * NF, 3 * NM>(s * NM + m, [&](int r) { load_item(st_nxt, 0, 0, r); });  // past the end this reads a stale stage; the result is never used
        deal<NPIECES, 4 * NM>(s * NM + m, [&](int q) { issue_piece(dma_lds, src, q); });
      });
    st_cur = st_nxt;
    st_nxt = ring_next(st_nxt);
    st_dma = ring_next(st_dma);
    advance(kt);
  }
  AC4K_LTL(2, wall_clock64());
#ifdef AC4K_LINEAR_TIMELINE
  AC4K_LTL(4, __builtin_readcyclecounter() - tl_c0);
  {
    uint32_t xcc, hwid;
    asm volatile("s_getreg_b32 %0, hwreg(HW_REG_XCC_ID)" : "=s"(xcc));
    asm volatile("s_getreg_b32 %0, hwreg(HW_REG_HW_ID)" : "=s"(hwid));
    AC4K_LTL(5, (xcc & 0xf) | (hwid << 8));
  }
#endif

  // ---- epilogue.  The MFMAs were issued with the operands swapped, so acc[i][j] holds the
  // TRANSPOSED 32x32 block: lane l, element e <-> n = j*32 + (e>>2)*8 + (l>>5)*4 + (e&3),
  // m = i*32 + (l&31): four consecutive n per lane.
  const int64_t m0 = m_first + (swave >> 1) * (32 * MI), n0 = tn * BN + (swave & 1) * (32 * NJ);
  // the last iterations' LDS-DMA fetches (into a stage nobody reads) must have landed before the
  // stages are reused, and every wave must be done reading them
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  auto store = [&](const f32x16 (&sums)[MI][NJ]) {
    if (!GROUPED && sk.partial) {  // split-K: raw fp32 sums of this K range; the reduce kernel scales and converts
      store_tile<AC4K_DTYPE_FP32, BIAS_NONE, true, MI, NJ, PL::LDS_BYTES, false>(
          sums, plds, sk.partial + (int64_t)blockIdx.y * a.M * a.N, nullptr, 1.0f, a.M, a.N, m0, n0, tn * BN, 0);
    } else if constexpr (BIAS_DT == BIAS_EPILOGUE) {
      store_tile_epilogue<D_DT, MI, NJ, PL::LDS_BYTES>(sums, plds, a, (*a.A_gs) * (*a.B_gs), m0, n0);
    } else {
      store_tile<D_DT, BIAS_DT, false, MI, NJ, PL::LDS_BYTES, GROUPED>(sums, plds, a.D, a.bias, (*a.A_gs) * (*a.B_gs), a.M, a.N,
                                                             m0, n0, tn * BN, tr.lo);
    }
  };
  const auto &acc = w.acc;
  if constexpr (KW == 1) {
    store(acc);
  } else {
    // the waves of a pair exchange halves of their blocks and add them: wave (wm, wn) of the 2 x 2 grid keeps its own
    static_assert(4 * MI * NJ * 4096 <= PL::LDS_BYTES, "the exchanged halves must fit in LDS");
    float4 *xch = reinterpret_cast<float4 *>(plds) + lane;
    auto xch_at = [&](int w, int i, int j, int g) { return xch + ((w * MI * NJ + i * NJ + j) * 4 + g) * 64; };
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x16 &o = acc[PAIR_M ? MI + i : i][PAIR_N ? NJ + j : j];
          *xch_at(swave ^ (PAIR_M ? 2 : 1), i, j, g) = make_float4(o[4 * g], o[4 * g + 1], o[4 * g + 2], o[4 * g + 3]);
        }
    __syncthreads();
    f32x16 sums[MI][NJ];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const float4 t = *xch_at(swave, i, j, g);
          sums[i][j][4 * g] = acc[i][j][4 * g] + t.x;
          sums[i][j][4 * g + 1] = acc[i][j][4 * g + 1] + t.y;
          sums[i][j][4 * g + 2] = acc[i][j][4 * g + 2] + t.z;
          sums[i][j][4 * g + 3] = acc[i][j][4 * g + 3] + t.w;
        }
    __syncthreads();  // what follows lies over the halves
    store(sums);
  }
}

// Raises a kernel's dynamic LDS limit once per (kernel instantiation, device): the attribute belongs
// to the device the call is made on.
template <typename Kernel>
static int allow_dynamic_lds(Kernel *kern, std::atomic<uint32_t> &done_mask, int bytes) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) dev = 0;
  const uint32_t bit = 1u << (dev & 31);
  if (done_mask.load(std::memory_order_relaxed) & bit) return 0;
  hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != hipSuccess) return set_error("hipFuncSetAttribute(LDS=%d): %s", bytes, hipGetErrorString(e));
  done_mask.fetch_or(bit, std::memory_order_relaxed);
  return 0;
}

// LDS stages per tile shape: enough k-steps in flight to cover the memory latency
constexpr int tile_stages(int mi, int nj, int kw) { return mi * nj >= 16 ? 3 : mi * nj > 8 ? 4 : mi * nj == 8 ? 3 + kw : mi * nj >= 4 ? 6 : 8; }

}  // namespace ac4k

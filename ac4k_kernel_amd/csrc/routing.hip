// Routing of tokens to experts with the plan that the grouped linears read, and the weighted return of the experts' rows to their tokens.
//
//   score_e = exp(l_e) / sum exp(l), or 1 / (1 + exp(-l_e))      key_e = score_e + bias_e
// A token takes the `k` experts of largest key, ties to the lowest index; with groups only those of the `top_groups` groups whose `best` (1 or 2)
// largest keys have the largest sum.  An expert whose logit or key is -inf is never taken; a NaN counts as the largest key.  weight = score, over the sum of the
// chosen ones with renormalize, times scale.
//
// Without a bias and without sums of two keys the order of the keys is that of the logits, which are compared as they are: no rounding decides.
// Otherwise scores and keys are held in 64 bits, so that keys next to each other are told apart as the formula does.
//
// The plan is a counting sort by expert that keeps the order of the tokens: a block of 16 tokens keeps, for each expert, the set of its tokens as bits;
// counts of the blocks in front and bits below a token's own are its place.  Bits are set by atomic ors, whose order does not matter, so every
// call gives the same plan.
//
// Bound by launches and by vector instructions, not by bytes: 16 tokens of 64 experts 3.7 us in one workgroup; 16384 tokens to 4 of 128 experts 6.0 + 7.1 us (choice, plan)
// where 5.2 MB of bytes need one; 4001 to 8 of 256 with groups and a bias 11.1 + 6.7: 940 vector instructions a wave, a third of them the choice's eight rounds, a
// quarter scores in 64 bits (the port busy for 72 %).  Scores in 64 bits take 2.3 us there, each round 0.35 to 0.43.
#include "elements.h"

namespace ac4k {

struct RouteArgs {
  const void *logits;
  int64_t stride;           // elements between rows
  const float *bias;        // or null
  float *weights;           // [T, k]
  int32_t *experts;         // [T, k]
  int32_t *offsets;         // [E + 1]
  int32_t *rows;            // [T * k]
  int32_t *places;          // [T, k]
  uint16_t *masks;          // [blocks, Ep]: tokens of the block that take the expert; rows of whole vectors
  uint8_t *counts;          // [blocks, Ep]: how many
  int32_t *bases;           // [blocks, E]: rows of the expert in front of the block
  int32_t *totals;          // [E]
  int64_t T, blocks;
  int E, Ep, k, groups, top_groups, best, group_size, group_lanes;
  bool sigmoid, renormalize;
  double scale;
};

constexpr int ROUTE_TOKENS = 16;        // of a block
constexpr int ROUTE_ROW_EXPERTS = 128;  // up to so many, without groups and up to 16 a token, 16 lanes take a token; otherwise a wave
static int route_lanes(int64_t E, int64_t k, int64_t groups) { return groups == 1 && k <= 16 && E <= ROUTE_ROW_EXPERTS ? 16 : 64; }
// Tokens of a call that one workgroup takes: 128 to 8 of 64 experts 9.4 us on the GPU and 13.4 for the caller, where two launches of 129 need 8.2 and 17.3;
// 256 would need 16.8 and 16.8.
constexpr int route_one_tokens(int lanes) { return lanes == 16 ? 128 : 64; }
constexpr int ROUTE_PLAN_BLOCKS = 16;   // of a workgroup that makes the plan in one launch, where all of them read at most so many counts
constexpr int64_t ROUTE_PLAN_COUNTS = 1 << 25;
constexpr int ROUTE_SCAN_EXPERTS = 16;  // of a workgroup of the scan

// Floats and doubles as unsigned numbers of the same order; 0 is -inf (not to be taken), all ones NaN
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);  // -0 is 0
  uint32_t k = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
  k = x == -__builtin_inff() ? 0u : k;
  return x != x ? 0xffffffffu : k;
}
__device__ __forceinline__ float unordered(uint32_t k) {
  return k == 0u ? -__builtin_inff() : k == 0xffffffffu ? __builtin_nanf("") : __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ uint64_t ordered(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x + 0.0);
  uint64_t k = b ^ ((uint64_t)((int64_t)b >> 63) | 0x8000000000000000ull);
  k = x == -__builtin_inf() ? 0ull : k;
  return x != x ? ~0ull : k;
}
__device__ __forceinline__ double unordered(uint64_t k) {
  return k == 0ull ? -__builtin_inf() : k == ~0ull ? __builtin_nan("") : __builtin_bit_cast(double, k >> 63 ? k & 0x7fffffffffffffffull : ~k);
}

// what the lane at the other end of a step of a reduction holds
template <int STEP, typename U>
__device__ __forceinline__ U lane_step(U v) {
  auto move = [](uint32_t w) {
    if constexpr (STEP == 1) return dpp_u32<DPP_QUAD_XOR1>(w);
    else if constexpr (STEP == 2) return dpp_u32<DPP_QUAD_XOR2>(w);
    else if constexpr (STEP == 4) return dpp_u32<DPP_ROW_HALF_MIRROR>(w);
    else if constexpr (STEP == 8) return dpp_u32<DPP_ROW_MIRROR>(w);
    else if constexpr (STEP == 16) return (uint32_t)__builtin_amdgcn_ds_swizzle((int)w, 0x401F);
    else return (uint32_t)__shfl_xor((int)w, 32);
  };
  if constexpr (sizeof(U) == 4) {
    return __builtin_bit_cast(U, move(__builtin_bit_cast(uint32_t, v)));
  } else {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(U, (uint64_t)move((uint32_t)(b >> 32)) << 32 | move((uint32_t)b));
  }
}
// reduction over aligned groups of `lanes` (a power of two, the same in the whole wave), in every lane of the group; MOST: of any call
template <int MOST, typename U, typename F>
__device__ __forceinline__ U lanes_reduce(U v, int lanes, F f) {
  if (lanes > 1) v = f(v, lane_step<1>(v));
  if (lanes > 2) v = f(v, lane_step<2>(v));
  if (lanes > 4) v = f(v, lane_step<4>(v));
  if (lanes > 8) v = f(v, lane_step<8>(v));
  if constexpr (MOST > 16) {
    if (lanes > 16) v = f(v, lane_step<16>(v));
    if (lanes > 32) v = f(v, lane_step<32>(v));
  }
  return v;
}

// The largest of a wave's unsigned numbers, a scalar: inside rows of 16 lanes, then the four rows.
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
  v = lanes_reduce<16>(v, 16, [](uint32_t p, uint32_t q) { return umax32(p, q); });
  const uint32_t a = (uint32_t)__builtin_amdgcn_readlane((int)v, 0), b = (uint32_t)__builtin_amdgcn_readlane((int)v, 16);
  const uint32_t c = (uint32_t)__builtin_amdgcn_readlane((int)v, 32), d = (uint32_t)__builtin_amdgcn_readlane((int)v, 48);
  return umax32(umax32(a, b), umax32(c, d));
}
// The largest key of the L lanes of a token and the lowest expert that has it, from each lane's largest key m and its expert e; experts rise with
// the lanes.  64-bit keys: the high words first, the low ones of those that share it.
template <int L, typename Key>
__device__ __forceinline__ Key choose(Key m, int e, int &taken) {
  if constexpr (L == 64) {
    const uint32_t hi = sizeof(Key) == 8 ? (uint32_t)((uint64_t)m >> 32) : (uint32_t)m;
    const uint32_t most = wave_umax(hi);
    uint64_t lanes = __ballot(hi == most);
    if constexpr (sizeof(Key) == 8) {
      if (lanes & (lanes - 1)) {
        const uint32_t lo = hi == most ? (uint32_t)m : 0u;
        lanes &= __ballot(lo == wave_umax(lo));
      }
    }
    taken = __builtin_amdgcn_readlane(e, __builtin_ctzll(lanes));
    return most;  // (of 64 bits the high ones: they are 0 for no allowed key)
  } else {
    const Key most = lanes_reduce<L>(m, L, [](Key p, Key q) { return p > q ? p : q; });
    taken = lanes_reduce<L>(m == most ? e : 0x7fffffff, L, [](int p, int q) { return p < q ? p : q; });
    return most;
  }
}

// One token on L lanes, PER experts each, the experts of a group in neighbouring lanes.  Lane s < k returns the token's s-th expert (-1: none) and its weight.
// All lanes of the wave take part; `valid` false: a token behind the last one.
template <int DT, int L, int PER, bool WIDE>
__device__ __forceinline__ void route_token(const RouteArgs &a, int64_t token, bool valid, int sub, int &my_expert, float &my_weight) {
  using Key = typename std::conditional<WIDE, uint64_t, uint32_t>::type;
  using T = typename Elem<DT>::T;
  const T *row = static_cast<const T *>(a.logits) + token * a.stride;
  const int lg = L == 64 ? a.group_lanes : L;  // (fewer lanes have one group)
  const int group = L == 64 ? sub / lg : 0, at = (sub - group * lg) * PER, e0 = group * a.group_size + at;
  float x[PER];
  const int here = valid && group < a.groups ? a.group_size - at : 0;
  if (here >= PER) {
    typedef T Run __attribute__((ext_vector_type(PER)));
    typedef Run RunElem __attribute__((aligned(sizeof(T))));  // global memory takes vector accesses at any address
    Run v;
    if constexpr (PER > 1) v = *reinterpret_cast<const RunElem *>(row + e0);
    else v[0] = row[e0];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const T one = v[j];
      x[j] = Elem<DT>::load(&one, 0);
    }
  } else {
#pragma unroll
    for (int j = 0; j < PER; ++j) x[j] = j < here ? Elem<DT>::load(row, e0 + j) : -__builtin_inff();
  }
  auto larger = [](Key p, Key q) { return p > q ? p : q; };
  auto add = [](double p, double q) { return p + q; };
  Key key[PER];
  float top;         // the largest logit
  double sum = 1.0;  // of the softmax
  if constexpr (WIDE) {
    double score[PER];
    if (a.sigmoid) {
#pragma unroll
      for (int j = 0; j < PER; ++j) score[j] = 1.0 / (1.0 + exp(-(double)x[j]));
      top = 0.0f;
    } else {
      top = x[0];
#pragma unroll
      for (int j = 1; j < PER; ++j) top = fmaxf(top, x[j]);
      top = lanes_reduce<L>(top, L, [](float p, float q) { return fmaxf(p, q); });
      sum = 0.0;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        score[j] = exp(x[j] == -__builtin_inff() ? -1000.0 : (double)x[j] - (double)top);  // (0 for an expert that is not allowed)
        sum += score[j];
      }
      sum = lanes_reduce<L>(sum, L, add);
      const double share = 1.0 / sum;
#pragma unroll
      for (int j = 0; j < PER; ++j) score[j] *= share;
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int e = e0 + j < a.E ? e0 + j : a.E - 1;
      const double v = a.bias ? score[j] + (double)a.bias[e] : score[j];
      key[j] = x[j] != -__builtin_inff() ? ordered(v) : 0;
    }
  } else {
    Key m = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      key[j] = ordered(x[j]);
      m = larger(m, key[j]);
    }
    top = unordered(lanes_reduce<L>(m, L, larger));
    if (!a.sigmoid && !a.renormalize) {
      float s = 0.0f;
#pragma unroll
      for (int j = 0; j < PER; ++j) s += x[j] == -__builtin_inff() ? 0.0f : expf(x[j] - top);
      sum = lanes_reduce<L>((double)s, L, add);
    }
  }
  // the lane's largest key and the expert that has it, the lowest one
  auto best_of = [&](const Key(&k)[PER], Key &m, int &e) {
    m = k[0], e = e0;
#pragma unroll
    for (int j = 1; j < PER; ++j)
      if (k[j] > m) m = k[j], e = e0 + j;
  };
  if (L == 64 && a.groups > 1) {
    Key m;
    int e;
    best_of(key, m, e);
    Key total = lanes_reduce<L>(m, lg, larger);
    if (WIDE && a.best == 2 && a.group_size > 1) {
      // the second one: the largest of all but the first
      const int first = lanes_reduce<L>(m == total ? e : 0x7fffffff, lg, [](int p, int q) { return p < q ? p : q; });
      Key second = 0;
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (e0 + j != first) second = larger(second, key[j]);
      second = lanes_reduce<L>(second, lg, larger);
      if constexpr (WIDE)
        if (second) total = ordered(unordered(total) + unordered(second));
    }
    int rank = 0;  // groups in front of this one
    for (int g = 0; g < a.groups; ++g) {
      Key other;
      if constexpr (WIDE)
        other = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(total >> 32), g * lg) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)total, g * lg);
      else
        other = (uint32_t)__builtin_amdgcn_readlane((int)total, g * lg);
      rank += other > total || (other == total && g < group) ? 1 : 0;
    }
    if (rank >= a.top_groups) {
#pragma unroll
      for (int j = 0; j < PER; ++j) key[j] = 0;
    }
  }
  my_expert = -1;
  float my_logit = 0.0f;
  for (int s = 0; s < a.k; ++s) {
    Key m;
    int e;
    best_of(key, m, e);
    int taken;
    const Key most = choose<L>(m, e, taken);
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (e0 + j == taken) key[j] = 0;
    if (sub == s && most != 0) {
      my_expert = taken;
      if constexpr (!WIDE) my_logit = unordered(most);
    }
  }
  double w = 0.0;
  if (my_expert >= 0) {
    if constexpr (WIDE) my_logit = Elem<DT>::load(row, my_expert);
    const double v = (double)my_logit;
    const double power = exp(a.sigmoid ? -v : v - (double)top);
    w = a.sigmoid ? 1.0 / (1.0 + power) : power / sum;
  }
  if (a.renormalize) {
    const double all = lanes_reduce<L>(w, L, add);
    w = all == 0.0 ? 0.0 : w / all;
  }
  my_weight = (float)(w * a.scale);
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

// The places of a block's tokens: `base` rows of expert e in front of the block (its range's start among them)
template <typename Base>
__device__ __forceinline__ void route_place(const RouteArgs &a, int64_t t, int slot, int e, uint64_t mask, int in_block, Base base) {
  const int64_t i = t * a.k + slot;
  int place = -1;
  if (e >= 0) {
    place = base(e) + __popcll(mask & ((1ull << in_block) - 1));
    a.rows[place] = (int32_t)t;
  }
  a.places[i] = place;
}

// Start of each expert's range from the counts in `count` [E] (LDS), in place, behind a barrier; returns the number of rows.  Whole workgroup.
template <int THREADS>
__device__ __forceinline__ int route_starts(int *count, int E, int *wave_sum) {
  constexpr int MOST = (AC4K_ROUTE_MAX_EXPERTS + THREADS - 1) / THREADS;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int c[MOST], sum = 0;
#pragma unroll
  for (int j = 0; j < MOST; ++j) {
    const int e = tid * MOST + j;
    c[j] = e < E ? count[e] : 0;
    sum += c[j];
  }
  int before = wave_prefix(sum);
  if (lane == 63) wave_sum[wave] = before;
  __syncthreads();
  int total = 0;
  before -= sum;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) {
    if (w < wave) before += wave_sum[w];
    total += wave_sum[w];
  }
#pragma unroll
  for (int j = 0; j < MOST; ++j) {
    const int e = tid * MOST + j;
    if (e < E) count[e] = before;
    before += c[j];
  }
  __syncthreads();
  return total;
}

// Scores, choice and weights of a block's tokens and the sets of its experts
template <int DT, int L, int PER, bool WIDE>
__global__ __launch_bounds__(ROUTE_TOKENS * L) void route_kernel(RouteArgs a) {
  __shared__ uint32_t mask[AC4K_ROUTE_MAX_EXPERTS];
  constexpr int THREADS = ROUTE_TOKENS * L;
  const int tid = threadIdx.x, sub = tid % L, b = tid / L;
  for (int e = tid; e < a.Ep; e += THREADS) mask[e] = 0;
  __syncthreads();
  const int64_t t = (int64_t)blockIdx.x * ROUTE_TOKENS + b;
  int e;
  float w;
  route_token<DT, L, PER, WIDE>(a, t, t < a.T, sub, e, w);
  if (t < a.T && sub < a.k) {
    a.experts[t * a.k + sub] = e;
    a.weights[t * a.k + sub] = w;
    if (e >= 0) atomicOr(&mask[e], 1u << b);
  }
  __syncthreads();
  for (int e = tid; e < a.Ep; e += THREADS) {
    a.masks[(int64_t)blockIdx.x * a.Ep + e] = (uint16_t)mask[e];
    a.counts[(int64_t)blockIdx.x * a.Ep + e] = (uint8_t)__popc(mask[e]);
  }
}

// Counts of each expert in the blocks in front of each block: 64 runs of blocks and 16 experts a workgroup
__global__ __launch_bounds__(64 * ROUTE_SCAN_EXPERTS) void route_scan_kernel(RouteArgs a) {
  __shared__ int part[64][ROUTE_SCAN_EXPERTS];
  const int x = threadIdx.x % ROUTE_SCAN_EXPERTS, run = threadIdx.x / ROUTE_SCAN_EXPERTS;
  const int e = blockIdx.x * ROUTE_SCAN_EXPERTS + x;
  const int64_t length = ceil_div(a.blocks, 64), b0 = run * length, b1 = b0 + length < a.blocks ? b0 + length : a.blocks;
  int sum = 0;
  if (e < a.E) {
#pragma unroll 8
    for (int64_t b = b0; b < b1; ++b) sum += a.counts[b * a.Ep + e];
  }
  part[run][x] = sum;
  __syncthreads();
  int before = 0;
  for (int r = 0; r < run; ++r) before += part[r][x];
  if (e >= a.E) return;
  if (run == 63) a.totals[e] = before + sum;
#pragma unroll 8
  for (int64_t b = b0; b < b1; ++b) {
    a.bases[b * a.E + e] = before;
    before += a.counts[b * a.Ep + e];
  }
}

__global__ __launch_bounds__(256) void route_place_kernel(RouteArgs a) {
  __shared__ int start[AC4K_ROUTE_MAX_EXPERTS];
  __shared__ int wave_sum[4];
  const int tid = threadIdx.x;
  for (int e = tid; e < a.E; e += 256) start[e] = a.totals[e];
  __syncthreads();
  const int total = route_starts<256>(start, a.E, wave_sum);
  if (blockIdx.x == 0) {
    for (int e = tid; e < a.E; e += 256) a.offsets[e] = start[e];
    if (tid == 0) a.offsets[a.E] = total;
  }
  const int64_t t0 = (int64_t)blockIdx.x * ROUTE_TOKENS;
  const int here = (int)(a.T - t0 < ROUTE_TOKENS ? a.T - t0 : ROUTE_TOKENS) * a.k;
  const int64_t row = (int64_t)blockIdx.x * a.E, mask_row = (int64_t)blockIdx.x * a.Ep;
  for (int i = tid; i < here; i += 256) {
    const int b = i / a.k, slot = i - b * a.k;
    const int e = a.experts[t0 * a.k + i];
    route_place(a, t0 + b, slot, e, e >= 0 ? a.masks[mask_row + e] : 0, b, [&](int x) { return start[x] + a.bases[row + x]; });
    if (t0 * a.k + i >= total) a.rows[t0 * a.k + i] = -1;
  }
}

// The same in one launch where there are few blocks: every workgroup counts all of them itself and places the tokens of ROUTE_PLAN_BLOCKS
// blocks.  A thread adds the counts of 16 experts in every runs-th block, as bytes (eight blocks of 16 tokens at a time) and then as pairs of 16 bits (at most 2^25 masks
// read in all workgroups: under 1500 a thread).  (With the bits counted here, a vector's eight experts one by one, 1164 vector instructions a wave took 11.4 us at
// 16384 x 128.)
__global__ __launch_bounds__(1024) void route_plan_kernel(RouteArgs a) {
  constexpr int THREADS = 1024;
  __shared__ int total[AC4K_ROUTE_MAX_EXPERTS];   // rows of the expert, then the start of its range
  __shared__ int before[AC4K_ROUTE_MAX_EXPERTS];  // of them, in front of this workgroup's blocks
  __shared__ uint16_t base[ROUTE_PLAN_BLOCKS][AC4K_ROUTE_MAX_EXPERTS];
  __shared__ __attribute__((aligned(16))) uint16_t mask[ROUTE_PLAN_BLOCKS * AC4K_ROUTE_MAX_EXPERTS];  // [block][Ep], as they lie in memory
  __shared__ uint32_t part[2][THREADS * 8];       // [run][pair of experts e, e + 2]
  __shared__ int wave_sum[THREADS / 64];
  const int tid = threadIdx.x, E = a.E, columns = a.Ep / 16, runs = THREADS / columns, pairs = columns * 8;
  const int64_t b0 = (int64_t)blockIdx.x * ROUTE_PLAN_BLOCKS;
  const int mine = (int)(a.blocks - b0 < ROUTE_PLAN_BLOCKS ? a.blocks - b0 : ROUTE_PLAN_BLOCKS);
  // the experts of the first slots are under way while the masks are counted
  const int64_t t0 = b0 * ROUTE_TOKENS;
  const int slots = (int)(a.T - t0 < ROUTE_PLAN_BLOCKS * ROUTE_TOKENS ? a.T - t0 : ROUTE_PLAN_BLOCKS * ROUTE_TOKENS) * a.k;
  int expert[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) expert[i] = tid + i * THREADS < slots ? a.experts[t0 * a.k + tid + i * THREADS] : -1;
  for (int e = tid; e < E; e += THREADS) total[e] = before[e] = 0;
  const u32x4 *masks = reinterpret_cast<const u32x4 *>(a.masks + b0 * a.Ep);
  const int vectors = mine * a.Ep / 8;  // at most two a thread
  u32x4 own[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) own[i] = tid + i * THREADS < vectors ? masks[tid + i * THREADS] : (u32x4){0, 0, 0, 0};
  const int run = tid / columns, column = tid - run * columns;
  if (run < runs) {
    uint32_t all[8] = {}, front[8] = {};
    constexpr int CHUNK = 8;  // loads under way at once: the counts come from other XCDs, a microsecond away
    for (int64_t b = run; b < a.blocks; b += CHUNK * runs) {
      u32x4 v[CHUNK], bytes = {0, 0, 0, 0}, front_bytes = {0, 0, 0, 0};
#pragma unroll
      for (int c = 0; c < CHUNK; ++c) {
        const int64_t at = b + c * runs;
        v[c] = at < a.blocks ? *reinterpret_cast<const u32x4 *>(a.counts + at * a.Ep + column * 16) : (u32x4){0, 0, 0, 0};
      }
#pragma unroll
      for (int c = 0; c < CHUNK; ++c) {
        bytes += v[c];
        if (b + c * runs < b0) front_bytes += v[c];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        all[i] += bytes[i / 2] >> (8 * (i & 1)) & 0x00ff00ffu;
        front[i] += front_bytes[i / 2] >> (8 * (i & 1)) & 0x00ff00ffu;
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      part[0][run * pairs + column * 8 + i] = front[i];
      part[1][run * pairs + column * 8 + i] = all[i];
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (tid + i * THREADS < vectors) reinterpret_cast<u32x4 *>(mask)[tid + i * THREADS] = own[i];
  __syncthreads();
  {
    const int shares = THREADS / pairs, share = tid / pairs, pair = tid - share * pairs;
    if (share < shares) {
      uint32_t f0 = 0, f1 = 0, t0 = 0, t1 = 0;
      for (int r = share; r < runs; r += shares) {
        const uint32_t f = part[0][r * pairs + pair], t = part[1][r * pairs + pair];
        f0 += f & 0xffffu, f1 += f >> 16, t0 += t & 0xffffu, t1 += t >> 16;
      }
      const int e = pair / 8 * 16 + pair % 8 / 2 * 4 + pair % 2;
      if (e < E) {
        atomicAdd(&before[e], (int)f0);
        atomicAdd(&total[e], (int)t0);
      }
      if (e + 2 < E) {
        atomicAdd(&before[e + 2], (int)f1);
        atomicAdd(&total[e + 2], (int)t1);
      }
    }
  }
  for (int e = tid; e < E; e += THREADS) {
    int sum = 0, m[ROUTE_PLAN_BLOCKS];
#pragma unroll
    for (int b = 0; b < ROUTE_PLAN_BLOCKS; ++b) m[b] = b < mine ? mask[b * a.Ep + e] : 0;
#pragma unroll
    for (int b = 0; b < ROUTE_PLAN_BLOCKS; ++b) {
      base[b][e] = (uint16_t)sum;
      sum += __popc((uint32_t)m[b]);
    }
  }
  __syncthreads();
  const int rows = route_starts<THREADS>(total, E, wave_sum);
  if (blockIdx.x == 0) {
    for (int e = tid; e < E; e += THREADS) a.offsets[e] = total[e];
    if (tid == 0) a.offsets[E] = rows;
  }
  for (int i = tid, n = 0; i < slots; i += THREADS, ++n) {
    const int t = i / a.k, slot = i - t * a.k, b = t / ROUTE_TOKENS;
    const int e = n == 0 ? expert[0] : n == 1 ? expert[1] : a.experts[t0 * a.k + i];
    route_place(a, t0 + t, slot, e, e >= 0 ? mask[b * a.Ep + e] : 0, t % ROUTE_TOKENS, [&](int x) { return total[x] + before[x] + base[b][x]; });
    if (t0 * a.k + i >= rows) a.rows[t0 * a.k + i] = -1;
  }
}

// All of a small call in one workgroup, THREADS / L tokens at a time
template <int DT, int L, int PER, bool WIDE, int THREADS>
__global__ __launch_bounds__(THREADS) void route_one_kernel(RouteArgs a) {
  constexpr int AT_ONCE = THREADS / L, TURNS = THREADS == 256 ? 1 : route_one_tokens(L) / AT_ONCE, WORDS = (AT_ONCE * TURNS + 63) / 64;
  constexpr int EXPERTS = L == 16 ? ROUTE_ROW_EXPERTS : AC4K_ROUTE_MAX_EXPERTS;
  __shared__ unsigned long long mask[WORDS][EXPERTS];  // tokens of each expert
  __shared__ int start[EXPERTS];
  __shared__ int16_t chosen[TURNS * THREADS];
  __shared__ int wave_sum[THREADS / 64];
  const int tid = threadIdx.x, sub = tid % L;
  for (int e = tid; e < a.E; e += THREADS) {
#pragma unroll
    for (int w = 0; w < WORDS; ++w) mask[w][e] = 0;
  }
  __syncthreads();
#pragma unroll 1
  for (int i = 0; i * AT_ONCE < a.T && i < TURNS; ++i) {
    const int t = i * AT_ONCE + tid / L;
    int mine = -1;
    if (i * AT_ONCE + (tid & ~63) / L < a.T) {  // a whole wave
      float w;
      route_token<DT, L, PER, WIDE>(a, t, t < a.T, sub, mine, w);
      if (t < a.T && sub < a.k) {
        a.experts[(int64_t)t * a.k + sub] = mine;
        a.weights[(int64_t)t * a.k + sub] = w;
        if (mine >= 0) atomicOr(&mask[t >> 6][mine], 1ull << (t & 63));
      }
    }
    chosen[i * THREADS + tid] = (int16_t)mine;
  }
  __syncthreads();
  for (int e = tid; e < a.E; e += THREADS) {
    int sum = 0;
#pragma unroll
    for (int w = 0; w < WORDS; ++w) sum += __popcll(mask[w][e]);
    start[e] = sum;
  }
  __syncthreads();
  const int total = route_starts<THREADS>(start, a.E, wave_sum);
  for (int e = tid; e < a.E; e += THREADS) a.offsets[e] = start[e];
  if (tid == 0) a.offsets[a.E] = total;
#pragma unroll 1
  for (int i = 0; i * AT_ONCE < a.T && i < TURNS; ++i) {
    const int t = i * AT_ONCE + tid / L, e = chosen[i * THREADS + tid];
    if (t < a.T && sub < a.k)
      route_place(a, t, sub, e, e >= 0 ? mask[t >> 6][e] : 0, t & 63, [&](int x) {
        int base = start[x];
        for (int w = 0; w < t >> 6; ++w) base += __popcll(mask[w][x]);
        return base;
      });
  }
  for (int i = total + tid; i < a.T * a.k; i += THREADS) a.rows[i] = -1;
}

template <int DT, int L, int PER, bool WIDE>
static void launch_route(const RouteArgs &a, hipStream_t st) {
  if (a.T <= route_one_tokens(L)) {
    if (a.T * L <= 256) hipLaunchKernelGGL((route_one_kernel<DT, L, PER, WIDE, 256>), dim3(1), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((route_one_kernel<DT, L, PER, WIDE, 1024>), dim3(1), dim3(1024), 0, st, a);
    return;
  }
  hipLaunchKernelGGL((route_kernel<DT, L, PER, WIDE>), dim3((unsigned)a.blocks), dim3(ROUTE_TOKENS * L), 0, st, a);
  const int64_t groups = ceil_div(a.blocks, ROUTE_PLAN_BLOCKS);
  if (groups * a.blocks * a.E <= ROUTE_PLAN_COUNTS) {
    hipLaunchKernelGGL(route_plan_kernel, dim3((unsigned)groups), dim3(1024), 0, st, a);
    return;
  }
  hipLaunchKernelGGL(route_scan_kernel, dim3((unsigned)ceil_div(a.E, ROUTE_SCAN_EXPERTS)), dim3(64 * ROUTE_SCAN_EXPERTS), 0, st, a);
  hipLaunchKernelGGL(route_place_kernel, dim3((unsigned)a.blocks), dim3(256), 0, st, a);
}
template <int DT, bool WIDE>
static int route_shape(RouteArgs a, hipStream_t st) {
  if (route_lanes(a.E, a.k, a.groups) == 16) {
    a.group_lanes = 16;
    if (a.E <= 16) launch_route<DT, 16, 1, WIDE>(a, st);
    else if (a.E <= 32) launch_route<DT, 16, 2, WIDE>(a, st);
    else if (a.E <= 64) launch_route<DT, 16, 4, WIDE>(a, st);
    else launch_route<DT, 16, 8, WIDE>(a, st);
    return 0;
  }
  a.group_lanes = 64;
  while (a.group_lanes * a.groups > 64) a.group_lanes /= 2;
  const int64_t per = ceil_div(a.group_size, a.group_lanes);
  if (per <= 1) launch_route<DT, 64, 1, WIDE>(a, st);
  else if (per <= 2) launch_route<DT, 64, 2, WIDE>(a, st);
  else if (per <= 4) launch_route<DT, 64, 4, WIDE>(a, st);
  else if (per <= 8) launch_route<DT, 64, 8, WIDE>(a, st);
  else if (per <= 16) launch_route<DT, 64, 16, WIDE>(a, st);
  else launch_route<DT, 64, 32, WIDE>(a, st);
  return 0;
}
template <int DT>
static int route_width(const RouteArgs &a, hipStream_t st) {
  const bool wide = a.bias || (a.groups > 1 && a.best == 2);
  return wide ? route_shape<DT, true>(a, st) : route_shape<DT, false>(a, st);
}

static int64_t route_workspace(int64_t T, int64_t E, int64_t k, int64_t groups) {
  if (T <= route_one_tokens(route_lanes(E, k, groups))) return 0;
  const int64_t blocks = ceil_div(T, ROUTE_TOKENS);
  return 4 * align_up(E, 4) + 4 * align_up(blocks * E, 4) + 3 * blocks * align_up(E, 16);
}

// ---------------------------------------------------------------------------
// the experts' rows back to their tokens
// ---------------------------------------------------------------------------
struct CombineArgs {
  void *out;
  const void *y, *residual;
  const float *weights;
  const int32_t *places;
  int64_t T, M, N, y_stride, residual_stride, out_stride;
  int k;
};

// A thread takes eight columns of a token; its places and weights are scalars of the wave.  Rows are read eight at a time.  Bound by memory: 8192 tokens of 8 rows of 4096
// with a residual 130 us, 5.2 TB/s, the rate of a copy; every row is read once, whole.  16 tokens 3.7 us, a chain of places, rows and store.
template <int DT>
__global__ __launch_bounds__(256) void combine_kernel(CombineArgs a, uint32_t spans) {
  using T = typename Elem<DT>::T;
  const uint32_t token = blockIdx.x / spans, span = blockIdx.x - token * spans;
  const int64_t c = (int64_t)span * 2048 + threadIdx.x * 8;
  if (c >= a.N) return;
  const int32_t *places = a.places + (int64_t)token * a.k;
  const float *weights = a.weights + (int64_t)token * a.k;
  float sum[8] = {};
  if (a.residual) {
    Vec8<DT> r;
    vec8_load(r, static_cast<const T *>(a.residual) + token * a.residual_stride, c, a.N);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i] = vec8_get(r, i);
  }
  for (int s0 = 0; s0 < a.k; s0 += 8) {
    Vec8<DT> v[8];
    float w[8];
    bool here[8];
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      const int64_t place = s0 + s < a.k ? places[s0 + s] : -1;
      here[s] = place >= 0 && place < a.M;
      w[s] = here[s] ? weights[s0 + s] : 0.0f;
      if (here[s]) vec8_load(v[s], static_cast<const T *>(a.y) + place * a.y_stride, c, a.N);
    }
#pragma unroll
    for (int s = 0; s < 8; ++s)
      if (here[s]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] = __builtin_fmaf(vec8_get(v[s], i), w[s], sum[i]);
      }
  }
  Vec8<DT> o;
  vec8_set(o, sum);
  vec8_store(static_cast<T *>(a.out) + token * a.out_stride, o, c, a.N);
}

}  // namespace ac4k

using namespace ac4k;

static bool float_tag(int d) { return d == AC4K_DTYPE_BF16 || d == AC4K_DTYPE_FP16 || d == AC4K_DTYPE_FP32; }

extern "C" __attribute__((visibility("default"))) int64_t ac4k_route_experts_workspace_bytes(int64_t T, int64_t E, int64_t k, int64_t groups, int64_t top_groups) {
  if (T < 1 || E < 1 || E > AC4K_ROUTE_MAX_EXPERTS || k < 1 || k > AC4K_ROUTE_MAX_K) return 0;
  return route_workspace(T, E, k, top_groups == groups ? 1 : groups);
}

extern "C" __attribute__((visibility("default"))) int ac4k_route_experts(
    float *weights, int32_t *experts, int32_t *offsets, int32_t *rows, int32_t *places, const void *logits, int dtype, int64_t stride, const float *bias,
    int64_t T, int64_t E, int64_t k, int scoring, int64_t groups, int64_t top_groups, int best, int renormalize, double scale, void *workspace,
    int64_t workspace_bytes, ac4k_stream_t stream) {
  AC4K_REQUIRE(weights && experts && offsets && rows && places && logits, "null pointer argument");
  AC4K_REQUIRE(float_tag(dtype), "logits must be bfloat16, half or float (dtype tag %d)", dtype);
  AC4K_REQUIRE(T >= 1 && E >= 1 && E <= AC4K_ROUTE_MAX_EXPERTS, "tokens must be positive and experts 1 to %d (T=%lld E=%lld)", (int)AC4K_ROUTE_MAX_EXPERTS,
               (long long)T, (long long)E);
  AC4K_REQUIRE(scoring == AC4K_SCORE_SOFTMAX || scoring == AC4K_SCORE_SIGMOID, "unknown scoring %d", scoring);
  AC4K_REQUIRE(groups >= 1 && groups <= 64 && E % groups == 0, "groups must be 1 to 64 and divide the %lld experts, got %lld", (long long)E, (long long)groups);
  AC4K_REQUIRE(top_groups >= 1 && top_groups <= groups, "top_groups must be 1 to %lld, got %lld", (long long)groups, (long long)top_groups);
  AC4K_REQUIRE(best == 1 || best == 2, "a group's score is that of its best one or two, not %d", best);
  AC4K_REQUIRE(k >= 1 && k <= AC4K_ROUTE_MAX_K && k <= E / groups * top_groups, "k must be 1 to %d and at most the %lld experts of the groups taken, got %lld",
               (int)AC4K_ROUTE_MAX_K, (long long)(E / groups * top_groups), (long long)k);
  AC4K_REQUIRE(T * k < (1ll << 27) && T <= (1ll << 26) - ROUTE_TOKENS, "too many tokens (%lld of %lld experts)", (long long)T,
               (long long)k);  // 2^32 threads a launch
  const int64_t need = route_workspace(T, E, k, top_groups == groups ? 1 : groups);
  AC4K_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0), "workspace of %lld bytes needed, on 16 bytes", (long long)need);
  RouteArgs a{};
  a.logits = logits, a.stride = stride, a.bias = bias, a.weights = weights, a.experts = experts, a.offsets = offsets, a.rows = rows, a.places = places;
  a.T = T, a.blocks = ceil_div(T, ROUTE_TOKENS), a.E = (int)E, a.Ep = (int)align_up(E, 16), a.k = (int)k;
  a.groups = (int)(top_groups == groups ? 1 : groups), a.top_groups = (int)top_groups, a.best = best, a.group_size = (int)(E / a.groups);
  a.sigmoid = scoring == AC4K_SCORE_SIGMOID, a.renormalize = renormalize != 0, a.scale = scale;
  a.totals = static_cast<int32_t *>(workspace);
  a.bases = a.totals + align_up(E, 4);
  a.masks = reinterpret_cast<uint16_t *>(a.bases + align_up(a.blocks * E, 4));
  a.counts = reinterpret_cast<uint8_t *>(a.masks + a.blocks * a.Ep);
  hipStream_t st = (hipStream_t)stream;
  int rc;
  if (dtype == AC4K_DTYPE_BF16) rc = route_width<AC4K_DTYPE_BF16>(a, st);
  else if (dtype == AC4K_DTYPE_FP16) rc = route_width<AC4K_DTYPE_FP16>(a, st);
  else rc = route_width<AC4K_DTYPE_FP32>(a, st);
  if (rc) return rc;
  return check_launch("ac4k_route_experts");
}

extern "C" __attribute__((visibility("default"))) int ac4k_combine_experts(
    void *out, int64_t out_stride, const void *y, int64_t y_stride, const float *weights, const int32_t *places, const void *residual, int64_t residual_stride,
    int64_t T, int64_t k, int64_t M, int64_t N, int dtype, ac4k_stream_t stream) {
  AC4K_REQUIRE(out && (y || M == 0) && weights && places, "null pointer argument");
  AC4K_REQUIRE(float_tag(dtype), "y must be bfloat16, half or float (dtype tag %d)", dtype);
  AC4K_REQUIRE(T >= 1 && k >= 1 && M >= 0 && N >= 1, "sizes must be positive (T=%lld k=%lld N=%lld)", (long long)T, (long long)k, (long long)N);
  const int64_t spans = ceil_div(N, 2048);
  AC4K_REQUIRE(k < (1ll << 16) && M < (1ll << 31) && T < (1ll << 24) && spans < (1ll << 24) && T * spans < (1ll << 24), "problem too large");  // 2^32 threads a launch
  const CombineArgs a{out, y, residual, weights, places, T, M, N, y_stride, residual_stride, out_stride, (int)k};
  hipStream_t st = (hipStream_t)stream;
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)(T * spans)), dim3(256), 0, st, a, (uint32_t)spans); };
  if (dtype == AC4K_DTYPE_BF16) go(combine_kernel<AC4K_DTYPE_BF16>);
  else if (dtype == AC4K_DTYPE_FP16) go(combine_kernel<AC4K_DTYPE_FP16>);
  else go(combine_kernel<AC4K_DTYPE_FP32>);
  return check_launch("ac4k_combine_experts");
}

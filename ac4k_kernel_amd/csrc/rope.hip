// Rotary positions with several axes: every pair (a, b) of a head's elements turns by the angle of its token's position along the pair's axis,
//
//   (a, b) -> (a c - b s, b c + a s),   c, s = table[position along the pair's axis][pair]
//
// in fp32, rounded once to the type of x.  Pair j is elements (2j, 2j + 1) of a head (interleaved) or (j, j + pairs); elements behind the
// last pair are copied.  The table holds cosines and sines in fp32, made from angles in 64 bits: a product of a far position and a
// frequency in 32 bits would be off by more than the rounding of the result.
//
// Bound by memory: every element is read and written once.  A thread keeps its token and its place inside the head and goes over the heads, so
// that it reads its four to eight entries of the table once, while the first heads are under way.  75600 tokens of 80 heads of 128, bf16, 535 us, 5.8 TB/s,
// every byte read and written once; fp32 2 x 4001 x 24 heads of 64 19-20 us, 4.9-5.1 TB/s; 32 tokens of 48 heads 4.7 us: position, table row and store,
// one after the other.
#include "elements.h"

namespace ac4k {

struct RopeTensor {
  const void *in;
  void *out;
  int64_t in_b, in_n, in_h, out_b, out_n, out_h;  // strides in elements; a head is contiguous
  int heads;
};

struct RopeArgs {
  RopeTensor t[2];
  const float2 *table;  // [length][pairs]
  const void *positions;
  int64_t pos_axis, pos_b, pos_n;  // strides; positions null: the token's place in a grid
  uint32_t grid[AC4K_ROPE_MAX_AXES];
  uint32_t N;
  int64_t length;
  int D, pairs, axes, pos_bytes;
  int end[AC4K_ROPE_MAX_AXES];  // first pair behind each axis
  uint32_t rot_vecs, vecs;      // vectors of a head: those that hold pairs, and with those that are copied
  uint32_t vecs_inverse;        // ceil(2^16 / vecs)
  uint32_t blocks_b;            // workgroups of a batch
  uint32_t once_log, across;    // 2^once_log tokens a workgroup, `across` heads of each at a time
  bool heads_first;             // neighbouring threads are on neighbouring heads of a token, otherwise on neighbouring tokens of a head
  float sign;                   // of the sines
};

// WHOLE: no vector is cut by the end of the pairs or of the head, or the last one is moved back to end there, and two threads write the same
// values to what lies in both (not in place, where one could read what the other has turned).  Four vectors are under way at a time then, with
// no branch between their loads (with the loads of cut vectors in between, every load was waited for by itself: 20000 x 48 heads of 40, halves, 54 us, now 36; in place still 54).
template <int DT, bool INTERLEAVED, bool WHOLE>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a) {
  using T = typename Elem<DT>::T;
  constexpr int AHEAD = WHOLE ? 4 : 1;
  // INTERLEAVED: a vector holds four pairs; otherwise the first elements of eight, their partners `pairs` further on
  constexpr int NP = INTERLEAVED ? 4 : 8;
  const int rot = 2 * a.pairs;
  const uint32_t u = threadIdx.x * a.vecs_inverse >> 16, v = threadIdx.x - u * a.vecs;  // (exact: both under 2^8)
  uint32_t my, head0;
  if (a.heads_first) {
    my = 0, head0 = u;
    if (a.once_log) my = u / a.across, head0 = u - my * a.across;
  } else {
    my = u & ((1u << a.once_log) - 1), head0 = u >> a.once_log;
  }
  const uint32_t b = blockIdx.x / a.blocks_b, n = ((blockIdx.x - b * a.blocks_b) << a.once_log) + my;
  if (my >> a.once_log || head0 >= a.across || n >= a.N) return;

  // first element of what the thread moves of a head, and the end of its kind
  const bool turned = v < a.rot_vecs;
  const int k1 = !turned ? a.D : INTERLEAVED ? rot : a.pairs;
  int k0 = turned ? v * 8 : rot + (v - a.rot_vecs) * 8;
  if (WHOLE && k0 > k1 - 8) k0 = k1 - 8;
  const uint32_t first = a.t[0].heads, heads = first + a.t[1].heads;
  const T *in[2];
  T *out[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    in[i] = static_cast<const T *>(a.t[i].in) + b * a.t[i].in_b + n * a.t[i].in_n;
    out[i] = static_cast<T *>(a.t[i].out) + b * a.t[i].out_b + n * a.t[i].out_n;
  }
  Vec8<DT> x[AHEAD], y[AHEAD];  // y: the partners, where they are apart
  auto move_in = [&](Vec8<DT> &to, const T *p) {
    if constexpr (WHOLE) vec8_load_all(to, p + k0);
    else vec8_load(to, p, k0, k1);
  };
  auto move_out = [&](T *p, const Vec8<DT> &from) {
    if constexpr (WHOLE) vec8_store_all(p + k0, from);
    else vec8_store(p, from, k0, k1);
  };
  auto load = [&](uint32_t h0) {  // heads past the last one: the last one again
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const uint32_t h = h0 + i * a.across < heads ? h0 + i * a.across : heads - 1;
      const T *p = h < first ? in[0] + h * a.t[0].in_h : in[1] + (h - first) * a.t[1].in_h;
      move_in(x[i], p);
      if constexpr (!INTERLEAVED) move_in(y[i], p + (turned ? a.pairs : 0));
    }
  };
  load(head0);  // under way while positions and angles are looked up

  float c[NP], s[NP];
  bool stay = false;
  const int pair0 = INTERLEAVED ? k0 / 2 : k0;
  int64_t at[NP];
  int axis_end = 0;  // of the first pair
  {
    int64_t pos[AC4K_ROPE_MAX_AXES];
    if (a.positions) {
      const int64_t i = b * a.pos_b + n * a.pos_n;
#pragma unroll
      for (int axis = 0; axis < AC4K_ROPE_MAX_AXES; ++axis)
        if (axis < a.axes)
          pos[axis] = a.pos_bytes == 8 ? static_cast<const int64_t *>(a.positions)[i + axis * a.pos_axis] : static_cast<const int32_t *>(a.positions)[i + axis * a.pos_axis];
    } else {
      uint32_t place = n;  // by the last axis first
#pragma unroll
      for (int axis = AC4K_ROPE_MAX_AXES - 1; axis >= 0; --axis)
        if (axis < a.axes) {
          const uint32_t q = place / a.grid[axis];
          pos[axis] = place - q * a.grid[axis];
          place = q;
        }
      stay = place > 0;  // behind the last place
    }
#pragma unroll
    for (int i = 0; i < NP; ++i) at[i] = 0;
#pragma unroll
    for (int axis = AC4K_ROPE_MAX_AXES - 1; axis >= 0; --axis)
      if (axis < a.axes) {
        stay |= pos[axis] < 0;
#pragma unroll
        for (int i = 0; i < NP; ++i)
          if (pair0 + i < a.end[axis]) at[i] = pos[axis];  // (axes in front overwrite)
        if (pair0 < a.end[axis]) axis_end = a.end[axis];
      }
  }
#pragma unroll
  for (int i = 0; i < NP; ++i) c[i] = 1.0f, s[i] = 0.0f;
  if (turned && !stay) {
    // a position that the table does not have has no angle: NaN, and nothing behind the table is read
    if (pair0 + NP <= axis_end && at[0] < a.length) {  // one row of the table
      const char *row = reinterpret_cast<const char *>(a.table + at[0] * a.pairs + pair0);
#pragma unroll
      for (int i = 0; i < NP; i += 2) {
        const f32x4 cs = *reinterpret_cast<const f32x4_elem *>(row + i * 8);
        c[i] = cs.x, s[i] = cs.y, c[i + 1] = cs.z, s[i + 1] = cs.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < NP; ++i)
        if (pair0 + i < a.pairs) {
          float2 cs = make_float2(__builtin_nanf(""), __builtin_nanf(""));
          if (at[i] < a.length) cs = a.table[at[i] * a.pairs + pair0 + i];
          c[i] = cs.x, s[i] = cs.y;
        }
    }
#pragma unroll
    for (int i = 0; i < NP; ++i) s[i] *= a.sign;
  }
  for (uint32_t h0 = head0; h0 < heads;) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const uint32_t h = h0 + i * a.across;
      if (turned && !stay) {
        float f[8], g[8];
        if constexpr (INTERLEAVED) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float p = vec8_get(x[i], 2 * j), q = vec8_get(x[i], 2 * j + 1);
            f[2 * j] = __builtin_fmaf(p, c[j], -(q * s[j]));
            f[2 * j + 1] = __builtin_fmaf(q, c[j], p * s[j]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float p = vec8_get(x[i], j), q = vec8_get(y[i], j);
            f[j] = __builtin_fmaf(p, c[j], -(q * s[j]));
            g[j] = __builtin_fmaf(q, c[j], p * s[j]);
          }
          vec8_set(y[i], g);
        }
        vec8_set(x[i], f);
      }
      if (h < heads) {
        T *p = h < first ? out[0] + h * a.t[0].out_h : out[1] + (h - first) * a.t[1].out_h;
        move_out(p, x[i]);
        if constexpr (!INTERLEAVED)
          if (turned) move_out(p + a.pairs, y[i]);
      }
    }
    h0 += AHEAD * a.across;
    if (h0 < heads) load(h0);
  }
}

template <int DT>
static void launch_rope(RopeArgs a, int64_t B, bool interleaved, hipStream_t st) {
  a.rot_vecs = interleaved ? (2 * a.pairs + 7) / 8 : (a.pairs + 7) / 8;
  a.vecs = a.rot_vecs + (a.D - 2 * a.pairs + 7) / 8;
  a.vecs_inverse = (65536 + a.vecs - 1) / a.vecs;
  const uint32_t across = 256 / a.vecs, heads = a.t[0].heads + a.t[1].heads;
  // Threads side by side are on the neighbours in memory: heads of a token, or tokens of a head.  A workgroup takes tokens enough that a
  // thread has four heads to go over (and eight tokens where they are the neighbours), as long as a thousand workgroups remain.  us, one
  // token at a time / two / four / eight: 8002 x 24 heads of 64, fp32 31 / 27 / 23 / 21; 8192 x 48 of 128, halves 39 / 36 / 34 / 34;
  // 75600 x 80 of 128 552 / 573 / 589 / 596.
  a.heads_first = a.t[0].in_h <= a.t[0].in_n;
  while ((2u << a.once_log) <= across && (1u << a.once_log) < a.N && ((heads << a.once_log) < 4 * across || (!a.heads_first && a.once_log < 3)) &&
         B * a.N >> (a.once_log + 1) >= 1000)
    ++a.once_log;
  a.across = across >> a.once_log;
  a.blocks_b = (a.N + (1u << a.once_log) - 1) >> a.once_log;
  const dim3 grid((unsigned)(B * a.blocks_b));
  const bool apart = a.t[0].in != a.t[0].out && (a.t[1].heads == 0 || a.t[1].in != a.t[1].out);  // (they do not overlap otherwise)
  auto fits = [&](int n) { return n % 8 == 0 || (n >= 8 && apart); };
  const bool whole = fits(interleaved ? 2 * a.pairs : a.pairs) && fits(a.D - 2 * a.pairs);
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, st, a); };
  if (interleaved) whole ? go(rope_kernel<DT, true, true>) : go(rope_kernel<DT, true, false>);
  else whole ? go(rope_kernel<DT, false, true>) : go(rope_kernel<DT, false, false>);
}

}  // namespace ac4k

using namespace ac4k;

extern "C" __attribute__((visibility("default"))) int ac4k_rope(
    const ac4k_rope_tensor *tensors, int count, int dtype, int64_t B, int64_t N, int64_t D, const float *table, int64_t length, int64_t pairs,
    const int64_t *sections, int axes, const void *positions, int positions_bytes, int64_t pos_axis_stride, int64_t pos_b_stride,
    int64_t pos_n_stride, const int64_t *grid, int interleaved, int inverse, ac4k_stream_t stream) {
  AC4K_REQUIRE(tensors && table && sections, "null pointer argument");
  AC4K_REQUIRE(count == 1 || count == 2, "one or two tensors a call, got %d", count);
  AC4K_REQUIRE(axes >= 1 && axes <= AC4K_ROPE_MAX_AXES, "1 to %d axes, got %d", (int)AC4K_ROPE_MAX_AXES, axes);
  AC4K_REQUIRE(!positions != !grid, "positions or a grid, one of them");
  AC4K_REQUIRE(!positions || positions_bytes == 4 || positions_bytes == 8, "positions of 4 or 8 bytes");
  AC4K_REQUIRE(B >= 1 && N >= 1 && length >= 1 && pairs >= 1, "sizes must be positive");
  AC4K_REQUIRE(D >= 2 && D <= AC4K_ROPE_MAX_DIM, "head dim from 2 to %d, got %lld", (int)AC4K_ROPE_MAX_DIM, (long long)D);
  AC4K_REQUIRE(2 * pairs <= D, "%lld pairs do not fit a head of %lld", (long long)pairs, (long long)D);
  AC4K_REQUIRE(((uintptr_t)table & 7) == 0, "the table must be on 8 bytes");
  AC4K_REQUIRE(B < (1ll << 24) && N < (1ll << 24) && B * N < (1ll << 24), "too many tokens");  // 2^32 threads a launch
  AC4K_REQUIRE(dtype == AC4K_DTYPE_BF16 || dtype == AC4K_DTYPE_FP16 || dtype == AC4K_DTYPE_FP32, "x must be bfloat16, half or float (dtype tag %d)", dtype);
  RopeArgs a{};
  int64_t sum = 0;
  for (int x = 0; x < axes; ++x) {
    AC4K_REQUIRE(sections[x] >= 0 && sections[x] <= pairs, "a section has 0 to all pairs");
    a.end[x] = (int)(sum += sections[x]);
    if (grid) {
      AC4K_REQUIRE(grid[x] >= 1, "a grid has at least one place along every axis");
      AC4K_REQUIRE(grid[x] <= length, "the table has %lld positions, the grid %lld", (long long)length, (long long)grid[x]);
      AC4K_REQUIRE(grid[x] < (1ll << 31), "grid too large");
      a.grid[x] = (uint32_t)grid[x];
    }
  }
  AC4K_REQUIRE(sum == pairs, "sections of %lld pairs, the table has %lld", (long long)sum, (long long)pairs);
  for (int i = 0; i < count; ++i) {
    const ac4k_rope_tensor &t = tensors[i];
    AC4K_REQUIRE(t.in && t.out, "null pointer argument");
    AC4K_REQUIRE(t.heads >= 1 && t.heads < (1 << 20), "1 to 2^20 heads, got %lld", (long long)t.heads);
    a.t[i] = RopeTensor{t.in, t.out, t.in_b_stride, t.in_n_stride, t.in_h_stride, t.out_b_stride, t.out_n_stride, t.out_h_stride, (int)t.heads};
  }
  a.table = reinterpret_cast<const float2 *>(table);
  a.positions = positions, a.pos_axis = pos_axis_stride, a.pos_b = pos_b_stride, a.pos_n = pos_n_stride, a.pos_bytes = positions_bytes;
  a.N = (uint32_t)N, a.length = length, a.sign = inverse ? -1.0f : 1.0f, a.D = (int)D, a.pairs = (int)pairs, a.axes = axes;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == AC4K_DTYPE_BF16) launch_rope<AC4K_DTYPE_BF16>(a, B, interleaved, st);
  else if (dtype == AC4K_DTYPE_FP16) launch_rope<AC4K_DTYPE_FP16>(a, B, interleaved, st);
  else launch_rope<AC4K_DTYPE_FP32>(a, B, interleaved, st);
  return check_launch("ac4k_rope");
}

// Rotary positions with several axes: every pair (a, b) of a head's elements turns by the angle of its token's position along the pair's axis,
//
//   (a, b) -> (a c - b s, b c + a s),   c, s = table[position along the pair's axis][pair]
//
// in fp32, rounded once to the type of x.  Pair j is elements (2j, 2j + 1) of a head (interleaved) or (j, j + pairs); elements behind the
// last pair are copied.  The table holds cosines and sines in fp32, made from angles in 64 bits: a product of a far position and a
// frequency in 32 bits would be off by more than the rounding of the result.
//
// Bound by memory: every element is read and written once.  A thread keeps its place inside the head and goes over the heads of its token,
// so that it reads the four to eight entries of the table once per token.
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
  int64_t grid[AC4K_ROPE_MAX_AXES];
  int64_t B, N, length;
  int D, pairs, axes, pos_bytes;
  int end[AC4K_ROPE_MAX_AXES];  // first pair behind each axis
};

// Position of token n of batch b along an axis; negative: the token stays as it is.
__device__ __forceinline__ int64_t rope_position(const RopeArgs &a, int64_t b, int64_t n, int axis) {
  if (a.positions) {
    const int64_t i = axis * a.pos_axis + b * a.pos_b + n * a.pos_n;
    return a.pos_bytes == 8 ? static_cast<const int64_t *>(a.positions)[i] : static_cast<const int32_t *>(a.positions)[i];
  }
  int64_t at = n;
  for (int x = a.axes - 1; x > axis; --x) at /= a.grid[x];
  return axis == 0 ? (at < a.grid[0] ? at : -1) : at % a.grid[axis];
}

template <int DT, bool INTERLEAVED, bool INVERSE>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a) {
  using T = typename Elem<DT>::T;
  // vectors of a head: those that hold pairs (INTERLEAVED: 4 pairs each; otherwise 8 first elements, their partners `pairs` further on),
  // then those that are copied
  const int rot = 2 * a.pairs;
  const int rot_vecs = INTERLEAVED ? (rot + 7) / 8 : (a.pairs + 7) / 8;
  const int vecs = rot_vecs + (a.D - rot + 7) / 8;
  const int across = 256 / vecs;  // heads at a time
  const int v = threadIdx.x % vecs, head0 = threadIdx.x / vecs;
  const int64_t n = blockIdx.x % a.N, b = blockIdx.x / a.N;
  if (head0 >= across) return;
  constexpr int NP = INTERLEAVED ? 4 : 8;
  float c[NP], s[NP];
  bool stay = false;
  for (int x = 0; x < a.axes; ++x) stay |= rope_position(a, b, n, x) < 0;
  const int pair0 = v * NP;
  if (v < rot_vecs) {
    int axis = 0;
    while (axis + 1 < a.axes && pair0 >= a.end[axis]) ++axis;
    int64_t at = rope_position(a, b, n, axis);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int pair = pair0 + i;
      while (axis + 1 < a.axes && pair >= a.end[axis]) at = rope_position(a, b, n, ++axis);
      c[i] = 1.0f, s[i] = 0.0f;
      if (pair < a.pairs && !stay) {
        // a position that the table does not have has no angle: NaN, and nothing behind the table is read
        float2 cs = make_float2(__builtin_nanf(""), __builtin_nanf(""));
        if (at < a.length) cs = a.table[at * a.pairs + pair];
        c[i] = cs.x, s[i] = INVERSE ? -cs.y : cs.y;
      }
    }
  }
  const int heads = a.t[0].heads + a.t[1].heads;
  for (int h = head0; h < heads; h += across) {
    const bool second = h >= a.t[0].heads;
    const RopeTensor &t = second ? a.t[1] : a.t[0];
    const int hh = second ? h - a.t[0].heads : h;
    const T *in = static_cast<const T *>(t.in) + b * t.in_b + n * t.in_n + hh * t.in_h;
    T *out = static_cast<T *>(t.out) + b * t.out_b + n * t.out_n + hh * t.out_h;
    if (v >= rot_vecs) {  // copied
      Vec8<DT> x;
      const int k = rot + (v - rot_vecs) * 8;
      vec8_load(x, in, k, a.D);
      vec8_store(out, x, k, a.D);
    } else if constexpr (INTERLEAVED) {
      Vec8<DT> x;
      vec8_load(x, in, v * 8, rot);
      float f[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p = vec8_get(x, 2 * i), q = vec8_get(x, 2 * i + 1);
        f[2 * i] = stay ? p : p * c[i] - q * s[i];
        f[2 * i + 1] = stay ? q : q * c[i] + p * s[i];
      }
      vec8_set(x, f);
      vec8_store(out, x, v * 8, rot);
    } else {
      Vec8<DT> x, y;
      vec8_load(x, in, v * 8, a.pairs);
      vec8_load(y, in + a.pairs, v * 8, a.pairs);
      float f[8], g[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p = vec8_get(x, i), q = vec8_get(y, i);
        f[i] = stay ? p : p * c[i] - q * s[i];
        g[i] = stay ? q : q * c[i] + p * s[i];
      }
      vec8_set(x, f);
      vec8_set(y, g);
      vec8_store(out, x, v * 8, a.pairs);
      vec8_store(out + a.pairs, y, v * 8, a.pairs);
    }
  }
}

template <int DT>
static void launch_rope(const RopeArgs &a, bool interleaved, bool inverse, hipStream_t st) {
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)(a.B * a.N)), dim3(256), 0, st, a); };
  if (interleaved) inverse ? go(rope_kernel<DT, true, true>) : go(rope_kernel<DT, true, false>);
  else inverse ? go(rope_kernel<DT, false, true>) : go(rope_kernel<DT, false, false>);
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
      a.grid[x] = grid[x];
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
  a.B = B, a.N = N, a.length = length, a.D = (int)D, a.pairs = (int)pairs, a.axes = axes;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == AC4K_DTYPE_BF16) launch_rope<AC4K_DTYPE_BF16>(a, interleaved, inverse, st);
  else if (dtype == AC4K_DTYPE_FP16) launch_rope<AC4K_DTYPE_FP16>(a, interleaved, inverse, st);
  else launch_rope<AC4K_DTYPE_FP32>(a, interleaved, inverse, st);
  return check_launch("ac4k_rope");
}

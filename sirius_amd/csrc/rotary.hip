// Rotary positions: the first `rot` elements of every head are r / 2 pairs, and pair i of a row at position p is turned by t = p f_i:
//   y_a = s (x_a cos t - x_b sin t),   y_b = s (x_b cos t + x_a sin t)
// with pairs (i, i + r / 2) or (2 i, 2 i + 1); the other elements are copied.  A rotation's gradient is the rotation back (-t) times
// the same s.
//
// Bound by memory: every element is read and written once.  The sines and cosines belong to a row and all its heads share them, so
// a workgroup takes whole rows (or a run of one row's heads), has each of its threads make some of the r / 2 pairs of factors a row, and
// keeps those in LDS.  p f is taken in fp64 (a position of 2^20 times a frequency of 1 leaves 2^-33 of a turn of error), whole turns come off
// there, and what is left goes through fp32 sine and cosine with the part that rounding it took off put back.  131072 rows of 40 x 128 in bf16 457 us
// (5.9 TB/s), 8192 of 24 x 64 9.4 (5.4), one of 40 x 128 2.6.
//
// Reference call site: the causal language models that train/gpt2.py:26 builds have learned positions; this is the form next to
// them.
#include <algorithm>
#include <climits>

#include "context.h"
#include "linear_epilogue.h"
#include "ops.h"

namespace tch {
namespace {

constexpr int kMaxPairs = 2048;   // of a workgroup: 16 KB of factors
constexpr int kUnitsAtOnce = 4;   // of a thread, on their way together

struct RotaryArgs {
  const void* x;
  void* y;
  const double* freqs;      // [rot / 2] radians a position
  const void* positions;    // [rows] int32 or int64, or null: start + row % seq
  int64_t ldx, ldy, rows, start;
  FastDiv seq, units, group_heads;   // units: of a head; group_heads: heads of a workgroup
  FastDiv pairs;
  int heads, head_dim, rot;
  int group_rows;
  int wide_positions;       // int64
  int copy;                 // the elements behind the rotated ones are copied (not where y is x)
  float scale, sign;
};

template <int BYTES>
struct Raw;
template <> struct Raw<16> { typedef unsigned int type __attribute__((ext_vector_type(4))); };
template <> struct Raw<8> { typedef unsigned int type __attribute__((ext_vector_type(2))); };
template <> struct Raw<4> { typedef unsigned int type; };
template <> struct Raw<2> { typedef unsigned short type; };

// V neighbouring elements as they lie in memory, and as numbers
template <typename T, int V>
struct Piece {
  typename Raw<V * sizeof(T)>::type raw;
  __device__ __forceinline__ void load(const T* p) { raw = *reinterpret_cast<const decltype(raw)*>(p); }
  template <bool STREAM>
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (STREAM)
      __builtin_nontemporal_store(raw, reinterpret_cast<std::remove_const_t<decltype(raw)>*>(p));
    else
      *reinterpret_cast<std::remove_const_t<decltype(raw)>*>(p) = raw;
  }
  __device__ __forceinline__ void get(float* v) const {
    if constexpr (sizeof(T) == 4) {
      __builtin_memcpy(v, &raw, V * 4);
    } else {
      uint16_t b[V];
      __builtin_memcpy(b, &raw, V * 2);
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = bf16_bits_to_float(b[i]);
    }
  }
  __device__ __forceinline__ void set(const float* v) {
    if constexpr (sizeof(T) == 4) {
      __builtin_memcpy(&raw, v, V * 4);
    } else if constexpr (V == 8) {
      const Chunk c = float_to_chunk<bf16>(v);
      __builtin_memcpy(&raw, &c, 16);
    } else {
      uint16_t b[V];
#pragma unroll
      for (int i = 0; i < V; ++i) b[i] = float_to_bf16_bits(v[i]);
      __builtin_memcpy(&raw, b, V * 2);
    }
  }
};

__device__ inline int64_t position_of(const RotaryArgs& p, int64_t row) {
  if (p.positions)
    return p.wide_positions ? static_cast<const int64_t*>(p.positions)[row] : static_cast<const int32_t*>(p.positions)[row];
  uint32_t q, r;
  p.seq.divmod(static_cast<uint32_t>(row), q, r);
  return p.start + r;
}

// s (cos, sin) of a pair at a position
__device__ inline float2 factors(const RotaryArgs& p, int64_t position, int pair) {
  const double turns = static_cast<double>(position) * (p.freqs[pair] * 0.15915494309189533577);   // 1 / (2 pi)
  const double half_turns = 2.0 * (turns - rint(turns));       // [-1, 1]
  const float h = static_cast<float>(half_turns);
  const float rest = static_cast<float>(half_turns - static_cast<double>(h)) * 3.14159265f;
  float s, c;
  sincospif(h, &s, &c);
  return make_float2(p.scale * fmaf(-rest, s, c), p.scale * p.sign * fmaf(rest, c, s));
}

// A unit is what a thread takes at a time: V pairs from two places of a head (HALVES, and V 1 of either layout), V / 2 pairs from V neighbours, or
// V elements that are copied.
template <typename T, int V, bool HALVES, bool STREAM>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs p) {
  constexpr bool TWO = HALVES || V == 1;
  __shared__ float2 lds[kMaxPairs];
  const int half = p.rot >> 1;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * p.group_rows;
  const int rows = static_cast<int>(min(static_cast<int64_t>(p.group_rows), p.rows - row0));
  const int head0 = blockIdx.y * p.group_heads.d, heads = min(static_cast<int>(p.group_heads.d), p.heads - head0);
  const uint32_t total = static_cast<uint32_t>(rows) * p.group_heads.d * p.units.d;
  const uint32_t rotated = TWO ? half / V : p.rot / V;

  struct Unit {
    Piece<T, V> a, b;
    int64_t to;          // of the unit's first element in y; -1: none
    int pair;            // in LDS; -1: copied
  };
  const int b_at = HALVES ? half : 1;
  auto request = [&](uint32_t q, Unit& u) {
    u.to = -1;
    if (q >= total) return;
    uint32_t line, unit, row, head;
    p.units.divmod(q, line, unit);
    p.group_heads.divmod(line, row, head);
    if (static_cast<int>(head) >= heads) return;
    const bool turned = unit < rotated;
    if (!turned && !p.copy) return;
    const int e = turned ? (TWO && !HALVES ? 2 * static_cast<int>(unit) : static_cast<int>(unit) * V)
                         : p.rot + static_cast<int>(unit - rotated) * V;
    const int64_t col = static_cast<int64_t>(head0 + head) * p.head_dim + e;
    u.pair = turned ? static_cast<int>(row) * half + (TWO && !HALVES ? static_cast<int>(unit) : HALVES ? e : e / 2) : -1;
    const T* from = static_cast<const T*>(p.x) + (row0 + row) * p.ldx + col;
    u.a.load(from);
    if (TWO && turned) u.b.load(from + b_at);
    u.to = (row0 + row) * p.ldy + col;
  };
  auto finish = [&](Unit& u) {
    if (u.to < 0) return;
    T* to = static_cast<T*>(p.y) + u.to;
    if (u.pair >= 0) {
      float a[V], b[V];
      u.a.get(a);
      if constexpr (TWO) {
        u.b.get(b);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float2 f = lds[u.pair + i];
          const float x = a[i];
          a[i] = x * f.x - b[i] * f.y;
          b[i] = b[i] * f.x + x * f.y;
        }
        u.b.set(b);
        u.b.template store<STREAM>(to + b_at);
      } else {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
          const float2 f = lds[u.pair + i];
          const float x = a[2 * i];
          a[2 * i] = x * f.x - a[2 * i + 1] * f.y;
          a[2 * i + 1] = a[2 * i + 1] * f.x + x * f.y;
        }
      }
      u.a.set(a);
    }
    u.a.template store<STREAM>(to);
  };

  Unit u[kUnitsAtOnce];
#pragma unroll
  for (int i = 0; i < kUnitsAtOnce; ++i) request(threadIdx.x + 256 * i, u[i]);   // on their way while the factors are made
  for (int i = threadIdx.x; i < rows * half; i += 256) {
    uint32_t row, pair;
    p.pairs.divmod(i, row, pair);
    lds[i] = factors(p, position_of(p, row0 + row), pair);
  }
  __syncthreads();
  for (uint32_t base = threadIdx.x;;) {
#pragma unroll
    for (int i = 0; i < kUnitsAtOnce; ++i) finish(u[i]);
    base += 256 * kUnitsAtOnce;
    if (base >= total) break;
#pragma unroll
    for (int i = 0; i < kUnitsAtOnce; ++i) request(base + 256 * i, u[i]);
  }
}

template <typename T, int V>
int launch_rotary(Context* ctx, const RotaryArgs& a, bool halves, dim3 grid, const char* name, double bytes) {
  if constexpr (V * sizeof(T) == 16)
    if (bytes > kStreamBytes)   // (131072 x 40 x 128 in bf16: 456 us, 469 without)
      return halves ? launch(ctx, rotary_kernel<T, V, true, true>, grid, dim3(256), a, name, bytes, 1)
                    : launch(ctx, rotary_kernel<T, V, false, true>, grid, dim3(256), a, name, bytes, 1);
  return halves ? launch(ctx, rotary_kernel<T, V, true, false>, grid, dim3(256), a, name, bytes, 1)
                : launch(ctx, rotary_kernel<T, V, false, false>, grid, dim3(256), a, name, bytes, 1);
}

}  // namespace

int rotary(Context* ctx, int dtype, const Rows& x, const Rows& y, const double* freqs, const void* positions, int wide_positions, int64_t start,
           int64_t seq, int64_t rows, int heads, int head_dim, int rot, int interleaved, float scale, int back) {
  TCH_CHECK_ARG(dtype == kBF16 || dtype == kF32, "rotary: dtype must be f32(0) or bf16(1)");
  TCH_CHECK_ARG(rows >= 0 && rows <= INT_MAX && heads > 0 && head_dim > 0 && static_cast<int64_t>(heads) * head_dim <= INT_MAX, "rotary: bad shape");
  TCH_CHECK_ARG(rot > 0 && rot % 2 == 0 && rot <= head_dim && rot <= 2 * kMaxPairs, "rotary: an even number of a head's elements is rotated, at most 4096");
  TCH_CHECK_ARG(positions || (seq > 0 && seq <= INT_MAX), "rotary: positions, or the length of a sequence");
  // (whole turns come off in fp64; further out less than 2^-12 of a turn would be right)
  TCH_CHECK_ARG(start >= -(1ll << 40) && start <= (1ll << 40), "rotary: start out of range");
  const int64_t width = static_cast<int64_t>(heads) * head_dim;
  const int eb = dtype == kBF16 ? 2 : 4;
  if (rows == 0) return 0;
  TCH_CHECK_ARG(x.ptr && y.ptr && freqs, "rotary: null tensor");
  TCH_CHECK_ARG((rows == 1 || (x.ld >= width && y.ld >= width)) && x.ld >= 0 && y.ld >= 0 && x.ld <= (1ll << 31) && y.ld <= (1ll << 31), "rotary: rows overlap");
  const uintptr_t px = reinterpret_cast<uintptr_t>(x.ptr), py = reinterpret_cast<uintptr_t>(y.ptr);
  TCH_CHECK_ARG((px | py) % eb == 0 && reinterpret_cast<uintptr_t>(freqs) % 8 == 0 &&
                    reinterpret_cast<uintptr_t>(positions) % (wide_positions ? 8 : 4) == 0, "rotary: a tensor is not aligned to its elements");
  const Span in{x.ptr, x.ld * eb, width * eb, rows}, out{y.ptr, y.ld * eb, width * eb, rows};
  const int pairs = rot / 2;
  TCH_CHECK_ARG(apart(out, in, true) && apart(out, {freqs, pairs * 8, pairs * 8, 1}) &&
                    apart(out, {positions, rows * (wide_positions ? 8 : 4), rows * (wide_positions ? 8 : 4), 1}),
                "rotary: the output overlaps an input (it may be the input itself)");
  // elements of an access: a whole chunk where heads, halves, rows and addresses allow it, two or one otherwise
  auto fits = [&](int v) {
    return (interleaved ? rot : pairs) % v == 0 && head_dim % v == 0 && rot % v == 0 && (rows == 1 || (x.ld % v == 0 && y.ld % v == 0)) && (px | py) % (v * eb) == 0;
  };
  const int chunk = 16 / eb, v = fits(chunk) ? chunk : fits(2) ? 2 : 1;
  const bool two = !interleaved || v == 1;
  RotaryArgs a{};
  a.x = x.ptr, a.ldx = x.ld;
  a.y = y.ptr, a.ldy = y.ld;
  a.freqs = freqs;
  a.positions = positions, a.wide_positions = wide_positions;
  a.start = start;
  a.rows = rows;
  a.heads = heads, a.head_dim = head_dim, a.rot = rot;
  a.copy = x.ptr != y.ptr;
  a.scale = scale, a.sign = back ? -1.f : 1.f;
  a.seq = FastDiv(static_cast<uint32_t>(positions ? 1 : seq));
  a.pairs = FastDiv(static_cast<uint32_t>(pairs));
  const int units = (two ? pairs : rot) / v + (head_dim - rot) / v;
  a.units = FastDiv(static_cast<uint32_t>(units));
  // A workgroup's share: what its threads take in one go, as whole rows or as a run of one row's heads; less where that leaves fewer
  // than six workgroups a compute unit (8192 x 24 x 64 in bf16: 9.3 us, 10.4 with 820 workgroups; 131072 x 40 x 128 512 with half the share, 457).
  const int64_t most = 256 * kUnitsAtOnce, of_row = static_cast<int64_t>(heads) * units;
  const int64_t share = std::min(std::max(rows * of_row / 1536, static_cast<int64_t>(256)), most);
  int group_heads = heads;
  a.group_rows = 1;
  if (of_row >= most)
    group_heads = static_cast<int>(std::max<int64_t>(most / units, 1));
  else
    a.group_rows = static_cast<int>(std::max<int64_t>(std::min<int64_t>({share / of_row, kMaxPairs / pairs, rows}), 1));
  const int64_t runs = (heads + group_heads - 1) / group_heads;
  TCH_CHECK_ARG(runs <= 65535, "rotary: too many heads");
  a.group_heads = FastDiv(static_cast<uint32_t>(group_heads));
  TCH_CHECK_ARG((rows + a.group_rows - 1) / a.group_rows < (1 << 24), "rotary: too many rows");   // (2^32 threads along a grid's side)
  const dim3 grid(static_cast<unsigned>((rows + a.group_rows - 1) / a.group_rows), static_cast<unsigned>(runs));
  const double bytes = 2.0 * rows * (a.copy ? width : static_cast<int64_t>(heads) * rot) * eb;
  const bool halves = !interleaved;
  if (dtype == kBF16)
    return v == 8   ? launch_rotary<bf16, 8>(ctx, a, halves, grid, "rotary_kernel<bf16>", bytes)
           : v == 2 ? launch_rotary<bf16, 2>(ctx, a, halves, grid, "rotary_kernel<bf16,2>", bytes)
                    : launch_rotary<bf16, 1>(ctx, a, halves, grid, "rotary_kernel<bf16,1>", bytes);
  return v == 4   ? launch_rotary<float, 4>(ctx, a, halves, grid, "rotary_kernel<f32>", bytes)
         : v == 2 ? launch_rotary<float, 2>(ctx, a, halves, grid, "rotary_kernel<f32,2>", bytes)
                  : launch_rotary<float, 1>(ctx, a, halves, grid, "rotary_kernel<f32,1>", bytes);
}

}  // namespace tch

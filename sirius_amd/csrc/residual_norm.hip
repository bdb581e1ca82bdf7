// The boundary between two blocks of a transformer, in one pass: the norm behind a block, its gate, the residual and its scale, and
// the norm in front of the next block.
//   n = pw . b^ + pb      b^ = (b - mean) / deviation of the block's output b (post norm; without one n = b)
//   t = s x + g . n       g: none, a vector, or a vector per sample
//   y = w . t^ + c        t^ = (t - mean) / deviation of t as it is stored
// with the mean and the deviation of a row (LayerNorm), or a mean of 0 (RMS).  Backward, from dy and the gradient dt0 that t has from
// elsewhere, with k = w . dy:
//   dt = dt0 + (k - mean(k) - t^ mean(k t^)) / deviation,   dx = s dt,   dn = g . dt,   db: through the post norm likewise
//   dw = sum dy t^,  dc = sum dy;  over the rows of a gate A = sum dt b^, B = sum dt:  dg = pw A + pb B,  dpw = sum g A,  dpb = sum g B
//
// Bound by memory: four tensors forward, six backward.  A lane has eight neighbours of a row, a row as many wavefronts as that takes (short
// rows share one), the vectors stay in registers while a workgroup walks its rows, and the next row is on its way while this one is
// worked on.  Means, deviations and sums are fp32 in registers; a wavefront's part of a deviation is taken about its own mean, and the
// parts are joined about the row's.  What a workgroup adds up over its rows goes to the workspace, where a second launch adds the
// workgroups up in fp64 in their order: the same bits every run.
// In bf16 with RMS norms and a gate 8192 x 4096 forward 47 us (5.7 TB/s), backward 77 (5.2); 16384 x 8192 189 (5.7) and 280 (5.8); in fp32 8192 x 4096
// 89 (6.0) and 140 (5.8); 8192 x 1024 with a LayerNorm and a gate forward 12.5; one token of 4096 3.5.
//
// Reference call sites: the blocks that train/gpt2.py:26 and train/swin_b.py:38 build have a LayerNorm in front of each half and a
// plain residual.
#include <algorithm>
#include <climits>

#include "context.h"
#include "linear_epilogue.h"
#include "ops.h"
#include "pack8.h"

namespace tch {
namespace {

constexpr int kEach = 8;             // neighbours of a lane
constexpr int kMaxWidth = 8192;      // sixteen wavefronts a row
enum Branch : int { kNoBranch = 0, kBranch = 1, kPostNorm = 2 };

struct RowsPtr {
  void* at;
  int64_t ld;   // elements
};

struct NormArgs {
  RowsPtr x, branch, total, y;            // forward
  RowsPtr dy, dtotal, dx, dbranch;        // backward, with total and branch
  float4* stats;                          // [rows] mean and 1 / deviation of the branch, of the total
  const float* weight;                    // null: there is no norm behind the sum
  const float* bias;
  const float* post_weight;
  const float* post_bias;
  const void* gate;
  unsigned char* packed;                  // forward: y in 8 bits too
  unsigned char* codes;
  int64_t rows, gate_rows;                // gate_rows: rows that share a gate
  FastDiv gate_div;                       // forward: by them
  int C, waves, groups;                   // wavefronts of a row, rows at a time of a workgroup
  int layer, gate_f32, format;
  float scale, eps;
  // backward
  float* sums;                            // [workgroups][planes][C]
  float* dgate;                           // [gates][C]: written here where a workgroup has all rows of its gates
  int planes, plane_of[4];                // -1: nobody wants it
  int split_gates, pieces;                // several workgroups have a part of a gate's rows: so many
  int gates_each;                         // otherwise: gates of a workgroup
  int gates, add_gates;
};

// the sum over the L lanes of a row, in every lane of it; L = 64: over the wavefront
template <int L>
__device__ __forceinline__ float lane_sum(float v) {
  auto plus = [&](auto ctrl) {
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  plus(std::integral_constant<int, 0xb1>{});     // lane ^ 1
  plus(std::integral_constant<int, 0x4e>{});     // lane ^ 2
  plus(std::integral_constant<int, 0x141>{});    // the other half of eight
  plus(std::integral_constant<int, 0x140>{});    // the other half of sixteen
  auto both = [&](auto r) { v = __uint_as_float(r[0]) + __uint_as_float(r[1]); };
  if constexpr (L > 16) both(__builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  if constexpr (L > 32) both(__builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  return v;
}

// What the wavefronts of a row tell each other: two numbers each, in turn in two places, so that one barrier a time is enough.
struct Meeting {
  float2 (*said)[16];
  int turn, first, waves, lane, wave;
  // what wavefront lane % 16 of the row said; 0 of one that is not there
  __device__ __forceinline__ float2 say(float a, float b) {
    float2* here = said[turn];
    turn ^= 1;
    if (lane == 0) here[wave] = make_float2(a, b);
    __syncthreads();
    return (lane & 15) < waves ? here[first + (lane & 15)] : make_float2(0.f, 0.f);
  }
  // both sums over the row, of sums over the wavefronts
  __device__ __forceinline__ void add(float& a, float& b) {
    if (waves == 1) return;
    const float2 h = say(a, b);
    a = lane_sum<16>(h.x);
    b = lane_sum<16>(h.y);
  }
};

// A lane's eight neighbours of a row in bf16, or in fp32 twice four, a row of lanes apart: an access of the lanes is whole lines either way.
struct Cols {
  int at[2];     // of the first and the second four
  bool on[2];    // whether they are there: bf16 rows are whole eights, fp32 rows whole fours
  __device__ __forceinline__ Cols in(bool row) const { return {{at[0], at[1]}, {on[0] && row, on[1] && row}}; }
};

// What the lanes of a row know of its wavefronts' elements: divided once for all rows (LayerNorms 8192 x 4096 53 us for 59).
struct Counts {
  float inv, inv_here, there, inv_there;   // 1 / C, 1 / those of this wavefront, those of wavefront lane % 16 of the row and 1 / them
};
template <int L>
__device__ __forceinline__ Counts counts(const NormArgs& p, int row_wave, int lane) {
  auto elements = [&](int w) { return L < 64 ? p.C : max(min(p.C - w * 64 * kEach, 64 * kEach), 1); };
  const float there = static_cast<float>(elements(lane & 15));
  return {1.f / static_cast<float>(p.C), 1.f / static_cast<float>(elements(row_wave)), there, 1.f / there};
}

// mean and 1 / deviation of a row
template <int L>
__device__ __forceinline__ float2 row_stats(const float* v, const Cols& cols, int layer, float eps, const Counts& n, Meeting& meet) {
  if (!layer) {
    float q = 0.f, none = 0.f;
#pragma unroll
    for (int e = 0; e < kEach; ++e) q = cols.on[e / 4] ? fmaf(v[e], v[e], q) : q;
    q = lane_sum<L>(q);
    meet.add(q, none);
    return make_float2(0.f, rsqrtf(q * n.inv + eps));
  }
  float s = 0.f;
#pragma unroll
  for (int e = 0; e < kEach; ++e) s += cols.on[e / 4] ? v[e] : 0.f;
  s = lane_sum<L>(s);
  const float mine = s * n.inv_here;
  float q = 0.f;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const float d = v[e] - mine;
    q = cols.on[e / 4] ? fmaf(d, d, q) : q;
  }
  q = lane_sum<L>(q);
  if (meet.waves == 1) return make_float2(mine, rsqrtf(q * n.inv + eps));
  const float2 h = meet.say(s, q);
  const float mean = lane_sum<16>(h.x) * n.inv, d = h.x * n.inv_there - mean;
  q = lane_sum<16>((meet.lane & 15) < meet.waves ? fmaf(n.there * d, d, h.y) : 0.f);
  return make_float2(mean, rsqrtf(q * n.inv + eps));
}

// A lane's eight as they lie in memory.
template <typename T, bool STREAM = false>
struct Eight {
  static constexpr int N = sizeof(T) / 2;   // chunks
  Chunk c[N];
  __device__ __forceinline__ void load(const RowsPtr& t, int64_t row, const Cols& cols) {
    const T* from = static_cast<const T*>(t.at) + row * t.ld;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      c[i] = zero_chunk();
      const uint4* chunk = reinterpret_cast<const uint4*>(from + cols.at[i]);
      if (cols.on[i]) c[i].u = STREAM ? load_streaming_u4(chunk, 0) : *chunk;
    }
  }
  __device__ __forceinline__ void get(float* v) const {
#pragma unroll
    for (int i = 0; i < N; ++i) chunk_to_float<T>(c[i], v + i * (kEach / N));
  }
  __device__ __forceinline__ void set(const float* v) {
#pragma unroll
    for (int i = 0; i < N; ++i) c[i] = float_to_chunk<T>(v + i * (kEach / N));
  }
  __device__ __forceinline__ void store(const RowsPtr& t, int64_t row, const Cols& cols) const {
    T* to = static_cast<T*>(t.at) + row * t.ld;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (cols.on[i]) store_u4<STREAM>(to + cols.at[i], 0, c[i].u);
  }
};

__device__ __forceinline__ void load_vector(const float* from, const Cols& cols, float otherwise, float* v) {
#pragma unroll
  for (int i = 0; i < kEach; i += 4) {
    float4 f = make_float4(otherwise, otherwise, otherwise, otherwise);
    if (from && cols.on[i / 4]) f = *reinterpret_cast<const float4*>(from + cols.at[i / 4]);
    v[i] = f.x, v[i + 1] = f.y, v[i + 2] = f.z, v[i + 3] = f.w;
  }
}
template <typename T>
__device__ __forceinline__ void load_gate(const NormArgs& p, int64_t gate, const Cols& cols, float* v) {
  if (!p.gate || p.gate_f32) {
    load_vector(static_cast<const float*>(p.gate) + (p.gate ? gate * p.C : 0), cols, 1.f, v);
  } else {
    Eight<T> g;
    g.load({const_cast<void*>(p.gate), p.C}, gate, cols);
    g.get(v);
  }
}

// y in 8 bits, as it is stored: the lanes of 32 neighbours are neighbours, four of them in bf16, eight in fp32
template <typename T, int FORMAT>
__device__ __forceinline__ void keep(const NormArgs& p, int64_t row, const Cols& cols, const float* v, int lane) {
  unsigned char* data = p.packed + row * p.C;
  unsigned char* codes = p.codes + row * ((p.C + kPackGroup - 1) / kPackGroup);
  if constexpr (sizeof(T) == 2) {
    uint32_t words[2];
    const uint32_t code = pack8_lane<FORMAT>(v, cols.on[0] ? 8 : 0, words);
    if (cols.on[0]) *reinterpret_cast<uint2*>(data + cols.at[0]) = make_uint2(words[0], words[1]);
    if (cols.on[0] && lane % 4 == 0) codes[cols.at[0] / kPackGroup] = static_cast<unsigned char>(code);
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t word;
      const uint32_t code = pack8_four<FORMAT>(v + 4 * i, cols.on[i], &word);
      if (cols.on[i]) *reinterpret_cast<uint32_t*>(data + cols.at[i]) = word;
      if (cols.on[i] && lane % 8 == 0) codes[cols.at[i] / kPackGroup] = static_cast<unsigned char>(code);
    }
  }
}

struct Place {   // of a lane
  int lane, wave, row_wave, group;
  Cols cols;
};
template <typename T, int L>
__device__ __forceinline__ Place place(const NormArgs& p) {
  Place a;
  a.lane = threadIdx.x & 63;
  a.wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  a.row_wave = 0;
  if (L < 64) {
    a.group = threadIdx.x / L;
  } else {
    a.group = a.wave / p.waves;
    a.row_wave = a.wave - a.group * p.waves;
  }
  const int first = a.row_wave * 64 * kEach, sub = a.lane % L;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    a.cols.at[i] = first + (sizeof(T) == 2 ? sub * 8 + i * 4 : (i * L + sub) * 4);
    a.cols.on[i] = a.cols.at[i] < p.C;
  }
  if (sizeof(T) == 2) a.cols.on[1] = a.cols.on[0];
  return a;
}

// WIDE: rows of more than eight wavefronts
template <typename T, int L, bool WIDE, int BR, bool STREAM>
__global__ __launch_bounds__(L < 64 ? 256 : WIDE ? 1024 : 512) void residual_norm_fwd_kernel(NormArgs p) {
  __shared__ float2 said[2][16];
  const Place at = place<T, L>(p);
  Meeting meet{said, 0, at.group * p.waves, p.waves, at.lane, at.wave};
  const Counts count = counts<L>(p, at.row_wave, at.lane);
  const bool samples = p.gate_rows < p.rows;
  float w[kEach], c[kEach], pw[kEach], pb[kEach], g[kEach];
  load_vector(p.weight, at.cols, 1.f, w);
  load_vector(p.bias, at.cols, 0.f, c);
  if constexpr (BR != kNoBranch) load_gate<T>(p, 0, at.cols, g);
  if constexpr (BR == kPostNorm) {
    load_vector(p.post_weight, at.cols, 1.f, pw);
    load_vector(p.post_bias, at.cols, 0.f, pb);
  }
  const int64_t step = static_cast<int64_t>(gridDim.x) * p.groups;
  int64_t row = static_cast<int64_t>(blockIdx.x) * p.groups + at.group;
  // The next row is on its way, of a wide one, which has the compute unit to itself, the one behind that too (16384 x 8192 in bf16: 199 us, 220
  // with one; 8192 x 1024 13.9, 13.2 with one).
  constexpr int AHEAD = WIDE ? 2 : 1;
  Eight<T, STREAM> xs[AHEAD], bs[AHEAD];
  auto request = [&](Eight<T, STREAM>& x, Eight<T, STREAM>& b, int64_t r) {
    const Cols cols = at.cols.in(r < p.rows);
    x.load(p.x, r, cols);
    if constexpr (BR != kNoBranch) b.load(p.branch, r, cols);
  };
  request(xs[0], bs[0], row);
  if constexpr (WIDE) request(xs[AHEAD - 1], bs[AHEAD - 1], row + step);
  // (every wavefront of the workgroup makes as many rounds: they meet in each)
  auto round = [&](Eight<T, STREAM>& x, Eight<T, STREAM>& b) __attribute__((always_inline)) {
    const Cols cols = at.cols.in(row < p.rows);
    float t[kEach], n[kEach];
    x.get(t);
    if constexpr (BR != kNoBranch) b.get(n);
    if (BR != kNoBranch && samples && row < p.rows) load_gate<T>(p, p.gate_div.div(static_cast<uint32_t>(row)), cols, g);
    request(x, b, row + AHEAD * step);
    float4 stats = make_float4(0.f, 0.f, 0.f, 0.f);
    if constexpr (BR == kPostNorm) {
      const float2 s = row_stats<L>(n, at.cols, p.layer, p.eps, count, meet);
      stats.x = s.x, stats.y = s.y;
#pragma unroll
      for (int e = 0; e < kEach; ++e) n[e] = fmaf((n[e] - s.x) * s.y, pw[e], pb[e]);
    }
    if constexpr (BR != kNoBranch) {
#pragma unroll
      for (int e = 0; e < kEach; ++e) t[e] = fmaf(g[e], n[e], p.scale * t[e]);
      Eight<T, STREAM> sum;
      sum.set(t);
      sum.store(p.total, row, cols);
      sum.get(t);
    }
    if (p.weight) {
      const float2 s = row_stats<L>(t, at.cols, p.layer, p.eps, count, meet);
      stats.z = s.x, stats.w = s.y;
#pragma unroll
      for (int e = 0; e < kEach; ++e) t[e] = fmaf((t[e] - s.x) * s.y, w[e], c[e]);
      Eight<T, STREAM> y;
      y.set(t);
      y.store(p.y, row, cols);
      if (p.packed) {   // what is kept is y as it is stored
        y.get(t);
        p.format == kPackInt8 ? keep<T, kPackInt8>(p, row, cols, t, at.lane) : keep<T, kPackE4m3>(p, row, cols, t, at.lane);
      }
    }
    if (row < p.rows && at.cols.at[0] == 0) p.stats[row] = stats;
  };
  for (int64_t first = static_cast<int64_t>(blockIdx.x) * p.groups; first < p.rows; first += step, row += step) {
    round(xs[0], bs[0]);
    if constexpr (WIDE) {
      if ((first += step) >= p.rows) break;
      row += step;
      round(xs[AHEAD - 1], bs[AHEAD - 1]);
    }
  }
}

// What a call asks for, as far as it is worth a kernel of its own: kFullRms and kFullLayer have the norm behind the sum, and a workgroup's rows
// have one gate, whose sums of dt b^ and dt go out as they are (what the gate makes of them the second launch does, once for all of
// its rows); kFullRms adds no rows of dy and dt up (there are no biases).  kAnything is told the rest by its arguments: among it several
// gates in a workgroup, where what each has to itself is taken here.  (Branches at run time and accumulators that nobody asked for make 10 to
// 110 registers of a wide row's spill; what is only loaded or stored on request costs none.)
enum BwdMode : int { kAnything = 0, kFullRms = 1, kFullLayer = 2 };
template <typename T, int L, bool WIDE, int BR, int MODE, bool STREAM>
__global__ __launch_bounds__(L < 64 ? 256 : WIDE ? 1024 : 512) void residual_norm_bwd_kernel(NormArgs p) {
  constexpr int kLds = WIDE ? 1 : 256 * kEach;   // (rows of more than four wavefronts come one at a time: there is nothing to add up here)
  const bool has_norm = MODE != kAnything || p.weight, has_dtotal = p.dtotal.at, has_dx = p.dx.at;
  const bool layer = MODE == kAnything ? p.layer != 0 : MODE == kFullLayer;
  const bool many = MODE == kAnything && !p.split_gates;
  const bool rows_of_dy = MODE == kAnything ? p.plane_of[1] >= 0 : MODE == kFullLayer, rows_of_dt = MODE == kAnything || MODE == kFullLayer;
  __shared__ float2 said[2][16];
  __shared__ float lds[kLds];
  const Place at = place<T, L>(p);
  Meeting meet{said, 0, at.group * p.waves, p.waves, at.lane, at.wave};
  const float inv = 1.f / static_cast<float>(p.C);
  float w[kEach], k2[kEach];   // k2: what dt is multiplied by in front of the post norm, g . pw; the gate where there is none
  // Where a wide row's lanes would spill they have what they need once a row or once a gate in places of their own there (256 gates of 16384 x
  // 8192 with LayerNorms in bf16 382 -> 331 us, 4096 x 8192 in fp32 161 -> 158; bf16 with one gate 281 -> 289 us, so not there).
  constexpr bool OWN = WIDE && (MODE == kAnything || sizeof(T) == 4);
  __shared__ float4 own[!OWN ? 1 : MODE == kAnything ? 8 : 4][OWN ? 1024 : 1];
  auto hold = [&](int i, const float* v) {
    if constexpr (OWN) {
      own[2 * i][threadIdx.x] = make_float4(v[0], v[1], v[2], v[3]);
      own[2 * i + 1][threadIdx.x] = make_float4(v[4], v[5], v[6], v[7]);
    }
  };
  auto fetch = [&](int i, float* v) {
    if constexpr (OWN) {
      const float4 lo = own[2 * i][threadIdx.x], hi = own[2 * i + 1][threadIdx.x];
      v[0] = lo.x, v[1] = lo.y, v[2] = lo.z, v[3] = lo.w, v[4] = hi.x, v[5] = hi.y, v[6] = hi.z, v[7] = hi.w;
    }
  };
  load_vector(p.weight, at.cols, 0.f, w);
  hold(0, w);
  float sum[4][kEach], gated[2][kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e) sum[0][e] = sum[1][e] = sum[2][e] = sum[3][e] = gated[0][e] = gated[1][e] = 0.f;
  if constexpr (MODE == kAnything) {
    hold(2, gated[0]);
    hold(3, gated[1]);
  }

  // The lanes' eight sums over the row groups of the workgroup, to `to` [C].
  auto add_up = [&](const float* v, float* to, bool add) {
    if (WIDE || p.groups == 1) {
#pragma unroll
      for (int i = 0; i < kEach; i += 4) {
        if (!at.cols.on[i / 4]) break;
        float4* out = reinterpret_cast<float4*>(to + at.cols.at[i / 4]);
        float4 s = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        if (add) {
          const float4 old = *out;
          s = make_float4(s.x + old.x, s.y + old.y, s.z + old.z, s.w + old.w);
        }
        *out = s;
      }
      return;
    }
    const int span = (L < 64 ? L : p.waves * 64) * kEach;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kEach; ++e) lds[at.group * span + at.cols.at[e / 4] + e % 4] = v[e];
    __syncthreads();
    for (int c = threadIdx.x; c < p.C; c += blockDim.x) {
      float s = 0.f;
      for (int q = 0; q < p.groups; ++q) s += lds[q * span + c];
      to[c] = add ? to[c] + s : s;
    }
  };

  // The workgroups of a gate's rows take them in turn, so that what the chip works on at a time lies together (each with a run of its
  // own rows the 16384 x 8192 case runs at 5.1 TB/s).
  int gate = 0, behind_gate = 1;
  int64_t offset = 0, step = p.groups;
  if (p.split_gates) {
    gate = blockIdx.x / p.pieces;
    behind_gate = gate + 1;
    offset = static_cast<int64_t>(blockIdx.x - gate * p.pieces) * p.groups;
    step *= p.pieces;
  } else {
    gate = blockIdx.x * p.gates_each;
    behind_gate = min(gate + p.gates_each, p.gates);
  }
  for (; gate < behind_gate; ++gate) {
    const int64_t r0 = gate * p.gate_rows + offset, r1 = min((gate + 1) * p.gate_rows, p.rows);
    if constexpr (BR != kNoBranch) {
      load_gate<T>(p, gate, at.cols, k2);
      if constexpr (BR == kPostNorm) {
        float pw[kEach];
        load_vector(p.post_weight, at.cols, 0.f, pw);
#pragma unroll
        for (int e = 0; e < kEach; ++e) k2[e] *= pw[e];
      }
      hold(1, k2);
    }
    Eight<T, STREAM> dy, d0, t, b;
    float4 stats, next_stats;
    auto request = [&](int64_t row) {
      const Cols cols = at.cols.in(row < r1);
      if (has_norm) {
        dy.load(p.dy, row, cols);
        t.load(p.total, row, cols);
      }
      d0.load(p.dtotal, row, cols.in(has_dtotal));
      if constexpr (BR != kNoBranch) b.load(p.branch, row, cols);
      next_stats = make_float4(0.f, 0.f, 0.f, 0.f);
      if (row < r1) next_stats = p.stats[row];
    };
    request(r0 + at.group);
    for (int64_t first = r0; first < r1; first += step) {
      const int64_t row = first + at.group;
      const Cols cols = at.cols.in(row < r1);
      stats = next_stats;
      float d[kEach], h[kEach], k[kEach], bh[kEach];
      d0.get(d);
      if (has_norm) {
        dy.get(k);
        t.get(h);
      }
      if constexpr (BR != kNoBranch) b.get(bh);
      request(row + step);
      if (has_norm) {
        float a = 0.f, q = 0.f;
        fetch(0, w);
        if (layer)
#pragma unroll
          for (int e = 0; e < kEach; ++e) h[e] -= stats.z;
        if (rows_of_dy)
#pragma unroll
          for (int e = 0; e < kEach; ++e) sum[1][e] += k[e];      // (rows and columns that are not there have a gradient of 0)
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
          h[e] *= stats.w;
          sum[0][e] = fmaf(k[e], h[e], sum[0][e]);
          k[e] *= w[e];
          q = fmaf(k[e], h[e], q);
        }
        if (layer) {
#pragma unroll
          for (int e = 0; e < kEach; ++e) a += k[e];
          a = lane_sum<L>(a);
        }
        q = lane_sum<L>(q);
        meet.add(a, q);
        q *= inv;
        if (layer) {
          a *= inv;
#pragma unroll
          for (int e = 0; e < kEach; ++e) k[e] -= a;
        }
        const float r_lo = cols.on[0] ? stats.w : 0.f, r_hi = cols.on[1] ? stats.w : 0.f;   // (d stays 0 where nothing is)
#pragma unroll
        for (int e = 0; e < kEach; ++e) d[e] = fmaf(e < 4 ? r_lo : r_hi, fmaf(-h[e], q, k[e]), d[e]);
      }
      if (has_dx) {
        Eight<T, STREAM> dx;
        if (p.scale != 1.f) {
#pragma unroll
          for (int e = 0; e < kEach; ++e) h[e] = p.scale * d[e];
          dx.set(h);
        } else {
          dx.set(d);
        }
        dx.store(p.dx, row, cols);
      }
      if constexpr (BR != kNoBranch) {
        fetch(1, k2);
        if (BR == kPostNorm && layer)
#pragma unroll
          for (int e = 0; e < kEach; ++e) bh[e] -= stats.x;
        if (rows_of_dt)
#pragma unroll
          for (int e = 0; e < kEach; ++e) sum[3][e] += d[e];
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
          if constexpr (BR == kPostNorm) bh[e] *= stats.y;
          sum[2][e] = fmaf(d[e], bh[e], sum[2][e]);
          k[e] = d[e] * k2[e];
        }
        if constexpr (BR == kPostNorm) {
          float a = 0.f, q = 0.f;
#pragma unroll
          for (int e = 0; e < kEach; ++e) q = fmaf(k[e], bh[e], q);
          if (layer) {
#pragma unroll
            for (int e = 0; e < kEach; ++e) a += k[e];
            a = lane_sum<L>(a);
          }
          q = lane_sum<L>(q);
          meet.add(a, q);
          q *= inv;
          if (layer) {
            a *= inv;
#pragma unroll
            for (int e = 0; e < kEach; ++e) k[e] -= a;
          }
#pragma unroll
          for (int e = 0; e < kEach; ++e) k[e] = stats.y * fmaf(-bh[e], q, k[e]);
        }
        Eight<T, STREAM> db;
        db.set(k);
        db.store(p.dbranch, row, cols);
      }
    }
    if (many) {
      // dg of these rows, and what the post norm's gradients have from them
      float g[kEach], dg[kEach], pw[kEach], pb[kEach];
      load_gate<T>(p, gate, at.cols, g);
      load_vector(p.post_weight, at.cols, 1.f, pw);
      load_vector(p.post_bias, at.cols, 0.f, pb);
      if constexpr (MODE == kAnything) {
        fetch(2, gated[0]);
        fetch(3, gated[1]);
      }
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        dg[e] = fmaf(pw[e], sum[2][e], pb[e] * sum[3][e]);
        gated[0][e] = fmaf(g[e], sum[2][e], gated[0][e]);
        gated[1][e] = fmaf(g[e], sum[3][e], gated[1][e]);
        sum[2][e] = sum[3][e] = 0.f;
      }
      if constexpr (MODE == kAnything) {
        hold(2, gated[0]);
        hold(3, gated[1]);
      }
      if (p.dgate) add_up(dg, p.dgate + static_cast<int64_t>(gate) * p.C, p.add_gates);
    }
  }
  if (many) {
    if constexpr (MODE == kAnything) {
      fetch(2, gated[0]);
      fetch(3, gated[1]);
    }
#pragma unroll
    for (int e = 0; e < kEach; ++e) sum[2][e] = gated[0][e], sum[3][e] = gated[1][e];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (p.plane_of[i] >= 0) add_up(sum[i], p.sums + (static_cast<int64_t>(blockIdx.x) * p.planes + p.plane_of[i]) * p.C, false);
}

// The workgroups' sums added up: 32 columns a workgroup, kLines threads a column, in fp64 in a fixed order.  blockIdx.y 0: the norm's two
// gradients; 1: those of the post norm; 2 and on: of gate blockIdx.y - 2.
struct NormSumArgs {
  const float* sums;
  const float* post_weight;
  const float* post_bias;
  const void* gate;         // [gates][C] where the sums are still without it, or null
  float* dweight;
  float* dbias;
  float* dpost_weight;
  float* dpost_bias;
  float* dgate;
  int C, blocks, planes, plane_of[4];
  int pieces;               // workgroups of a gate's rows
  FastDiv div;              // by them
  int gate_f32, add;
};
template <int kLines>
__global__ __launch_bounds__(32 * kLines) void residual_norm_sum_kernel(NormSumArgs p) {
  __shared__ double meet[2][kLines][32];
  const int lane = threadIdx.x & 31, line = threadIdx.x >> 5, c = blockIdx.x * 32 + lane, job = blockIdx.y;
  double s[2] = {0.0, 0.0};
  if (c < p.C) {
    const int first = job < 2 ? 0 : (job - 2) * p.pieces, behind = job < 2 ? p.blocks : first + p.pieces;
    const int64_t ld = static_cast<int64_t>(p.planes) * p.C;
    constexpr int U = 8;   // workgroups of a thread, on their way together; behind the last one it is read again, for nothing
    const int plane0 = p.plane_of[job == 0 ? 0 : 2], plane1 = p.plane_of[job == 0 ? 1 : 3];
    auto add_up = [&](auto planes_c, int plane, int other, double* sum, auto weight_of) {
      constexpr int N = decltype(planes_c)::value;
      const float* at[2] = {p.sums + static_cast<int64_t>(plane) * p.C + c, p.sums + static_cast<int64_t>(other) * p.C + c};
      for (int b = first + line; b < behind; b += U * kLines) {
        float v[U][N], g[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int block = min(b + u * kLines, behind - 1);
#pragma unroll
          for (int i = 0; i < N; ++i) v[u][i] = at[i][block * ld];
          g[u] = weight_of(block);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int i = 0; i < N; ++i) sum[i] += b + u * kLines < behind ? static_cast<double>(g[u]) * v[u][i] : 0.0;
      }
    };
    auto with_weight = [&](auto weight_of) {
      if (plane0 >= 0 && plane1 >= 0)
        add_up(std::integral_constant<int, 2>{}, plane0, plane1, s, weight_of);
      else if (plane0 >= 0)
        add_up(std::integral_constant<int, 1>{}, plane0, plane0, s, weight_of);
      else if (plane1 >= 0)
        add_up(std::integral_constant<int, 1>{}, plane1, plane1, s + 1, weight_of);
    };
    auto gate_at = [&](int block) { return static_cast<int64_t>(p.div.div(static_cast<uint32_t>(block))) * p.C + c; };
    if (job != 1 || !p.gate)
      with_weight([](int) { return 1.f; });
    else if (p.gate_f32)
      with_weight([&](int block) { return static_cast<const float*>(p.gate)[gate_at(block)]; });
    else
      with_weight([&](int block) { return Elem<bf16>::load(static_cast<const bf16*>(p.gate) + gate_at(block)); });
  }
  meet[0][line][lane] = s[0];
  meet[1][line][lane] = s[1];
  for (int half = kLines / 2; half > 0; half /= 2) {
    __syncthreads();
    if (line < half)
#pragma unroll
      for (int i = 0; i < 2; ++i) meet[i][line][lane] += meet[i][line + half][lane];
  }
  if (line != 0 || c >= p.C) return;
  s[0] = meet[0][0][lane], s[1] = meet[1][0][lane];
  auto put = [&](float* to, int64_t i, double v) {
    if (to) to[i] = p.add ? static_cast<float>(to[i] + v) : static_cast<float>(v);
  };
  if (job == 0) {
    put(p.dweight, c, s[0]);
    put(p.dbias, c, s[1]);
  } else if (job == 1) {
    put(p.dpost_weight, c, s[0]);
    put(p.dpost_bias, c, s[1]);
  } else {
    const double w = p.post_weight ? p.post_weight[c] : 1.0, b = p.post_bias ? p.post_bias[c] : 0.0;
    put(p.dgate, static_cast<int64_t>(job - 2) * p.C + c, w * s[0] + b * s[1]);
  }
}

struct Shape {
  int lanes, waves, groups, threads;   // lanes: 16, 32, or 64 (as many wavefronts as it takes)
};
// As many rows at a time as make four wavefronts, where there are that many.
Shape shape_of(int64_t rows, int C) {
  if (C <= 16 * kEach) return {16, 1, 16, 256};
  if (C <= 32 * kEach) return {32, 1, 8, 256};
  const int waves = (C + 64 * kEach - 1) / (64 * kEach);
  const int groups = static_cast<int>(std::min<int64_t>(std::max(4 / waves, 1), std::max<int64_t>(rows, 1)));
  return {64, waves, groups, waves * groups * 64};
}

// The backward's workgroups: 512 of four wavefronts or fewer, 256 of more, with equally many rounds each.  A compute unit has eight wavefronts of
// rows of up to 1024, of 2048 and of 4096 elements and sixteen of 8192; in between it has what the row leaves it (six at 1536, five at 2560, nine at
// 4608).  (Twelve are resident, but every workgroup leaves its sums: 8192 x 4096 in bf16 84 us with 512 of eight, 78 with 256.  Other counts for the
// widths in between are not measured: 16384 x 1536 with LayerNorms runs at 4.8 TB/s.)  From half as many gates as workgroups on, a workgroup has all
// rows of its gates, and with 130 or 300 gates some compute units none: 8320 x 8192 with 130 gates 236 us, 8192 x 8192 with 256 171.
struct Cut {
  Shape shape;
  int64_t blocks, pieces;   // pieces: workgroups of a gate's rows
  int gates_each;           // gates of a workgroup
  bool split;               // a gate's rows are several workgroups'; otherwise a workgroup has all rows of its gates
};
Cut cut_rows(int64_t rows, int C, int64_t gates) {
  Cut c{};
  c.shape = shape_of(rows, C);
  const int64_t want = c.shape.threads > 256 ? 256 : 512, rounds = (rows / gates + c.shape.groups - 1) / c.shape.groups;
  const int64_t most = std::max<int64_t>(want / gates, 1), each = (rounds + most - 1) / most;
  c.pieces = (rounds + each - 1) / each;
  c.gates_each = static_cast<int>((gates + want - 1) / want);
  c.split = gates == 1 || c.pieces > 1;   // (256 gates of 8192 x 4096 from their sums in a second launch 110 us, with all their rows in a workgroup 91)
  c.blocks = c.split ? gates * c.pieces : (gates + c.gates_each - 1) / c.gates_each;
  return c;
}

int check_shape(const char* what, int dtype, int64_t rows, int64_t C, int64_t gates) {
  const std::string name(what);
  TCH_CHECK_ARG(dtype == kBF16 || dtype == kF32, name + ": dtype must be f32(0) or bf16(1)");
  TCH_CHECK_ARG(rows >= 0 && rows <= INT_MAX && C > 0 && C <= kMaxWidth, name + ": rows of 1 to 8192 elements");
  TCH_CHECK_ARG(C % (dtype == kBF16 ? 8 : 4) == 0, name + ": rows must be whole 16-byte chunks");
  TCH_CHECK_ARG(gates >= 1 && (rows == 0 || (gates <= rows && rows % gates == 0)), name + ": every gate is shared by as many rows");
  return 0;
}
bool fits(const Rows& t, int64_t C, int eb) {
  return !t.ptr || (t.ld >= C && t.ld % (16 / eb) == 0 && t.ld <= (1ll << 31) && (reinterpret_cast<uintptr_t>(t.ptr) & 15) == 0);
}
bool aligned(std::initializer_list<const void*> all) {
  uintptr_t bits = 0;
  for (const void* p : all) bits |= reinterpret_cast<uintptr_t>(p);
  return (bits & 15) == 0;
}

// (Rows of up to 256 elements, however many, and backward what only kAnything does are not streamed; what it would give there beyond the cache is not
// measured.  131072 x 256 in fp32 103 us forward, 5.2 TB/s, and 158 backward, 5.1; a quarter of the rows, which the cache holds, 21 and 39.)
template <typename T, int L, bool WIDE, bool STREAM>
int launch_fwd(Context* ctx, const NormArgs& a, int br, dim3 grid, dim3 block, const char* name, double bytes) {
  if (br == kNoBranch) return launch(ctx, residual_norm_fwd_kernel<T, L, WIDE, kNoBranch, STREAM>, grid, block, a, name, bytes, 1);
  if (br == kBranch) return launch(ctx, residual_norm_fwd_kernel<T, L, WIDE, kBranch, STREAM>, grid, block, a, name, bytes, 1);
  return launch(ctx, residual_norm_fwd_kernel<T, L, WIDE, kPostNorm, STREAM>, grid, block, a, name, bytes, 1);
}
template <typename T>
int launch_fwd_of(Context* ctx, const NormArgs& a, const Shape& s, int br, dim3 grid, const char* const* names, double bytes) {
  const dim3 block(s.threads);
  const bool stream = bytes > kStreamBytes;
  if (s.lanes == 16) return launch_fwd<T, 16, false, false>(ctx, a, br, grid, block, names[0], bytes);
  if (s.lanes == 32) return launch_fwd<T, 32, false, false>(ctx, a, br, grid, block, names[1], bytes);
  if (s.waves > 8)
    return stream ? launch_fwd<T, 64, true, true>(ctx, a, br, grid, block, names[3], bytes) : launch_fwd<T, 64, true, false>(ctx, a, br, grid, block, names[3], bytes);
  return stream ? launch_fwd<T, 64, false, true>(ctx, a, br, grid, block, names[2], bytes) : launch_fwd<T, 64, false, false>(ctx, a, br, grid, block, names[2], bytes);
}
template <typename T, int L, bool WIDE, int BR, bool STREAM>
int launch_bwd(Context* ctx, const NormArgs& a, int mode, dim3 grid, dim3 block, const char* name, double bytes) {
  if (mode == kFullRms) return launch(ctx, residual_norm_bwd_kernel<T, L, WIDE, BR, kFullRms, STREAM>, grid, block, a, name, bytes, 1);
  if (mode == kFullLayer) return launch(ctx, residual_norm_bwd_kernel<T, L, WIDE, BR, kFullLayer, STREAM>, grid, block, a, name, bytes, 1);
  return launch(ctx, residual_norm_bwd_kernel<T, L, WIDE, BR, kAnything, false>, grid, block, a, name, bytes, 1);
}
template <typename T, int BR>
int launch_bwd_of(Context* ctx, const NormArgs& a, const Shape& s, int mode, dim3 grid, const char* const* names, double bytes) {
  const dim3 block(s.threads);
  const bool stream = bytes > kStreamBytes;
  if (s.lanes == 16) return launch_bwd<T, 16, false, BR, false>(ctx, a, mode, grid, block, names[0], bytes);
  if (s.lanes == 32) return launch_bwd<T, 32, false, BR, false>(ctx, a, mode, grid, block, names[1], bytes);
  if (s.waves > 8)
    return stream ? launch_bwd<T, 64, true, BR, true>(ctx, a, mode, grid, block, names[3], bytes)
                  : launch_bwd<T, 64, true, BR, false>(ctx, a, mode, grid, block, names[3], bytes);
  return stream ? launch_bwd<T, 64, false, BR, true>(ctx, a, mode, grid, block, names[2], bytes)
                : launch_bwd<T, 64, false, BR, false>(ctx, a, mode, grid, block, names[2], bytes);
}
template <typename T>
int launch_bwd_branch(Context* ctx, const NormArgs& a, const Shape& s, int br, int mode, dim3 grid, const char* const* names, double bytes) {
  if (br == kNoBranch) return launch_bwd_of<T, kNoBranch>(ctx, a, s, mode, grid, names, bytes);
  if (br == kBranch) return launch_bwd_of<T, kBranch>(ctx, a, s, mode, grid, names, bytes);
  return launch_bwd_of<T, kPostNorm>(ctx, a, s, mode, grid, names, bytes);
}
const char* const kFwdNames[2][4] = {
    {"residual_norm_fwd_kernel<f32,16>", "residual_norm_fwd_kernel<f32,32>", "residual_norm_fwd_kernel<f32>", "residual_norm_fwd_kernel<f32,wide>"},
    {"residual_norm_fwd_kernel<bf16,16>", "residual_norm_fwd_kernel<bf16,32>", "residual_norm_fwd_kernel<bf16>", "residual_norm_fwd_kernel<bf16,wide>"}};
const char* const kBwdNames[2][4] = {
    {"residual_norm_bwd_kernel<f32,16>", "residual_norm_bwd_kernel<f32,32>", "residual_norm_bwd_kernel<f32>", "residual_norm_bwd_kernel<f32,wide>"},
    {"residual_norm_bwd_kernel<bf16,16>", "residual_norm_bwd_kernel<bf16,32>", "residual_norm_bwd_kernel<bf16>", "residual_norm_bwd_kernel<bf16,wide>"}};

}  // namespace

int residual_norm_fwd(Context* ctx, int dtype, const ResidualNorm& n, const Rows& x, const Rows& branch, const Rows& total, const Rows& y, float* stats,
                      void* packed, void* codes, int format, int64_t rows, int64_t C) {
  if (int rc = check_shape("residual_norm_fwd", dtype, rows, C, n.gates)) return rc;
  if (rows == 0) return 0;
  const int eb = dtype == kBF16 ? 2 : 4;
  TCH_CHECK_ARG(x.ptr && stats, "residual_norm_fwd: null tensor");
  TCH_CHECK_ARG((branch.ptr != nullptr) == (total.ptr != nullptr), "residual_norm_fwd: a branch and the sum come together");
  TCH_CHECK_ARG((n.weight != nullptr) == (y.ptr != nullptr), "residual_norm_fwd: a norm's weight and its output come together");
  TCH_CHECK_ARG(branch.ptr || n.weight, "residual_norm_fwd: nothing to do");
  TCH_CHECK_ARG(branch.ptr || (!n.post_weight && !n.gate && n.scale == 1.f), "residual_norm_fwd: a post norm, a gate and a scale go with a branch");
  TCH_CHECK_ARG((n.weight || !n.bias) && (n.post_weight || !n.post_bias), "residual_norm_fwd: a bias goes with a weight");
  TCH_CHECK_ARG((packed != nullptr) == (codes != nullptr) && (!packed || (y.ptr && format >= 0 && format < kPackFormats)),
                "residual_norm_fwd: what is kept of y in 8 bits comes with its scales, and with y");
  TCH_CHECK_ARG(n.gate || n.gates == 1, "residual_norm_fwd: gates without their values");
  TCH_CHECK_ARG(n.eps >= 0.f, "residual_norm_fwd: eps must not be negative");
  TCH_CHECK_ARG(fits(x, C, eb) && fits(branch, C, eb) && fits(total, C, eb) && fits(y, C, eb), "residual_norm_fwd: rows must start on 16-byte boundaries and not overlap");
  TCH_CHECK_ARG(aligned({n.weight, n.bias, n.post_weight, n.post_bias, n.gate, stats, packed}),
                "residual_norm_fwd: vectors, statistics and kept activations must start on a 16-byte boundary");
  const int64_t gate_bytes = n.gates * C * (n.gate_f32 ? 4 : eb), groups32 = (C + kPackGroup - 1) / kPackGroup;
  const Span in[7] = {{x.ptr, x.ld * eb, C * eb, rows}, {branch.ptr, branch.ld * eb, C * eb, rows}, {n.weight, C * 4, C * 4, 1}, {n.bias, C * 4, C * 4, 1},
                      {n.post_weight, C * 4, C * 4, 1}, {n.post_bias, C * 4, C * 4, 1}, {n.gate, gate_bytes, gate_bytes, 1}};
  const Span out[5] = {{total.ptr, total.ld * eb, C * eb, rows}, {y.ptr, y.ld * eb, C * eb, rows}, {stats, 16, 16, rows}, {packed, C, C, rows},
                       {codes, groups32, groups32, rows}};
  for (int o = 0; o < 5; ++o) {
    bool ok = true;
    for (int i = 0; i < 7; ++i) ok = ok && apart(out[o], in[i], o < 2 && i < 2);
    for (int i = 0; i < o; ++i) ok = ok && apart(out[o], out[i]);
    TCH_CHECK_ARG(ok, "residual_norm_fwd: an output overlaps another tensor (the sum and y may be x or the branch)");
  }
  const Shape s = shape_of(rows, static_cast<int>(C));
  NormArgs a{};
  a.x = {x.ptr, x.ld}, a.branch = {branch.ptr, branch.ld}, a.total = {total.ptr, total.ld}, a.y = {y.ptr, y.ld};
  a.stats = reinterpret_cast<float4*>(stats);
  a.weight = n.weight, a.bias = n.bias, a.post_weight = n.post_weight, a.post_bias = n.post_bias;
  a.gate = n.gate, a.gate_f32 = n.gate_f32 || dtype == kF32, a.gate_rows = rows / n.gates;
  a.gate_div = FastDiv(static_cast<uint32_t>(a.gate_rows));
  a.packed = static_cast<unsigned char*>(packed), a.codes = static_cast<unsigned char*>(codes), a.format = format;
  a.rows = rows, a.C = static_cast<int>(C);
  a.waves = s.waves, a.groups = s.groups;
  a.layer = n.layer, a.scale = n.scale, a.eps = n.eps;
  const int64_t blocks = (rows + s.groups - 1) / s.groups;
  // (sixteen wavefronts a compute unit at most and equally many workgroups on each: 16384 x 7168 in bf16 172 us, 259 with 292 workgroups)
  const dim3 grid(static_cast<unsigned>(std::min<int64_t>(blocks, 256 * (1024 / s.threads))));
  const int br = !branch.ptr ? kNoBranch : n.post_weight ? kPostNorm : kBranch;
  const double bytes = static_cast<double>(rows) * C * (eb * (1.0 + (branch.ptr ? 2 : 0) + (y.ptr ? 1 : 0)) + (packed ? 33.0 / 32 : 0));
  return dtype == kBF16 ? launch_fwd_of<bf16>(ctx, a, s, br, grid, kFwdNames[1], bytes) : launch_fwd_of<float>(ctx, a, s, br, grid, kFwdNames[0], bytes);
}

int64_t residual_norm_bwd_workspace_bytes(int64_t rows, int64_t C, int64_t gates) {
  if (rows <= 0 || rows > INT_MAX || C <= 0 || C > kMaxWidth || gates < 1 || gates > rows || rows % gates != 0) return 0;
  const Cut c = cut_rows(rows, static_cast<int>(C), gates);
  return c.blocks * C * 4 * 4;
}

int residual_norm_bwd(Context* ctx, int dtype, const ResidualNorm& n, const Rows& dy, const Rows& dtotal, const Rows& total, const Rows& branch, const Rows& dx,
                      const Rows& dbranch, const float* stats, const ResidualNormGrads& g, int accumulate, int64_t rows, int64_t C, void* workspace,
                      int64_t workspace_bytes) {
  if (int rc = check_shape("residual_norm_bwd", dtype, rows, C, n.gates)) return rc;
  const int eb = dtype == kBF16 ? 2 : 4;
  const int64_t grads[5] = {C, C, C, C, C * n.gates};
  float* const grad[5] = {g.weight, g.bias, g.post_weight, g.post_bias, g.gate};
  TCH_CHECK_ARG(aligned({n.weight, n.post_weight, n.post_bias, n.gate, stats, g.weight, g.bias, g.post_weight, g.post_bias, g.gate, workspace}),
                "residual_norm_bwd: vectors, statistics and the workspace must start on a 16-byte boundary");
  if (rows == 0) {
    if (!accumulate)
      for (int i = 0; i < 5; ++i)
        if (grad[i])
          if (int rc = fill_zero(ctx, grad[i], grads[i] * 4)) return rc;
    return 0;
  }
  TCH_CHECK_ARG(stats && (n.weight != nullptr) == (dy.ptr != nullptr) && (!n.weight || total.ptr), "residual_norm_bwd: a norm's weight, the gradient of its output and the sum come together");
  TCH_CHECK_ARG(n.weight || dtotal.ptr, "residual_norm_bwd: no gradient");
  TCH_CHECK_ARG((branch.ptr != nullptr) == (dbranch.ptr != nullptr), "residual_norm_bwd: a branch and its gradient come together");
  TCH_CHECK_ARG(branch.ptr || dx.ptr, "residual_norm_bwd: nothing to do");
  TCH_CHECK_ARG(branch.ptr || (!n.post_weight && !n.gate && n.scale == 1.f), "residual_norm_bwd: a post norm, a gate and a scale go with a branch");
  TCH_CHECK_ARG(n.gate || n.gates == 1, "residual_norm_bwd: gates without their values");
  TCH_CHECK_ARG((n.weight || (!g.weight && !g.bias)) && (n.post_weight || (!g.post_weight && !g.post_bias && !n.post_bias)) && (n.gate || !g.gate),
                "residual_norm_bwd: a gradient of what is not there");
  TCH_CHECK_ARG(fits(dy, C, eb) && fits(dtotal, C, eb) && fits(total, C, eb) && fits(branch, C, eb) && fits(dx, C, eb) && fits(dbranch, C, eb),
                "residual_norm_bwd: rows must start on 16-byte boundaries and not overlap");
  const Cut cut = cut_rows(rows, static_cast<int>(C), n.gates);
  const Shape& s = cut.shape;
  const bool many = !cut.split;      // (and the gates' gradients are written where the rows are)
  NormArgs a{};
  const bool gates_later = g.gate && !many;
  const bool wanted[4] = {g.weight != nullptr, g.bias != nullptr, g.post_weight || gates_later, g.post_bias || (gates_later && n.post_bias)};
  for (int i = 0; i < 4; ++i) a.plane_of[i] = wanted[i] ? a.planes++ : -1;
  const int64_t need = cut.blocks * C * 4 * a.planes;
  TCH_CHECK_ARG(need <= (workspace ? workspace_bytes : 0), "residual_norm_bwd: workspace too small");
  const int64_t gate_bytes = n.gates * C * (n.gate_f32 ? 4 : eb);
  auto rows_of = [&](const Rows& t) { return Span{t.ptr, t.ld * eb, C * eb, rows}; };
  const Span in[9] = {rows_of(dy), rows_of(dtotal), rows_of(total), rows_of(branch), {n.weight, C * 4, C * 4, 1}, {n.post_weight, C * 4, C * 4, 1},
                      {n.post_bias, C * 4, C * 4, 1}, {n.gate, gate_bytes, gate_bytes, 1}, {stats, 16, 16, rows}};
  const Span out[8] = {rows_of(dx), rows_of(dbranch), {g.weight, C * 4, C * 4, 1}, {g.bias, C * 4, C * 4, 1}, {g.post_weight, C * 4, C * 4, 1},
                       {g.post_bias, C * 4, C * 4, 1}, {g.gate, C * 4, C * 4, n.gates}, {workspace, need, need, need ? 1 : 0}};
  for (int o = 0; o < 8; ++o) {
    bool ok = true;
    for (int i = 0; i < 9; ++i) ok = ok && apart(out[o], in[i], o < 2 && i < 4);
    for (int i = 0; i < o; ++i) ok = ok && apart(out[o], out[i]);
    TCH_CHECK_ARG(ok, "residual_norm_bwd: an output or the workspace overlaps another tensor (dx and dbranch may be dy, dtotal, the sum or the branch)");
  }
  a.dy = {dy.ptr, dy.ld}, a.dtotal = {dtotal.ptr, dtotal.ld}, a.total = {total.ptr, total.ld}, a.branch = {branch.ptr, branch.ld};
  a.dx = {dx.ptr, dx.ld}, a.dbranch = {dbranch.ptr, dbranch.ld};
  a.stats = reinterpret_cast<float4*>(const_cast<float*>(stats));
  a.weight = n.weight, a.post_weight = n.post_weight, a.post_bias = n.post_bias;
  a.gate = n.gate, a.gate_f32 = n.gate_f32 || dtype == kF32, a.gate_rows = rows / n.gates;
  a.gates = static_cast<int>(n.gates);
  a.rows = rows, a.C = static_cast<int>(C);
  a.split_gates = cut.split, a.pieces = static_cast<int>(cut.pieces), a.gates_each = cut.gates_each;
  a.waves = s.waves, a.groups = s.groups;
  a.layer = n.layer, a.scale = n.scale, a.eps = n.eps;
  a.sums = static_cast<float*>(workspace);
  a.dgate = g.gate;
  a.add_gates = accumulate;
  const int br = !branch.ptr ? kNoBranch : n.post_weight ? kPostNorm : kBranch;
  const double bytes = static_cast<double>(rows) * C * eb * ((dy.ptr ? 2.0 : 0) + (dtotal.ptr ? 1 : 0) + (dx.ptr ? 1 : 0) + (branch.ptr ? 2 : 0)) + need;
  const dim3 grid(static_cast<unsigned>(cut.blocks));
  const bool full = n.weight && !many;
  const int mode = full && n.layer ? kFullLayer : full && a.plane_of[1] < 0 && a.plane_of[3] < 0 ? kFullRms : kAnything;
  const int rc = dtype == kBF16 ? launch_bwd_branch<bf16>(ctx, a, s, br, mode, grid, kBwdNames[1], bytes)
                                : launch_bwd_branch<float>(ctx, a, s, br, mode, grid, kBwdNames[0], bytes);
  if (rc || a.planes == 0) return rc;
  NormSumArgs f{};
  f.sums = a.sums;
  f.post_weight = n.post_weight, f.post_bias = n.post_bias;
  f.gate = many ? nullptr : n.gate, f.gate_f32 = a.gate_f32;
  f.dweight = g.weight, f.dbias = g.bias, f.dpost_weight = g.post_weight, f.dpost_bias = g.post_bias, f.dgate = g.gate;
  f.C = static_cast<int>(C), f.blocks = static_cast<int>(cut.blocks), f.planes = a.planes;
  for (int i = 0; i < 4; ++i) f.plane_of[i] = a.plane_of[i];
  f.pieces = static_cast<int>(cut.pieces), f.add = accumulate;
  f.div = FastDiv(static_cast<uint32_t>(cut.pieces));
  // (gates whose rows are several workgroups' are half as many as workgroups at most)
  const dim3 blocks(static_cast<unsigned>((C + 31) / 32), static_cast<unsigned>(gates_later ? 2 + n.gates : 2));
  return cut.blocks > 256 ? launch(ctx, residual_norm_sum_kernel<16>, blocks, dim3(512), f, "residual_norm_sum_kernel<16>", static_cast<double>(need), 1)
                          : launch(ctx, residual_norm_sum_kernel<8>, blocks, dim3(256), f, "residual_norm_sum_kernel<8>", static_cast<double>(need), 1);
}

}  // namespace tch

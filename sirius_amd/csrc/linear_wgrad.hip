// Weight and bias gradients of linear layers in bf16: dw (+)= dy^T x over the rows, dbias (+)= column sums of dy, in fp32.
//
// One of the operands may come with a low part (what rounding to bf16 took off it: linear_epilogue.h, rounded_off); the gradient is
// then that of the unrounded operand, in twice the multiplies.  Both parts add to the same accumulators, and share the other
// operand's tile in LDS and in registers: a step moves 1.5 times the bytes for twice the multiplies.
//
// Both operands are contiguous along the output's axes and strided along the reduction, the opposite of what an MFMA operand wants:
// tiles of 32 rows are kept as they come, [row][column], and read transposed (ds_read_b64_tr_b16: sixteen lanes fetch a patch of 4
// rows x 16 columns, each keeps 4 rows of one column).  The 16-byte slot of a column is XOR-ed by four times the row, so that
// the 64-byte patches of the eight rows of a read lie in different banks.  Element 4t + i of lane half h is row 8t + 4h + i of a
// sixteen-row slice, for both operands alike.
#include "direct_load.h"
#include "fp32_split.h"
#include "linear_epilogue.h"

#include <algorithm>
#include <numeric>

#include "context.h"
#include "ops.h"

namespace tch {
namespace {

// As many workgroups as the chip holds, and all of them busy to the end however many tiles there are: each takes `rounds` whole
// tiles, and an equal run of the steps of the tiles that are left, tile by tile.  A tile that lies within one run is stored; of a
// tile that is cut, every workgroup leaves its part in the workspace (the first of its run in slot 2 g, the second in 2 g + 1), and a
// second launch adds them up in the order of the runs.
//
// The operands come through L2 32 rows at a time, and what no neighbour on the XCD wants at about the same time is read again from
// further away (6 TB/s in all).  So whole tiles lie in blocks (locate_tile) that the workgroups of an XCD walk down together, and the runs are dealt
// to the workgroups in the order of the row that they begin with: run r begins (left r mod runs) / runs of the way down a tile, so that
// with g = gcd(left, runs) and q = runs / g the runs r = v inverse(left / g) mod q + c q, c < g, are those that begin v / q down.
struct LinearWgradArgs {
  const void* a;        // dy [M][N]
  const void* a_low;
  const void* b;        // x [M][K]
  const void* b_low;
  float* out;           // dw [N][K]
  float* bias;          // dbias [N]; may be null
  float* slots;         // partial tiles [2 runs][tile]
  float* bias_slots;    // and their column sums [2 runs][rows of a tile]
  int64_t M, units;     // units: steps of the tiles that are left
  int N, K;
  int tiles_n, tiles_k, steps;
  int groups, rounds, runs;   // tiles behind groups * rounds are left, for the first `runs` workgroups
  int accumulate;       // out and bias are added to
  int same_start, period, inverse;   // g, q, inverse(left / g) mod q
};
__host__ __device__ inline int64_t run_start(int64_t units, int runs, int run) { return units * run / runs; }
// four tiles down, then one to the right
__device__ inline void locate_tile(const LinearWgradArgs& p, int tile, int& tile_n, int& tile_k) {
  const int band = tile / (4 * p.tiles_k), rest = tile - band * (4 * p.tiles_k), rows = min(4, p.tiles_n - 4 * band);
  tile_k = rest / rows;
  tile_n = 4 * band + rest - tile_k * rows;
}

enum Pair : int { kNoLow = 0, kLowA = 1, kLowB = 2 };
constexpr int kRows = 32;   // of a reduction step

// WM x WN wavefronts of TM x TN MFMA tiles (32 x 32).  NBUF tiles in LDS, one barrier per step; the sixteen-row slice that is multiplied
// next is read while this one is multiplied, and the direct loads of the step NBUF - 1 ahead go out between the multiplies.
// 2048 x 11264 over 8192 rows with a low part: 548-576 us, 1.31-1.38 PFLOP/s, which is what the chip's power allows; with runs dealt out as they
// come, 4 GB through L2 in 661 us.  4096 x 1024: 110-116 us and 17 to add up four parts a tile.
template <int PAIR, int WM, int WN, int TM, int TN, int NBUF, int PER_CU>
__global__ __launch_bounds__(WM* WN * 64, PER_CU* WM* WN / 4) void linear_wgrad_kernel(LinearWgradArgs p) {
  constexpr int BM = WM * TM * 32, BN = WN * TN * 32, NW = WM * WN;
  constexpr int PA = PAIR == kLowA ? 2 : 1, PB = PAIR == kLowB ? 2 : 1;
  constexpr int RA = BM * 2, RB = BN * 2;                       // bytes of an LDS row
  constexpr int A_PLANE = kRows * RA, B_PLANE = kRows * RB, B_AT = PA * A_PLANE, BUF_BYTES = B_AT + PB * B_PLANE;
  constexpr int A_LD = BM / 16 / NW, B_LD = BN / 16 / NW;       // direct loads (1 KB) per wavefront, plane and step
  constexpr int LOADS = PA * A_LD + PB * B_LD, AHEAD = (NBUF - 2) * LOADS;
  static_assert(BM % (16 * NW) == 0 && BN % (16 * NW) == 0 && AHEAD < 64 && NBUF >= 3, "tile/loader mismatch");
  static_assert(BUF_BYTES <= 65536, "operand reads reach a buffer's planes with their immediate offset");
  __shared__ __attribute__((aligned(1024))) unsigned char lds[NBUF * BUF_BYTES];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int group = static_cast<int>(xcd_remap(blockIdx.x, gridDim.x));
  const int run = __builtin_amdgcn_readfirstlane(group < p.runs ? group / p.same_start * p.inverse % p.period + group % p.same_start * p.period : 0);
  int64_t unit = group < p.runs ? run_start(p.units, p.runs, run) : 0;
  const int64_t run_end = group < p.runs ? run_start(p.units, p.runs, run + 1) : 0;

  // ---- the walk of the loads: the resources move down the rows, the lanes' offsets stay; rows behind the last one are outside ----
  auto lane_offset = [&](int load, int row_bytes, int ld, int col0) {   // of 1 KB number `load` of a plane
    const int per_row = row_bytes / 16, row = load * (1024 / row_bytes) + lane / per_row;
    const int chunk = (lane % per_row) ^ ((row & 3) << 2);
    return (row * ld + col0 + chunk * 8) * 2;
  };
  int a_off[A_LD], b_off[B_LD];
  const int64_t a_step = static_cast<int64_t>(kRows) * p.N * 2, b_step = static_cast<int64_t>(kRows) * p.K * 2;
  int64_t a_at = 0, b_at = 0;
  int left = 0;
  __amdgpu_buffer_rsrc_t rsrc_a[PA], rsrc_b[PB];
  auto resources = [&]() LINEAR_INLINE {
    const int here = __builtin_amdgcn_readfirstlane(left < 0 ? 0 : left < kRows ? left : kRows);
    const uint32_t a_bytes = static_cast<uint32_t>(here) * static_cast<uint32_t>(p.N) * 2, b_bytes = static_cast<uint32_t>(here) * static_cast<uint32_t>(p.K) * 2;
    rsrc_a[0] = make_rsrc(static_cast<const unsigned char*>(p.a) + a_at, a_bytes);
    if constexpr (PA == 2) rsrc_a[1] = make_rsrc(static_cast<const unsigned char*>(p.a_low) + a_at, a_bytes);
    rsrc_b[0] = make_rsrc(static_cast<const unsigned char*>(p.b) + b_at, b_bytes);
    if constexpr (PB == 2) rsrc_b[1] = make_rsrc(static_cast<const unsigned char*>(p.b_low) + b_at, b_bytes);
  };
  auto next_step = [&]() LINEAR_INLINE {
    left -= kRows;
    if (left > 0) a_at += a_step, b_at += b_step;   // (behind the last row the resources are empty)
    resources();
  };
  auto issue_load = [&](uint32_t buf, int j) LINEAR_INLINE {
    if (j < PA * A_LD) {
      const int plane = j / A_LD, i = j % A_LD;
      load_to_lds(rsrc_a[plane], lds + buf + plane * A_PLANE + (wave * A_LD + i) * 1024, a_off[i], 0);
    } else {
      const int plane = (j - PA * A_LD) / B_LD, i = (j - PA * A_LD) % B_LD;
      load_to_lds(rsrc_b[plane], lds + buf + B_AT + plane * B_PLANE + (wave * B_LD + i) * 1024, b_off[i], 0);
    }
  };

  // ---- operand reads ----
  const int half = lane >> 5, patch_row = (lane & 15) >> 2, patch_slot = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  const uint32_t lds_base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds));
  uint32_t rd[TM + TN];
#pragma unroll
  for (int i = 0; i < TM + TN; ++i) {
    const bool is_a = i < TM;
    const int ct = is_a ? wm * TM + i : wn * TN + i - TM;
    rd[i] = lds_base + (is_a ? 0 : B_AT) + (4 * half + patch_row) * (is_a ? RA : RB) + (4 * (ct ^ patch_row) + patch_slot) * 16 + (lane & 1) * 8;
  }
  constexpr int FRAGS = PA * TM + PB * TN, READS = 2 * FRAGS;
  uint2_t frag[2][FRAGS][2];   // [set][operand tile: A's planes, B's planes][rows 0-7, 8-15 of the slice]
  auto read_one = [&](auto kk_c, uint32_t buf, auto set_c, auto i_c) LINEAR_INLINE {
    constexpr int kk = decltype(kk_c)::value, set = decltype(set_c)::value, i = decltype(i_c)::value, f = i >> 1, t = i & 1;
    constexpr bool is_a = f < PA * TM;
    constexpr int plane = is_a ? f / TM : (f - PA * TM) / TN, which = is_a ? f % TM : TM + (f - PA * TM) % TN;
    constexpr int ROW = kk * 16 + 8 * t, OFF = is_a ? plane * A_PLANE + ROW * RA : plane * B_PLANE + ROW * RB;
    const uint32_t from = rd[which] + buf;
    uint2_t v;
    asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(v) : "v"(from), "n"(OFF));
    frag[set][f][t] = v;
  };
  auto hold_set = [&](int set) LINEAR_INLINE {
#pragma unroll
    for (int f = 0; f < FRAGS; ++f)
#pragma unroll
      for (int t = 0; t < 2; ++t) asm volatile("" : "+v"(frag[set][f][t]));
  };
  auto operand = [&](int set, int f) LINEAR_INLINE {
    Chunk c;
    c.w[0] = frag[set][f][0][0];
    c.w[1] = frag[set][f][0][1];
    c.w[2] = frag[set][f][1][0];
    c.w[3] = frag[set][f][1][1];
    return c.h;
  };

  f32x16_t acc[TM][TN];
  // the bias gradient: the wavefronts of the first column of tiles add up the dy operands that they multiply anyway
  bool sums = false;
  float col_sum[TM];

  // multiplies the slice in `set`; meanwhile slice kk of the step in `buf` is read into the other set and half q of the loads goes
  // to `ld_buf`
  auto slice = [&](auto set_c, uint32_t buf, auto kk_c, auto q_c, uint32_t ld_buf) LINEAR_INLINE {
    constexpr int set = decltype(set_c)::value, q = decltype(q_c)::value;
    constexpr int PARTS = PA > PB ? PA : PB, MF = TM * TN * PARTS, FIRST = q * LOADS / 2, AUX = READS + (q + 1) * LOADS / 2 - FIRST;
    constexpr int PER = (AUX + MF - 1) / MF;
    unrolled<MF>([&](auto m_c) LINEAR_INLINE {
      constexpr int m = decltype(m_c)::value, part = m / (TM * TN), tm = m % (TM * TN) / TN, tn = m % TN;
      constexpr int fa = (PA == 2 ? part * TM : 0) + tm, fb = PA * TM + (PB == 2 ? part * TN : 0) + tn;
      acc[tm][tn] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(operand(set, fa), operand(set, fb), acc[tm][tn], 0, 0, 0);
      unrolled<PER>([&](auto a_c) LINEAR_INLINE {
        constexpr int a = m * PER + decltype(a_c)::value;
        if constexpr (a < READS)
          read_one(kk_c, buf, std::integral_constant<int, set ^ 1>{}, std::integral_constant<int, a>{});
        else if constexpr (a < AUX)
          issue_load(ld_buf, FIRST + a - READS);
      });
      __builtin_amdgcn_sched_barrier(0);
    });
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    hold_set(set ^ 1);
    if (sums) {
#pragma unroll
      for (int f = 0; f < PA * TM; ++f)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t w = frag[set][f][t][i];
            col_sum[f % TM] += __uint_as_float(w << 16) + __uint_as_float(w & 0xffff0000u);
          }
    }
  };

  std::integral_constant<int, 0> zero;
  std::integral_constant<int, 1> one;
  // behind the last barrier of a part nobody reads what counts, and every wavefront waits for its own loads: the next part's may
  // go to the same buffers
  int slot = 2 * run;
  for (int round = 0; round < p.rounds || unit < run_end; ++round) {
    int tile = round * p.groups + group, from = 0, to = p.steps;
    if (round >= p.rounds) {
      // (quotients and 64-bit minima come out of the vector unit: back in scalar registers, or every load of the loop becomes a
      // loop over its resources)
      const int left_tile = __builtin_amdgcn_readfirstlane(static_cast<int>(unit / p.steps));
      tile = p.rounds * p.groups + left_tile;
      from = __builtin_amdgcn_readfirstlane(static_cast<int>(unit - static_cast<int64_t>(left_tile) * p.steps));
      to = __builtin_amdgcn_readfirstlane(static_cast<int>(min(static_cast<int64_t>(p.steps), from + (run_end - unit))));
      unit += to - from;
    }
    int tile_n, tile_k;
    locate_tile(p, tile, tile_n, tile_k);
    tile_n = __builtin_amdgcn_readfirstlane(tile_n), tile_k = __builtin_amdgcn_readfirstlane(tile_k);
    const int n0 = tile_n * BM, k0 = tile_k * BN;
    const int64_t row0 = static_cast<int64_t>(from) * kRows;
#pragma unroll
    for (int j = 0; j < A_LD; ++j) a_off[j] = lane_offset(wave * A_LD + j, RA, p.N, n0);
#pragma unroll
    for (int j = 0; j < B_LD; ++j) b_off[j] = lane_offset(wave * B_LD + j, RB, p.K, k0);
    a_at = row0 * p.N * 2;
    b_at = row0 * p.K * 2;
    left = __builtin_amdgcn_readfirstlane(static_cast<int>(min(static_cast<int64_t>(to - from) * kRows, p.M - row0)));
    sums = p.bias && tile_k == 0 && wn == 0;
    clear(acc);
#pragma unroll
    for (int i = 0; i < TM; ++i) col_sum[i] = 0.f;

    resources();
#pragma unroll
    for (int s = 0; s < NBUF - 1; ++s) {
#pragma unroll
      for (int j = 0; j < LOADS; ++j) issue_load(s * BUF_BYTES, j);
      next_step();
    }
#pragma unroll
    for (int j = 0; j < LOADS / 2; ++j) issue_load((NBUF - 1) * BUF_BYTES, j);
    wait_and_meet<AHEAD + LOADS / 2>();
    unrolled<READS>([&](auto i_c) LINEAR_INLINE { read_one(zero, 0u, zero, i_c); });
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    hold_set(0);
    uint32_t buf = 0, before = (NBUF - 1) * BUF_BYTES;
    for (int s = from; s < to; ++s) {
      slice(zero, buf, one, one, before);
      next_step();
      wait_and_meet<AHEAD>();
      before = buf;
      buf = buf == (NBUF - 1) * BUF_BYTES ? 0 : buf + BUF_BYTES;
      slice(one, buf, zero, zero, before);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the zeros behind the last step have landed

    // ---- a lane's accumulators are one column of dw (x) and rows 8 (e / 4) + 4 half + e % 4: whole lines of 128 bytes a store ----
    const bool whole = to - from == p.steps;
    const int ld = whole ? p.K : BN;
    const bool add = whole && p.accumulate;
    float* out = whole ? p.out + static_cast<int64_t>(n0) * p.K + k0 : p.slots + static_cast<int64_t>(slot) * (BM * BN);
    const int rows = whole ? min(BM, p.N - n0) : BM, cols = whole ? min(BN, p.K - k0) : BN;
    const __amdgpu_buffer_rsrc_t rsrc_out = make_rsrc(out, static_cast<uint32_t>((rows - 1) * ld + cols) * 4u);
#pragma unroll
    for (int tm = 0; tm < TM; ++tm)
#pragma unroll
      for (int tn = 0; tn < TN; ++tn) {
        const int col = (wn * TN + tn) * 32 + (lane & 31), row = (wm * TM + tm) * 32 + 4 * half;
        const int at = col < cols ? (row * ld + col) * 4 : static_cast<int>(kOutOfRange);
        auto off = [&](int e) { return at + (8 * (e >> 2) + (e & 3)) * ld * 4; };
        if (add) {
          float old[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) old[e] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rsrc_out, off(e), 0, 0));
#pragma unroll
          for (int e = 0; e < 16; ++e) acc[tm][tn][e] += old[e];
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(acc[tm][tn][e]), rsrc_out, off(e), 0, 0);
      }
    if (sums) {
#pragma unroll
      for (int tm = 0; tm < TM; ++tm) {
        const float s = col_sum[tm] + __shfl_xor(col_sum[tm], 32, 64);
        const int n = (wm * TM + tm) * 32 + (lane & 31);
        if (lane < 32 && n < rows) {
          float* b = whole ? p.bias + n0 + n : p.bias_slots + static_cast<int64_t>(slot) * BM + n;
          *b = add ? *b + s : s;
        }
      }
    }
    if (round >= p.rounds) ++slot;
  }
}

// The tiles that several workgroups had a part of: dw (+)= their sum in the workgroups' order.  A workgroup here has a band of
// kBand rows of a tile; the loads of kPartsAtOnce parts are on their way together (few tiles have many parts each: 272 x 176 over 4115
// rows 85, 33 us a part at a time in bands of 32 rows).
constexpr int kBand = 8, kPartsAtOnce = 8;
template <int SIDE>
__global__ __launch_bounds__(256) void linear_wgrad_sum_kernel(LinearWgradArgs p) {
  constexpr int BANDS = SIDE / kBand;
  const int left_tile = blockIdx.x / BANDS, band = blockIdx.x % BANDS;
  const int64_t first = static_cast<int64_t>(left_tile) * p.steps, behind = first + p.steps;
  // the runs that have the tile's first and its last step, and the slot of a run's part
  int g0 = static_cast<int>(first * p.runs / p.units);
  while (run_start(p.units, p.runs, g0 + 1) <= first) ++g0;
  if (run_start(p.units, p.runs, g0 + 1) >= behind) return;   // one workgroup had all of it
  int g1 = static_cast<int>((behind - 1) * p.runs / p.units);
  while (run_start(p.units, p.runs, g1 + 1) < behind) ++g1;
  // (the first of them may have begun in the tile before: its part of this one is its second)
  auto slot_of = [&](int g) { return static_cast<int64_t>(2 * g + (g > g0 || run_start(p.units, p.runs, g0) == first ? 0 : 1)); };
  int tile_n, tile_k;
  locate_tile(p, p.rounds * p.groups + left_tile, tile_n, tile_k);
  const int n0 = tile_n * SIDE + band * kBand, k0 = tile_k * SIDE;
  constexpr int QUADS = kBand * SIDE / 4 / 256;
  float4 sum[QUADS];
#pragma unroll
  for (int i = 0; i < QUADS; ++i) sum[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int g = g0; g <= g1; g += kPartsAtOnce) {
    float4 v[kPartsAtOnce][QUADS];
#pragma unroll
    for (int b = 0; b < kPartsAtOnce; ++b) {
      if (g + b > g1) continue;
      const float* from = p.slots + slot_of(g + b) * (SIDE * SIDE) + band * kBand * SIDE;
#pragma unroll
      for (int i = 0; i < QUADS; ++i) v[b][i] = load_streaming_f4(from + (i * 256 + threadIdx.x) * 4);
    }
#pragma unroll
    for (int b = 0; b < kPartsAtOnce; ++b) {
      if (g + b > g1) continue;
#pragma unroll
      for (int i = 0; i < QUADS; ++i)
        sum[i] = make_float4(sum[i].x + v[b][i].x, sum[i].y + v[b][i].y, sum[i].z + v[b][i].z, sum[i].w + v[b][i].w);
    }
  }
#pragma unroll
  for (int i = 0; i < QUADS; ++i) {
    const int q = i * 256 + threadIdx.x, row = q / (SIDE / 4), col = q % (SIDE / 4) * 4;
    if (n0 + row >= p.N || k0 + col >= p.K) continue;
    float* to = p.out + static_cast<int64_t>(n0 + row) * p.K + k0 + col;
    float4 s = sum[i];
    if (p.accumulate) {
      const float4 v = *reinterpret_cast<const float4*>(to);
      s = make_float4(s.x + v.x, s.y + v.y, s.z + v.z, s.w + v.w);
    }
    store_streaming_f4(to, s);
  }
  if (p.bias && tile_k == 0 && threadIdx.x < kBand && n0 + static_cast<int>(threadIdx.x) < p.N) {
    float s = 0.f;
#pragma unroll 4
    for (int g = g0; g <= g1; ++g) s += p.bias_slots[slot_of(g) * SIDE + band * kBand + threadIdx.x];
    float* to = p.bias + n0 + threadIdx.x;
    *to = p.accumulate ? *to + s : s;
  }
}

int tiles_over(int n, int tile) { return (n + tile - 1) / tile; }

// The tiling and the number of workgroups with the shortest estimate: the steps of a run, a start and an end, and the partial tiles'
// way through memory.  Steps in microseconds, with a low part: 256 x 256 1.43; 128 x 128 0.95 alone on a compute unit, 0.97 where
// two share it.
struct Choice {
  bool big, cut;       // cut: some tiles are shared, the workspace is needed
  int groups;
};
Choice choose(int64_t M, int N, int K, bool low, bool may_cut) {
  const int64_t steps = (M + kRows - 1) / kRows;
  Choice best{false, false, 1};
  float best_us = INFINITY;
  auto consider = [&](bool big, int64_t groups) {
    const int side = big ? 256 : 128;
    const int64_t tiles = static_cast<int64_t>(tiles_over(N, side)) * tiles_over(K, side), units = tiles * steps;
    if (groups < 1 || groups > units || groups > 0x3fffffff) return;
    const bool cut = tiles % groups != 0;
    if (cut && (!may_cut || groups > (big ? 256 : 512))) return;
    const int64_t slots = big ? 256 : 512, rounds = (groups + slots - 1) / slots, run = (units + groups - 1) / groups;
    const float step_us = (big ? 1.43f : groups > 256 ? 0.97f : 0.95f) * (low ? 1.f : 0.6f);
    float us = static_cast<float>(rounds) * (run * step_us + (big ? 8.f : 5.f) * ((run + steps - 1) / steps));
    if (cut) {
      const float parts = static_cast<float>(groups + tiles % groups);
      us += 5.f + 0.1f * parts / (tiles % groups) + (parts * side * side * 8.f + static_cast<float>(N) * K * 4.f) / 5e6f;
    }
    if (us < best_us) {
      best_us = us;
      best = Choice{big, cut, static_cast<int>(groups)};
    }
  };
  for (int big = 0; big < 2; ++big) {
    const int side = big ? 256 : 128;
    consider(big, static_cast<int64_t>(tiles_over(N, side)) * tiles_over(K, side));
    for (int64_t groups = big ? 256 : 512; groups >= 8; groups /= 2) {
      consider(big, groups);
      consider(big, groups / 4 * 3);
    }
  }
  return best;
}
int64_t slot_floats(const Choice& c) {
  const int64_t side = c.big ? 256 : 128;
  return c.cut ? 2 * static_cast<int64_t>(c.groups) * (side * side + side) : 0;
}

template <int PAIR>
int launch_wgrad_pair(Context* ctx, const LinearWgradArgs& a, bool big, unsigned grid, double flops, double bytes) {
  static const char* const names[2][3] = {
      {"linear_wgrad_kernel<128x128>", "linear_wgrad_kernel<128x128,dy_low>", "linear_wgrad_kernel<128x128,x_low>"},
      {"linear_wgrad_kernel<256x256>", "linear_wgrad_kernel<256x256,dy_low>", "linear_wgrad_kernel<256x256,x_low>"}};
  const char* name = names[big][PAIR];
  if (!big) return launch(ctx, linear_wgrad_kernel<PAIR, 2, 2, 2, 2, 3, 2>, dim3(grid), dim3(256), a, name, flops, 0, bytes);
  if constexpr (PAIR == kLowB)
    return launch(ctx, linear_wgrad_kernel<PAIR, 2, 4, 4, 2, 3, 1>, dim3(grid), dim3(512), a, name, flops, 0, bytes);
  else
    return launch(ctx, linear_wgrad_kernel<PAIR, 4, 2, 2, 4, 3, 1>, dim3(grid), dim3(512), a, name, flops, 0, bytes);
}

}  // namespace

int64_t linear_wgrad_workspace_bytes(int64_t M, int64_t K, int64_t N) {
  if (M <= 0 || K <= 0 || N <= 0 || K > INT32_MAX || N > INT32_MAX) return 0;
  int64_t most = 0;
  for (int low = 0; low < 2; ++low) most = std::max(most, slot_floats(choose(M, static_cast<int>(N), static_cast<int>(K), low != 0, true)) * 4);
  return most;
}

int linear_wgrad(Context* ctx, const void* x, const void* x_low, const void* dy, const void* dy_low, float* dw, float* dbias, int accumulate, int64_t M,
                 int64_t K, int64_t N, void* workspace, int64_t workspace_bytes) {
  TCH_CHECK_ARG(M >= 0 && K > 0 && N > 0 && M <= INT32_MAX - 1024, "linear_wgrad: bad shape");
  TCH_CHECK_ARG(K % 8 == 0 && N % 8 == 0, "linear_wgrad: the layer's sizes must be multiples of a 16-byte chunk");
  TCH_CHECK_ARG(K < (1 << 21) && N < (1 << 21) && N * K < (1ll << 40), "linear_wgrad: layer too large");
  TCH_CHECK_ARG(x && dy && dw, "linear_wgrad: null tensor");
  TCH_CHECK_ARG(!x_low || !dy_low, "linear_wgrad: one low part at a time");
  TCH_CHECK_ARG(((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(x_low) | reinterpret_cast<uintptr_t>(dy) |
                  reinterpret_cast<uintptr_t>(dy_low) | reinterpret_cast<uintptr_t>(dw) | reinterpret_cast<uintptr_t>(dbias) |
                  reinterpret_cast<uintptr_t>(workspace)) & 15) == 0,
                "linear_wgrad: tensors must start on 16-byte boundaries");
  if (M == 0) {
    if (accumulate) return 0;
    if (int rc = fill_zero(ctx, dw, N * K * 4)) return rc;
    return dbias ? fill_zero(ctx, dbias, N * 4) : 0;
  }
  const int n = static_cast<int>(N), k = static_cast<int>(K);
  const bool low = x_low || dy_low;
  Choice c = choose(M, n, k, low, workspace != nullptr);
  TCH_CHECK_ARG(slot_floats(c) * 4 <= (workspace ? workspace_bytes : 0), "linear_wgrad: workspace too small");
  const Span in[4] = {{x, K * 2, K * 2, M}, {x_low, K * 2, K * 2, M}, {dy, N * 2, N * 2, M}, {dy_low, N * 2, N * 2, M}};
  const Span out[3] = {{dw, K * 4, K * 4, N}, {dbias, N * 4, N * 4, 1}, {workspace, slot_floats(c) * 4, slot_floats(c) * 4, c.cut ? 1 : 0}};
  for (int o = 0; o < 3; ++o) {
    bool ok = true;
    for (const Span& i : in) ok = ok && apart(out[o], i);
    for (int i = 0; i < o; ++i) ok = ok && apart(out[o], out[i]);
    TCH_CHECK_ARG(ok, "linear_wgrad: an output or the workspace overlaps another tensor");
  }
  const int side = c.big ? 256 : 128;
  LinearWgradArgs a{};
  a.a = dy, a.a_low = dy_low;
  a.b = x, a.b_low = x_low;
  a.out = dw;
  a.bias = dbias;
  a.slots = static_cast<float*>(workspace);
  a.bias_slots = a.slots + 2 * static_cast<int64_t>(c.groups) * side * side;
  a.M = M, a.N = n, a.K = k;
  a.tiles_n = tiles_over(n, side);
  a.tiles_k = tiles_over(k, side);
  const int64_t tiles = static_cast<int64_t>(a.tiles_n) * a.tiles_k;
  TCH_CHECK_ARG(tiles <= 0x3fffffff, "linear_wgrad: grid out of range");
  a.steps = static_cast<int>((M + kRows - 1) / kRows);
  a.groups = c.groups;
  a.rounds = static_cast<int>(tiles / c.groups);
  const int left = static_cast<int>(tiles % c.groups);
  a.units = static_cast<int64_t>(left) * a.steps;
  a.runs = static_cast<int>(std::min<int64_t>(a.units, c.groups));   // (a run has a step at least)
  a.same_start = std::max(std::gcd(left, a.runs), 1);
  a.period = std::max(a.runs / a.same_start, 1);
  while (a.period > 1 && static_cast<int64_t>(left / a.same_start) * a.inverse % a.period != 1) ++a.inverse;
  a.accumulate = accumulate;
  const unsigned grid = static_cast<unsigned>(c.groups);
  const double flops = 2.0 * M * N * K * (low ? 2.0 : 1.0);
  const double bytes = 2.0 * M * (N * (dy_low ? 2 : 1) + K * (x_low ? 2 : 1)) + 4.0 * N * K;
  int rc = dy_low   ? launch_wgrad_pair<kLowA>(ctx, a, c.big, grid, flops, bytes)
           : x_low ? launch_wgrad_pair<kLowB>(ctx, a, c.big, grid, flops, bytes)
                   : launch_wgrad_pair<kNoLow>(ctx, a, c.big, grid, flops, bytes);
  if (rc || !c.cut) return rc;
  const dim3 blocks(static_cast<unsigned>(left * (side / kBand)));
  const double sum_bytes = 4.0 * (a.runs + 2.0 * left) * side * side;
  return c.big ? launch(ctx, linear_wgrad_sum_kernel<256>, blocks, dim3(256), a, "linear_wgrad_sum_kernel<256>", sum_bytes, 1)
               : launch(ctx, linear_wgrad_sum_kernel<128>, blocks, dim3(256), a, "linear_wgrad_sum_kernel<128>", sum_bytes, 1);
}

}  // namespace tch

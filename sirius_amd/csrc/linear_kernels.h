// Device code of the linear layers: a product of two row-major operands, out(m, n) = sum_k A(m, k) B(n, k), with everything a
// feed-forward layer does to it in the epilogue (linear_epilogue.h).  A has its own row stride, B (the weights) is dense.
// Compiled once per element type (linear_bf16.hip, linear_f32.hip).
//
// LOW: a data gradient of bf16 gradients that come with what rounding took off them, or one that keeps what rounding takes off its own.  The product of the rounded gradient alone has an error of its
// own of about 2^-9.3 of dx, next to the 2^-9.3 of rounding dx.  The reduction is walked twice, over a and then over its low part, into the
// same accumulators: a tile's steps are twice as many, and so is its time where the multiplies bound it (8192 x 2048 over 11264 293 us, with the
// low part of a 551-566; 8192 x 1024 over 4096 59 and 117; 1023 x 1024 over 5472 25 and 45).  A low part that is stored: 8192 x 4096 over 1024
// through GELU 80 and 96.
//
// Gated modes multiply both projections in one tile: 32 (in the narrowest tiles 16) rows of the gate's weights lie next to the same rows of the up
// projection's, so that a lane ends up with both products of its columns and the epilogue needs nobody else's.
#pragma once

#include "direct_load.h"
#include "fp32_split.h"
#include "linear_epilogue.h"

namespace tch {

struct LinearArgs {
  const void* a;      // [M][K], row stride lda (elements)
  const void* a_low;  // data gradient, bf16: what rounding took off a, laid out like it (may be null); both are multiplied
  const void* b;      // [N][K] dense; gated forward: [2N][K], gate rows first
  const float* bias;  // forward: [N] or [2N], may be null
  const void* add;    // residual, laid out by ldadd; may be null
  const void* z;      // backward: pre-activations [M][N] or [M][2N]
  void* out;          // [M][N]; gated backward: [M][2N]
  void* out2;         // forward: pre (may be null); gated backward: h (may be null)
  void* low;          // data gradients, bf16: what rounding took off out and out2 (may be null), laid out like them
  void* low2;
  int64_t lda, ldadd, ldz, ldo, ldo2;
  int M, N, K, act;
  uint32_t b_bytes;
  int tiles_m, tiles_n, group_rows;
  FastDiv div_tiles_n, div_group, div_rows;
};

namespace {

// What a tile's epilogue reads and writes beside the accumulators: buffer resources that begin at the tile's first row and end
// behind its last existing one, so that a row beyond M is dropped by its offset and 64-bit offsets stay out of the lanes.
struct TileTensors {
  __amdgpu_buffer_rsrc_t add, z, out, out2, low, low2;
};
template <typename T>
__device__ inline __amdgpu_buffer_rsrc_t rows_from(const void* base, int64_t ld, int row0, int rows, int width) {
  const int64_t bytes = rows > 0 && base ? ((rows - 1) * ld + width) * static_cast<int64_t>(sizeof(T)) : 0;
  return make_rsrc(base ? static_cast<const T*>(base) + row0 * ld : nullptr, static_cast<uint32_t>(bytes));
}
template <typename T, int MODE, bool LOW>
__device__ inline TileTensors tile_tensors(const LinearArgs& p, int m0, int rows) {
  constexpr int kWide = is_gated(MODE) ? 2 : 1;
  TileTensors t;
  t.add = rows_from<T>(p.add, p.ldadd, m0, rows, p.N);
  t.z = rows_from<T>(p.z, p.ldz, m0, rows, kWide * p.N);
  t.out = rows_from<T>(p.out, p.ldo, m0, rows, MODE == kGatedBwd ? 2 * p.N : p.N);
  t.out2 = rows_from<T>(p.out2, p.ldo2, m0, rows, MODE == kGatedFwd ? 2 * p.N : p.N);
  if constexpr (LOW || MODE == kGatedBwd) t.low = rows_from<T>(p.low, p.ldo, m0, rows, kWide * p.N);
  if constexpr (MODE == kGatedBwd) t.low2 = rows_from<T>(p.low2, p.ldo2, m0, rows, p.N);
  return t;
}

template <typename T>
__device__ inline int at(int row, int64_t ld, int col, bool ok) {   // byte offset of a chunk in a tile's tensor
  return ok ? (row * static_cast<int>(ld) + col) * static_cast<int>(sizeof(T)) : static_cast<int>(kOutOfRange);
}
__device__ inline Chunk read_chunk(__amdgpu_buffer_rsrc_t rsrc, int off) {
  const uint4_t v = __builtin_amdgcn_raw_buffer_load_b128(rsrc, off, 0, 0);
  Chunk c;
  c.w[0] = v[0];
  c.w[1] = v[1];
  c.w[2] = v[2];
  c.w[3] = v[3];
  return c;
}
template <typename T, int AUX = 0>
__device__ inline void write_chunk(__amdgpu_buffer_rsrc_t rsrc, int off, const float* v) {
  const Chunk c = float_to_chunk<T>(v);
  const uint4_t w = {c.w[0], c.w[1], c.w[2], c.w[3]};
  __builtin_amdgcn_raw_buffer_store_b128(w, rsrc, off, 0, AUX);
}

// One 16-byte chunk of the output (E columns of a row) in two steps: what it reads, and the rest.
template <typename T, int MODE, bool LOW>
struct ChunkOperands {
  Chunk zg, zu, add;
  __device__ __forceinline__ void request(const LinearArgs& p, const TileTensors& t, int row, int col) {
    const bool ok = col < p.N;
    if constexpr (MODE == kLinBwd || MODE == kGatedBwd) {
      if (MODE == kGatedBwd || p.act != kActNone) zg = read_chunk(t.z, at<T>(row, p.ldz, col, ok));
      if constexpr (MODE == kGatedBwd) zu = read_chunk(t.z, at<T>(row, p.ldz, p.N + col, ok));
    }
    if constexpr (!is_gated(MODE))
      if (p.add) add = read_chunk(t.add, at<T>(row, p.ldadd, col, ok));
  }
  // STREAM: forward outputs go past L2 (non-temporal) and leave it to the operands: the tile kernel, 8192 x 4096 over 1024 with the kept
  // pre-activation 78 -> 74 us (the outputs of a gated data gradient that way are 6 % slower)
  template <int ACT, bool STREAM>
  __device__ __forceinline__ void finish(const LinearArgs& p, const TileTensors& t, int row, int col, const float* v, float* u) {
    constexpr int E = Elem<T>::kPerChunk, AUX = STREAM && (MODE == kLinFwd || MODE == kGatedFwd) ? 2 : 0;
    const bool ok = col < p.N;
    float fg[E], fu[E], o[E], h[E];
    if constexpr (MODE == kLinBwd || MODE == kGatedBwd) chunk_to_float<T>(zg, fg);
    if constexpr (MODE == kGatedBwd) chunk_to_float<T>(zu, fu);
    if constexpr (MODE == kLinFwd || MODE == kGatedFwd) {
      if (p.out2) {
        write_chunk<T, AUX>(t.out2, at<T>(row, p.ldo2, col, ok), v);
        if constexpr (MODE == kGatedFwd) write_chunk<T, AUX>(t.out2, at<T>(row, p.ldo2, p.N + col, ok), u);
      }
    }
    combine<T, MODE, ACT, E>(v, u, fg, fu, o, h);
    if constexpr (!is_gated(MODE)) {
      if (p.add) {
        float r[E];
        chunk_to_float<T>(add, r);
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] += r[e];
      }
    }
    write_chunk<T, AUX>(t.out, at<T>(row, p.ldo, col, ok), o);
    if constexpr (LOW) {
      if (p.low) {
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = rounded_off(o[e]);
        write_chunk<T>(t.low, at<T>(row, p.ldo, col, ok), o);
      }
    }
    if constexpr (MODE == kGatedBwd) {
      write_chunk<T>(t.out, at<T>(row, p.ldo, p.N + col, ok), u);
      if (p.out2) write_chunk<T>(t.out2, at<T>(row, p.ldo2, col, ok), h);
      if constexpr (sizeof(T) == 2) {
        if (p.low) {
#pragma unroll
          for (int e = 0; e < E; ++e) o[e] = rounded_off(o[e]), u[e] = rounded_off(u[e]);
          write_chunk<T>(t.low, at<T>(row, p.ldo, col, ok), o);
          write_chunk<T>(t.low, at<T>(row, p.ldo, p.N + col, ok), u);
        }
        if (p.low2) {
#pragma unroll
          for (int e = 0; e < E; ++e) h[e] = rounded_off(h[e]);
          write_chunk<T>(t.low2, at<T>(row, p.ldo2, col, ok), h);
        }
      }
    }
  }
};

template <typename T>
__device__ inline void mma32(const uint4_t& first, const uint4_t& second, f32x16_t& acc) {
  if constexpr (sizeof(T) == 2) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, first), __builtin_bit_cast(bf16x8_t, second), acc, 0, 0, 0);
  } else {
    // a lane holds four neighbouring reduction elements: instruction e multiplies element e of both halves of the lanes
    const f32x4_t x = __builtin_bit_cast(f32x4_t, first), y = __builtin_bit_cast(f32x4_t, second);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], y[e], acc, 0, 0, 0);
  }
}

// ---------------------------------------------------------------------------
// large products: a persistent grid whose workgroups walk output tiles as one sequence of reduction steps
// ---------------------------------------------------------------------------
// WM x WN wavefronts of TM x TN MFMA tiles (32 x 32).  Operand tiles go from global memory straight into LDS (16 bytes a lane,
// rows of 128 bytes, the 16-byte slot XOR-ed by the row so that an operand read touches every bank once), NBUF of them; the
// slice of 32 bytes that is multiplied next is read while this one is multiplied, and the direct loads of the tile NBUF - 1
// steps ahead go out between the multiplies.  The tiles of a workgroup are one sequence: the next tile's first loads are on
// their way during this tile's last steps and its epilogue.  A row of the operands that does not exist is outside its buffer
// resource and lands as zeros; a chunk behind K is turned away by its lane's offset in the last step of a tile.
// Measured: gated forward 16384 x 11008 over 4096 2.12-2.27 ms, 1.30-1.39 PFLOP/s, bound by power (matrix pipes 79 % busy; a library product
// of this size 1.35); data gradient 8192 x 2048 over 11264 293 us, 1.29.  Where the reduction is short the epilogue counts, in which the
// matrix pipes stand: forward 8192 x 4096 over 1024 with GELU and the kept pre-activation 72-74 us, about 25 of them epilogue (134 MB written);
// the gated data gradient 8192 x 5632 over 2048 with its low parts 287-293 us, half of them (740 MB at 5.5 TB/s).  fp32 4096 x 4096 over 1024: 247 us, 0.139 of 0.157 PFLOP/s.
template <typename T, int MODE, bool LOW, int WM, int WN, int TM, int TN, int NBUF, int PER_CU>
__global__ __launch_bounds__(WM* WN * 64, PER_CU* WM* WN / 4) void linear_tile_kernel(LinearArgs p) {
  constexpr int E = Elem<T>::kPerChunk, EB = sizeof(T), RB = 128;
  constexpr int KS = RB / EB, SL = RB / 32, SLOTS = RB / 16, LD_ROWS = 1024 / RB;
  constexpr int BM = WM * TM * 32, BN = WN * TN * 32, NW = WM * WN;
  constexpr bool GATED_FWD = MODE == kGatedFwd;
  constexpr int BN_OUT = GATED_FWD ? BN / 2 : BN;
  static_assert(TN == 2, "a wavefront has 64 columns: gate and up tiles, or the whole lines of the epilogue");
  static_assert(BM % (LD_ROWS * NW) == 0 && BN % (LD_ROWS * NW) == 0, "tile/loader mismatch");
  constexpr int A_LD = BM / LD_ROWS / NW, B_LD = BN / LD_ROWS / NW, LOADS = A_LD + B_LD;
  constexpr bool OWN_STAGE = NBUF == 2;   // the epilogue's staging has a place of its own
  static_assert(OWN_STAGE || A_LD >= 4, "4 KB of a wavefront's own loads stage its epilogue");
  constexpr int A_BYTES = BM * RB, BUF_BYTES = A_BYTES + BN * RB;
  // with two buffers the requested tile is waited for at the end of the step: all requests go out in its first half
  constexpr int LOAD_SL = NBUF == 2 ? (SL + 1) / 2 : SL;
  constexpr int AHEAD = (NBUF - 2) * LOADS;
  static_assert(AHEAD < 48, "vmcnt range");
  constexpr bool BIAS = MODE == kLinFwd || MODE == kGatedFwd;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[NBUF * BUF_BYTES + (OWN_STAGE ? NW * 4096 : 0)];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const int frag_row = lane & 31, frag_half = lane >> 5;
  const int nk = (p.K + KS - 1) / KS, steps = LOW && p.a_low ? 2 * nk : nk;   // the steps of a, and then those of its low part
  const int tiles = p.tiles_m * p.tiles_n;
  const int first = static_cast<int>(xcd_remap(blockIdx.x, gridDim.x));
  auto swizzle = [](int row) { return (row >> 1) & 7; };

  // consecutive tiles walk down group_rows row tiles before they move one column tile on: the tiles an XCD works on at one time
  // form a block, with fewer distinct operand rows through its L2
  auto locate = [&](int id, int& m0, int& n0) LINEAR_INLINE {
    uint32_t q, rem;
    if (p.group_rows <= 1) {
      p.div_tiles_n.divmod(static_cast<uint32_t>(id), q, rem);
      m0 = static_cast<int>(q) * BM;
      n0 = static_cast<int>(rem) * BN_OUT;
      return;
    }
    p.div_group.divmod(static_cast<uint32_t>(id), q, rem);
    const uint32_t row0 = q * p.group_rows, rows = min(static_cast<uint32_t>(p.group_rows), static_cast<uint32_t>(p.tiles_m) - row0);
    const uint32_t col = rows == static_cast<uint32_t>(p.group_rows) ? p.div_rows.div(rem) : rem / rows;
    m0 = static_cast<int>(row0 + (rem - col * rows)) * BM;
    n0 = static_cast<int>(col) * BN_OUT;
  };

  // ---- the walk of the loads: offsets are the same for every tile, the resources move ----
  const int sub_row = lane / SLOTS, slot = lane % SLOTS;
  uint32_t a_off[A_LD], b_off[B_LD];
  uint32_t behind_k[2] = {0u, 0u};   // the lane's chunk of an even / odd direct load lies behind K in the last step
#pragma unroll
  for (int j = 0; j < A_LD; ++j) {
    const int trow = (wave * A_LD + j) * LD_ROWS + sub_row;
    a_off[j] = (static_cast<uint32_t>(trow) * static_cast<uint32_t>(p.lda) + (slot ^ swizzle(trow)) * E) * EB;
  }
#pragma unroll
  for (int j = 0; j < B_LD; ++j) {
    const int trow = (wave * B_LD + j) * LD_ROWS + sub_row;
    const int block = trow >> 5;
    const uint32_t row = GATED_FWD ? static_cast<uint32_t>((block & 1) * p.N + (block >> 1) * 32 + (trow & 31)) : static_cast<uint32_t>(trow);
    b_off[j] = (row * static_cast<uint32_t>(p.K) + (slot ^ swizzle(trow)) * E) * EB;
  }
#pragma unroll
  for (int odd = 0; odd < 2; ++odd)
    behind_k[odd] = (nk - 1) * KS + (slot ^ swizzle(odd * LD_ROWS + sub_row)) * E >= p.K ? kOutOfRange : 0u;
  const bool ragged_k = p.K % KS != 0;

  __amdgpu_buffer_rsrc_t rsrc_a, rsrc_b;
  const __amdgpu_buffer_rsrc_t rsrc_bias = make_rsrc(p.bias, BIAS && p.bias ? static_cast<uint32_t>(p.N) * (GATED_FWD ? 8u : 4u) : 0u);
  int ld_id = first, ld_kt = 0;
  bool ld_low = false;   // the walk is in the low part
  auto mark_tail = [&]() LINEAR_INLINE {
#pragma unroll
    for (int j = 0; j < A_LD; ++j) a_off[j] |= behind_k[(wave * A_LD + j) & 1];
#pragma unroll
    for (int j = 0; j < B_LD; ++j) b_off[j] |= behind_k[(wave * B_LD + j) & 1];
  };
  auto enter_tile = [&]() LINEAR_INLINE {   // or its low part
    int m0 = 0, n0 = 0;
    const bool any = ld_id < tiles;
    if (any) locate(ld_id, m0, n0);
    const int rows = min(BM, p.M - m0);
    rsrc_a = make_rsrc(static_cast<const T*>(LOW && ld_low ? p.a_low : p.a) + m0 * p.lda, static_cast<uint32_t>(((rows - 1) * p.lda + p.K) * EB));
    const uint32_t skip = static_cast<uint32_t>(n0) * static_cast<uint32_t>(p.K) * EB;
    rsrc_b = make_rsrc(static_cast<const unsigned char*>(p.b) + skip, p.b_bytes - skip);
    if (ragged_k || !any) {   // behind the last tile every offset is out of range: zeros land
      const uint32_t set = any ? 0u : kOutOfRange;
#pragma unroll
      for (int j = 0; j < A_LD; ++j) a_off[j] = (a_off[j] & ~kOutOfRange) | set;
#pragma unroll
      for (int j = 0; j < B_LD; ++j) b_off[j] = (b_off[j] & ~kOutOfRange) | set;
      if (ragged_k && nk == 1) mark_tail();
    }
  };
  auto issue_load = [&](uint32_t buf, int j) LINEAR_INLINE {   // direct load j of the step the walk stands at
    if (j < A_LD)
      load_to_lds(rsrc_a, lds + buf + (wave * A_LD + j) * 1024, static_cast<int>(a_off[j]), ld_kt * RB);
    else
      load_to_lds(rsrc_b, lds + buf + A_BYTES + (wave * B_LD + j - A_LD) * 1024, static_cast<int>(b_off[j - A_LD]), ld_kt * RB);
  };
  auto next_step = [&]() LINEAR_INLINE {
    if (++ld_kt == nk) {
      ld_kt = 0;
      ld_low = LOW && p.a_low && !ld_low;
      if (!ld_low) ld_id += gridDim.x;
      enter_tile();
    } else if (ragged_k && ld_kt == nk - 1) {
      mark_tail();
    }
  };

  f32x16_t acc[TM][TN];
  clear(acc);
  const int swz = swizzle(frag_row);
  const uint32_t lds_base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds));
  const uint32_t a_rd = lds_base + (wm * TM * 32 + frag_row) * RB + swz * 16;
  const uint32_t b_rd = lds_base + A_BYTES + (wn * TN * 32 + frag_row) * RB + swz * 16;
  uint4_t fa[2][TM], fb[2][TN];
  // The operand reads are asm: the compiler would put a wait for every direct load in flight in front of an LDS read it can see.
  auto read_one = [&](uint32_t pa, uint32_t pb, int set, int i) {
    if (i < TM)
      asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(fa[set][i]) : "v"(pa), "n"(i * 32 * RB));
    else
      asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(fb[set][i - TM]) : "v"(pb), "n"((i - TM) * 32 * RB));
  };
  auto hold_set = [&](int set) {
#pragma unroll
    for (int i = 0; i < TM; ++i) asm volatile("" : "+v"(fa[set][i]));
#pragma unroll
    for (int i = 0; i < TN; ++i) asm volatile("" : "+v"(fb[set][i]));
  };
  // multiplies the slice in `set`; meanwhile slice kk of the step in `buf` is read into the other set and part `q` of the loads
  // (-1: all of them) goes to `ld_buf`
  auto slice = [&](auto set_c, uint32_t buf, auto kk_c, auto q_c, uint32_t ld_buf) LINEAR_INLINE {
    constexpr int set = decltype(set_c)::value, kk = decltype(kk_c)::value, q = decltype(q_c)::value;
    constexpr int READS = TM + TN, MF = TM * TN, FIRST = q < 0 ? 0 : (q < LOAD_SL ? q : LOAD_SL) * LOADS / LOAD_SL;
    constexpr int AUX = READS + (q < 0 ? LOADS : q < LOAD_SL ? (q + 1) * LOADS / LOAD_SL - FIRST : 0);
    constexpr int PER = (AUX + MF - 1) / MF > 2 ? (AUX + MF - 1) / MF : 2;
    const uint32_t pa = (a_rd ^ static_cast<uint32_t>((2 * kk + frag_half) * 16)) + buf;
    const uint32_t pb = (b_rd ^ static_cast<uint32_t>((2 * kk + frag_half) * 16)) + buf;
    unrolled<MF>([&](auto m_c) LINEAR_INLINE {
      constexpr int m = decltype(m_c)::value, tm = m / TN, tn = m % TN;
      mma32<T>(fb[set][tn], fa[set][tm], acc[tm][tn]);
      unrolled<PER>([&](auto a_c) LINEAR_INLINE {
        constexpr int a = m * PER + decltype(a_c)::value;
        if constexpr (a < READS) read_one(pa, pb, set ^ 1, a);
        else if constexpr (a < AUX) issue_load(ld_buf, FIRST + a - READS);
      });
      __builtin_amdgcn_sched_barrier(0);
    });
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    hold_set(set ^ 1);
  };

  // ---- the output: sixteen rows of a wavefront's accumulators at a time go through LDS (fp32, 16-byte slots XOR-ed by the row) and
  // come back row by row, so that every load and store of the epilogue moves whole cache lines ----
  // A lane's accumulators are four columns of one row at a time, 32 rows apart in memory: stored from there, a line is written in
  // four pieces over the whole epilogue, and the output of the tiles at work is more than L2 holds.
  // The 4 KB lie behind the buffers where there are two.  Where there are three, they are this wavefront's own part of the buffer
  // that the tile's last step was read from: nobody else touches it before this wavefront requests the step that goes there,
  // behind the epilogue.
  auto epilogue = [&](int id, uint32_t stage) LINEAR_INLINE {
    int m0, n0;
    locate(id, m0, n0);
    const TileTensors t = tile_tensors<T, MODE, LOW>(p, m0, min(BM, p.M - m0));
    constexpr int COLS = GATED_FWD ? 32 : 64;             // output columns of a wavefront
    constexpr int LANES = COLS / E, ROWS = 64 / LANES;    // lanes per row, rows per pass
    constexpr int PASSES = 16 / ROWS, BLOCKS = TM * 2, TOTAL = BLOCKS * PASSES;
    constexpr int DEPTH = TM <= 2 ? 4 : MODE == kGatedBwd ? 1 : 2;                 // passes whose operands are on their way, as the registers allow
    const int lane_row = lane / LANES, lane_col = lane % LANES * E;
    const int col = n0 + wn * COLS + lane_col;
    ChunkOperands<T, MODE, LOW> operands[DEPTH];
    auto row_of = [&](int pass) {
      int row = (wm * BLOCKS + pass / PASSES) * 16 + pass % PASSES * ROWS + lane_row;
      asm volatile("" : "+v"(row));   // offsets are made where they are used, not all of them ahead of the first
      return row;
    };
    auto request = [&](int pass) LINEAR_INLINE { operands[pass % DEPTH].request(p, t, row_of(pass), col); };
    float bv[E], bu[E];
#pragma unroll
    for (int e = 0; e < E; ++e) bv[e] = bu[e] = 0.f;
    if (BIAS && p.bias) {
#pragma unroll
      for (int e = 0; e < E; e += 4) {
        const int off = col < p.N ? (col + e) * 4 : static_cast<int>(kOutOfRange);
        const uint4_t b = __builtin_amdgcn_raw_buffer_load_b128(rsrc_bias, off, 0, 0);
        const uint4_t c = GATED_FWD ? __builtin_amdgcn_raw_buffer_load_b128(rsrc_bias, col < p.N ? off + p.N * 4 : off, 0, 0) : b;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          bv[e + i] = __uint_as_float(b[i]);
          bu[e + i] = __uint_as_float(c[i]);
        }
      }
    }
    // slot of four columns: (column / 4) ^ row; columns of the up projection lie behind the gate's 32
    const uint32_t mine = lds_base + (OWN_STAGE ? NBUF * BUF_BYTES + wave * 4096 : stage + wave * A_LD * 1024);
    const uint32_t wr = mine + (frag_row & 15) * 256;
    auto stage_block = [&](auto block_c) LINEAR_INLINE {   // 16 rows: half the lanes
      constexpr int block = decltype(block_c)::value, tm = block >> 1;
      if ((frag_row >> 4) == (block & 1)) {
#pragma unroll
        for (int tn = 0; tn < 2; ++tn)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint4_t v = {__float_as_uint(acc[tm][tn][4 * j]), __float_as_uint(acc[tm][tn][4 * j + 1]), __float_as_uint(acc[tm][tn][4 * j + 2]),
                               __float_as_uint(acc[tm][tn][4 * j + 3])};
            const uint32_t to = wr + (static_cast<uint32_t>((tn * 8 + j * 2 + frag_half) ^ (frag_row & 15)) << 4);
            asm volatile("ds_write_b128 %0, %1" ::"v"(to), "v"(v) : "memory");
          }
      }
    };
    auto from_stage = [&](int row16, int first_col, float* v) LINEAR_INLINE {   // E columns of a row; LDS accesses of a wavefront keep their order
      if constexpr (E == 8) {
        uint4_t x, y;
        const uint32_t s0 = mine + row16 * 256 + (((first_col >> 2) ^ row16) << 4), s1 = mine + row16 * 256 + (((first_col >> 2) + 1 ^ row16) << 4);
        asm volatile("ds_read_b128 %0, %2\n\tds_read_b128 %1, %3\n\ts_waitcnt lgkmcnt(0)" : "=&v"(x), "=&v"(y) : "v"(s0), "v"(s1) : "memory");
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v[i] = __uint_as_float(x[i]);
          v[4 + i] = __uint_as_float(y[i]);
        }
      } else {
        uint4_t x;
        asm volatile("ds_read_b128 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=&v"(x) : "v"(mine + row16 * 256 + (((first_col >> 2) ^ row16) << 4)) : "memory");
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(x[i]);
      }
    };
    // the multiplies are done before their results are read by hand-written instructions
    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
    with_activation(p.act, [&](auto act_c) LINEAR_INLINE {
      constexpr int ACT = decltype(act_c)::value;
#pragma unroll
      for (int pass = 0; pass < DEPTH; ++pass) request(pass);
      unrolled<BLOCKS>([&](auto block_c) LINEAR_INLINE {
        stage_block(block_c);
#pragma unroll
        for (int i = 0; i < PASSES; ++i) {
          const int pass = decltype(block_c)::value * PASSES + i;
          float v[E], u[E];
          from_stage(i * ROWS + lane_row, lane_col, v);
          if constexpr (GATED_FWD) from_stage(i * ROWS + lane_row, 32 + lane_col, u);
          if constexpr (BIAS) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
              v[e] += bv[e];
              if constexpr (GATED_FWD) u[e] += bu[e];
            }
          }
          operands[pass % DEPTH].template finish<ACT, true>(p, t, row_of(pass), col, v, u);
          if (pass + DEPTH < TOTAL) request(pass + DEPTH);
          __builtin_amdgcn_sched_barrier(0);   // one pass at a time: the registers are the accumulators'
        }
      });
    });
    clear(acc);
  };

  // Behind an epilogue its stores (this many of an output; one that is turned away counts too) are newer requests than the step that
  // has to land: they are not waited for.  With two buffers all of that step is requested ahead of the epilogue for this.
  constexpr int STORES = TM * 32 * (GATED_FWD ? 32 : 64) / (64 * E);
  constexpr int NEWER = NBUF == 2 ? 0 : AHEAD;
  constexpr int OUTPUTS = MODE == kGatedBwd ? 2 : 1, MORE = MODE == kGatedFwd ? 2 : MODE == kLinBwd && !LOW ? 0 : 1;   // `out`; `out2` or `low`
  constexpr int AFTER_ONE = NEWER + STORES * OUTPUTS < 63 ? NEWER + STORES * OUTPUTS : 63;
  constexpr int AFTER_BOTH = NEWER + STORES * (OUTPUTS + MORE) < 63 ? NEWER + STORES * (OUTPUTS + MORE) : 63;
  enter_tile();
#pragma unroll
  for (int s = 0; s < NBUF - 1; ++s) {
#pragma unroll
    for (int j = 0; j < LOADS; ++j) issue_load(s * BUF_BYTES, j);
    next_step();
  }
  constexpr int STARTED = NBUF == 2 ? LOADS : LOADS / LOAD_SL;
#pragma unroll
  for (int j = 0; j < STARTED; ++j) issue_load((NBUF - 1) * BUF_BYTES, j);
  if (NBUF == 2) next_step();
  wait_and_meet<AHEAD + STARTED>();
#pragma unroll
  for (int i = 0; i < TM + TN; ++i) read_one(a_rd ^ static_cast<uint32_t>(frag_half * 16), b_rd ^ static_cast<uint32_t>(frag_half * 16), 0, i);
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  hold_set(0);
  uint32_t buf = 0, before = (NBUF - 1) * BUF_BYTES;
  // One step: its last slice is multiplied behind the barrier that hands over the next one, with the first part of the requests
  // for the step that takes its buffer.  Behind a tile's last step: all of them where there are two buffers (the first step of
  // the next tile then requests nothing), none where there are three (the buffer stages the epilogue).
  constexpr int NONE = LOAD_SL, ALL = -1;
  auto step = [&](int after_stores, auto first_c, auto last_part) LINEAR_INLINE {
    unrolled<SL - 1>([&](auto s_c) LINEAR_INLINE {
      constexpr int s = decltype(s_c)::value, part = decltype(first_c)::value && NBUF == 2 ? NONE : s + 1;
      slice(std::integral_constant<int, (s & 1)>{}, buf, std::integral_constant<int, s + 1>{}, std::integral_constant<int, part>{}, before);
    });
    if (!(decltype(first_c)::value && NBUF == 2)) next_step();
    if (after_stores == 0)
      wait_and_meet<AHEAD>();
    else if (after_stores == 1)
      wait_and_meet<AFTER_ONE>();
    else
      wait_and_meet<AFTER_BOTH>();
    before = buf;
    buf = buf == (NBUF - 1) * BUF_BYTES ? 0 : buf + BUF_BYTES;
    slice(std::integral_constant<int, ((SL - 1) & 1)>{}, buf, std::integral_constant<int, 0>{}, last_part, before);
  };
  std::integral_constant<int, 0> middle;
  std::integral_constant<int, 1> start;
  std::integral_constant<int, NBUF == 2 ? ALL : NONE> finish;
  constexpr bool ONE_STEP = TM <= 2;   // reductions of one step; with 128 accumulators the second way there costs registers (spilled)
  const int outputs = p.out2 || (LOW && p.low) ? 2 : 1;
  int stored = 0;
  for (int id = first; id < tiles; id += gridDim.x) {
    if (ONE_STEP && steps == 1) {
      step(stored, start, finish);
    } else {
      step(stored, start, middle);
      for (int kt = 1; kt < steps - 1; ++kt) step(0, middle, middle);
      step(0, middle, finish);
    }
    if (NBUF == 2) next_step();
    epilogue(id, before);
    if (NBUF > 2) {
#pragma unroll
      for (int j = 0; j < LOADS / LOAD_SL; ++j) issue_load(before, j);
    }
    stored = outputs;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the zeros behind the last tile land before the LDS goes
}

// ---------------------------------------------------------------------------
// few tiles: every wavefront of a workgroup has the whole tile for every KG-th reduction step
// ---------------------------------------------------------------------------
// Each wavefront has a ring of NBUF operand tiles (rows of RB bytes) of its own, filled with direct loads, and waits for its own loads
// only: no barrier before the partial tiles meet in LDS, where they are added in the order of the wavefronts.  What that buys
// where workgroups are few: KG * (NBUF - 1) operand tiles in flight per compute unit and a chain of nk / KG steps instead of nk.
// Bound by the bytes of the weights where there are many (7 rows through 2048 -> 2 x 5632 gated: 9.3 us, 5.0 TB/s; 32 through 8192 -> 8192:
// 23.6 us, 5.7 TB/s), by the latency of a chain of steps where there are few.
template <typename T, int MODE, bool LOW, int TM, int TN, int KG, int NBUF, int RB>
__global__ __launch_bounds__(KG * 64) void linear_split_kernel(LinearArgs p) {
  constexpr int E = Elem<T>::kPerChunk, EB = sizeof(T), KS = RB / EB, SL = RB / 32, SLOTS = RB / 16, LD_ROWS = 1024 / RB;
  constexpr bool GATED_FWD = MODE == kGatedFwd;
  constexpr int BM = TM * 32, BN = TN * 32, BN_OUT = GATED_FWD ? BN / 2 : BN;
  constexpr int HALF = TN == 1 ? 16 : 32;   // gated: columns of the gate that lie together, in front of the same of the up projection
  constexpr int A_LD = BM / LD_ROWS, B_LD = BN / LD_ROWS, A_BYTES = BM * RB, BUF_BYTES = (BM + BN) * RB;
  constexpr int NT = KG * 64, LD = BN + 4;
  constexpr int RED_BYTES = KG * BM * LD * 4, RING_BYTES = KG * NBUF * BUF_BYTES;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[RED_BYTES > RING_BYTES ? RED_BYTES : RING_BYTES];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // consecutive tiles (one XCD) share the rows of the larger operand: group_rows != 0: walk down the row tiles of a column tile
  uint32_t slow, fast;
  p.div_tiles_n.divmod(xcd_remap(blockIdx.x, gridDim.x), slow, fast);
  const int m0 = static_cast<int>(p.group_rows ? fast : slow) * BM, n0 = static_cast<int>(p.group_rows ? slow : fast) * BN_OUT;
  const int rows = min(BM, p.M - m0);
  const int nk = (p.K + KS - 1) / KS, steps = LOW && p.a_low ? 2 * nk : nk;   // the steps of a, and then those of its low part
  const int my_steps = steps > wave ? (steps - wave + KG - 1) / KG : 0;

  auto swizzle = [](int row) { return RB == 128 ? (row >> 1) & 7 : (row >> 2) & 3; };
  const int sub_row = lane / SLOTS, slot = lane % SLOTS;
  int chunk[2];   // of an even and an odd direct load
#pragma unroll
  for (int odd = 0; odd < 2; ++odd) chunk[odd] = slot ^ swizzle(odd * LD_ROWS + sub_row);
  uint32_t a_off[A_LD], b_off[B_LD];
#pragma unroll
  for (int j = 0; j < A_LD; ++j) a_off[j] = (static_cast<uint32_t>(j * LD_ROWS + sub_row) * static_cast<uint32_t>(p.lda) + chunk[j & 1] * E) * EB;
#pragma unroll
  for (int j = 0; j < B_LD; ++j) {
    const int trow = j * LD_ROWS + sub_row, block = trow / HALF;
    const uint32_t row = GATED_FWD ? static_cast<uint32_t>((block & 1) * p.N + (block >> 1) * HALF + trow % HALF) : static_cast<uint32_t>(trow);
    b_off[j] = (row * static_cast<uint32_t>(p.K) + chunk[j & 1] * E) * EB;
  }
  const uint32_t skip = static_cast<uint32_t>(n0) * static_cast<uint32_t>(p.K) * EB;
  const __amdgpu_buffer_rsrc_t rsrc_b = make_rsrc(static_cast<const unsigned char*>(p.b) + skip, p.b_bytes - skip);

  unsigned char* ring = lds + wave * (NBUF * BUF_BYTES);
  int ld_kt = wave;
  auto issue_loads = [&](int buf) {
    const bool low = LOW && ld_kt >= nk;
    const int kt = low ? ld_kt - nk : ld_kt;
    const __amdgpu_buffer_rsrc_t rsrc_a =
        make_rsrc(static_cast<const T*>(low ? p.a_low : p.a) + m0 * p.lda, static_cast<uint32_t>(((rows - 1) * p.lda + p.K) * EB));
    uint32_t behind[2];   // the chunk lies behind K
#pragma unroll
    for (int odd = 0; odd < 2; ++odd) behind[odd] = kt * KS + chunk[odd] * E >= p.K ? kOutOfRange : 0u;
    unsigned char* dst = ring + buf * BUF_BYTES;
#pragma unroll
    for (int j = 0; j < A_LD; ++j) load_to_lds(rsrc_a, dst + j * 1024, static_cast<int>(a_off[j] | behind[j & 1]), kt * RB);
#pragma unroll
    for (int j = 0; j < B_LD; ++j) load_to_lds(rsrc_b, dst + A_BYTES + j * 1024, static_cast<int>(b_off[j] | behind[j & 1]), kt * RB);
    ld_kt += KG;
  };

  f32x16_t acc[TM][TN];
  clear(acc);
  const int frag_row = lane & 31, frag_half = lane >> 5;
  const uint32_t rd = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(ring)) + frag_row * RB + swizzle(frag_row) * 16;
  auto read_frags = [&](int buf, int kk, uint4_t* fa, uint4_t* fb) {
    const uint32_t pa = (rd ^ static_cast<uint32_t>((2 * kk + frag_half) * 16)) + buf * BUF_BYTES;
#pragma unroll
    for (int tm = 0; tm < TM; ++tm) asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(fa[tm]) : "v"(pa), "n"(tm * 32 * RB));
#pragma unroll
    for (int tn = 0; tn < TN; ++tn) asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(fb[tn]) : "v"(pa), "n"(A_BYTES + tn * 32 * RB));
  };
  auto multiply = [&](uint4_t* fa, uint4_t* fb) {
#pragma unroll
    for (int tm = 0; tm < TM; ++tm) asm volatile("" : "+v"(fa[tm]));
#pragma unroll
    for (int tn = 0; tn < TN; ++tn) asm volatile("" : "+v"(fb[tn]));
#pragma unroll
    for (int tm = 0; tm < TM; ++tm)
#pragma unroll
      for (int tn = 0; tn < TN; ++tn) mma32<T>(fb[tn], fa[tm], acc[tm][tn]);
  };
  // The tile of step i has landed when at most the NBUF - 2 requested behind it are outstanding (near the end fewer follow: wait
  // for everything).  The reads of step i - 1 were waited for before its multiplies, so its buffer is free.
  constexpr int AHEAD = (NBUF - 2) * (A_LD + B_LD);
  static_assert(AHEAD < 64, "vmcnt range");
  auto step = [&](int i, int buf) {
    if (i + NBUF - 1 <= my_steps)
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(AHEAD) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (i + NBUF - 1 < my_steps) issue_loads((buf + NBUF - 1) % NBUF);
    // a slice is read while the one before it is multiplied
    uint4_t fa[2][TM], fb[2][TN];
    read_frags(buf, 0, fa[0], fb[0]);
#pragma unroll
    for (int kk = 0; kk < SL; ++kk) {
      if (kk + 1 < SL) {
        read_frags(buf, kk + 1, fa[(kk + 1) & 1], fb[(kk + 1) & 1]);
        asm volatile("s_waitcnt lgkmcnt(%0)" ::"n"(TM + TN) : "memory");
      } else {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
      multiply(fa[kk & 1], fb[kk & 1]);
    }
  };
#pragma unroll
  for (int i = 0; i < NBUF - 1; ++i)
    if (i < my_steps) issue_loads(i);
  int i0 = 0;
  for (; i0 + NBUF <= my_steps; i0 += NBUF) {
#pragma unroll
    for (int u = 0; u < NBUF; ++u) step(i0 + u, u);
  }
#pragma unroll
  for (int u = 0; u < NBUF - 1; ++u)
    if (i0 + u < my_steps) step(i0 + u, u);

  // ---- the partial tiles meet: [wave][BM][LD] fp32, over the rings ----
  float* red = reinterpret_cast<float*>(lds);
  const TileTensors t = tile_tensors<T, MODE, LOW>(p, m0, rows);
  constexpr int CH = BN_OUT / E, ITEMS = BM * CH, VISITS = (ITEMS + NT - 1) / NT;
  ChunkOperands<T, MODE, LOW> operands[VISITS];
#pragma unroll
  for (int visit = 0; visit < VISITS; ++visit) {
    const int q = tid + visit * NT;
    operands[visit].request(p, t, q / CH, q < ITEMS ? n0 + q % CH * E : p.N);
  }
  __syncthreads();   // every wavefront is done with its ring
#pragma unroll
  for (int tm = 0; tm < TM; ++tm)
#pragma unroll
    for (int tn = 0; tn < TN; ++tn)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<float4*>(red + wave * (BM * LD) + (tm * 32 + frag_row) * LD + tn * 32 + 8 * j + 4 * frag_half) =
            make_float4(acc[tm][tn][4 * j], acc[tm][tn][4 * j + 1], acc[tm][tn][4 * j + 2], acc[tm][tn][4 * j + 3]);
  __syncthreads();
  auto total = [&](int row, int col, float* v) {
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = 0.f;
#pragma unroll
    for (int g = 0; g < KG; ++g)
#pragma unroll
      for (int e = 0; e < E; e += 4) {
        const float4 s = *reinterpret_cast<const float4*>(red + (g * BM + row) * LD + col + e);
        v[e] += s.x;
        v[e + 1] += s.y;
        v[e + 2] += s.z;
        v[e + 3] += s.w;
      }
  };
  auto add_bias = [&](int col, float* v) {
#pragma unroll
    for (int e = 0; e < E; e += 4) {
      const float4 b = *reinterpret_cast<const float4*>(p.bias + col + e);
      v[e] += b.x;
      v[e + 1] += b.y;
      v[e + 2] += b.z;
      v[e + 3] += b.w;
    }
  };
  with_activation(p.act, [&](auto act_c) {
    constexpr int ACT = decltype(act_c)::value;
#pragma unroll
    for (int visit = 0; visit < VISITS; ++visit) {
      const int q = tid + visit * NT;
      const int row = q / CH, c = q % CH * E;
      if (q >= ITEMS || n0 + c >= p.N) continue;
      float v[E], u[E];
      if constexpr (GATED_FWD) {
        total(row, c / HALF * (2 * HALF) + c % HALF, v);
        total(row, c / HALF * (2 * HALF) + HALF + c % HALF, u);
      } else {
        total(row, c, v);
      }
      if constexpr (MODE == kLinFwd || MODE == kGatedFwd) {
        if (p.bias) {
          add_bias(n0 + c, v);
          if constexpr (GATED_FWD) add_bias(p.N + n0 + c, u);
        }
      }
      operands[visit].template finish<ACT, false>(p, t, row, n0 + c, v, u);
    }
  });
}

// ---------------------------------------------------------------------------
// few rows (tokens that decode together), or few outputs: operands straight into registers
// ---------------------------------------------------------------------------
// A workgroup has 16 rows and 16 output columns; its KG wavefronts take 256-byte pieces of the reduction in turn.  Weight rows are the rows and the tokens the columns of 16 x 16 MFMA tiles; lane l holds the 16-byte
// chunk l / 16 (of four) of row l % 16, so that a load covers 64 neighbouring bytes of sixteen rows.  The next piece is
// requested before this one is multiplied.  Up to 16 rows it is bound by the bytes of the weights; beyond, by what a compute unit
// loads into registers (32 or 64 rows a workgroup, for fewer loads of the weights, were slower throughout, and so were gate and up tiles
// next to each other against 32 x 32 tiles with a ring in LDS).  One token through 4096 x 4096 bf16: 7.4 us, 4.5 TB/s.
template <typename T>
__device__ inline void mma16(const uint4_t& first, const uint4_t& second, f32x4_t& acc) {
  if constexpr (sizeof(T) == 2) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, first), __builtin_bit_cast(bf16x8_t, second), acc, 0, 0, 0);
  } else {
    const f32x4_t x = __builtin_bit_cast(f32x4_t, first), y = __builtin_bit_cast(f32x4_t, second);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], acc, 0, 0, 0);
  }
}

template <typename T>
__device__ inline void load_four(const T* p, float* v) {
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = Elem<T>::load(p + e);
}
template <typename T>
__device__ inline void store_four(T* p, const float* v) {
#pragma unroll
  for (int e = 0; e < 4; ++e) Elem<T>::store(p + e, v[e]);
}

template <typename T, int MODE, bool LOW, int KG>
__global__ __launch_bounds__(KG * 64) void linear_rows_kernel(LinearArgs p) {
  constexpr int E = Elem<T>::kPerChunk, EB = sizeof(T);
  static_assert(MODE != kGatedFwd, "gate and up projections need another layout");
  constexpr int U = 4, PIECE = U * 4 * E;   // loads per piece and tile; elements of a piece
  constexpr int LD = 20;                    // floats of a row of 16 partial sums
  __shared__ float red[KG][16 * LD];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  // consecutive workgroups (one XCD) share the weights of a column tile
  uint32_t tile_n, tile_m;
  p.div_tiles_n.divmod(xcd_remap(blockIdx.x, gridDim.x), tile_n, tile_m);   // divided by the row tiles
  const int n0 = static_cast<int>(tile_n) * 16, m0 = static_cast<int>(tile_m) * 16;
  const bool with_low = LOW && p.a_low;
  const int nk = (p.K + PIECE - 1) / PIECE, pieces = with_low ? 2 * nk : nk;   // those of a, and then those of its low part
  const int row16 = lane & 15, quarter = lane >> 4;

  const uint32_t skip = static_cast<uint32_t>(n0) * static_cast<uint32_t>(p.K) * EB;
  const __amdgpu_buffer_rsrc_t rsrc_b = make_rsrc(static_cast<const unsigned char*>(p.b) + skip, p.b_bytes - skip);
  const uint32_t a_off = (static_cast<uint32_t>(row16) * static_cast<uint32_t>(p.lda) + quarter * E) * EB;
  const uint32_t b_off = (static_cast<uint32_t>(row16) * static_cast<uint32_t>(p.K) + quarter * E) * EB;
  f32x4_t acc = {0.f, 0.f, 0.f, 0.f};

  uint4_t fa[2][U], fb[2][U];
  auto request = [&](int piece, int set) LINEAR_INLINE {
    const bool low = with_low && piece >= nk;
    const __amdgpu_buffer_rsrc_t rsrc_a = rows_from<T>(low ? p.a_low : p.a, p.lda, m0, min(16, p.M - m0), p.K);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = (low ? piece - nk : piece) * PIECE + u * (4 * E);
      const uint32_t behind = k + quarter * E >= p.K ? kOutOfRange : 0u, from = static_cast<uint32_t>(k) * EB;
      fb[set][u] = __builtin_amdgcn_raw_buffer_load_b128(rsrc_b, static_cast<int>((b_off + from) | behind), 0, 0);
      fa[set][u] = __builtin_amdgcn_raw_buffer_load_b128(rsrc_a, static_cast<int>((a_off + from) | behind), 0, 0);
    }
  };
  auto multiply = [&](int set) LINEAR_INLINE {
#pragma unroll
    for (int u = 0; u < U; ++u) mma16<T>(fb[set][u], fa[set][u], acc);
  };
  // pieces behind the last one are requested out of range and add zeros: no branch around the loads in flight
  request(wave, 0);
  for (int piece = wave; piece < pieces; piece += 2 * KG) {
    request(piece + KG, 1);
    multiply(0);
    request(piece + 2 * KG, 0);
    multiply(1);
  }

  // acc[e] is column 4 * quarter + e of the tile, token row16; the wavefronts' sums meet in LDS, added in their order
  *reinterpret_cast<float4*>(&red[wave][row16 * LD + quarter * 4]) = make_float4(acc[0], acc[1], acc[2], acc[3]);
  __syncthreads();
  for (int q = tid; q < 64; q += KG * 64) {   // four columns of one token a thread
    const int in_tile = q >> 2, row = m0 + in_tile, c = (q & 3) * 4, col = n0 + c;
    if (row >= p.M || col >= p.N) continue;
    float v[4] = {0.f, 0.f, 0.f, 0.f}, u[4], zg[4], zu[4], o[4], h[4];
#pragma unroll
    for (int g = 0; g < KG; ++g) {
      const float4 s = *reinterpret_cast<const float4*>(&red[g][in_tile * LD + c]);
      v[0] += s.x;
      v[1] += s.y;
      v[2] += s.z;
      v[3] += s.w;
    }
    T* out = static_cast<T*>(p.out) + row * p.ldo + col;
    T* out2 = static_cast<T*>(p.out2) + row * p.ldo2 + col;
    if constexpr (MODE == kLinFwd) {
      if (p.bias) {
        float b[4];
        load_four(p.bias + col, b);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += b[e];
      }
      if (p.out2) store_four(out2, v);
    } else {
      const T* z = static_cast<const T*>(p.z) + row * p.ldz + col;
      if (MODE == kGatedBwd || p.act != kActNone) load_four(z, zg);
      if constexpr (MODE == kGatedBwd) load_four(z + p.N, zu);
    }
    with_activation(p.act, [&](auto act_c) { combine<T, MODE, decltype(act_c)::value, 4>(v, u, zg, zu, o, h); });
    if constexpr (!is_gated(MODE)) {
      if (p.add) {
        float r[4];
        load_four(static_cast<const T*>(p.add) + row * p.ldadd + col, r);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] += r[e];
      }
    }
    store_four(out, o);
    if constexpr (LOW) {
      if (p.low) {
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = rounded_off(o[e]);
        store_four(static_cast<T*>(p.low) + row * p.ldo + col, o);
      }
    }
    if constexpr (MODE == kGatedBwd) {
      store_four(out + p.N, u);
      if (p.out2) store_four(out2, h);
      if constexpr (sizeof(T) == 2) {
        if (p.low) {
          T* low = static_cast<T*>(p.low) + row * p.ldo + col;
#pragma unroll
          for (int e = 0; e < 4; ++e) o[e] = rounded_off(o[e]), u[e] = rounded_off(u[e]);
          store_four(low, o);
          store_four(low + p.N, u);
        }
        if (p.low2) {
#pragma unroll
          for (int e = 0; e < 4; ++e) h[e] = rounded_off(h[e]);
          store_four(static_cast<T*>(p.low2) + row * p.ldo2 + col, h);
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
template <typename T>
constexpr const char* type_name() { return sizeof(T) == 2 ? "bf16," : "f32,"; }
inline std::string mode_name(int mode, bool low) {
  static const char* const names[] = {"fwd,", "dgrad,", "gated_fwd,", "gated_dgrad,"};
  return low ? "dgrad_low," : names[mode];
}
inline double linear_flops(const LinearArgs& a, int mode) { return (mode == kGatedFwd || a.a_low ? 4.0 : 2.0) * a.M * a.N * a.K; }
inline double linear_bytes(const LinearArgs& a, int mode, int eb) {
  const double mn = static_cast<double>(a.M) * a.N, wide = is_gated(mode) ? 2.0 : 1.0;
  double elems = (a.a_low ? 2.0 : 1.0) * a.M * a.K + mn;
  if (a.add) elems += mn;
  if (mode == kLinBwd || mode == kGatedBwd) elems += a.z ? wide * mn : 0.0;
  if (mode == kGatedBwd) elems += mn;
  if (a.out2) elems += mode == kGatedFwd ? 2.0 * mn : mn;
  elems += (a.low ? wide * mn : 0.0) + (a.low2 ? mn : 0.0);
  return elems * eb + a.b_bytes;
}
inline int tiles_over(int n, int tile) { return (n + tile - 1) / tile; }

template <typename T, int MODE, bool LOW, int WM, int WN, int TM, int TN, int NBUF, int PER_CU>
int launch_linear_tile(Context* ctx, LinearArgs& a) {
  constexpr int BM = WM * TM * 32, BN = WN * TN * 32, BN_OUT = MODE == kGatedFwd ? BN / 2 : BN;
  static const std::string name = std::string("linear_tile_kernel<") + type_name<T>() + mode_name(MODE, LOW) + std::to_string(BM) + "x" +
                                  std::to_string(BN) + "," + std::to_string(NBUF) + "buf>";
  a.tiles_m = tiles_over(a.M, BM);
  a.tiles_n = tiles_over(a.N, BN_OUT);
  const int64_t tiles = static_cast<int64_t>(a.tiles_m) * a.tiles_n;
  TCH_CHECK_ARG(tiles <= 0x3fffffff, "linear: grid out of range");
  a.group_rows = a.tiles_n > 8 ? 4 : 0;
  a.div_tiles_n = FastDiv(a.tiles_n);
  a.div_group = FastDiv(static_cast<uint32_t>(a.group_rows > 1 ? a.group_rows * a.tiles_n : 1));
  a.div_rows = FastDiv(a.group_rows > 1 ? a.group_rows : 1);
  // bf16: the workgroups that the chip holds walk the tiles.  fp32 tiles take so long that their number per compute unit is what
  // counts: a workgroup per tile, and who is done makes room (768 x 6216 over 3480: 308 us, walked 404)
  const int64_t most = sizeof(T) == 2 ? 256 * PER_CU : tiles;
  const unsigned grid = static_cast<unsigned>(tiles < most ? tiles : most);
  return launch(ctx, linear_tile_kernel<T, MODE, LOW, WM, WN, TM, TN, NBUF, PER_CU>, dim3(grid), dim3(WM * WN * 64), a, name.c_str(),
                linear_flops(a, MODE), 0, linear_bytes(a, MODE, sizeof(T)));
}

template <typename T, int MODE, bool LOW, int TM, int TN, int KG, int NBUF, int RB>
int launch_linear_split(Context* ctx, LinearArgs& a) {
  constexpr int BM = TM * 32, BN = TN * 32, BN_OUT = MODE == kGatedFwd ? BN / 2 : BN;
  static const std::string name = std::string("linear_split_kernel<") + type_name<T>() + mode_name(MODE, LOW) + std::to_string(BM) + "x" +
                                  std::to_string(BN) + "," + std::to_string(KG) + "way," + std::to_string(RB) + ">";
  a.tiles_m = tiles_over(a.M, BM);
  a.tiles_n = tiles_over(a.N, BN_OUT);
  const int64_t tiles = static_cast<int64_t>(a.tiles_m) * a.tiles_n;
  TCH_CHECK_ARG(tiles <= 0x3fffffff, "linear: grid out of range");
  // the larger operand is the one an XCD should fetch once
  a.group_rows = (MODE == kGatedFwd ? 2.0 : 1.0) * a.N > a.M ? 1 : 0;
  a.div_tiles_n = FastDiv(a.group_rows ? a.tiles_m : a.tiles_n);
  return launch(ctx, linear_split_kernel<T, MODE, LOW, TM, TN, KG, NBUF, RB>, dim3(static_cast<unsigned>(tiles)), dim3(KG * 64), a, name.c_str(),
                linear_flops(a, MODE), 0, linear_bytes(a, MODE, sizeof(T)));
}

template <typename T, int MODE, bool LOW, int KG>
int launch_linear_rows(Context* ctx, LinearArgs& a) {
  static const std::string name = std::string("linear_rows_kernel<") + type_name<T>() + mode_name(MODE, LOW) + "16x16," + std::to_string(KG) + "way>";
  a.tiles_m = tiles_over(a.M, 16);
  a.tiles_n = tiles_over(a.N, 16);
  const int64_t tiles = static_cast<int64_t>(a.tiles_m) * a.tiles_n;
  TCH_CHECK_ARG(tiles <= 0x3fffffff, "linear: grid out of range");
  a.div_tiles_n = FastDiv(static_cast<uint32_t>(a.tiles_m));
  return launch(ctx, linear_rows_kernel<T, MODE, LOW, KG>, dim3(static_cast<unsigned>(tiles)), dim3(KG * 64), a, name.c_str(),
                linear_flops(a, MODE), 0, linear_bytes(a, MODE, sizeof(T)));
}

// Which kernel: the one with the shortest estimate, (rounds of workgroups) x (reduction steps of a wavefront x microseconds a step +
// start and end).  The constants are measured on products of 1-16384 rows, 64-11264 outputs and 256-11104 reduction elements, and
// take the best kernel or one within 10 % of it for nearly all of them: bf16, M x N over K: 1 x 4096 over 4096 7.4 us with 16-row tiles (7.6
// as 32 x 32), 17 x 1024 over 4096 6.7 as 32 x 32 (16-row tiles 9.2, 32 x 64 8.9), 512 x 1024 over 8192 20 as 32 x 64 (27 as 64 x 64),
// 1024 x 1024 over 1024 7.9 as 64 x 64 (8.3 as 128 x 64, 10.2 as 128 x 128), 512 x 4096 over 4096 23 as 128 x 64 (25 as 128 x 128, 29 as
// 64 x 64, 38 as 256 x 128), 512 x 8192 over 8192 73 as 128 x 128 (97 as 128 x 64, 93 as 256 x 128), 4096 x 4096 over 1024 31 as 256 x 256
// (33 as 256 x 128, 37 as 128 x 128).  Gated, 7 rows, 2048 outputs over 8192: 11.8 as 32 x 32 (32 x 64 15.0).  fp32: 8 x 4096 over 8192 27
// with 16-row tiles (40 as 32 x 32), 4096 x 4096 over 1024 247 as 128 x 64 (314 as 64 x 64).  (One run of replayed programs on warm operands.)
enum Kernel : int { kRows16, kSplit32, kSplit32x64, kSplit64, kTile128x64, kTile128, kTile256x128, kTile256, kKernels };
struct KernelCost {
  int bm, bn;      // tile; gated forward: half as many output columns
  int step;        // reduction bytes of a step
  int ways;        // wavefronts that share a tile's steps
  float step_us, full_us;   // a step where there is one workgroup; where there are 256 (16-row tiles: where 16 rows are filled)
  float fixed_us, again_us; // start and end; what a further round costs beyond that
};
template <typename T, bool GATED_FWD>
const KernelCost* kernel_costs() {
  static constexpr KernelCost kBf16[kKernels] = {{GATED_FWD ? 0 : 16, 16, 256, 8, 0.85f, 1.45f, 1.2f, 0.f},
                                                 {32, 32, 128, 4, 0.22f, 0.45f, 0.6f, 0.f},
                                                 {32, 64, 128, 4, 0.4f, 0.75f, 0.6f, 0.f},
                                                 {64, 64, 128, 3, 0.78f, 0.78f, 0.9f, 0.f},
                                                 {128, 64, 128, 1, 0.39f, 0.44f, 2.5f, 0.f},
                                                 {128, 128, 128, 1, 0.5f, 0.58f, 3.5f, 0.f},
                                                 {256, 128, 128, 1, 0.84f, 1.f, 3.2f, 0.f},
                                                 {256, 256, 128, 1, 1.45f, 1.62f, 6.f, 0.f}};
  // (128 x 64: two share a compute unit at half the rate each)
  static constexpr KernelCost kF32[kKernels] = {{GATED_FWD ? 0 : 16, 16, 256, 8, 1.45f, 1.45f, 1.2f, 0.f},
                                                {32, 32, 128, 4, 0.65f, 0.65f, 0.8f, 2.f},
                                                {32, 64, 128, 4, 1.2f, 1.2f, 0.8f, 3.5f},
                                                {64, 64, 64, 4, 1.18f, 1.18f, 1.2f, 3.5f},
                                                {128, 64, 128, 1, 1.f, 1.f, 2.8f, 0.f}};
  return sizeof(T) == 2 ? kBf16 : kF32;
}
template <typename T, bool GATED_FWD>
float kernel_us(int kernel, int M, const LinearArgs& a) {
  const KernelCost& c = kernel_costs<T, GATED_FWD>()[kernel];
  if (!c.bm) return INFINITY;
  const int all_steps = tiles_over(a.K * static_cast<int>(sizeof(T)), c.step) * (a.a_low ? 2 : 1);
  if (kernel == kTile256 && all_steps < 2) return INFINITY;   // (it takes two steps at least)
  const double tiles = static_cast<double>(tiles_over(M, c.bm)) * tiles_over(a.N, GATED_FWD ? c.bn / 2 : c.bn);
  const int steps = tiles_over(all_steps, c.ways);
  const double rounds = kernel < kTile128x64 && tiles > 8 * 256 ? tiles / 256 : ceil(tiles / 256);
  const float load = kernel == kRows16 ? static_cast<float>(min(M, 16)) / 16.f : tiles < 256 ? static_cast<float>(tiles) / 256.f : 1.f;
  const float step_us = c.step_us + load * (c.full_us - c.step_us);
  return static_cast<float>(rounds) * (steps * step_us + c.fixed_us) + static_cast<float>(rounds - 1.0) * c.again_us;
}
template <typename T, bool GATED_FWD>
Kernel choose_kernel(int M, const LinearArgs& a, float* us) {
  Kernel best = kSplit32;
  *us = INFINITY;
  for (int k = 0; k < kKernels; ++k) {
    const float t = kernel_us<T, GATED_FWD>(k, M, a);
    if (t < *us) {
      *us = t;
      best = static_cast<Kernel>(k);
    }
  }
  return best;
}

template <typename T, int MODE, bool LOW>
int launch_linear_kernel(Context* ctx, Kernel kernel, LinearArgs& a) {
  constexpr bool kWide = MODE == kGatedFwd, kBf = sizeof(T) == 2;
  switch (kernel) {
    case kRows16:
      if constexpr (!kWide) return launch_linear_rows<T, MODE, LOW, 8>(ctx, a);
      break;
    case kSplit32: return launch_linear_split<T, MODE, LOW, 1, 1, 4, 3, 128>(ctx, a);
    case kSplit32x64: return launch_linear_split<T, MODE, LOW, 1, 2, 4, 3, 128>(ctx, a);
    case kSplit64:
      if constexpr (kBf) return launch_linear_split<T, MODE, LOW, 2, 2, 3, 3, 128>(ctx, a);
      else return launch_linear_split<T, MODE, LOW, 2, 2, 4, 4, 64>(ctx, a);
    case kTile128x64:
      if constexpr (kBf) return launch_linear_tile<T, MODE, LOW, 4, 1, 1, 2, 4, 1>(ctx, a);
      else return launch_linear_tile<T, MODE, LOW, 4, 1, 1, 2, 2, 2>(ctx, a);
    case kTile128:
      if constexpr (kBf) return launch_linear_tile<T, MODE, LOW, 2, 2, 2, 2, 3, 1>(ctx, a);
      break;
    case kTile256x128:
      if constexpr (kBf) return launch_linear_tile<T, MODE, LOW, 4, 2, 2, 2, 3, 1>(ctx, a);
      break;
    case kTile256:
      if constexpr (kBf) return launch_linear_tile<T, MODE, LOW, 2, 4, 4, 2, 2, 1>(ctx, a);
      break;
    default: break;
  }
  set_error("linear: no kernel");
  return -22;
}

// Large tiles rarely fill their last round.  Where it is estimated to be shorter by more than the estimate is good for, the rows that
// fill whole rounds are one launch and the others a second one, with tiles as small as suit them: bf16 9729 x 3456 over 15184 1128 ->
// 990 us, fp32 1568 x 4096 over 1024 124 -> 103, 768 x 6216 over 3480 297 -> 268.
constexpr float kSecondLaunchUs = 3.f, kWorthwhile = 0.93f;
template <typename T, int MODE, bool LOW = false>
int launch_linear_mode(Context* ctx, LinearArgs& a) {
  constexpr bool kWide = MODE == kGatedFwd;
  float us;
  Kernel kernel = choose_kernel<T, kWide>(a.M, a, &us), rest_kernel = kernel;
  us *= kWorthwhile;
  int rows = a.M;
  for (int k = kTile128x64; k < kKernels; ++k) {
    const KernelCost& c = kernel_costs<T, kWide>()[k];
    if (!c.bm) continue;
    const int64_t tiles_n = tiles_over(a.N, kWide ? c.bn / 2 : c.bn), rounds = tiles_over(a.M, c.bm) * tiles_n / 256;
    const int64_t main_rows = rounds * 256 / tiles_n * c.bm;
    if (main_rows <= 0 || main_rows >= a.M) continue;
    float rest_us;
    const Kernel rest = choose_kernel<T, kWide>(a.M - static_cast<int>(main_rows), a, &rest_us);
    const float both_us = kernel_us<T, kWide>(k, static_cast<int>(main_rows), a) + rest_us + kSecondLaunchUs;
    if (both_us < us) {
      us = both_us;
      kernel = static_cast<Kernel>(k);
      rest_kernel = rest;
      rows = static_cast<int>(main_rows);
    }
  }
  if (rows == a.M) return launch_linear_kernel<T, MODE, LOW>(ctx, kernel, a);
  LinearArgs rest = a;
  auto skip = [&](const void* t, int64_t ld) -> const void* { return t ? static_cast<const T*>(t) + rows * ld : nullptr; };
  rest.M = a.M - rows;
  rest.a = skip(a.a, a.lda);
  rest.a_low = skip(a.a_low, a.lda);
  rest.add = skip(a.add, a.ldadd);
  rest.z = skip(a.z, a.ldz);
  rest.out = const_cast<void*>(skip(a.out, a.ldo));
  rest.out2 = const_cast<void*>(skip(a.out2, a.ldo2));
  rest.low = const_cast<void*>(skip(a.low, a.ldo));
  rest.low2 = const_cast<void*>(skip(a.low2, a.ldo2));
  a.M = rows;
  if (int rc = launch_linear_kernel<T, MODE, LOW>(ctx, kernel, a)) return rc;
  return launch_linear_kernel<T, MODE, LOW>(ctx, rest_kernel, rest);
}

template <typename T>
int launch_linear_typed(Context* ctx, int mode, LinearArgs& a) {
  switch (mode) {
    case kLinFwd: return launch_linear_mode<T, kLinFwd>(ctx, a);
    case kLinBwd:
      // low parts have kernels of their own: with the choice at run time the others are slower (8192 x 4096 over 1024 81 -> 87 us)
      if constexpr (sizeof(T) == 2)
        if (a.a_low || a.low) return launch_linear_mode<T, kLinBwd, true>(ctx, a);
      return launch_linear_mode<T, kLinBwd>(ctx, a);
    case kGatedFwd: return launch_linear_mode<T, kGatedFwd>(ctx, a);
    default: return launch_linear_mode<T, kGatedBwd>(ctx, a);
  }
}

}  // namespace

int launch_linear_bf16(Context* ctx, int mode, LinearArgs& a);   // linear_bf16.hip
int launch_linear_f32(Context* ctx, int mode, LinearArgs& a);    // linear_f32.hip

}  // namespace tch

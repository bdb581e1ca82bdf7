// Linear layers with bias, activation and residual in one launch, gated feed-forward layers, and their data gradients: argument
// checks, and the derivative of an activation as a pass of its own for a gradient that no product of this library ends in.
// The products are in linear_kernels.h.
//
// Reference call sites: the feed-forward halves of the transformer blocks that train/gpt2.py:26 and train/swin_b.py:38 build
// (a projection, an activation, a projection and the residual).
#include "linear_kernels.h"

#include <algorithm>
#include <climits>

#include "context.h"
#include "ops.h"
#include "pack8.h"

namespace tch {
namespace {

// ---------------------------------------------------------------------------
// dz = dy * act'(z), and the gated form (dg, du, and h again on request) from dh and (g | u)
// ---------------------------------------------------------------------------
// Bound by memory: 6 (gated 10, with h 12; with low parts 8 and 14) bytes per element in bf16, a byte less for every kept pre-activation.  A thread has
// kAtOnce chunks on their way at a time.  8192 x 4096 with the low part: 44.5 us, 6.0 TB/s; from 8 bits with column sums 35 us, 4.8 TB/s, gated 8192 x 2 x
// 5632 with h 74, 6.3 TB/s.
struct ActBwdArgs {
  const void* dy;
  const void* z;
  void* dz;
  void* h;
  void* low;   // bf16: what rounding took off dz, laid out like it; may be null
  int64_t lddy, ldz, lddz, ldh;
  uint32_t chunks;    // rows * row_chunks
  int row_chunks, N, act;
  FastDiv div;        // by row_chunks
  // act_bwd_sum_kernel
  float* sums;        // [row blocks][N, gated 2 N]; one row block: dbias itself
  int64_t M, block_rows;
  int lanes_log;      // 2^lanes_log threads of a workgroup share a row
  int add;            // sums is added to
  // pre-activations kept in 8 bits (pack8.h): z is [M][ldz] bytes
  const unsigned char* codes;
  int64_t code_groups;   // of a row
};
constexpr int kAtOnce = 4;
constexpr int kDense = -1;   // z is of the tensors' type; otherwise a Pack8Format

// the pre-activations of a chunk of dy
template <typename T, int FORMAT>
struct ActBwdZ {
  static constexpr int E = Elem<T>::kPerChunk;
  Chunk z;
  __device__ __forceinline__ void request(const ActBwdArgs& p, int64_t row, uint32_t col, int64_t from) {
    z.u = load_streaming_u4(static_cast<const T*>(p.z) + row * p.ldz + from, col);
  }
  __device__ __forceinline__ void get(float* v) const { chunk_to_float<T>(z, v); }
};
template <typename T, int FORMAT>
struct ActBwdKept {
  static constexpr int E = Elem<T>::kPerChunk;
  uint32_t words[E / 4], code;
  __device__ __forceinline__ void request(const ActBwdArgs& p, int64_t row, uint32_t col, int64_t from) {
    const int64_t at = from + static_cast<int64_t>(col) * E;
    const uint32_t* data = reinterpret_cast<const uint32_t*>(static_cast<const unsigned char*>(p.z) + row * p.ldz + at);
    if constexpr (E == 8) {
      const uint2 v = *reinterpret_cast<const uint2*>(data);
      words[0] = v.x, words[1] = v.y;
    } else {
      words[0] = data[0];
    }
    code = p.codes[row * p.code_groups + at / kPackGroup];
  }
  __device__ __forceinline__ void get(float* v) const {
    const float unit = pack8_unit(code);
#pragma unroll
    for (int i = 0; i < E / 4; ++i) unpack8_word<FORMAT>(words[i], unit, v + 4 * i);
  }
};

// The chunks of one place: what is read, and the gradients from it, stored and (unrounded) returned in o and u.
template <typename T, int GATED, int FORMAT, bool STREAM>
struct ActBwdChunks {
  static constexpr int E = Elem<T>::kPerChunk;
  Chunk dy;
  std::conditional_t<FORMAT == kDense, ActBwdZ<T, FORMAT>, ActBwdKept<T, FORMAT>> zg, zu;
  __device__ __forceinline__ void request(const ActBwdArgs& p, int64_t row, uint32_t col) {
    const T* from = static_cast<const T*>(p.dy) + row * p.lddy;
    dy.u = FORMAT == kDense || STREAM ? load_streaming_u4(from, col) : reinterpret_cast<const uint4*>(from)[col];
    zg.request(p, row, col, 0);
    if (GATED) zu.request(p, row, col, p.N);
  }
  template <int ACT>
  __device__ __forceinline__ void finish(const ActBwdArgs& p, int64_t row, uint32_t col, float* o, float* u) {
    float v[E], fg[E], fu[E], h[E];
    chunk_to_float<T>(dy, v);
    zg.get(fg);
    if (GATED) zu.get(fu);
    combine<T, GATED ? kGatedBwd : kLinBwd, ACT, E>(v, u, fg, fu, o, h);
    T* dz = static_cast<T*>(p.dz) + row * p.lddz;
    store_u4<STREAM>(dz, col, float_to_chunk<T>(o).u);
    if (GATED) {
      store_u4<STREAM>(dz + p.N, col, float_to_chunk<T>(u).u);
      if (p.h) store_u4<STREAM>(static_cast<T*>(p.h) + row * p.ldh, col, float_to_chunk<T>(h).u);
    } else if (FORMAT != kDense && p.h) {
#pragma unroll
      for (int e = 0; e < E; ++e) h[e] = act_value<T, ACT>(fg[e]);
      store_u4<STREAM>(static_cast<T*>(p.h) + row * p.ldh, col, float_to_chunk<T>(h).u);
    }
    if constexpr (sizeof(T) == 2) {
      if (p.low) {
        T* low = static_cast<T*>(p.low) + row * p.lddz;
        float o_low[E], u_low[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
          o_low[e] = rounded_off(o[e]);
          if (GATED) u_low[e] = rounded_off(u[e]);
        }
        reinterpret_cast<uint4*>(low)[col] = float_to_chunk<T>(o_low).u;
        if (GATED) reinterpret_cast<uint4*>(low + p.N)[col] = float_to_chunk<T>(u_low).u;
      }
    }
  }
};

template <typename T, int GATED, int FORMAT, bool STREAM>
__global__ __launch_bounds__(256) void act_bwd_kernel(ActBwdArgs p) {
  constexpr int E = Elem<T>::kPerChunk;
  with_activation(p.act, [&](auto act_c) {
    constexpr int ACT = decltype(act_c)::value;
    const uint64_t stride = static_cast<uint64_t>(gridDim.x) * (256 * kAtOnce);
    for (uint64_t base = static_cast<uint64_t>(blockIdx.x) * (256 * kAtOnce) + threadIdx.x; base < p.chunks; base += stride) {
      ActBwdChunks<T, GATED, FORMAT, STREAM> c[kAtOnce];
      uint32_t row[kAtOnce], col[kAtOnce];
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const uint64_t q = base + 256 * i;
        if (q >= p.chunks) break;
        p.div.divmod(static_cast<uint32_t>(q), row[i], col[i]);
        c[i].request(p, row[i], col[i]);
      }
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        if (base + 256 * i >= p.chunks) break;
        float o[E], u[E];
        c[i].template finish<ACT>(p, row[i], col[i], o, u);
      }
    }
  });
}

// The same with the column sums of the unrounded gradients, which are the bias gradient: added up from their rounded parts they would be as far off
// as the parts (8192 rows: 2.5e-6 of the result; this way 1.1e-7).  A workgroup has a block of rows and 2^lanes_log chunks of columns; a thread walks down the
// rows of its chunk, the threads of a column meet in LDS in their order, and the row blocks' sums are added up by a second launch.
template <typename T, int GATED, int FORMAT, bool STREAM>
__global__ __launch_bounds__(256) void act_bwd_sum_kernel(ActBwdArgs p) {
  constexpr int E = Elem<T>::kPerChunk, PARTS = GATED ? 2 : 1;
  __shared__ float meet[PARTS][256 * E];
  const int lanes = 1 << p.lanes_log, lane = threadIdx.x & (lanes - 1), line = threadIdx.x >> p.lanes_log, lines = 256 >> p.lanes_log;
  const int col = blockIdx.x * lanes + lane;
  const int64_t row0 = blockIdx.y * p.block_rows, behind = min(row0 + p.block_rows, p.M);
  float sum[PARTS][E];
#pragma unroll
  for (int e = 0; e < E; ++e) sum[0][e] = sum[PARTS - 1][e] = 0.f;
  with_activation(p.act, [&](auto act_c) {
    constexpr int ACT = decltype(act_c)::value;
    if (col < p.row_chunks)
      for (int64_t base = row0 + line; base < behind; base += kAtOnce * lines) {
        ActBwdChunks<T, GATED, FORMAT, STREAM> c[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i)
          if (base + i * lines < behind) c[i].request(p, base + i * lines, col);
#pragma unroll
        for (int i = 0; i < kAtOnce; ++i) {
          if (base + i * lines >= behind) break;
          float o[E], u[E];
          c[i].template finish<ACT>(p, base + i * lines, col, o, u);
#pragma unroll
          for (int e = 0; e < E; ++e) {
            sum[0][e] += o[e];
            if (GATED) sum[PARTS - 1][e] += u[e];
          }
        }
      }
  });
  // [line][column] of the workgroup: thread t adds up columns t, t + 256, ...
#pragma unroll
  for (int part = 0; part < PARTS; ++part)
#pragma unroll
    for (int e = 0; e < E; ++e) meet[part][(line * lanes + lane) * E + e] = sum[part][e];
  __syncthreads();
  const int cols = lanes * E, first = blockIdx.x * cols;
#pragma unroll
  for (int part = 0; part < PARTS; ++part)
    for (int c = threadIdx.x; c < cols && first + c < p.N; c += 256) {
      float s = 0.f;
      for (int l = 0; l < lines; ++l) s += meet[part][l * cols + c];
      float* to = p.sums + blockIdx.y * static_cast<int64_t>(PARTS * p.N) + part * p.N + first + c;
      *to = p.add ? *to + s : s;
    }
}

// dbias (+)= the sum of the row blocks' sums: 32 columns a workgroup, eight threads a column, in a fixed order
struct BiasSumArgs {
  const float* sums;
  float* out;
  int blocks, cols, add;
};
__global__ __launch_bounds__(256) void act_bwd_bias_kernel(BiasSumArgs p) {
  __shared__ double meet[8][32];
  const int lane = threadIdx.x & 31, line = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
  double s = 0.0;
  if (col < p.cols) {
#pragma unroll 8
    for (int b = line; b < p.blocks; b += 8) s += p.sums[static_cast<int64_t>(b) * p.cols + col];
  }
  meet[line][lane] = s;
  __syncthreads();
  if (line != 0 || col >= p.cols) return;
#pragma unroll
  for (int l = 1; l < 8; ++l) s += meet[l][lane];
  p.out[col] = p.add ? static_cast<float>(p.out[col] + s) : static_cast<float>(s);
}

// How the rows of a derivative pass with column sums are cut: enough workgroups for the chip, kAtOnce rows a thread at least.  `split`: there is a
// workspace for the row blocks' sums; without it a workgroup has all rows, of one 128-byte line's columns.
struct RowBlocks {
  int lanes_log, col_blocks, blocks;
  int64_t rows;
};
// (8192 x 4096 with its low part and both launches: 49 us, 44.5 without the sums; 53 with 1024 workgroups, 61 with 1024 of 64 chunks wide.  1023 x 2 x 2736
// gated 14.7, 10.6 without.)
constexpr int kSumGroups = 4096, kMaxRowBlocks = 1024, kSumLanesLog = 5;
RowBlocks row_blocks(int64_t M, int row_chunks, bool split) {
  RowBlocks r{split ? kSumLanesLog : 3, 0, 1, M};
  while (r.lanes_log > 0 && (1 << (r.lanes_log - 1)) >= row_chunks) --r.lanes_log;
  r.col_blocks = (row_chunks + (1 << r.lanes_log) - 1) >> r.lanes_log;
  if (!split) return r;
  const int64_t lines = 256 >> r.lanes_log, want = std::min(std::max(kSumGroups / r.col_blocks, 1), kMaxRowBlocks);
  const int64_t each = std::max((M + want - 1) / want, kAtOnce * lines);
  r.rows = (each + lines - 1) / lines * lines;
  r.blocks = static_cast<int>((M + r.rows - 1) / r.rows);
  return r;
}

// a tensor [M][width] with rows ld elements apart: aligned for 16-byte accesses, and within reach of a tile's 32-bit offsets
bool rows_fit(const void* t, int64_t ld, int64_t width, int eb) {
  return !t || (ld >= width && ld % (16 / eb) == 0 && (reinterpret_cast<uintptr_t>(t) & 15) == 0 && ld * eb < (1ll << 31) / 512);
}

int check_common(const char* what, int dtype, int64_t M, int64_t K, int64_t N, int act) {
  const std::string name(what);
  TCH_CHECK_ARG(dtype == kBF16 || dtype == kF32, name + ": dtype must be f32(0) or bf16(1)");
  const int E = dtype == kBF16 ? 8 : 4;
  TCH_CHECK_ARG(M >= 0 && M <= INT_MAX - 1024 && K > 0 && N > 0, name + ": bad shape");
  TCH_CHECK_ARG(K % E == 0 && N % E == 0, name + ": the layer's sizes must be multiples of a 16-byte chunk");
  TCH_CHECK_ARG(act >= 0 && act < kActCount, name + ": unknown activation");
  return 0;
}

int linear_launch(Context* ctx, const char* what, int dtype, int mode, LinearArgs& a, int64_t M, int64_t K, int64_t N) {
  const std::string name(what);
  if (int rc = check_common(what, dtype, M, K, N, a.act)) return rc;
  if (M == 0) return 0;
  const int eb = dtype == kBF16 ? 2 : 4;
  const int64_t wide = is_gated(mode) ? 2 : 1;
  const int64_t weight_rows = mode == kGatedFwd ? 2 * N : N;
  TCH_CHECK_ARG(a.a && a.b && a.out, name + ": null tensor");
  TCH_CHECK_ARG(weight_rows * K * eb < (1ll << 31) && K * eb < (1ll << 31) / 512, name + ": the weights exceed the 2 GiB reach of a buffer offset");
  TCH_CHECK_ARG((reinterpret_cast<uintptr_t>(a.b) & 15) == 0 && (reinterpret_cast<uintptr_t>(a.bias) & 15) == 0,
                name + ": weights and bias must start on a 16-byte boundary");
  TCH_CHECK_ARG(rows_fit(a.a, a.lda, K, eb) && rows_fit(a.a_low, a.lda, K, eb) && rows_fit(a.out, a.ldo, mode == kGatedBwd ? 2 * N : N, eb) && rows_fit(a.add, a.ldadd, N, eb) &&
                    rows_fit(a.z, a.ldz, wide * N, eb) && rows_fit(a.out2, a.ldo2, mode == kGatedFwd ? 2 * N : N, eb) &&
                    rows_fit(a.low, a.ldo, wide * N, eb) && rows_fit(a.low2, a.ldo2, N, eb),
                name + ": rows must start on 16-byte boundaries, not overlap, and be less than 4 MiB apart");
  auto rows_of = [&](const void* t, int64_t ld, int64_t width) { return Span{t, ld * eb, width * eb, M}; };
  const Span in[5] = {rows_of(a.a, a.lda, K), rows_of(a.add, a.ldadd, N), rows_of(a.z, a.ldz, wide * N), {a.b, K * eb, K * eb, weight_rows},
                      rows_of(a.a_low, a.lda, K)};
  const Span out[4] = {rows_of(a.out, a.ldo, mode == kGatedBwd ? 2 * N : N), rows_of(a.out2, a.ldo2, mode == kGatedFwd ? 2 * N : N),
                       rows_of(a.low, a.ldo, wide * N), rows_of(a.low2, a.ldo2, N)};
  const Span bias{a.bias, weight_rows * 4, weight_rows * 4, 1};
  for (int o = 0; o < 4; ++o) {
    bool ok = apart(out[o], bias);
    for (int i = 0; i < 5; ++i) ok = ok && apart(out[o], in[i], o == 0 && (i == 1 || i == 2));
    for (int i = 0; i < o; ++i) ok = ok && apart(out[o], out[i]);
    TCH_CHECK_ARG(ok, name + ": an output overlaps another tensor (it may be the residual or the pre-activations themselves)");
  }
  a.M = static_cast<int>(M);
  a.N = static_cast<int>(N);
  a.K = static_cast<int>(K);
  a.b_bytes = static_cast<uint32_t>(weight_rows * K * eb);
  return dtype == kBF16 ? launch_linear_bf16(ctx, mode, a) : launch_linear_f32(ctx, mode, a);
}

// a derivative pass, with (SUMS) or without the column sums
template <bool SUMS, typename T, int GATED, int FORMAT>
int launch_act_bwd_of(Context* ctx, dim3 grid, const ActBwdArgs& a, double bytes) {
  static const char* const names[2][2][2][3] = {
      {{{"act_bwd_kernel<f32>", "act_bwd_kernel<f32,int8>", "act_bwd_kernel<f32,e4m3>"},
        {"act_bwd_kernel<f32,gated>", "act_bwd_kernel<f32,gated,int8>", "act_bwd_kernel<f32,gated,e4m3>"}},
       {{"act_bwd_kernel<bf16>", "act_bwd_kernel<bf16,int8>", "act_bwd_kernel<bf16,e4m3>"},
        {"act_bwd_kernel<bf16,gated>", "act_bwd_kernel<bf16,gated,int8>", "act_bwd_kernel<bf16,gated,e4m3>"}}},
      {{{"act_bwd_sum_kernel<f32>", "act_bwd_sum_kernel<f32,int8>", "act_bwd_sum_kernel<f32,e4m3>"},
        {"act_bwd_sum_kernel<f32,gated>", "act_bwd_sum_kernel<f32,gated,int8>", "act_bwd_sum_kernel<f32,gated,e4m3>"}},
       {{"act_bwd_sum_kernel<bf16>", "act_bwd_sum_kernel<bf16,int8>", "act_bwd_sum_kernel<bf16,e4m3>"},
        {"act_bwd_sum_kernel<bf16,gated>", "act_bwd_sum_kernel<bf16,gated,int8>", "act_bwd_sum_kernel<bf16,gated,e4m3>"}}}};
  const char* name = names[SUMS][sizeof(T) == 2][GATED][FORMAT + 1];
  auto of = [&](auto stream_c) {
    constexpr bool STREAM = decltype(stream_c)::value;
    if constexpr (SUMS)
      return launch(ctx, act_bwd_sum_kernel<T, GATED, FORMAT, STREAM>, grid, dim3(256), a, name, bytes, 1);
    else
      return launch(ctx, act_bwd_kernel<T, GATED, FORMAT, STREAM>, grid, dim3(256), a, name, bytes, 1);
  };
  if constexpr (FORMAT != kDense)
    if (bytes > kStreamBytes) return of(std::true_type{});   // (8192 x 2 x 5632 in bf16 with h: 74 us, 82 without)
  return of(std::false_type{});
}
template <bool SUMS, typename T, int GATED>
int launch_act_bwd_format(Context* ctx, int format, dim3 grid, const ActBwdArgs& a, double bytes) {
  if (format == kPackInt8) return launch_act_bwd_of<SUMS, T, GATED, kPackInt8>(ctx, grid, a, bytes);
  if (format == kPackE4m3) return launch_act_bwd_of<SUMS, T, GATED, kPackE4m3>(ctx, grid, a, bytes);
  return launch_act_bwd_of<SUMS, T, GATED, kDense>(ctx, grid, a, bytes);
}
template <bool SUMS>
int launch_act_bwd(Context* ctx, int dtype, int gated, int format, dim3 grid, const ActBwdArgs& a, double bytes) {
  if (dtype == kBF16)
    return gated ? launch_act_bwd_format<SUMS, bf16, 1>(ctx, format, grid, a, bytes) : launch_act_bwd_format<SUMS, bf16, 0>(ctx, format, grid, a, bytes);
  return gated ? launch_act_bwd_format<SUMS, float, 1>(ctx, format, grid, a, bytes) : launch_act_bwd_format<SUMS, float, 0>(ctx, format, grid, a, bytes);
}

}  // namespace

int linear_fwd(Context* ctx, int dtype, const Rows& x, const void* w, const Rows& y, const float* bias, int act, const Rows& residual,
               const Rows& pre, int64_t M, int64_t K, int64_t N) {
  LinearArgs a{};
  a.a = x.ptr, a.lda = x.ld;
  a.b = w;
  a.bias = bias;
  a.add = residual.ptr, a.ldadd = residual.ld;
  a.out = y.ptr, a.ldo = y.ld;
  a.out2 = pre.ptr, a.ldo2 = pre.ld;
  a.act = act;
  return linear_launch(ctx, "linear_fwd", dtype, kLinFwd, a, M, K, N);
}

int linear_dgrad(Context* ctx, int dtype, const Rows& dy, const void* dy_low, const void* wt, const Rows& dx, void* dx_low, int act,
                 const Rows& pre, const Rows& residual, int64_t M, int64_t K, int64_t N) {
  TCH_CHECK_ARG(act == kActNone || pre.ptr || M == 0, "linear_dgrad: an activation's derivative needs its pre-activations");
  TCH_CHECK_ARG(dtype == kBF16 || (!dy_low && !dx_low), "linear_dgrad: fp32 gradients are not rounded: there is no low part");
  LinearArgs a{};
  a.a = dy.ptr, a.lda = dy.ld;
  a.a_low = dy_low;
  a.b = wt;
  a.add = residual.ptr, a.ldadd = residual.ld;
  a.z = act == kActNone ? nullptr : pre.ptr, a.ldz = pre.ld;
  a.out = dx.ptr, a.ldo = dx.ld;
  a.low = dx_low;
  a.act = act;
  return linear_launch(ctx, "linear_dgrad", dtype, kLinBwd, a, M, K, N);
}

int gated_linear_fwd(Context* ctx, int dtype, const Rows& x, const void* w, const Rows& h, const float* bias, int act, const Rows& pre, int64_t M,
                     int64_t K, int64_t F) {
  LinearArgs a{};
  a.a = x.ptr, a.lda = x.ld;
  a.b = w;
  a.bias = bias;
  a.out = h.ptr, a.ldo = h.ld;
  a.out2 = pre.ptr, a.ldo2 = pre.ld;
  a.act = act;
  return linear_launch(ctx, "gated_linear_fwd", dtype, kGatedFwd, a, M, K, F);
}

int linear_dgrad_gated(Context* ctx, int dtype, const Rows& dy, const void* wt, const Rows& pre, const Rows& dpre, void* dpre_low, const Rows& h,
                       void* h_low, int act, int64_t M, int64_t K, int64_t F) {
  TCH_CHECK_ARG(pre.ptr || M == 0, "linear_dgrad_gated: null tensor");
  TCH_CHECK_ARG(dtype == kBF16 || (!dpre_low && !h_low), "linear_dgrad_gated: fp32 gradients are not rounded: there is no low part");
  TCH_CHECK_ARG(h.ptr || !h_low, "linear_dgrad_gated: the low part of h comes with h");
  LinearArgs a{};
  a.a = dy.ptr, a.lda = dy.ld;
  a.b = wt;
  a.z = pre.ptr, a.ldz = pre.ld;
  a.out = dpre.ptr, a.ldo = dpre.ld;
  a.out2 = h.ptr, a.ldo2 = h.ld;
  a.low = dpre_low;
  a.low2 = h_low;
  a.act = act;
  return linear_launch(ctx, "linear_dgrad_gated", dtype, kGatedBwd, a, M, K, F);
}

int64_t act_bwd_workspace_bytes(int dtype, int64_t M, int64_t N, int gated) {
  if ((dtype != kBF16 && dtype != kF32) || M <= 0 || N <= 0 || M > INT_MAX || N > INT_MAX) return 0;
  const int E = dtype == kBF16 ? 8 : 4;
  if (N % E != 0) return 0;   // no layer: the call is refused
  const RowBlocks r = row_blocks(M, static_cast<int>(N / E), true);
  return r.blocks > 1 ? r.blocks * N * (gated ? 2 : 1) * 4 : 0;
}

namespace {

// pre: [M][N, gated 2 N] of the tensors' type, or kept in 8 bits (format >= 0: pre.ptr the numbers, dense, and `codes`)
int act_bwd_launch(Context* ctx, int dtype, const Rows& dy, const Rows& pre, const void* codes, int format, const Rows& dz, void* dz_low, const Rows& h,
                   int gated, int act, int64_t M, int64_t N, float* dbias, int accumulate, void* workspace, int64_t workspace_bytes) {
  if (int rc = check_common("act_bwd", dtype, M, 16, N, act)) return rc;
  TCH_CHECK_ARG(dtype == kBF16 || !dz_low, "act_bwd: fp32 gradients are not rounded: there is no low part");
  const bool kept = format != kDense;
  const int64_t wide = gated ? 2 : 1;
  if (M == 0) return dbias && !accumulate ? fill_zero(ctx, dbias, wide * N * 4) : 0;
  const int eb = dtype == kBF16 ? 2 : 4;
  TCH_CHECK_ARG(dy.ptr && pre.ptr && dz.ptr, "act_bwd: null tensor");
  TCH_CHECK_ARG(!kept || (codes && (reinterpret_cast<uintptr_t>(pre.ptr) & 15) == 0 && wide * N < (1ll << 31)),
                "act_bwd: kept pre-activations need their scales, and start on a 16-byte boundary");
  TCH_CHECK_ARG(rows_fit(dy.ptr, dy.ld, N, eb) && (kept || rows_fit(pre.ptr, pre.ld, wide * N, eb)) && rows_fit(dz.ptr, dz.ld, wide * N, eb) &&
                    rows_fit(h.ptr, h.ld, N, eb) && rows_fit(dz_low, dz.ld, wide * N, eb),
                "act_bwd: rows must start on 16-byte boundaries, not overlap, and be less than 4 MiB apart");
  TCH_CHECK_ARG(((reinterpret_cast<uintptr_t>(dbias) | reinterpret_cast<uintptr_t>(workspace)) & 3) == 0,
                "act_bwd: dbias and the workspace must start on a 4-byte boundary");
  const int row_chunks = static_cast<int>(N * eb / 16);
  TCH_CHECK_ARG(M * row_chunks < (1ll << 31), "act_bwd: tensor exceeds 2^31 chunks");
  const RowBlocks cut = row_blocks(M, row_chunks, workspace != nullptr);
  const int64_t sums_bytes = dbias && cut.blocks > 1 ? cut.blocks * wide * N * 4 : 0;
  TCH_CHECK_ARG(sums_bytes <= (workspace ? workspace_bytes : 0), "act_bwd: workspace too small");
  const int64_t groups = (wide * N + kPackGroup - 1) / kPackGroup;
  const Span in[3] = {{dy.ptr, dy.ld * eb, N * eb, M},
                      kept ? Span{pre.ptr, wide * N, wide * N, M} : Span{pre.ptr, pre.ld * eb, wide * N * eb, M},
                      {codes, groups, groups, kept ? M : 0}};
  const Span out[5] = {{dz.ptr, dz.ld * eb, wide * N * eb, M}, {h.ptr, h.ld * eb, N * eb, M}, {dz_low, dz.ld * eb, wide * N * eb, M},
                       {dbias, wide * N * 4, wide * N * 4, 1}, {workspace, sums_bytes, sums_bytes, sums_bytes ? 1 : 0}};
  for (int o = 0; o < 5; ++o) {
    bool ok = apart(out[o], in[0], o == 0) && apart(out[o], in[1], o == 0 && !kept) && apart(out[o], in[2]);
    for (int i = 0; i < o; ++i) ok = ok && apart(out[o], out[i]);
    TCH_CHECK_ARG(ok, "act_bwd: an output overlaps another tensor (the gradient may be the one it is made of, or the pre-activations)");
  }
  ActBwdArgs a{dy.ptr, pre.ptr, dz.ptr, h.ptr, dz_low, dy.ld, pre.ld, dz.ld, h.ld, static_cast<uint32_t>(M * row_chunks), row_chunks, static_cast<int>(N), act,
               FastDiv(static_cast<uint32_t>(row_chunks))};
  if (kept) {
    a.ldz = wide * N;
    a.codes = static_cast<const unsigned char*>(codes), a.code_groups = groups;
  }
  const double z_bytes = wide * (kept ? 33.0 / 32 : eb);
  const double bytes = static_cast<double>(M) * N * (z_bytes + eb * (1.0 + wide + (h.ptr ? 1 : 0) + (dz_low ? wide : 0)));
  if (dbias) {
    const bool split = cut.blocks > 1;
    a.sums = split ? static_cast<float*>(workspace) : dbias;
    a.M = M, a.block_rows = cut.rows;
    a.lanes_log = cut.lanes_log;
    a.add = accumulate && !split;
    const dim3 blocks(static_cast<unsigned>(cut.col_blocks), static_cast<unsigned>(cut.blocks));
    const int rc = launch_act_bwd<true>(ctx, dtype, gated, format, blocks, a, bytes);
    if (rc || !split) return rc;
    const int cols = static_cast<int>(wide * N);
    BiasSumArgs b{a.sums, dbias, cut.blocks, cols, accumulate};
    return launch(ctx, act_bwd_bias_kernel, dim3(static_cast<unsigned>((cols + 31) / 32)), dim3(256), b, "act_bwd_bias_kernel", 4.0 * cut.blocks * cols, 1);
  }
  const int64_t workgroups = (M * row_chunks + 256 * kAtOnce - 1) / (256 * kAtOnce);
  const dim3 grid(static_cast<unsigned>(workgroups < (1 << 20) ? workgroups : (1 << 20)));
  return launch_act_bwd<false>(ctx, dtype, gated, format, grid, a, bytes);
}

}  // namespace

int act_bwd(Context* ctx, int dtype, const Rows& dy, const Rows& pre, const Rows& dz, void* dz_low, const Rows& h, int gated, int act, int64_t M,
            int64_t N, float* dbias, int accumulate, void* workspace, int64_t workspace_bytes) {
  return act_bwd_launch(ctx, dtype, dy, pre, nullptr, kDense, dz, dz_low, h, gated, act, M, N, dbias, accumulate, workspace, workspace_bytes);
}

int act_bwd_packed(Context* ctx, int dtype, const Rows& dy, const void* data, const void* codes, int format, const Rows& dz, void* dz_low, const Rows& h,
                   int gated, int act, int64_t M, int64_t N, float* dbias, int accumulate, void* workspace, int64_t workspace_bytes) {
  TCH_CHECK_ARG(format >= 0 && format < kPackFormats, "act_bwd_packed: unknown 8-bit format");
  return act_bwd_launch(ctx, dtype, dy, {const_cast<void*>(data), 0}, codes, format, dz, dz_low, h, gated, act, M, N, dbias, accumulate, workspace,
                        workspace_bytes);
}

}  // namespace tch

// The global norm of many gradient tensors, and clipping by it:
//   norm = sqrt(sum g^2),   coef = min(1, max_norm / (norm + 1e-6)),   g <- coef g
//
// The tensors are cut into pieces of at most kPieceElems elements, listed in a table in device memory.  Squares are added in fp64
// (nothing overflows: the largest fp32 squared is 1e77) by a fixed assignment of pieces to workgroups, and the workgroups' sums in a
// fixed order, so that a norm is the same bit for bit every run.  Bound by memory: a clip reads everything twice and writes it
// once; the second reading goes from the last piece to the first, so that what the 256 MB cache still holds is read from there.
// 124 million fp32 gradients: norm 91 us (5.5 TB/s), clip 162 (6.1 TB/s).  A few short tensors: two launches of 3-4 us.
#include "context.h"
#include "kernels.h"
#include "ops.h"

namespace tch {
namespace {

constexpr int kPieceElems = 8192;
constexpr int kMaxGroups = 2048;

struct Piece {   // one row of the table
  const void* src;
  void* dst;
  int32_t n;        // elements, 1 .. kPieceElems
  int32_t src_bf16, dst_bf16;
  int32_t aligned;  // both sides start on the boundary of four elements
};
static_assert(sizeof(Piece) == 32, "the table's rows are four 64-bit words");

struct NormArgs {
  const Piece* pieces;
  double* partial;   // one per workgroup
  int64_t count;
};

__device__ inline double wave_sum_f64(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}
// the sum over the workgroup, in every thread; the wavefronts' sums are added in their order
__device__ inline double group_sum_f64(double v, double* scratch) {
  v = wave_sum_f64(v);
  if ((threadIdx.x & 63) == 0) scratch[threadIdx.x >> 6] = v;
  __syncthreads();
  return ((scratch[0] + scratch[1]) + scratch[2]) + scratch[3];
}

// LAST: nobody reads it again
template <bool LAST, typename T>
__device__ inline void load4(const T* p, int64_t i, float* v) {
  if constexpr (sizeof(T) == 4) {
    const float4 f = LAST ? load_streaming_f4(p + 4 * i) : reinterpret_cast<const float4*>(p)[i];
    v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
  } else {
    const uint2 u = reinterpret_cast<const uint2*>(p)[i];
    v[0] = __uint_as_float(u.x << 16), v[1] = __uint_as_float(u.x & 0xffff0000u);
    v[2] = __uint_as_float(u.y << 16), v[3] = __uint_as_float(u.y & 0xffff0000u);
  }
}

constexpr int kVisits = kPieceElems / 1024;   // groups of four elements per thread

template <typename T>
__device__ inline double piece_squares(const Piece& piece) {
  const T* src = static_cast<const T*>(piece.src);
  double s = 0.0;
  auto add = [&](float v) { s = fma(static_cast<double>(v), static_cast<double>(v), s); };
  const int quads = piece.aligned ? piece.n >> 2 : 0;
  float v[kVisits][4];
#pragma unroll
  for (int i = 0; i < kVisits; ++i) {
    const int q = i * 256 + threadIdx.x;
    if (q < quads) load4<false>(src, q, v[i]);
  }
#pragma unroll
  for (int i = 0; i < kVisits; ++i) {
    if (i * 256 + static_cast<int>(threadIdx.x) < quads)
#pragma unroll
      for (int e = 0; e < 4; ++e) add(v[i][e]);
  }
  for (int i = quads * 4 + threadIdx.x; i < piece.n; i += 256) add(Elem<T>::load(src + i));
  return s;
}

__global__ __launch_bounds__(256) void grad_norm_kernel(NormArgs p) {
  __shared__ double scratch[4];
  double s = 0.0;
  Piece piece = p.pieces[blockIdx.x];
  for (int64_t i = blockIdx.x; i < p.count; i += gridDim.x) {
    const Piece next = p.pieces[min(i + gridDim.x, p.count - 1)];   // on its way while this one is read
    s += piece.src_bf16 ? piece_squares<bf16>(piece) : piece_squares<float>(piece);
    piece = next;
  }
  s = group_sum_f64(s, scratch);
  if (threadIdx.x == 0) p.partial[blockIdx.x] = s;
}

struct ClipArgs {
  const Piece* pieces;
  const double* partial;
  int64_t count;
  int groups;        // partial sums
  float* norm;
  float* coef;       // may be null
  double max_norm;   // negative: no clipping (coef 1)
};

// Every workgroup adds the partial sums itself, in the same order.
__device__ inline float clip_coefficient(const ClipArgs& p, double* scratch) {
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < kMaxGroups / 256; ++i) {
    const int at = i * 256 + threadIdx.x;
    s += at < p.groups ? p.partial[at] : 0.0;
  }
  const double norm = sqrt(group_sum_f64(s, scratch));
  const double c = p.max_norm / (norm + 1e-6);
  const float coef = p.max_norm < 0.0 || c > 1.0 ? 1.f : static_cast<float>(c);   // a NaN stays one
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    *p.norm = static_cast<float>(norm);
    if (p.coef) *p.coef = coef;
  }
  return coef;
}

__global__ __launch_bounds__(256) void grad_norm_finish_kernel(ClipArgs p) {
  __shared__ double scratch[4];
  clip_coefficient(p, scratch);
}

template <typename S, typename D>
__device__ inline void scale_piece(const Piece& piece, float coef) {
  const S* src = static_cast<const S*>(piece.src);
  D* dst = static_cast<D*>(piece.dst);
  const int quads = piece.aligned ? piece.n >> 2 : 0;
  float v[kVisits][4];
#pragma unroll
  for (int i = 0; i < kVisits; ++i) {
    const int q = i * 256 + threadIdx.x;
    if (q < quads) load4<true>(src, q, v[i]);
  }
#pragma unroll
  for (int i = 0; i < kVisits; ++i) {
    const int q = i * 256 + threadIdx.x;
    if (q >= quads) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[i][e] *= coef;
    if constexpr (sizeof(D) == 4) {
      store_streaming_f4(dst + q * 4, make_float4(v[i][0], v[i][1], v[i][2], v[i][3]));
    } else {
      uint2 w;
      w.x = float_to_bf16_bits(v[i][0]) | (static_cast<uint32_t>(float_to_bf16_bits(v[i][1])) << 16);
      w.y = float_to_bf16_bits(v[i][2]) | (static_cast<uint32_t>(float_to_bf16_bits(v[i][3])) << 16);
      reinterpret_cast<uint2*>(dst)[q] = w;
    }
  }
  for (int i = quads * 4 + threadIdx.x; i < piece.n; i += 256) Elem<D>::store(dst + i, Elem<S>::load(src + i) * coef);
}

__global__ __launch_bounds__(256) void grad_clip_kernel(ClipArgs p) {
  __shared__ double scratch[4];
  Piece piece = p.pieces[p.count - 1 - blockIdx.x];
  const float coef = clip_coefficient(p, scratch);
  for (int64_t i = p.count - 1 - blockIdx.x; i >= 0; i -= gridDim.x) {
    const Piece next = p.pieces[max(i - gridDim.x, static_cast<int64_t>(0))];
    if (coef != 1.f || piece.src != piece.dst) {   // (times one, in place: nothing to do)
      if (piece.src_bf16)
        piece.dst_bf16 ? scale_piece<bf16, bf16>(piece, coef) : scale_piece<bf16, float>(piece, coef);
      else
        piece.dst_bf16 ? scale_piece<float, bf16>(piece, coef) : scale_piece<float, float>(piece, coef);
    }
    piece = next;
  }
}

}  // namespace

int64_t grad_table_piece_elems() { return kPieceElems; }
int64_t grad_norm_workspace_bytes(int64_t pieces) {
  return 8 * (pieces < 1 ? 1 : pieces < kMaxGroups ? pieces : kMaxGroups);
}

int grad_norm(Context* ctx, const void* table, int64_t pieces, int64_t bytes_read, int64_t bytes_written, int clip, double max_norm,
              float* norm, float* coef, void* workspace) {
  TCH_CHECK_ARG(pieces >= 0 && (table || pieces == 0) && norm && workspace, "grad_norm: null tensor");
  TCH_CHECK_ARG((reinterpret_cast<uintptr_t>(workspace) & 7) == 0, "grad_norm: the workspace must start on an 8-byte boundary");
  TCH_CHECK_ARG(!clip || max_norm >= 0.0, "grad_norm: max_norm must not be negative");
  const int groups = static_cast<int>(pieces < kMaxGroups ? pieces : kMaxGroups);
  if (groups > 0) {
    NormArgs n{static_cast<const Piece*>(table), static_cast<double*>(workspace), pieces};
    if (int rc = launch(ctx, grad_norm_kernel, dim3(groups), dim3(256), n, "grad_norm_kernel", static_cast<double>(bytes_read), 1)) return rc;
  }
  ClipArgs c{static_cast<const Piece*>(table), static_cast<const double*>(workspace), pieces, groups, norm, coef, max_norm};
  if (!clip || groups == 0) return launch(ctx, grad_norm_finish_kernel, dim3(1), dim3(256), c, "grad_norm_finish_kernel", 8.0 * groups, 1);
  return launch(ctx, grad_clip_kernel, dim3(groups), dim3(256), c, "grad_clip_kernel", static_cast<double>(bytes_read + bytes_written), 1);
}

}  // namespace tch

// Activations in 8 bits for the backward pass (pack8.h): kept, fetched, and kept by the pass that takes an activation of them.
// Bound by memory: an element is 2 or 4 bytes on one side and 1 + 1 / 32 on the other.  In bf16 8192 x 4096 kept with GELU on the way 31 us (5.4 TB/s),
// 8192 x 1024 fetched 6.5, 16384 x 11008 kept 107 (5.1) and fetched 82 (6.7).
//
// Reference call sites: what the backward pass of train/gpt2.py:90 and train/swin_b.py:118 finds of the forward pass, all of it in the types it was computed in.
#include <algorithm>
#include <climits>

#include "context.h"
#include "linear_epilogue.h"
#include "ops.h"
#include "pack8.h"

namespace tch {
namespace {

struct PackArgs {
  const void* x;          // kept: rows ldx apart
  void* h;                // act(x); may be null
  void* out;              // fetched: rows ldx apart
  unsigned char* data;    // [M][C]
  unsigned char* codes;   // [M][groups of 32]
  int64_t ldx, ldh;
  uint64_t total;         // rows * chunks of a row, whole groups
  int C, groups, act;
  FastDiv chunks;
};

// A lane has a 16-byte chunk: eight numbers in bf16, four in fp32, and the four or eight lanes of a group are neighbours (a row has whole groups of
// them; all lanes of a wavefront go round together).  One chunk a lane: with four on their way together 8192 x 4096 in bf16 with GELU takes 33
// us instead of 31, fetching 8192 x 1024 7.4 instead of 6.5, and small tensors leave the chip idle.
template <typename T>
struct At {
  static constexpr int E = Elem<T>::kPerChunk;
  int64_t row;
  int col;
  bool on;
  __device__ __forceinline__ At(const PackArgs& p, uint64_t q) : row(0), col(0), on(false) {
    if (q >= p.total) return;
    uint32_t r, chunk;
    p.chunks.divmod(static_cast<uint32_t>(q), r, chunk);
    row = r;
    col = static_cast<int>(chunk) * E;
    on = col < p.C;
  }
};

template <typename T, int FMT, bool STREAM>
__global__ __launch_bounds__(256) void pack8_kernel(PackArgs p) {
  constexpr int E = Elem<T>::kPerChunk;
  const uint64_t stride = static_cast<uint64_t>(gridDim.x) * 256;
  for (uint64_t base = static_cast<uint64_t>(blockIdx.x) * 256; base < p.total; base += stride) {
    const At<T> at(p, base + threadIdx.x);
    const uint4* from = reinterpret_cast<const uint4*>(static_cast<const T*>(p.x) + at.row * p.ldx + at.col);
    Chunk x = zero_chunk();
    if (at.on) x.u = STREAM ? load_streaming_u4(from, 0) : *from;
    float v[E];
    chunk_to_float<T>(x, v);
    unsigned char* data = p.data + at.row * p.C + at.col;
    uint32_t words[2], code;
    if constexpr (E == 8) {
      code = pack8_lane<FMT>(v, at.on ? 8 : 0, words);
      if (at.on) *reinterpret_cast<uint2*>(data) = make_uint2(words[0], words[1]);
    } else {
      code = pack8_four<FMT>(v, at.on, words);
      if (at.on) *reinterpret_cast<uint32_t*>(data) = words[0];
    }
    if (at.on && threadIdx.x % (kPackGroup / E) == 0) p.codes[at.row * p.groups + at.col / kPackGroup] = static_cast<unsigned char>(code);
    if (p.h)
      with_activation(p.act, [&](auto act_c) {
        constexpr int ACT = decltype(act_c)::value;
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = act_value<T, ACT>(v[e]);
        if (at.on) store_u4<STREAM>(static_cast<T*>(p.h) + at.row * p.ldh + at.col, 0, float_to_chunk<T>(v).u);
      });
  }
}

template <typename T, int FMT, bool STREAM>
__global__ __launch_bounds__(256) void unpack8_kernel(PackArgs p) {
  constexpr int E = Elem<T>::kPerChunk;
  const uint64_t stride = static_cast<uint64_t>(gridDim.x) * 256;
  for (uint64_t q = static_cast<uint64_t>(blockIdx.x) * 256 + threadIdx.x; q < p.total; q += stride) {
    const At<T> at(p, q);
    if (!at.on) continue;
    const unsigned char* data = p.data + at.row * p.C + at.col;
    const float unit = pack8_unit(p.codes[at.row * p.groups + at.col / kPackGroup]);
    float v[E];
    if constexpr (E == 8) {
      const uint2 w = *reinterpret_cast<const uint2*>(data);
      unpack8_word<FMT>(w.x, unit, v);
      unpack8_word<FMT>(w.y, unit, v + 4);
    } else {
      unpack8_word<FMT>(*reinterpret_cast<const uint32_t*>(data), unit, v);
    }
    store_u4<STREAM>(static_cast<T*>(p.out) + at.row * p.ldx + at.col, 0, float_to_chunk<T>(v).u);
  }
}

int bind(const char* what, PackArgs& a, int dtype, void* data, void* codes, int format, int64_t M, int64_t C) {
  const std::string name(what);
  TCH_CHECK_ARG(dtype == kBF16 || dtype == kF32, name + ": dtype must be f32(0) or bf16(1)");
  TCH_CHECK_ARG(format >= 0 && format < kPackFormats, name + ": unknown 8-bit format");
  TCH_CHECK_ARG(M >= 0 && M <= INT_MAX && C > 0 && C < (1 << 30), name + ": bad shape");
  TCH_CHECK_ARG(C % (dtype == kBF16 ? 8 : 4) == 0, name + ": rows must be whole 16-byte chunks");
  if (M == 0) return 0;
  TCH_CHECK_ARG(data && codes, name + ": null tensor");
  TCH_CHECK_ARG((reinterpret_cast<uintptr_t>(data) & 15) == 0, name + ": the kept numbers must start on a 16-byte boundary");
  a.data = static_cast<unsigned char*>(data), a.codes = static_cast<unsigned char*>(codes);
  a.C = static_cast<int>(C);
  a.groups = static_cast<int>((C + kPackGroup - 1) / kPackGroup);
  const int64_t chunks = a.groups * (dtype == kBF16 ? 4ll : 8ll);
  TCH_CHECK_ARG(M * chunks < (1ll << 31), name + ": tensor exceeds 2^31 chunks");
  a.total = static_cast<uint64_t>(M * chunks);
  a.chunks = FastDiv(static_cast<uint32_t>(chunks));
  return 0;
}

// fn(element type, format, whether to stream past the cache, the kernel's name)
template <typename T>
struct Type {
  typedef T type;
};
const char* const kNames[2][2][2] = {{{"pack8_kernel<f32,int8>", "pack8_kernel<f32,e4m3>"}, {"pack8_kernel<bf16,int8>", "pack8_kernel<bf16,e4m3>"}},
                                     {{"unpack8_kernel<f32,int8>", "unpack8_kernel<f32,e4m3>"}, {"unpack8_kernel<bf16,int8>", "unpack8_kernel<bf16,e4m3>"}}};
template <typename F>
int launch_of(int unpack, int dtype, int format, uint64_t total, double bytes, F&& fn) {
  const char* name = kNames[unpack][dtype == kBF16][format];
  const dim3 grid(static_cast<unsigned>(std::min<uint64_t>((total + 255) / 256, 1 << 20)));
  auto streamed = [&](auto t, auto format_c) {
    return bytes > kStreamBytes ? fn(t, format_c, std::true_type{}, grid, name) : fn(t, format_c, std::false_type{}, grid, name);
  };
  auto typed = [&](auto t) {
    return format == kPackInt8 ? streamed(t, std::integral_constant<int, kPackInt8>{}) : streamed(t, std::integral_constant<int, kPackE4m3>{});
  };
  return dtype == kBF16 ? typed(Type<bf16>{}) : typed(Type<float>{});
}

bool rows_ok(const void* t, int64_t ld, int64_t C, int eb) {
  return ld >= C && ld % (16 / eb) == 0 && ld <= (1ll << 31) && (reinterpret_cast<uintptr_t>(t) & 15) == 0;
}

}  // namespace

int pack8(Context* ctx, int dtype, const Rows& x, void* data, void* codes, int format, const Rows& h, int act, int64_t M, int64_t C) {
  PackArgs a{};
  if (int rc = bind("pack8", a, dtype, data, codes, format, M, C)) return rc;
  TCH_CHECK_ARG(act >= 0 && act < kActCount, "pack8: unknown activation");
  if (M == 0) return 0;
  const int eb = dtype == kBF16 ? 2 : 4;
  TCH_CHECK_ARG(x.ptr, "pack8: null tensor");
  TCH_CHECK_ARG(rows_ok(x.ptr, x.ld, C, eb) && (!h.ptr || rows_ok(h.ptr, h.ld, C, eb)), "pack8: rows must start on 16-byte boundaries and not overlap");
  const Span in{x.ptr, x.ld * eb, C * eb, M};
  const Span out[3] = {{h.ptr, h.ld * eb, C * eb, M}, {data, C, C, M}, {codes, a.groups, a.groups, M}};
  TCH_CHECK_ARG(apart(out[0], in, true) && apart(out[1], in) && apart(out[2], in) && apart(out[0], out[1]) && apart(out[0], out[2]) && apart(out[1], out[2]),
                "pack8: an output overlaps another tensor (the activations may be written over what they are taken of)");
  a.x = x.ptr, a.ldx = x.ld;
  a.h = h.ptr, a.ldh = h.ld;
  a.act = h.ptr ? act : kActNone;
  const double bytes = static_cast<double>(M) * C * (eb * (h.ptr ? 2.0 : 1.0) + 33.0 / 32);
  return launch_of(0, dtype, format, a.total, bytes, [&](auto t, auto format_c, auto stream_c, dim3 grid, const char* name) {
    return launch(ctx, pack8_kernel<typename decltype(t)::type, decltype(format_c)::value, decltype(stream_c)::value>, grid, dim3(256), a, name, bytes, 1);
  });
}

int unpack8(Context* ctx, int dtype, const void* data, const void* codes, int format, const Rows& x, int64_t M, int64_t C) {
  PackArgs a{};
  if (int rc = bind("unpack8", a, dtype, const_cast<void*>(data), const_cast<void*>(codes), format, M, C)) return rc;
  if (M == 0) return 0;
  const int eb = dtype == kBF16 ? 2 : 4;
  TCH_CHECK_ARG(x.ptr, "unpack8: null tensor");
  TCH_CHECK_ARG(rows_ok(x.ptr, x.ld, C, eb), "unpack8: rows must start on 16-byte boundaries and not overlap");
  const Span out{x.ptr, x.ld * eb, C * eb, M};
  TCH_CHECK_ARG(apart(out, {data, C, C, M}) && apart(out, {codes, a.groups, a.groups, M}), "unpack8: the output overlaps what is kept");
  a.out = x.ptr, a.ldx = x.ld;
  const double bytes = static_cast<double>(M) * C * (eb + 33.0 / 32);
  return launch_of(1, dtype, format, a.total, bytes, [&](auto t, auto format_c, auto stream_c, dim3 grid, const char* name) {
    return launch(ctx, unpack8_kernel<typename decltype(t)::type, decltype(format_c)::value, decltype(stream_c)::value>, grid, dim3(256), a, name, bytes, 1);
  });
}

}  // namespace tch

// Activations kept in 8 bits: 32 neighbours of a row share a power of two 2^e, e the smallest with which none of them is beyond the
// largest number L of the 8-bit type (127 of int8, 448 of e4m3), and each is kept as the nearest multiple of its step (ties to even):
//   |x - kept| <= 2^e / 2 (int8),   max(2^-4 |x|, 2^-10 2^e) (e4m3),   max |x| > L 2^(e - 1).
// A power of two and at most 8 significant bits: what is fetched is exact in bf16, so that a product of it multiplies what was kept.
// e is held between -117, with which every kept number is normal in fp32 and bf16, and the last value with which L 2^e is finite
// (larger numbers saturate); a byte holds 127 + e.  A group that holds an infinity or a NaN is marked 255 and comes back as NaN.
#pragma once

#include "kernels.h"

namespace tch {

enum Pack8Format : int { kPackInt8 = 0, kPackE4m3 = 1, kPackFormats = 2 };
constexpr int kPackGroup = 32;
constexpr uint32_t kPackNaN = 255;

// the group's byte from the bits of its largest magnitude
template <int FMT>
__device__ __forceinline__ uint32_t pack8_code(uint32_t top) {
  constexpr int kBelow = FMT == kPackInt8 ? 6 : 8;                            // L = 1.98 2^6, 1.75 2^8
  constexpr uint32_t kMost = FMT == kPackInt8 ? 0x7e0000u : 0x600000u;        // L's mantissa
  constexpr int kLast = 254 - kBelow;
  const int code = static_cast<int>(top >> 23) - kBelow + ((top & 0x7fffffu) > kMost ? 1 : 0);
  return top >= 0x7f800000u ? kPackNaN : static_cast<uint32_t>(code < 10 ? 10 : code > kLast ? kLast : code);
}

// four numbers in a word
template <int FMT>
__device__ __forceinline__ uint32_t pack8_word(const float* v, uint32_t code) {
  if (code == kPackNaN) return 0;
  const float unit = __uint_as_float((254u - code) << 23);   // 2^-e
  constexpr float kLargest = FMT == kPackInt8 ? 127.f : 448.f;
  float s[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) s[i] = __builtin_amdgcn_fmed3f(v[i] * unit, -kLargest, kLargest);
  if constexpr (FMT == kPackInt8) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= (static_cast<uint32_t>(static_cast<int>(rintf(s[i]))) & 0xffu) << (8 * i);
    return w;
  } else {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(s[0], s[1], 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(s[2], s[3], w, true));
  }
}

// 2^e; NaN of a group that is marked so
__device__ __forceinline__ float pack8_unit(uint32_t code) { return __uint_as_float(code == kPackNaN ? 0x7fc00000u : code << 23); }

template <int FMT>
__device__ __forceinline__ void unpack8_word(uint32_t w, float unit, float* v) {
  if constexpr (FMT == kPackInt8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = static_cast<float>(static_cast<int>(w << (24 - 8 * i)) >> 24) * unit;
  } else {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
    v[0] = lo[0] * unit, v[1] = lo[1] * unit, v[2] = hi[0] * unit, v[3] = hi[1] * unit;
  }
}

// the largest magnitude's bits over the four lanes (eight neighbours each) of a group
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  v = max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0xb1, 0xf, 0xf, true)));   // the neighbour
  return max(v, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), 0x4e, 0xf, 0xf, true)));   // the other pair
}

// A lane's eight neighbours (`live` of them from the first on are there) as two words; all four lanes of a group are here.
template <int FMT>
__device__ __forceinline__ uint32_t pack8_lane(const float* v, int live, uint32_t* words) {
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < live) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
  const uint32_t code = pack8_code<FMT>(quad_max(top));
  words[0] = pack8_word<FMT>(v, code);
  words[1] = pack8_word<FMT>(v + 4, code);
  return code;
}

// A lane's four neighbours as one word; all eight lanes of a group are here.
template <int FMT>
__device__ __forceinline__ uint32_t pack8_four(const float* v, bool live, uint32_t* word) {
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (live) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
  top = quad_max(top);
  top = max(top, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(top), 0x141, 0xf, 0xf, true)));   // the other quad of eight
  const uint32_t code = pack8_code<FMT>(top);
  *word = pack8_word<FMT>(v, code);
  return code;
}

}  // namespace tch

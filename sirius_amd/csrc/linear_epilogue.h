// Activations of the linear layers and what their kernels do with a product before it is stored.
//
//   kLinFwd    v = x W^T + b (kept in pre on request);         y  = act(v) + residual
//   kLinBwd    v = dy W;                                       dx = v * act'(z) + residual
//   kGatedFwd  g = x Wg^T + bg, u = x Wu^T + bu (pre = g | u); h  = act(g) * u
//   kGatedBwd  v = dy W (the gradient of h), z = g | u;        dg = v * u * act'(g), du = v * act(g), h again on request
//
// Everything here is fp32: products arrive in fp32 and are rounded once, when they are stored.  The activation is taken of the
// unrounded product, not of the rounded copy that is kept in pre: one rounding less in y.
#pragma once

#include <cstdint>

#include "kernels.h"

namespace tch {

// Left to itself the compiler stops inlining where a kernel gets long, and whatever a lambda refers to, accumulators too, is in memory then.
#define LINEAR_INLINE __attribute__((always_inline))

enum LinearMode : int { kLinFwd = 0, kLinBwd = 1, kGatedFwd = 2, kGatedBwd = 3 };
enum Activation : int { kActNone = 0, kActRelu = 1, kActGelu = 2, kActGeluTanh = 3, kActSilu = 4, kActCount = 5 };

constexpr bool is_gated(int mode) { return mode == kGatedFwd || mode == kGatedBwd; }

// T decides how exactly: bf16 results are off by up to 2^-8 of their size when they are stored (2^-16 in two parts), so the hardware's
// exponential and reciprocal (2^-23 each) do; fp32 results take the library's exponential and division.
template <typename T>
__device__ inline float fast_exp(float x) {
  if constexpr (sizeof(T) == 2)
    return __builtin_amdgcn_exp2f(x * 1.4426950408889634f);
  else
    return expf(x);
}
template <typename T>
__device__ inline float reciprocal(float x) {
  if constexpr (sizeof(T) == 2)
    return __builtin_amdgcn_rcpf(x);
  else
    return 1.f / x;
}
template <typename T>
__device__ inline float sigmoid(float x) {
  return reciprocal<T>(1.f + fast_exp<T>(-x));   // x -> -inf: 1 / inf = 0
}

// The normal distribution's integral and density at z.  Left of zero the integral is small and GELU is z times it, so it is its relative error
// that counts: 0.5 erfc(m / sqrt 2) = exp(-m^2 / 2) t Q(t), m = |z|, t = 1 / (1 + a m), Q the polynomial with the smallest relative error; the
// exponential is the density's as well.
// bf16: degree 6, 7.1e-7 (a linear program over 0 <= m <= 13.3).  With the roundings of the exponential's argument the integral is within
// (40 + 1.5 z^2) 2^-24 of its size: 1.1e-6 next to zero, 7.7e-6 at z = -13, behind which it is subnormal.
// fp32: degree 9, 2.7e-9 (an exchange, x = m / sqrt 2 <= 10.5); what rounding takes off z^2 / 2 goes back into the exponential.  Within 12 x 2^-24 of its
// size for z > -13 (4.5e-7 is the largest found); against a call of the library's erfc the epilogue of 1568 x 4096 over 1024 is 20 us shorter.
template <typename T>
__device__ inline void normal_cdf(float z, float& cdf, float& density) {
  if constexpr (sizeof(T) == 2) {
    const float e = __builtin_amdgcn_exp2f(z * z * -0.72134752044448170f);   // log2(e) / 2
    const float t = reciprocal<T>(fmaf(0.362f, fabsf(z), 1.f));
    constexpr float kQ[7] = {0.14450584f, 0.14266214f, 0.13957834f, 0.028423097f, 0.17721444f, -0.18045251f, 0.048069008f};
    float q = kQ[6];
#pragma unroll
    for (int i = 5; i >= 0; --i) q = fmaf(q, t, kQ[i]);
    const float half_erfc = e * t * q;
    cdf = z < 0.f ? half_erfc : 1.f - half_erfc;
    density = 0.3989422804014327f * e;
  } else {
    const float m = fminf(fabsf(z), 20.f);   // (exp(-200) is 0 already; a NaN comes back with the factor z)
    const float h = 0.5f * m, square = h * m, rest = fmaf(h, m, -square);
    float e = expf(-square);
    e = fmaf(-e, rest, e);
    const float t = 1.f / fmaf(0.42f, m * 0.7071067811865476f, 1.f);
    constexpr float kQ[10] = {0.2369725f,   0.23662911f, 0.21974683f,  0.15076452f, 0.21153738f,
                              -0.19304434f, 0.43176283f, -0.48242532f, 0.22883562f, -0.04077912f};
    float q = 0.5f * kQ[9];
#pragma unroll
    for (int i = 8; i >= 0; --i) q = fmaf(q, t, 0.5f * kQ[i]);
    const float half_erfc = e * (t * q);
    cdf = z < 0.f ? half_erfc : 1.f - half_erfc;
    density = 0.3989422804014327f * e;
  }
}

constexpr float kTanhA = 1.5957691216057308f;             // 2 sqrt(2 / pi): gelu_tanh(z) = z sigmoid(z (A + B z^2))
constexpr float kTanhB = 1.5957691216057308f * 0.044715f;

template <typename T, int ACT>
__device__ inline float act_value(float z) {
  if constexpr (ACT == kActRelu) return z > 0.f || z != z ? z : 0.f;   // a NaN stays one
  if constexpr (ACT == kActGelu) {
    float cdf, density;
    normal_cdf<T>(z, cdf, density);
    return z * cdf;
  }
  if constexpr (ACT == kActGeluTanh) return z * sigmoid<T>(z * (kTanhA + kTanhB * z * z));
  if constexpr (ACT == kActSilu) return z * sigmoid<T>(z);
  return z;
}

// The slope at z, and the value where it is asked for.  A slope is 0 or 1 to the last bit of fp32 from |z| = 16 (GELU) or 104 (SiLU)
// on; z is held to that range for it, so that z^2 does not overflow and an infinite z gives the limit and not 0 * inf.
template <typename T, int ACT>
__device__ inline float act_slope(float z, float* value = nullptr) {
  if constexpr (ACT == kActNone) {
    if (value) *value = z;
    return 1.f;
  } else if constexpr (ACT == kActRelu) {
    if (value) *value = act_value<T, ACT>(z);
    return z != z ? z : z > 0.f ? 1.f : 0.f;
  } else {
    constexpr float kFlat = ACT == kActSilu ? 104.f : 16.f;
    const float c = z > kFlat ? kFlat : z < -kFlat ? -kFlat : z;   // comparisons, not min / max: a NaN stays one
    if constexpr (ACT == kActGelu) {
      float cdf, density;
      normal_cdf<T>(c, cdf, density);
      if (value) *value = z * cdf;
      return cdf + c * density;
    } else {
      const float x = ACT == kActSilu ? c : c * (kTanhA + kTanhB * c * c);
      const float e = fast_exp<T>(-x), s = reciprocal<T>(1.f + e);
      if (value) *value = z * s;
      const float rest = x > 0.f ? e * s : 1.f - s;   // 1 - s without cancellation
      return s + c * s * rest * (ACT == kActSilu ? 1.f : kTanhA + 3.f * kTanhB * c * c);
    }
  }
}

// E neighbouring columns of one row: v (and u, gated forward) hold the products with their bias; zg, zu the kept pre-activations
// (backward).  out: what is stored first; u: the up half's gradient (gated backward); h: the layer's output again (gated backward).
template <typename T, int MODE, int ACT, int E>
__device__ inline void combine(const float* v, float* u, const float* zg, const float* zu, float* out, float* h) {
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if constexpr (MODE == kLinFwd) out[e] = act_value<T, ACT>(v[e]);
    if constexpr (MODE == kLinBwd) out[e] = ACT == kActNone ? v[e] : v[e] * act_slope<T, ACT>(zg[e]);
    if constexpr (MODE == kGatedFwd) out[e] = act_value<T, ACT>(v[e]) * u[e];
    if constexpr (MODE == kGatedBwd) {
      float value;
      const float slope = act_slope<T, ACT>(zg[e], &value);
      out[e] = v[e] * (zu[e] * slope);
      u[e] = v[e] * value;
      h[e] = value * zu[e];
    }
  }
}

// what rounding v to bf16 takes off (nothing of a value that becomes infinite): with it, a weight gradient is that of the unrounded v
__device__ inline float rounded_off(float v) {
  const float r = bf16_bits_to_float(float_to_bf16_bits(v));
  return fabsf(r) < INFINITY ? v - r : 0.f;
}

// What a call reads and writes: rows of `width` bytes, `ld` bytes apart.  A launch has no order among its tiles, so that what it
// writes may not be what another tile reads; a chunk that is read by the lane that then writes it may (`in_place`).
struct Span {
  const void* at;
  int64_t ld, width, rows;
};
inline bool apart(const Span& a, const Span& b, bool in_place = false) {
  if (!a.at || !b.at || a.rows <= 0 || b.rows <= 0) return true;
  const uintptr_t pa = reinterpret_cast<uintptr_t>(a.at), pb = reinterpret_cast<uintptr_t>(b.at);
  if (pa + (a.rows - 1) * a.ld + a.width <= pb || pb + (b.rows - 1) * b.ld + b.width <= pa) return true;
  const bool same_ld = a.ld == b.ld || (a.rows == 1 && b.rows == 1);
  if (pa == pb && same_ld && a.width == b.width) return in_place;
  if (a.ld != b.ld) return false;
  const int64_t ld = a.ld, shift = ((static_cast<int64_t>(pb) - static_cast<int64_t>(pa)) % ld + ld) % ld;   // columns of one matrix?
  return shift >= a.width && shift + b.width <= ld;
}

// fn with the activation as a constant
template <typename F>
__device__ __forceinline__ void with_activation(int act, F&& fn) {
  switch (act) {
    case kActRelu: fn(std::integral_constant<int, kActRelu>{}); break;
    case kActGelu: fn(std::integral_constant<int, kActGelu>{}); break;
    case kActGeluTanh: fn(std::integral_constant<int, kActGeluTanh>{}); break;
    case kActSilu: fn(std::integral_constant<int, kActSilu>{}); break;
    default: fn(std::integral_constant<int, kActNone>{}); break;
  }
}

}  // namespace tch

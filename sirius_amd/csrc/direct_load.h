// Operand loads of the matrix kernels: bounds-checked buffer loads, direct loads from global memory into LDS, and the waits and
// unrolled walks around them.
#pragma once

#include <utility>

#include "kernels.h"

namespace tch {

// Operand loads go through buffer instructions: an offset outside the declared extent
// returns zeros, so padding, ragged edges and the tail of the reduction need neither a
// branch nor a select, and the loads stay in flight across the multiply of earlier tiles.
typedef unsigned int uint4_t __attribute__((ext_vector_type(4)));
typedef unsigned int uint2_t __attribute__((ext_vector_type(2)));
constexpr uint32_t kOutOfRange = 0x80000000u;

__device__ inline __amdgpu_buffer_rsrc_t make_rsrc(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, static_cast<int>(bytes), 0x00020000);
}

__device__ inline Chunk load_chunk(__amdgpu_buffer_rsrc_t rsrc, uint32_t byte_off, bool valid) {
  uint4_t v = __builtin_amdgcn_raw_buffer_load_b128(rsrc, static_cast<int>(valid ? byte_off : kOutOfRange), 0, 0);
  Chunk c;
  c.w[0] = v[0];
  c.w[1] = v[1];
  c.w[2] = v[2];
  c.w[3] = v[3];
  return c;
}

typedef __attribute__((address_space(3))) void* lds_void_ptr;

// 16 bytes per lane from `rsrc` at byte offset voff (+ the wave-uniform soff) to dst + lane*16 in
// LDS; an offset outside the resource stores zeros.  (Kept in a device function: named directly
// in a kernel body, the builtin makes the host pass drop the kernel's launch stub.)
__device__ inline void load_to_lds(__amdgpu_buffer_rsrc_t rsrc, unsigned char* dst, int voff, int soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_void_ptr)dst, 16, voff, soff, 0, 0);
}

// the registers belong to their values up to this point of the program
template <int A, int B>
__device__ inline void hold(uint4_t (&r)[A][B]) {
#pragma unroll
  for (int i = 0; i < A; ++i)
#pragma unroll
    for (int j = 0; j < B; ++j) asm volatile("" : "+v"(r[i][j]));
}

__device__ inline const void* wave_uniform(const void* ptr) {
  const uint64_t v = reinterpret_cast<uint64_t>(ptr);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v >> 32));
  return reinterpret_cast<const void*>(static_cast<uint64_t>(hi) << 32 | lo);
}

// fn(0), fn(1), .. fn(N - 1) with the index as a constant
template <int... I, typename F>
__device__ __forceinline__ void unrolled_steps(std::integer_sequence<int, I...>, F&& fn) {
  (fn(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void unrolled(F&& fn) {
  unrolled_steps(std::make_integer_sequence<int, N>{}, fn);
}

// All but the newest N of this wave's direct loads have landed, all its LDS accesses are done, and every wave of the
// workgroup is here.  Not __syncthreads(): the compiler puts a wait for EVERY outstanding direct load in front of
// that (a direct load is an LDS write to it), which leaves no tile in flight across the barrier whatever NBUF is:
// each step then pays a whole trip to memory (a 64 x 64 tile: 0.47 us per 64-element step with two buffers or three).
template <int N>
__device__ inline void wait_and_meet() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

}  // namespace tch

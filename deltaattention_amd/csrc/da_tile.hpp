// What the matrix kernels on K/V tiles in LDS share: uniform pointers and buffer resources, hand-issued
// LDS reads with exact waits, exchanges between the halves of a wave.
#pragma once

#include <utility>

#include "da_common.hpp"

namespace da {

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// min(max(x, 0), hi) for a wave-uniform x, kept in scalar registers (the compiler would
// otherwise form a clamp that only exists as a vector instruction, v_med3).
__device__ __forceinline__ int clamp0_uniform(int x, int hi) {
  x = __builtin_amdgcn_readfirstlane(x < hi ? x : hi);
  asm volatile("" : "+s"(x));
  return x > 0 ? x : 0;
}

// Third dword of a raw buffer resource on gfx9 (32-bit data format, no swizzle).
constexpr int kBufferDword3 = 0x00020000;

// A wave-uniform pointer moved into scalar registers.
__device__ __forceinline__ const void* uniform_ptr(const void* p) {
  const uint64_t v = (uint64_t)p;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
  return (const void*)(((uint64_t)hi << 32) | lo);
}

typedef short i16x4 __attribute__((ext_vector_type(4)));

// LDS byte address of a pointer into the kernel's LDS.
__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)p;
}
// ds_read_b64_tr_b16 at addr + OFF: in each group of 16 lanes, lane i receives element
// i % 4 of the 8 bytes read by lanes 4e + i / 4, e = 0..3 (a 4 x 4 transpose of 16-bit
// elements per group of four lanes).  Issued as asm: the caller waits with lgkm_wait.
template <int OFF>
__device__ __forceinline__ i16x4 ds_read_tr16(uint32_t addr) {
  i16x4 v;
  asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(v) : "v"(addr), "i"(OFF));
  return v;
}
// s_waitcnt lgkmcnt(N) that the uses of a and b cannot move above.
template <int N>
__device__ __forceinline__ void lgkm_wait(i16x4& a, i16x4& b) {
  asm volatile("s_waitcnt lgkmcnt(%2)" : "+v"(a), "+v"(b) : "i"(N));
}
// ds_read_b128 issued as asm (waited for with lgkm_wait), so that the reads stay ahead
// of the MFMAs that use them.
__device__ __forceinline__ u32x4 ds_read_b128_asm(uint32_t addr) {
  u32x4 v;
  asm volatile("ds_read_b128 %0, %1" : "=v"(v) : "v"(addr));
  return v;
}
template <int N>
__device__ __forceinline__ void lgkm_wait(u32x4& a, u32x4& b) {
  asm volatile("s_waitcnt lgkmcnt(%2)" : "+v"(a), "+v"(b) : "i"(N));
}
template <int N>
__device__ __forceinline__ void lgkm_wait(u32x4& a) {
  asm volatile("s_waitcnt lgkmcnt(%1)" : "+v"(a) : "i"(N));
}
template <typename F, int... I>
__device__ __forceinline__ void static_for_impl(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
// f(integral_constant<int, i>) for i = 0 .. N-1, in order
template <int N, typename F>
__device__ __forceinline__ void static_for(F&& f) {
  static_for_impl(f, std::make_integer_sequence<int, N>{});
}

// Max / sum of x over lanes l and l ^ 32, without LDS (v_permlane32_swap); the order
// of the returned pair does not matter for either.
__device__ __forceinline__ float halves_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __builtin_fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float halves_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// s_waitcnt immediate (gfx9 encoding) that waits for vmcnt <= n only.
constexpr int vmcnt_only(int n) { return (n & 15) | ((n >> 4) << 14) | (7 << 4) | (15 << 8); }

}  // namespace da

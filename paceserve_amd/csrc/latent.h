// What the two forms of latent attention share.
#pragma once

#include "attention.h"

namespace pace_kv {

constexpr int kRope = 64;      // columns of the rotated part

// A score in units of log 2, rounded by itself: a difference of it and a maximum of
// others like it is exact where it matters, and 0 for the largest.
__device__ __forceinline__ float scaled(float s, float scale_log2) {
#pragma clang fp contract(off)
  return s * scale_log2;
}

__device__ __forceinline__ float unfused(float a, float b) {
#pragma clang fp contract(off)
  return a - b;
}

// Weights are rounded to the rows' type for their product, which takes nothing wider, and sums
// take them unrounded (attention.h).  The running maximum is exact, so that the largest weight is
// a power of two and not rounded: outputs are off by 0.0018 to 0.0021 of the values against 64
// bits (bfloat16, 2000 to 8192 tokens), of which their own rounding is 0.0016.  (MI355X: raising
// it only where a score passes it by 2^4 in weight saves a product of every sum, 4 to 8 % of
// prompts and of calls of 64 rows and more, but outputs were off by 0.0019 to 0.0023, and where
// one token stands out by up to twice as much.)

// The maximum of no scores: finite, so that differences from it are numbers.
constexpr float kLowest = -0x1.fffffep127f;

// log2 of the weight of a score that equals the maximum.  In float16 the largest weights are
// 2^15, which leaves those down to 2^-29 of the largest their 2^-11.  bfloat16 has float32's
// exponents: 2^-24, so that up to 2^24 values of the largest exponent have a finite sum.
template <int TYPE>
constexpr float kUnit = TYPE == PACE_KV_FP16 ? 15.f : -24.f;

// Matrix instructions' results, waited for: max3_of reads them in assembly, which the
// compiler does not do for.  20 cycles, more than any such instruction takes to write.
template <int N>
__device__ __forceinline__ void settle(f32x4 (&x)[N][2]) {
  static_assert(N == 1 || N == 2);
  if constexpr (N == 1) asm volatile("s_nop 15\n\ts_nop 3" : "+v"(x[0][0]), "+v"(x[0][1]));
  else asm volatile("s_nop 15\n\ts_nop 3" : "+v"(x[0][0]), "+v"(x[0][1]), "+v"(x[1][0]), "+v"(x[1][1]));
}

// A workgroup's barrier that waits for its LDS operations alone, not for rows on their way
// into LDS as __syncthreads does.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// One that waits for those rows too.
__device__ __forceinline__ void rows_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// LDS by offsets, whose swizzles are xors.  Its 64 banks serve 8-byte reads by 32 lanes in
// order, 16-byte reads by 16: lanes 0-3, 12-15 and 20-27, then 4-11, 16-19 and 28-31, and the
// upper 32 the same way (measured: the counter of conflicts is 0 for layouts that keep
// these lanes apart).  Of a fragment read by rows n = lane % 16, rows 0-3 and 12-15 of one
// 16-byte column thus meet rows 4-11 of the next: the rows whose pieces lie in the same 32
// bytes are of one set or the other, and, for values, not both of 0-7.
__device__ __forceinline__ uint32_t lds_offset(const void* x) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((const __attribute__((address_space(3))) char*)x));
}

template <class T>
__device__ __forceinline__ T lds_get(uint32_t at) {
  return *(const __attribute__((address_space(3))) T*)static_cast<uintptr_t>(at);
}

template <class T>
__device__ __forceinline__ void lds_put(uint32_t at, T x) {
  *(__attribute__((address_space(3))) T*)static_cast<uintptr_t>(at) = x;
}

// Transposing read: lanes of 16 hold four columns each of four rows, and get four rows
// of a column each.
__device__ __forceinline__ u32x2 lds_transposed(uint32_t at) {
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                       (__attribute__((address_space(3))) s16x4*)static_cast<uintptr_t>(at)));
}

// Each lane's 16 bytes at `from` into LDS, at `at` (the same for all lanes) + 16 * lane;
// there once vmcnt says so.
__device__ __forceinline__ void copy_to_lds(const char* from, uint32_t at) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                   (__attribute__((address_space(3))) void*)static_cast<uintptr_t>(at), 16, 0, 0);
}

// A word with its infinite and NaN halves as zeros.
template <int TYPE>
__device__ __forceinline__ uint32_t finite_halves(uint32_t x) {
  if (odd_word<TYPE>(x & 0xffffu)) x &= 0xffff0000u;
  if (odd_word<TYPE>(x >> 16)) x &= 0xffffu;
  return x;
}

// Natural logarithm of a row's sum of exponentials: l, its weights over the maximum m.
template <int TYPE>
__device__ __forceinline__ float log_total(float m, float l) {
  constexpr float kScale = TYPE == PACE_KV_FP16 ? 0x1p-15f : 0x1p24f;  // 2^-kUnit
  return l == 0.f ? -INFINITY : (m + __log2f(l * kScale)) * 0.69314718055994531f;
}

}  // namespace pace_kv

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

// The weight of a score s over the maximum m: at most 1, in float16 at most 2^15 (whose
// subnormals then lie below 2^-29 of the largest).
template <int TYPE>
__device__ __forceinline__ float weight_of(float s, float m) {
#pragma clang fp contract(off)
  return exp2_of((s - m) + kTopWeight<TYPE>);
}

// Natural logarithm of a row's sum of exponentials: l weights over the maximum m.
template <int TYPE>
__device__ __forceinline__ float log_total(float m, float l) {
  constexpr float kScale = TYPE == PACE_KV_FP16 ? 0x1p-15f : 1.f;
  return l == 0.f ? -INFINITY : (m + __log2f(l * kScale)) * 0.69314718055994531f;
}

}  // namespace pace_kv

// The quantised page format and its conversions.
//
// Blocks of 32 elements along head_dim share a power-of-two scale 2^e, held as
// the byte e + 127; elements are e4m3 (8 bits) or e2m1 (4 bits, two to a byte,
// the even one low).  e is the smallest exponent that brings the block's
// largest magnitude within the element type (448 or 6), so nothing is clamped,
// and x * 2^-e is exact: the one rounding is the element's, to nearest even
// (2^-4 of the value for e4m3, 2^-2 for e2m1, above the smallest normal
// element).  Bytes lie in [10, 254]: with 2^-117 at least, every non-zero
// element stands for a normal number in float32 and bfloat16.  A block with an
// infinity or a NaN has the byte 255 and zero elements, and reads as NaN.
//
// Half a page (its keys or its values) is [page_size, H, D] elements, then
// [page_size, H, D / 32] scale bytes, so block k's scale is byte k behind the
// elements and a page carries all that its values need.
//
// gfx950's scaled conversions (v_cvt_scalef32_pk_*) do both directions, two
// elements an instruction: they divide or multiply by the scale, whose float32
// form is its byte in the exponent's place, round to nearest even, keep
// subnormals, and give NaN for 255.
#pragma once

#include "internal.h"

namespace pace_kv {

constexpr int kMxBlock = 32;

// Elements that a lane carries: 16 bytes of a 16-bit type, so a block is four
// neighbouring lanes'.
constexpr int kLaneElems = 8;

constexpr int elem_bytes(int type) { return type == PACE_KV_FP32 ? 4 : 2; }
constexpr int mx_bits(int format) { return format == PACE_KV_MXFP8 ? 8 : 4; }

// Bytes of half a page of n elements.
inline int64_t mx_half_bytes(int64_t n, int format) { return n * mx_bits(format) / 8 + n / kMxBlock; }

inline bool is_elem_type(int type) { return type == PACE_KV_BF16 || type == PACE_KV_FP16 || type == PACE_KV_FP32; }
inline bool is_mx_format(int format) { return format == PACE_KV_MXFP8 || format == PACE_KV_MXFP4; }

#ifdef __HIP__

typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// kLaneElems consecutive values as they lie in memory.
template <int TYPE>
struct Run {
  static constexpr int kVecs = elem_bytes(TYPE) / 2;
  u32x4 v[kVecs];
};

// STREAM: nontemporally.
template <int TYPE, bool STREAM>
__device__ __forceinline__ Run<TYPE> load_run(const char* s) {
  Run<TYPE> r;
#pragma unroll
  for (int k = 0; k < Run<TYPE>::kVecs; ++k) {
    const u32x4* const at = reinterpret_cast<const u32x4*>(s) + k;
    r.v[k] = STREAM ? __builtin_nontemporal_load(at) : *at;
  }
  return r;
}

template <bool STREAM, class T>
__device__ __forceinline__ void put(T* to, T x) {
  if constexpr (STREAM) __builtin_nontemporal_store(x, to);
  else *to = x;
}

// Largest magnitude of the lane's block as float32 bits; infinities and NaN
// give at least an infinity's.  Magnitudes order as their bits do.
template <int TYPE>
__device__ __forceinline__ uint32_t block_amax(const Run<TYPE>& r) {
  uint32_t m;
  if constexpr (TYPE == PACE_KV_FP32) {
    m = 0;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) m = max(m, r.v[k][j] & 0x7fffffffu);
  } else {
    u16x2 p = {0, 0};
#pragma unroll
    for (int j = 0; j < 4; ++j) p = __builtin_elementwise_max(p, __builtin_bit_cast(u16x2, r.v[0][j] & 0x7fff7fffu));
    m = max(static_cast<uint32_t>(p[0]), static_cast<uint32_t>(p[1]));
  }
  m = max(m, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(m), 0xB1, 0xf, 0xf, true)));  // lane ^ 1
  m = max(m, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(m), 0x4E, 0xf, 0xf, true)));  // lane ^ 2
  if constexpr (TYPE == PACE_KV_BF16) return m << 16;
  if constexpr (TYPE == PACE_KV_FP16) {
    return __float_as_uint(static_cast<float>(__builtin_bit_cast(_Float16, static_cast<unsigned short>(m))));
  }
  return m;
}

// Scale byte of a block: the exponent of 448 = 1.75 * 2^8 (or 6 = 1.5 * 2^2)
// taken off amax's, one more where amax's fraction is the larger.
template <int FORMAT>
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax) {
  constexpr int kLead = FORMAT == PACE_KV_MXFP8 ? 8 : 2;
  constexpr uint32_t kFraction = FORMAT == PACE_KV_MXFP8 ? 0x600000u : 0x400000u;
  const int e = static_cast<int>(amax >> 23) - kLead + ((amax & 0x7fffffu) > kFraction ? 1 : 0);
  return amax >= 0x7f800000u ? 255u : static_cast<uint32_t>(min(max(e, 10), 254));
}

__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

// The two values at 2 * k of a run as elements: e4m3 into half HALF of `to`,
// or e2m1 into byte BYTE of it.
template <int TYPE, int FORMAT, int AT>
__device__ __forceinline__ uint32_t pair_down(uint32_t to, const Run<TYPE>& r, int k, float scale) {
  if constexpr (TYPE == PACE_KV_FP32) {
    const float a = __uint_as_float(r.v[k / 2][(k % 2) * 2]), b = __uint_as_float(r.v[k / 2][(k % 2) * 2 + 1]);
    if constexpr (FORMAT == PACE_KV_MXFP8)
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(__builtin_bit_cast(s16x2, to), a, b,
                                                                                    scale, AT != 0));
    else
      return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(to, a, b, scale, AT);
  } else if constexpr (TYPE == PACE_KV_BF16) {
    const uint32_t w = r.v[0][k];  // a bit cast of the vector's element itself takes element 0
    const bf16x2 x = __builtin_bit_cast(bf16x2, w);
    if constexpr (FORMAT == PACE_KV_MXFP8)
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(__builtin_bit_cast(s16x2, to), x,
                                                                                     scale, AT != 0));
    else
      return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(to, x, scale, AT);
  } else {
    const uint32_t w = r.v[0][k];
    const f16x2 x = __builtin_bit_cast(f16x2, w);
    if constexpr (FORMAT == PACE_KV_MXFP8)
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(__builtin_bit_cast(s16x2, to), x,
                                                                                    scale, AT != 0));
    else
      return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(to, x, scale, AT);
  }
}

// Stores a lane's run as elements at `data`, its place among the half page's
// elements, and the block's scale byte at `scale` (from the block's first lane).
template <int TYPE, int FORMAT, bool STREAM>
__device__ __forceinline__ void store_run(const Run<TYPE>& r, uint32_t byte, char* data, char* scale) {
  const float s = scale_of(byte);
  const uint32_t keep = byte == 255u ? 0u : ~0u;
  if constexpr (FORMAT == PACE_KV_MXFP8) {
    u32x2 q = {0, 0};
    q[0] = pair_down<TYPE, FORMAT, 0>(q[0], r, 0, s);
    q[0] = pair_down<TYPE, FORMAT, 1>(q[0], r, 1, s);
    q[1] = pair_down<TYPE, FORMAT, 0>(q[1], r, 2, s);
    q[1] = pair_down<TYPE, FORMAT, 1>(q[1], r, 3, s);
    put<STREAM>(reinterpret_cast<u32x2*>(data), q & keep);
  } else {
    uint32_t q = 0;
    q = pair_down<TYPE, FORMAT, 0>(q, r, 0, s);
    q = pair_down<TYPE, FORMAT, 1>(q, r, 1, s);
    q = pair_down<TYPE, FORMAT, 2>(q, r, 2, s);
    q = pair_down<TYPE, FORMAT, 3>(q, r, 3, s);
    put<STREAM>(reinterpret_cast<uint32_t*>(data), q & keep);
  }
  if (threadIdx.x % 4 == 0) *reinterpret_cast<uint8_t*>(scale) = static_cast<uint8_t>(byte);
}

// Two elements of `word` (its half AT of e4m3, or its byte AT of e2m1) as two
// 16-bit values.
template <int TYPE, int FORMAT, int AT>
__device__ __forceinline__ uint32_t pair_up(uint32_t word, float scale) {
  if constexpr (TYPE == PACE_KV_BF16) {
    if constexpr (FORMAT == PACE_KV_MXFP8)
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, scale, AT != 0));
    else
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, AT));
  } else {
    if constexpr (FORMAT == PACE_KV_MXFP8)
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, scale, AT != 0));
    else
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, scale, AT));
  }
}

template <int FORMAT, int AT>
__device__ __forceinline__ f32x2 pair_up_f32(uint32_t word, float scale) {
  if constexpr (FORMAT == PACE_KV_MXFP8) return __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(word, scale, AT != 0);
  else return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(word, scale, AT);
}

// The four words of eight 16-bit values from eight elements.
template <int TYPE, int FORMAT>
__device__ __forceinline__ u32x4 run_up(u32x2 q, float s) {
  if constexpr (FORMAT == PACE_KV_MXFP8)
    return u32x4{pair_up<TYPE, FORMAT, 0>(q[0], s), pair_up<TYPE, FORMAT, 1>(q[0], s),
                 pair_up<TYPE, FORMAT, 0>(q[1], s), pair_up<TYPE, FORMAT, 1>(q[1], s)};
  else
    return u32x4{pair_up<TYPE, FORMAT, 0>(q[0], s), pair_up<TYPE, FORMAT, 1>(q[0], s),
                 pair_up<TYPE, FORMAT, 2>(q[0], s), pair_up<TYPE, FORMAT, 3>(q[0], s)};
}

#endif  // __HIP__

}  // namespace pace_kv

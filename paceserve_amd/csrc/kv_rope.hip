// Queries and keys normalised per head and rotated by position, into tensors or,
// with the values, straight into a paged cache (16-bit or quantised); and the
// rows of a latent cache, normalised and rotated the same way.
//
//   y = x / sqrt(mean(x^2) + eps) * w                      (where there is a weight)
//   (y_i, y_{i + r/2}) -> (y_i c_i - y_{i + r/2} s_i, y_{i + r/2} c_i + y_i s_i), i < r / 2
//   interleaved: the pairs are (y_{2 i}, y_{2 i + 1})
// with c and s the token's row of a float32 table.  All in float32, rounded once:
// to the rows' type, or to a quantised cache's elements.
//
// Bound by HBM: each row is read and written once.  A lane holds two runs of eight
// elements that rotate against each other, [8 u, 8 u + 8) and the same behind
// r / 2 (of the columns that do not rotate, the same half of them apart), so a
// head is D / 16 lanes, its pairs never leave a lane, and its sum of squares takes
// log2(D / 16) exchanges.  The cosines and sines of a token are 64 bytes a lane
// against 32 of its rows: a lane loads them once and goes on over the token's heads.
#include <algorithm>
#include <cmath>

#include "mx.h"

namespace pace_kv {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int64_t kMaxGroupsPerLaunch = int64_t(1) << 24;

struct Rows {
  const char* in;
  int64_t in_token, in_head;   // bytes between tokens and heads
  char* out;                   // unless it goes to the cache
  int64_t out_token, out_head;
  const char* weight;          // [head_dim], or nullptr
  uint32_t heads;
};

struct RopeParams {
  Rows q, k, v;                // v only with a cache
  const int32_t* positions;
  const int64_t* slots;        // of a cache, else nullptr
  const float* table;          // [table_rows, rotary]
  char* cache;
  int32_t* err;
  int64_t nnz, table_rows, num_slots;
  int64_t page_bytes, half_bytes, scale_at;  // of a page, its half, and the scales within a half
  uint32_t head_dim, rotary, units;  // units = head_dim / 16 lanes
  uint32_t group_log2;         // lanes of a head: units to the next power of two
  uint32_t parts, part_heads;  // waves that a token's heads are dealt to, and heads of each
  uint32_t page_size;
  float eps, inv_dim;
  FastDiv by_page;
};

template <int TYPE>
__device__ __forceinline__ void widen(const u32x4& v, float* x) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t w = v[j];
    if constexpr (TYPE == PACE_KV_BF16) {
      x[2 * j] = __uint_as_float(w << 16);
      x[2 * j + 1] = __uint_as_float(w & 0xffff0000u);
    } else {
      const f16x2 h = __builtin_bit_cast(f16x2, w);
      x[2 * j] = static_cast<float>(h[0]);
      x[2 * j + 1] = static_cast<float>(h[1]);
    }
  }
}

template <int TYPE>
__device__ __forceinline__ u32x4 narrow(const float* x) {
  u32x4 v;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (TYPE == PACE_KV_BF16) {
      const bf16x2 h = {static_cast<__bf16>(x[2 * j]), static_cast<__bf16>(x[2 * j + 1])};
      v[j] = __builtin_bit_cast(uint32_t, h);
    } else {
      const f16x2 h = {static_cast<_Float16>(x[2 * j]), static_cast<_Float16>(x[2 * j + 1])};
      v[j] = __builtin_bit_cast(uint32_t, h);
    }
  }
  return v;
}

// Rotates the pairs of a lane's two runs a, b by the angles of its cosines and sines:
// pair j is (a[j], b[j]), or, interleaved, the neighbours of a and then those of b.
__device__ __forceinline__ void rotate(bool interleaved, float* a, float* b, const float* cos, const float* sin) {
  if (!interleaved) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float x = a[j], y = b[j];
      a[j] = x * cos[j] - y * sin[j];
      b[j] = y * cos[j] + x * sin[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float x = a[2 * j], y = a[2 * j + 1];
      a[2 * j] = x * cos[j] - y * sin[j];
      a[2 * j + 1] = y * cos[j] + x * sin[j];
      x = b[2 * j], y = b[2 * j + 1];
      b[2 * j] = x * cos[4 + j] - y * sin[4 + j];
      b[2 * j + 1] = y * cos[4 + j] + x * sin[4 + j];
    }
  }
}

// The eight cosines and sines of unit u of `rotary` columns, from a table row: those
// of its eight pairs, or, interleaved, four from 4 u and four from rotary / 4 + 4 u.
__device__ __forceinline__ void load_angles(const float* row, uint32_t rotary, bool interleaved, uint32_t u, float* cos,
                                            float* sin) {
  const float* const c = row + (interleaved ? 4 : 8) * u;
  const uint32_t second = interleaved ? rotary / 4 : 4;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    cos[j] = c[j];
    cos[4 + j] = c[second + j];
    sin[j] = c[rotary / 2 + j];
    sin[4 + j] = c[rotary / 2 + second + j];
  }
}

// A lane's run as float32 bits, for the quantising store.
__device__ __forceinline__ Run<PACE_KV_FP32> float_run(const float* x) {
  Run<PACE_KV_FP32> r;
#pragma unroll
  for (int j = 0; j < 8; ++j) r.v[j / 4][j % 4] = __float_as_uint(x[j]);
  return r;
}

// FORMAT: of the cache, or -1 without one.
template <int TYPE, int FORMAT, bool INTERLEAVED>
__global__ __launch_bounds__(kThreads) void rope_kernel(const RopeParams p) {
  const uint32_t lane = threadIdx.x % 64;
  const int64_t wave = static_cast<int64_t>(blockIdx.x) * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int64_t token = wave / p.parts;
  const uint32_t part = static_cast<uint32_t>(wave - token * p.parts);
  if (token >= p.nnz) return;
  int64_t page_at = 0, slot = 0;
  if constexpr (FORMAT >= 0) {
    const int64_t s = p.slots[token];
    if (s == -1) return;                                 // padding
    if (s < 0 || s >= p.num_slots) {
      if (p.err != nullptr && part == 0 && lane == 0) atomicAdd(p.err, 1);
      return;
    }
    const int64_t page = s / p.page_size;
    slot = s - page * p.page_size;
    page_at = page * p.page_bytes;
  }
  const int64_t position = p.positions[token];
  if (position < 0 || position >= p.table_rows) {
    if (p.err != nullptr && part == 0 && lane == 0) atomicAdd(p.err, 1);
    return;
  }
  const uint32_t group = 1u << p.group_log2, u = lane & (group - 1);
  const bool rotates = u < p.rotary / 16, active = u < p.units;
  // First elements of the lane's runs.
  const uint32_t tail = p.head_dim - p.rotary;
  const uint32_t ea = rotates ? 8 * u : p.rotary + 8 * (u - p.rotary / 16);
  const uint32_t eb = ea + (rotates ? p.rotary : tail) / 2;
  float cos[8], sin[8];
  if (rotates) load_angles(p.table + position * p.rotary, p.rotary, INTERLEAVED, u, cos, sin);
  const uint32_t qk = p.q.heads + p.k.heads, heads = qk + (FORMAT >= 0 ? p.v.heads : 0u);
  const uint32_t end = min((part + 1) * p.part_heads, heads);
  for (uint32_t h = part * p.part_heads + (lane >> p.group_log2); h < end; h += 64u >> p.group_log2) {
    const Rows& rows = h < p.q.heads ? p.q : h < qk ? p.k : p.v;
    const uint32_t head = h < p.q.heads ? h : h < qk ? h - p.q.heads : h - qk;
    const char* const in = rows.in + token * rows.in_token + head * rows.in_head;
    u32x4 ra = {0, 0, 0, 0}, rb = {0, 0, 0, 0};
    if (active) {
      ra = *reinterpret_cast<const u32x4*>(in + ea * 2);
      rb = *reinterpret_cast<const u32x4*>(in + eb * 2);
    }
    float a[8], b[8];
    if (h < qk) {
      widen<TYPE>(ra, a);
      widen<TYPE>(rb, b);
      if (rows.weight != nullptr) {
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += a[j] * a[j] + b[j] * b[j];
        for (uint32_t k = 1; k < group; k *= 2) sum += __shfl_xor(sum, k);
        const float inv = 1.f / sqrtf(sum * p.inv_dim + p.eps);
        if (active) {
          float wa[8], wb[8];
          widen<TYPE>(*reinterpret_cast<const u32x4*>(rows.weight + ea * 2), wa);
          widen<TYPE>(*reinterpret_cast<const u32x4*>(rows.weight + eb * 2), wb);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            a[j] = a[j] * inv * wa[j];
            b[j] = b[j] * inv * wb[j];
          }
        }
      }
      if (rotates) rotate(INTERLEAVED, a, b, cos, sin);
    }
    if (!active) continue;
    if (FORMAT < 0 || h < p.q.heads) {
      char* const out = rows.out + token * rows.out_token + head * rows.out_head;
      *reinterpret_cast<u32x4*>(out + ea * 2) = narrow<TYPE>(a);
      *reinterpret_cast<u32x4*>(out + eb * 2) = narrow<TYPE>(b);
    } else if constexpr (FORMAT >= 0) {
      const int64_t element = (slot * p.k.heads + head) * p.head_dim;
      char* const half = p.cache + page_at + (h < qk ? 0 : p.half_bytes);
      if constexpr (FORMAT == PACE_KV_PLAIN) {
        *reinterpret_cast<u32x4*>(half + (element + ea) * 2) = h < qk ? narrow<TYPE>(a) : ra;
        *reinterpret_cast<u32x4*>(half + (element + eb) * 2) = h < qk ? narrow<TYPE>(b) : rb;
      } else {
        // Blocks of 32 are four neighbouring lanes' runs: rotary and tail are multiples of 64.
        constexpr int kBits = mx_bits(FORMAT);
        const auto put_run = [&](const float* x, const u32x4& raw, uint32_t e) {
          Run<PACE_KV_FP32> r = float_run(x);
          if (h >= qk) {
            float f[8];
            widen<TYPE>(raw, f);
            r = float_run(f);
          }
          const uint32_t byte = scale_byte<FORMAT>(block_amax<PACE_KV_FP32>(r));
          store_run<PACE_KV_FP32, FORMAT, false>(r, byte, half + (element + e) * kBits / 8,
                                                 half + p.scale_at + (element + e) / kMxBlock);
        };
        put_run(a, ra, ea);
        put_run(b, rb, eb);
      }
    }
  }
}

struct LatentParams {
  const char* latent;
  const char* rope_key;
  int64_t latent_stride, rope_stride;  // bytes between tokens
  const char* weight;
  const int32_t* positions;
  const int64_t* slots;
  const float* table;
  char* cache;
  int32_t* err;
  int64_t nnz, table_rows, num_slots;
  float eps;
};

constexpr int kRope = 64;      // columns of a latent row's rotated part

// L / 8 lanes take a token: eight elements of the latent each, and the first four two
// runs of the rotated part.
template <int L, int TYPE, bool INTERLEAVED>
__global__ __launch_bounds__(kThreads) void latent_rows_kernel(const LatentParams p) {
  constexpr uint32_t kLanes = L / 8, kTokens = kThreads / kLanes;
  const uint32_t u = threadIdx.x % kLanes;
  const int64_t token = static_cast<int64_t>(blockIdx.x) * kTokens + threadIdx.x / kLanes;
  if (token >= p.nnz) return;
  const int64_t slot = p.slots[token];
  if (slot == -1) return;                                // padding
  const int64_t position = p.positions[token];
  if (slot < 0 || slot >= p.num_slots || position < 0 || position >= p.table_rows) {
    if (p.err != nullptr && u == 0) atomicAdd(p.err, 1);
    return;
  }
  u32x4 raw = *reinterpret_cast<const u32x4*>(p.latent + token * p.latent_stride + u * 16);
  u32x4 ra, rb;
  float cos[8], sin[8];
  if (u < kRope / 16) {
    const char* const in = p.rope_key + token * p.rope_stride;
    ra = *reinterpret_cast<const u32x4*>(in + u * 16);
    rb = *reinterpret_cast<const u32x4*>(in + u * 16 + kRope);
    load_angles(p.table + position * kRope, kRope, INTERLEAVED, u, cos, sin);
  }
  char* const row = p.cache + slot * ((L + kRope) * 2);
  if (p.weight != nullptr) {
    float x[8], w[8];
    widen<TYPE>(raw, x);
    widen<TYPE>(*reinterpret_cast<const u32x4*>(p.weight + u * 16), w);
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += x[j] * x[j];
#pragma unroll
    for (uint32_t k = 1; k < kLanes; k *= 2) sum += __shfl_xor(sum, k);
    const float inv = 1.f / sqrtf(sum * (1.f / L) + p.eps);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = x[j] * inv * w[j];
    raw = narrow<TYPE>(x);
  }
  *reinterpret_cast<u32x4*>(row + u * 16) = raw;
  if (u < kRope / 16) {
    float a[8], b[8];
    widen<TYPE>(ra, a);
    widen<TYPE>(rb, b);
    rotate(INTERLEAVED, a, b, cos, sin);
    *reinterpret_cast<u32x4*>(row + L * 2 + u * 16) = narrow<TYPE>(a);
    *reinterpret_cast<u32x4*>(row + L * 2 + u * 16 + kRope) = narrow<TYPE>(b);
  }
}

template <int TYPE, int FORMAT>
const void* pick_rope(bool interleaved) {
  return interleaved ? reinterpret_cast<const void*>(&rope_kernel<TYPE, FORMAT, true>)
                     : reinterpret_cast<const void*>(&rope_kernel<TYPE, FORMAT, false>);
}

template <int TYPE>
const void* pick_rope(int format, bool interleaved) {
  switch (format) {
    case -1: return pick_rope<TYPE, -1>(interleaved);
    case PACE_KV_PLAIN: return pick_rope<TYPE, PACE_KV_PLAIN>(interleaved);
    case PACE_KV_MXFP8: return pick_rope<TYPE, PACE_KV_MXFP8>(interleaved);
    default: return pick_rope<TYPE, PACE_KV_MXFP4>(interleaved);
  }
}

template <int L>
const void* pick_latent(int type, bool interleaved) {
  if (type == PACE_KV_BF16)
    return interleaved ? reinterpret_cast<const void*>(&latent_rows_kernel<L, PACE_KV_BF16, true>)
                       : reinterpret_cast<const void*>(&latent_rows_kernel<L, PACE_KV_BF16, false>);
  return interleaved ? reinterpret_cast<const void*>(&latent_rows_kernel<L, PACE_KV_FP16, true>)
                     : reinterpret_cast<const void*>(&latent_rows_kernel<L, PACE_KV_FP16, false>);
}

int check_rows(const char* call, const Rows& r, bool writes, uint32_t head_dim) {
  if (r.heads == 0) return PACE_KV_OK;
  if (!r.in || (writes && !r.out)) return fail(PACE_KV_EINVAL, "%s: NULL rows", call);
  uintptr_t bits = reinterpret_cast<uintptr_t>(r.in) | static_cast<uintptr_t>(r.in_token | r.in_head) |
                   reinterpret_cast<uintptr_t>(r.weight);
  if (writes) bits |= reinterpret_cast<uintptr_t>(r.out) | static_cast<uintptr_t>(r.out_token | r.out_head);
  if (bits & 15u) return fail(PACE_KV_EINVAL, "%s: rows, weights and strides must be multiples of 16 bytes", call);
  if (writes && r.heads > 1 && r.out_head < static_cast<int64_t>(head_dim) * 2 &&
      r.out_head > -static_cast<int64_t>(head_dim) * 2)
    return fail(PACE_KV_EINVAL, "%s: output heads overlap", call);
  return PACE_KV_OK;
}

int check_turn(const char* call, int elem_type, int64_t nnz, const int32_t* positions, const float* table,
               int64_t table_rows, float eps) {
  if (nnz < 0 || table_rows < 0) return fail(PACE_KV_EINVAL, "%s: negative size", call);
  if (elem_type != PACE_KV_BF16 && elem_type != PACE_KV_FP16)
    return fail(PACE_KV_EINVAL, "%s: rows must be bfloat16 or float16", call);
  if (!(eps >= 0.f) || !std::isfinite(eps)) return fail(PACE_KV_EINVAL, "%s: eps must be finite and >= 0", call);
  if (nnz > 0 && (!positions || (table_rows > 0 && !table))) return fail(PACE_KV_EINVAL, "%s: NULL argument", call);
  if (reinterpret_cast<uintptr_t>(table) & 15u)
    return fail(PACE_KV_EINVAL, "%s: the table must be 16-byte aligned", call);
  return PACE_KV_OK;
}

// Launches the kernel over p, whose rows, cache and table are set and checked.
int launch_rope(RopeParams& p, int elem_type, int format, int head_dim, int rotary_dim, int interleaved,
                hipStream_t stream) {
  p.head_dim = static_cast<uint32_t>(head_dim);
  p.rotary = static_cast<uint32_t>(rotary_dim);
  p.units = p.head_dim / 16;
  p.group_log2 = 0;
  while ((1u << p.group_log2) < p.units) ++p.group_log2;
  p.inv_dim = 1.f / static_cast<float>(head_dim);
  const uint32_t heads = p.q.heads + p.k.heads + p.v.heads, turn = 64u >> p.group_log2;
  // A wave for a token's heads, or several where the tokens are too few for the CUs.
  const uint32_t turns = (heads + turn - 1) / turn;
  uint32_t per = turns;
  while (per > 1 && p.nnz * ((turns + per - 1) / per) < 4096) per = (per + 1) / 2;
  p.part_heads = per * turn;
  p.parts = (heads + p.part_heads - 1) / p.part_heads;
  const int64_t groups = (p.nnz * p.parts + kWaves - 1) / kWaves;
  if (groups > kMaxGroupsPerLaunch) return fail(PACE_KV_ERANGE, "rope: too many tokens for one call");
  void* args[] = {&p};
  const void* kernel = elem_type == PACE_KV_BF16 ? pick_rope<PACE_KV_BF16>(format, interleaved != 0)
                                                 : pick_rope<PACE_KV_FP16>(format, interleaved != 0);
  return hip_status(hipLaunchKernel(kernel, dim3(static_cast<uint32_t>(groups)), dim3(kThreads), args, 0, stream),
                    "rope launch");
}

int check_dims(const char* call, int head_dim, int rotary_dim, int q_heads, int k_heads) {
  if (head_dim <= 0 || head_dim % 16 || head_dim > 1024 || rotary_dim <= 0 || rotary_dim % 16 || rotary_dim > head_dim)
    return fail(PACE_KV_EINVAL, "%s: head_dim (up to 1024) and rotary_dim (up to head_dim) must be multiples of 16, got "
                "%d and %d", call, head_dim, rotary_dim);
  if (q_heads < 0 || k_heads < 0 || q_heads > (1 << 20) || k_heads > (1 << 20))
    return fail(PACE_KV_EINVAL, "%s: bad number of heads", call);
  return PACE_KV_OK;
}

}  // namespace
}  // namespace pace_kv

extern "C" {

int pace_kv_norm_rotate(const void* q, int64_t q_token_stride, int64_t q_head_stride, int q_heads, void* q_out,
                        int64_t q_out_token_stride, int64_t q_out_head_stride, const void* q_weight, const void* k,
                        int64_t k_token_stride, int64_t k_head_stride, int k_heads, void* k_out,
                        int64_t k_out_token_stride, int64_t k_out_head_stride, const void* k_weight, int elem_type,
                        int head_dim, int64_t nnz, const int32_t* positions, const float* table, int64_t table_rows,
                        int rotary_dim, int interleaved, float eps, int32_t* err_count, void* stream) {
  using namespace pace_kv;
  const char* const call = "norm_rotate";
  PACE_KV_TRY(check_dims(call, head_dim, rotary_dim, q_heads, k_heads));
  PACE_KV_TRY(check_turn(call, elem_type, nnz, positions, table, table_rows, eps));
  if (nnz == 0 || (q_heads == 0 && k_heads == 0)) return PACE_KV_OK;
  RopeParams p = {};
  p.q = Rows{static_cast<const char*>(q), q_token_stride, q_head_stride, static_cast<char*>(q_out), q_out_token_stride,
             q_out_head_stride, static_cast<const char*>(q_weight), static_cast<uint32_t>(q_heads)};
  p.k = Rows{static_cast<const char*>(k), k_token_stride, k_head_stride, static_cast<char*>(k_out), k_out_token_stride,
             k_out_head_stride, static_cast<const char*>(k_weight), static_cast<uint32_t>(k_heads)};
  PACE_KV_TRY(check_rows(call, p.q, true, static_cast<uint32_t>(head_dim)));
  PACE_KV_TRY(check_rows(call, p.k, true, static_cast<uint32_t>(head_dim)));
  p.positions = positions;
  p.table = table;
  p.table_rows = table_rows;
  p.err = err_count;
  p.nnz = nnz;
  p.eps = eps;
  p.page_size = 1;
  return launch_rope(p, elem_type, -1, head_dim, rotary_dim, interleaved, static_cast<hipStream_t>(stream));
}

int pace_kv_append_rope(const void* q, int64_t q_token_stride, int64_t q_head_stride, int q_heads, void* q_out,
                        int64_t q_out_token_stride, int64_t q_out_head_stride, const void* q_weight, const void* k,
                        int64_t k_token_stride, int64_t k_head_stride, const void* k_weight, const void* v,
                        int64_t v_token_stride, int64_t v_head_stride, int kv_heads, int elem_type, int head_dim,
                        int64_t nnz, const int32_t* positions, const int64_t* slot_mapping, const float* table,
                        int64_t table_rows, int rotary_dim, int interleaved, float eps, void* cache, int format,
                        int64_t num_pages, int page_size, int32_t* err_count, void* stream) {
  using namespace pace_kv;
  const char* const call = "append_rope";
  PACE_KV_TRY(check_dims(call, head_dim, rotary_dim, q_heads, kv_heads));
  PACE_KV_TRY(check_turn(call, elem_type, nnz, positions, table, table_rows, eps));
  if (kv_heads == 0) return fail(PACE_KV_EINVAL, "%s: no KV heads", call);
  if (format != PACE_KV_PLAIN && !is_mx_format(format)) return fail(PACE_KV_EINVAL, "%s: unknown format %d", call, format);
  if (format != PACE_KV_PLAIN && (head_dim % 64 || rotary_dim % 64))
    return fail(PACE_KV_EINVAL, "%s: a quantised cache takes head_dim and rotary_dim in multiples of 64", call);
  if (num_pages < 0 || num_pages > INT32_MAX || page_size <= 0)
    return fail(PACE_KV_EINVAL, "%s: bad number of pages or page size", call);
  if (nnz == 0) return PACE_KV_OK;
  if (!slot_mapping || (num_pages > 0 && !cache)) return fail(PACE_KV_EINVAL, "%s: NULL argument", call);
  if ((reinterpret_cast<uintptr_t>(cache) & 15u) || (reinterpret_cast<uintptr_t>(slot_mapping) & 7u))
    return fail(PACE_KV_EINVAL, "%s: the cache must be 16-byte aligned, slot_mapping 8-byte", call);
  RopeParams p = {};
  p.q = Rows{static_cast<const char*>(q), q_token_stride, q_head_stride, static_cast<char*>(q_out), q_out_token_stride,
             q_out_head_stride, static_cast<const char*>(q_weight), static_cast<uint32_t>(q_heads)};
  p.k = Rows{static_cast<const char*>(k), k_token_stride, k_head_stride, nullptr, 0, 0,
             static_cast<const char*>(k_weight), static_cast<uint32_t>(kv_heads)};
  p.v = Rows{static_cast<const char*>(v), v_token_stride, v_head_stride, nullptr, 0, 0, nullptr,
             static_cast<uint32_t>(kv_heads)};
  PACE_KV_TRY(check_rows(call, p.q, true, static_cast<uint32_t>(head_dim)));
  PACE_KV_TRY(check_rows(call, p.k, false, static_cast<uint32_t>(head_dim)));
  PACE_KV_TRY(check_rows(call, p.v, false, static_cast<uint32_t>(head_dim)));
  const int64_t half = static_cast<int64_t>(page_size) * kv_heads * head_dim;
  if (half >= int64_t(1) << 36) return fail(PACE_KV_ERANGE, "%s: pages of 2^36 elements or more", call);
  p.half_bytes = format == PACE_KV_PLAIN ? half * 2 : mx_half_bytes(half, format);
  if (p.half_bytes % 16) return fail(PACE_KV_EINVAL, "%s: half a page must be a multiple of 16 bytes", call);
  p.page_bytes = 2 * p.half_bytes;
  p.scale_at = format == PACE_KV_PLAIN ? 0 : half * mx_bits(format) / 8;
  p.positions = positions;
  p.slots = slot_mapping;
  p.table = table;
  p.table_rows = table_rows;
  p.cache = static_cast<char*>(cache);
  p.err = err_count;
  p.nnz = nnz;
  p.num_slots = num_pages * page_size;
  p.page_size = static_cast<uint32_t>(page_size);
  p.eps = eps;
  return launch_rope(p, elem_type, format, head_dim, rotary_dim, interleaved, static_cast<hipStream_t>(stream));
}

int pace_kv_append_latent(const void* latent, int64_t latent_stride, const void* rope_key, int64_t rope_stride,
                          const void* weight, int elem_type, int latent_dim, int64_t nnz, const int32_t* positions,
                          const int64_t* slot_mapping, const float* table, int64_t table_rows, int interleaved, float eps,
                          void* cache, int64_t num_pages, int page_size, int32_t* err_count, void* stream) {
  using namespace pace_kv;
  const char* const call = "append_latent";
  PACE_KV_TRY(check_turn(call, elem_type, nnz, positions, table, table_rows, eps));
  if (latent_dim != 256 && latent_dim != 512)
    return fail(PACE_KV_EINVAL, "%s: latent_dim must be 256 or 512, got %d", call, latent_dim);
  if (num_pages < 0 || num_pages > INT32_MAX || page_size <= 0)
    return fail(PACE_KV_EINVAL, "%s: bad number of pages or page size", call);
  if (nnz == 0) return PACE_KV_OK;
  if (!latent || !rope_key || !slot_mapping || (num_pages > 0 && !cache))
    return fail(PACE_KV_EINVAL, "%s: NULL argument", call);
  if (((reinterpret_cast<uintptr_t>(latent) | reinterpret_cast<uintptr_t>(rope_key) | reinterpret_cast<uintptr_t>(cache) |
        reinterpret_cast<uintptr_t>(weight) | static_cast<uintptr_t>(latent_stride | rope_stride)) & 15u) ||
      (reinterpret_cast<uintptr_t>(slot_mapping) & 7u))
    return fail(PACE_KV_EINVAL, "%s: rows, strides, weight and cache must be multiples of 16 bytes, slot_mapping of 8", call);
  const int64_t tokens = kThreads / (latent_dim / 8), groups = (nnz + tokens - 1) / tokens;
  if (groups > kMaxGroupsPerLaunch) return fail(PACE_KV_ERANGE, "%s: too many tokens for one call", call);
  LatentParams p = {};
  p.latent = static_cast<const char*>(latent);
  p.rope_key = static_cast<const char*>(rope_key);
  p.latent_stride = latent_stride;
  p.rope_stride = rope_stride;
  p.weight = static_cast<const char*>(weight);
  p.positions = positions;
  p.slots = slot_mapping;
  p.table = table;
  p.cache = static_cast<char*>(cache);
  p.err = err_count;
  p.nnz = nnz;
  p.table_rows = table_rows;
  p.num_slots = num_pages * page_size;
  p.eps = eps;
  void* args[] = {&p};
  const void* kernel = latent_dim == 512 ? pick_latent<512>(elem_type, interleaved != 0)
                                         : pick_latent<256>(elem_type, interleaved != 0);
  return hip_status(hipLaunchKernel(kernel, dim3(static_cast<uint32_t>(groups)), dim3(kThreads), args, 0,
                                    static_cast<hipStream_t>(stream)), "append_latent launch");
}

}  // extern "C"

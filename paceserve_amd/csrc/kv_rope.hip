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
#include <type_traits>

#include "mx.h"

namespace pace_kv {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
// Workgroups of a launch, whose threads are counted in 32 bits.
constexpr int64_t kMostGroups = int64_t(1) << 24;
// Rows of more bytes than this are loaded nontemporally: what a projection has just written
// is still in the memory-side cache where it is smaller.  MI355X, 40 heads of 128: 40 MiB
// 17.2 us plain, 18.6 so, 160 MiB 71 and 61.
constexpr int64_t kStreamBytes = int64_t(64) << 20;
// Latent rows of a call from which on a lane group takes two.  MI355X, 65536 rows of 576 numbers
// 45 us by one, 39 by two, 16384 10.4 and 10.0, 2000 3.4 and 3.8.
constexpr int64_t kManyRows = 8192;
// Waves that a token's heads are dealt to while there are fewer than this: the CUs hold 8192, and
// a wave's turns wait for their rows one after another.  MI355X, 8190 tokens of 48 heads into
// an 8-bit cache: by 8190 waves 53 us, by 16380 41, by 49140 42; 16384 tokens of 40 heads,
// rotated alone, 62 us by as many waves, 65 by four times as many.
constexpr int64_t kEnoughWaves = 16384;

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
  FastDiv by_page, by_parts;
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

// The sum over aligned groups of `lanes` lanes, in each of them: within rows of 16 by
// exchanges that need no LDS.
__device__ __forceinline__ float sum_of_group(float x, uint32_t lanes) {
  const auto moved = [](float v, auto control) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), decltype(control)::value, 0xf, 0xf, true));
  };
  if (lanes >= 2) x += moved(x, std::integral_constant<int, 0xB1>{});    // lane ^ 1
  if (lanes >= 4) x += moved(x, std::integral_constant<int, 0x4E>{});    // lane ^ 2
  if (lanes >= 8) x += moved(x, std::integral_constant<int, 0x141>{});   // the other four of eight
  if (lanes >= 16) x += moved(x, std::integral_constant<int, 0x140>{});  // the other eight of sixteen
  for (uint32_t k = 16; k < lanes; k *= 2) x += __shfl_xor(x, k);
  return x;
}

// Sum of the squares of a lane's runs.
template <class... R>
__device__ __forceinline__ float squares(const R&... runs) {
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) sum += (... + (runs[j] * runs[j]));
  return sum;
}

// 1 / sqrt(mean(x^2) + eps) of the rows whose runs lie with groups of `lanes` lanes.  The root's
// instruction takes normal numbers alone, and squares of numbers below 2^-63 are none.  Where eps
// would not hide those (below kLeastEps, which is the same for all lanes), rows whose mean square
// does not either are scaled by 2^100 first, in place: what is returned is for the scaled runs.
constexpr float kLeastEps = 0x1p-90f;

template <class... R>
__device__ __forceinline__ float inverse_root(uint32_t lanes, float inv_dim, float eps, R&... runs) {
  float sum = sum_of_group(squares(runs...), lanes);
  if (eps < kLeastEps) {
    const float up = sum * inv_dim + eps < kLeastEps ? 0x1p100f : 1.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) (..., (runs[j] *= up));
    sum = sum_of_group(squares(runs...), lanes);
    eps = eps * up * up;
  }
  return __builtin_amdgcn_rsqf(sum * inv_dim + eps);
}

// Written through the L2 at device scope.  The asm carries the wait states that a store of
// more than 64 bits needs before its data registers change.
__device__ __forceinline__ void put_vec(char* to, u32x4 v) {
  asm volatile("global_store_dwordx4 %0, %1, off sc1\n\ts_nop 1" : : "v"(to), "v"(v) : "memory");
}

template <bool STREAM>
__device__ __forceinline__ u32x4 load_vec(const char* x) {
  const u32x4* const at = reinterpret_cast<const u32x4*>(x);
  return STREAM ? __builtin_nontemporal_load(at) : *at;
}

// FORMAT: of the cache, or -1 without one.  STREAM: rows are loaded nontemporally.
template <int TYPE, int FORMAT, bool INTERLEAVED, bool STREAM>
__global__ __launch_bounds__(kThreads) void rope_kernel(const RopeParams p) {
  const uint32_t lane = threadIdx.x % 64;
  const uint32_t wave = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t whole = over(p.by_parts, wave), part = wave - whole * p.parts;
  const int64_t token = whole;
  if (token >= p.nnz) return;
  const int64_t position = p.positions[token];
  int64_t page_at = 0, slot = 0;
  if constexpr (FORMAT >= 0) slot = p.slots[token];
  const uint32_t group = 1u << p.group_log2, u = lane & (group - 1);
  const bool rotates = u < p.rotary / 16, active = u < p.units;
  // First elements of the lane's runs.
  const uint32_t tail = p.head_dim - p.rotary;
  const uint32_t ea = rotates ? 8 * u : p.rotary + 8 * (u - p.rotary / 16);
  const uint32_t eb = ea + (rotates ? p.rotary : tail) / 2;
  const uint32_t qk = p.q.heads + p.k.heads, heads = qk + (FORMAT >= 0 ? p.v.heads : 0u);
  const uint32_t end = min((part + 1) * p.part_heads, heads);
  const uint32_t turn = 64u >> p.group_log2;
  uint32_t h = part * p.part_heads + (lane >> p.group_log2);
  const auto load = [&](uint32_t h, u32x4& ra, u32x4& rb) {
    ra = rb = u32x4{0, 0, 0, 0};
    if (!active || h >= end) return;
    const Rows& rows = h < p.q.heads ? p.q : h < qk ? p.k : p.v;
    const uint32_t head = h < p.q.heads ? h : h < qk ? h - p.q.heads : h - qk;
    const char* const in = rows.in + token * rows.in_token + head * rows.in_head;
    ra = load_vec<STREAM>(in + ea * 2);
    rb = load_vec<STREAM>(in + eb * 2);
  };
  // On the way to a cache the first rows do not wait for the slot.  (MI355X, 8190 tokens of 48
  // heads into an 8-bit cache 41 us instead of 44; without a cache there is nothing to wait
  // for but the position, and 16384 tokens took 71 us instead of 62.)
  constexpr bool kEarly = FORMAT >= 0;
  u32x4 ra, rb;
  if (kEarly) load(h, ra, rb);
  const uint32_t h0 = h;
  if constexpr (FORMAT >= 0) {
    if (slot == -1) return;                              // padding
    if (slot < 0 || slot >= p.num_slots) {
      if (p.err != nullptr && part == 0 && lane == 0) atomicAdd(p.err, 1);
      return;
    }
    const int64_t page = slot <= UINT32_MAX ? over(p.by_page, static_cast<uint32_t>(slot)) : slot / p.page_size;
    slot -= page * p.page_size;
    page_at = page * p.page_bytes;
  }
  if (position < 0 || position >= p.table_rows) {
    if (p.err != nullptr && part == 0 && lane == 0) atomicAdd(p.err, 1);
    return;
  }
  float cos[8], sin[8];
  if (rotates) load_angles(p.table + position * p.rotary, p.rotary, INTERLEAVED, u, cos, sin);
  for (; h < end; h += turn) {
    const Rows& rows = h < p.q.heads ? p.q : h < qk ? p.k : p.v;
    const uint32_t head = h < p.q.heads ? h : h < qk ? h - p.q.heads : h - qk;
    if (!kEarly || h != h0) load(h, ra, rb);
    float a[8], b[8];
    if (h < qk) {
      widen<TYPE>(ra, a);
      widen<TYPE>(rb, b);
      if (rows.weight != nullptr) {
        const float inv = inverse_root(group, p.inv_dim, p.eps, a, b);
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
      put_vec(out + ea * 2, narrow<TYPE>(a));
      put_vec(out + eb * 2, narrow<TYPE>(b));
    } else if constexpr (FORMAT >= 0) {
      const int64_t element = (slot * p.k.heads + head) * p.head_dim;
      char* const half = p.cache + page_at + (h < qk ? 0 : p.half_bytes);
      if constexpr (FORMAT == PACE_KV_PLAIN) {
        put_vec(half + (element + ea) * 2, h < qk ? narrow<TYPE>(a) : ra);
        put_vec(half + (element + eb) * 2, h < qk ? narrow<TYPE>(b) : rb);
      } else {
        // Blocks of 32 are four neighbouring lanes' runs: rotary and tail are multiples of 64.
        // Half a page may be of any multiple of 34 or 66 bytes, so that runs lie at even bytes:
        // packed stores, the same instructions as aligned ones.
        constexpr int kBits = mx_bits(FORMAT);
        const auto put_run = [&](const float* x, const u32x4& v, uint32_t e) {
          char* const data = half + (element + e) * kBits / 8;
          char* const scale = half + p.scale_at + (element + e) / kMxBlock;
          if (h < qk) {
            const Run<PACE_KV_FP32> r = float_run(x);
            store_run<PACE_KV_FP32, FORMAT, false, true>(r, scale_byte<FORMAT>(block_amax<PACE_KV_FP32>(r)), data, scale);
          } else {
            Run<TYPE> r;
            r.v[0] = v;
            store_run<TYPE, FORMAT, false, true>(r, scale_byte<FORMAT>(block_amax<TYPE>(r)), data, scale);
          }
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

// L / 8 lanes take ROWS tokens: eight elements of each latent a lane, and four lanes
// a token two runs of its rotated part.
template <int L, int TYPE, bool INTERLEAVED, uint32_t ROWS>
__global__ __launch_bounds__(kThreads) void latent_rows_kernel(const LatentParams p) {
  constexpr uint32_t kLanes = L / 8, kTokens = kThreads / kLanes * ROWS;
  const uint32_t u = threadIdx.x % kLanes;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kTokens + threadIdx.x / kLanes * ROWS;
  // Everything that does not wait for a slot or a position is asked for first.
  const int64_t rope_token = first + u / 4;
  const bool ropes = u < 4 * ROWS && rope_token < p.nnz;
  u32x4 raw[ROWS], ra, rb;
  int64_t slot[ROWS], rope_slot = -1;
  int32_t position[ROWS], rope_position = -1;
#pragma unroll
  for (uint32_t k = 0; k < ROWS; ++k) {
    slot[k] = -1;
    position[k] = -1;
    raw[k] = u32x4{0, 0, 0, 0};
    const int64_t token = first + k;
    if (token >= p.nnz) continue;
    slot[k] = p.slots[token];
    position[k] = p.positions[token];
    raw[k] = *reinterpret_cast<const u32x4*>(p.latent + token * p.latent_stride + u * 16);
  }
  if (ropes) {
    const char* const in = p.rope_key + rope_token * p.rope_stride + u % 4 * 16;
    ra = *reinterpret_cast<const u32x4*>(in);
    rb = *reinterpret_cast<const u32x4*>(in + kRope);
  }
#pragma unroll
  for (uint32_t k = 0; k < ROWS; ++k) {
    if (slot[k] == -1) continue;                         // padding
    if (slot[k] < 0 || slot[k] >= p.num_slots || position[k] < 0 || position[k] >= p.table_rows) {
      if (p.err != nullptr && u == 0) atomicAdd(p.err, 1);
      slot[k] = -1;
    } else if (u / 4 == k) {
      rope_slot = slot[k];
      rope_position = position[k];
    }
  }
  if (rope_slot >= 0) {
    float a[8], b[8], cos[8], sin[8];
    load_angles(p.table + static_cast<int64_t>(rope_position) * kRope, kRope, INTERLEAVED, u % 4, cos, sin);
    widen<TYPE>(ra, a);
    widen<TYPE>(rb, b);
    rotate(INTERLEAVED, a, b, cos, sin);
    char* const row = p.cache + rope_slot * ((L + kRope) * 2) + L * 2 + u % 4 * 16;
    put_vec(row, narrow<TYPE>(a));
    put_vec(row + kRope, narrow<TYPE>(b));
  }
  float w[8];
  if (p.weight != nullptr) widen<TYPE>(*reinterpret_cast<const u32x4*>(p.weight + u * 16), w);
#pragma unroll
  for (uint32_t k = 0; k < ROWS; ++k) {
    if (p.weight != nullptr) {
      float x[8];
      widen<TYPE>(raw[k], x);
      const float inv = inverse_root(kLanes, 1.f / L, p.eps, x);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = x[j] * inv * w[j];
      raw[k] = narrow<TYPE>(x);
    }
    if (slot[k] >= 0) put_vec(p.cache + slot[k] * ((L + kRope) * 2) + u * 16, raw[k]);
  }
}

template <int TYPE, int FORMAT, bool STREAM>
const void* pick_rope(bool interleaved) {
  return interleaved ? reinterpret_cast<const void*>(&rope_kernel<TYPE, FORMAT, true, STREAM>)
                     : reinterpret_cast<const void*>(&rope_kernel<TYPE, FORMAT, false, STREAM>);
}

template <int TYPE, bool STREAM>
const void* pick_rope(int format, bool interleaved) {
  switch (format) {
    case -1: return pick_rope<TYPE, -1, STREAM>(interleaved);
    case PACE_KV_PLAIN: return pick_rope<TYPE, PACE_KV_PLAIN, STREAM>(interleaved);
    case PACE_KV_MXFP8: return pick_rope<TYPE, PACE_KV_MXFP8, STREAM>(interleaved);
    default: return pick_rope<TYPE, PACE_KV_MXFP4, STREAM>(interleaved);
  }
}

template <bool STREAM>
const void* pick_rope(int type, int format, bool interleaved) {
  return type == PACE_KV_BF16 ? pick_rope<PACE_KV_BF16, STREAM>(format, interleaved)
                              : pick_rope<PACE_KV_FP16, STREAM>(format, interleaved);
}

template <int L, int TYPE, uint32_t ROWS>
const void* pick_latent(bool interleaved) {
  return interleaved ? reinterpret_cast<const void*>(&latent_rows_kernel<L, TYPE, true, ROWS>)
                     : reinterpret_cast<const void*>(&latent_rows_kernel<L, TYPE, false, ROWS>);
}

template <int L>
const void* pick_latent(int type, bool interleaved, bool many) {
  if (type == PACE_KV_BF16)
    return many ? pick_latent<L, PACE_KV_BF16, 2>(interleaved) : pick_latent<L, PACE_KV_BF16, 1>(interleaved);
  return many ? pick_latent<L, PACE_KV_FP16, 2>(interleaved) : pick_latent<L, PACE_KV_FP16, 1>(interleaved);
}

int check_rows(const char* call, const Rows& r, bool writes, int64_t nnz, uint32_t head_dim) {
  if (r.heads == 0) return PACE_KV_OK;
  if (!r.in || (writes && !r.out)) return fail(PACE_KV_EINVAL, "%s: NULL rows", call);
  uintptr_t bits = reinterpret_cast<uintptr_t>(r.in) | static_cast<uintptr_t>(r.in_token | r.in_head) |
                   reinterpret_cast<uintptr_t>(r.weight);
  if (writes) bits |= reinterpret_cast<uintptr_t>(r.out) | static_cast<uintptr_t>(r.out_token | r.out_head);
  if (bits & 15u) return fail(PACE_KV_EINVAL, "%s: rows, weights and strides must be multiples of 16 bytes", call);
  if (writes && rows_overlap(nnz, r.out_token, r.heads, r.out_head, int64_t(2) * head_dim))
    return fail(PACE_KV_EINVAL, "%s: output rows overlap", call);
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
  // More than any launch takes; below, products of the number with heads and sizes fit 64 bits.
  if (nnz > INT32_MAX) return fail(PACE_KV_ERANGE, "%s: too many tokens for one call", call);
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
  while (per > 1 && p.nnz * ((turns + per - 1) / per) < kEnoughWaves) per = (per + 1) / 2;
  p.part_heads = per * turn;
  p.parts = (heads + p.part_heads - 1) / p.part_heads;
  const int64_t groups = (p.nnz * p.parts + kWaves - 1) / kWaves;
  if (groups >= kMostGroups) return fail(PACE_KV_ERANGE, "rope: too many tokens for one call");
  void* args[] = {&p};
  p.by_parts = fast_div(p.parts);
  p.by_page = fast_div(p.page_size);
  const bool streams = p.nnz * heads * head_dim * 2 > kStreamBytes;
  const void* kernel = streams ? pick_rope<true>(elem_type, format, interleaved != 0)
                              : pick_rope<false>(elem_type, format, interleaved != 0);
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

// packed: half a page may be of any size.
int append_rope(bool packed, const void* q, int64_t q_token_stride, int64_t q_head_stride, int q_heads, void* q_out,
                int64_t q_out_token_stride, int64_t q_out_head_stride, const void* q_weight, const void* k,
                int64_t k_token_stride, int64_t k_head_stride, const void* k_weight, const void* v,
                int64_t v_token_stride, int64_t v_head_stride, int kv_heads, int elem_type, int head_dim, int64_t nnz,
                const int32_t* positions, const int64_t* slot_mapping, const float* table, int64_t table_rows,
                int rotary_dim, int interleaved, float eps, void* cache, int format, int64_t num_pages, int page_size,
                int32_t* err_count, void* stream) {
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
  PACE_KV_TRY(check_rows(call, p.q, true, nnz, static_cast<uint32_t>(head_dim)));
  PACE_KV_TRY(check_rows(call, p.k, false, nnz, static_cast<uint32_t>(head_dim)));
  PACE_KV_TRY(check_rows(call, p.v, false, nnz, static_cast<uint32_t>(head_dim)));
  const int64_t half = static_cast<int64_t>(page_size) * kv_heads * head_dim;
  if (half >= int64_t(1) << 36) return fail(PACE_KV_ERANGE, "%s: pages of 2^36 elements or more", call);
  p.half_bytes = format == PACE_KV_PLAIN ? half * 2 : mx_half_bytes(half, format);
  if (!packed && p.half_bytes % 16)
    return fail(PACE_KV_EINVAL, "%s: half a page must be a multiple of 16 bytes", call);
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
  PACE_KV_TRY(check_rows(call, p.q, true, nnz, static_cast<uint32_t>(head_dim)));
  PACE_KV_TRY(check_rows(call, p.k, true, nnz, static_cast<uint32_t>(head_dim)));
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
  return pace_kv::append_rope(false, q, q_token_stride, q_head_stride, q_heads, q_out, q_out_token_stride,
                              q_out_head_stride, q_weight, k, k_token_stride, k_head_stride, k_weight, v,
                              v_token_stride, v_head_stride, kv_heads, elem_type, head_dim, nnz, positions,
                              slot_mapping, table, table_rows, rotary_dim, interleaved, eps, cache, format, num_pages,
                              page_size, err_count, stream);
}

int pace_kv_append_rope_packed(const void* q, int64_t q_token_stride, int64_t q_head_stride, int q_heads, void* q_out,
                               int64_t q_out_token_stride, int64_t q_out_head_stride, const void* q_weight,
                               const void* k, int64_t k_token_stride, int64_t k_head_stride, const void* k_weight,
                               const void* v, int64_t v_token_stride, int64_t v_head_stride, int kv_heads,
                               int elem_type, int head_dim, int64_t nnz, const int32_t* positions,
                               const int64_t* slot_mapping, const float* table, int64_t table_rows, int rotary_dim,
                               int interleaved, float eps, void* cache, int format, int64_t num_pages, int page_size,
                               int32_t* err_count, void* stream) {
  return pace_kv::append_rope(true, q, q_token_stride, q_head_stride, q_heads, q_out, q_out_token_stride,
                              q_out_head_stride, q_weight, k, k_token_stride, k_head_stride, k_weight, v,
                              v_token_stride, v_head_stride, kv_heads, elem_type, head_dim, nnz, positions,
                              slot_mapping, table, table_rows, rotary_dim, interleaved, eps, cache, format, num_pages,
                              page_size, err_count, stream);
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
  const bool many = nnz >= kManyRows;
  const int64_t tokens = kThreads / (latent_dim / 8) * (many ? 2 : 1), groups = (nnz + tokens - 1) / tokens;
  if (groups >= kMostGroups) return fail(PACE_KV_ERANGE, "%s: too many tokens for one call", call);
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
  const void* kernel = latent_dim == 512 ? pick_latent<512>(elem_type, interleaved != 0, many)
                                         : pick_latent<256>(elem_type, interleaved != 0, many);
  return hip_status(hipLaunchKernel(kernel, dim3(static_cast<uint32_t>(groups)), dim3(kThreads), args, 0,
                                    static_cast<hipStream_t>(stream)), "append_latent launch");
}

}  // extern "C"

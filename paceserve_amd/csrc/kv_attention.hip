// Attention of each request's last tokens over its pages: single tokens of a
// decode step, or a tree of drafted tokens, over a 16-bit or a quantised cache.
//
//   request b: kv_len tokens in pages kv_indices[kv_indptr[b] .. kv_indptr[b+1]),
//   its last q_len are the queries; base = kv_len - q_len.
//   query i sees position t < base, and t = base + j where bit j of its mask row
//   is set (no mask: j <= i).
//   s = scale * q . k, or cap * tanh(scale * q . k / cap);  o = softmax(s) v
//
// One pass over the keys and values with a running maximum m, sum l and
// unnormalised output per query row (float32).  The queries of one KV head,
// q_len * group rows, share every key and value that a workgroup loads.
// Scores are computed transposed, S^T = K Q^T (v_mfma_f32_16x16x32: lane holds
// four tokens of one query), so that a lane's exponentials are already the
// operand of O^T = V^T P^T: its four tokens of two 16-token tiles are eight
// consecutive entries of the product's k, for which V's rows are read in the
// same order through the transposing LDS read.  P is rounded to the values'
// type for the product (within 2^-8 of each weight in bfloat16, 2^-11 in float16,
// errors that average out over the row); l sums the unrounded weights.
//
// Work split: a request's pages in chunks of C; chunk k of request b is work
// item floor(kv_indptr[b] / C) + b + k, which a workgroup inverts by counting
// the requests that start at or before its item, so a launch needs no plan and
// a captured one follows the tables.  A request of one chunk is written
// directly; the others leave (o, m, l) in a workspace for combine_kernel.
#include "mx.h"

namespace pace_kv {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = 4;
constexpr int kXcds = 8;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

struct AttnParams {
  const char* q;
  int64_t q_stride;            // bytes between tokens
  const int32_t* qo_indptr;    // batch + 1 entries, or nullptr: one token per request
  const char* cache;
  const int32_t* kv_indices;
  const int32_t* kv_indptr;
  const int32_t* kv_last_page_len;
  const uint64_t* mask;        // [nnz, mask_words], or nullptr
  char* out;
  int64_t out_stride;
  float* lse;                  // [nnz, heads * group], or nullptr
  float* part_o;               // [items, heads, row_tiles, rows of a tile, D]
  float* part_ml;              // [items, heads, row_tiles, rows of a tile, 2]
  int32_t* err;
  uint32_t num_indices, batch, nnz, heads, group, num_pages, page_size, max_q, mask_words;
  uint32_t chunk_pages, items, row_tiles, tile_rows;
  uint32_t page16, half16, row16;  // page, half page and token row, in 16-byte units
  uint32_t scale_at, scale_row;    // scales within a half page, scale bytes of a token
  FastDiv by_page, by_chunk, by_group, by_unit, by_tiles;
  float scale_log2;            // scale * log2(e); with a cap: scale / cap * 2 * log2(e)
  float cap_log2;              // cap * log2(e), or 0
};

// Swaps of half a wave and of neighbouring rows of 16 lanes bring the four
// lanes of one query together.
template <class F>
__device__ __forceinline__ float across_groups(float x, F f) {
  const uint32_t b = __float_as_uint(x);
  auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  const uint32_t y = __float_as_uint(f(__uint_as_float(r[0]), __uint_as_float(r[1])));
  r = __builtin_amdgcn_permlane16_swap(y, y, false, false);
  return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max_of(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ float sum_of(float a, float b) { return a + b; }

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// A request and the part of it that a work item covers.
struct Request {
  uint32_t b, chunk, chunks;
  int32_t first_page;          // in kv_indices
  uint32_t pages;
  uint32_t kv_len;
  uint32_t q0, q_len;
};

__device__ __forceinline__ uint32_t item_of(const AttnParams& p, uint32_t b, int32_t first) {
  return over(p.by_chunk, static_cast<uint32_t>(max(first, 0))) + b;
}

// The sizes of request b; false where its queries are not nnz's or exceed max_q.
__device__ __forceinline__ bool request_of(const AttnParams& p, uint32_t b, Request* r) {
  const int32_t k0 = max(p.kv_indptr[b], 0), k1 = p.kv_indptr[b + 1];
  r->b = b;
  r->first_page = k0;
  r->pages = k1 > k0 ? static_cast<uint32_t>(k1 - k0) : 0u;
  r->pages = min(r->pages, p.num_indices - min(static_cast<uint32_t>(k0), p.num_indices));
  const int64_t most = static_cast<int64_t>(r->pages) * p.page_size;
  const int64_t len = (most > p.page_size ? most - p.page_size : 0) + p.kv_last_page_len[b];
  r->kv_len = static_cast<uint32_t>(min(max(len, int64_t(0)), most));
  const uint32_t n = over(p.by_chunk, r->pages);
  r->chunks = max(n * p.chunk_pages < r->pages ? n + 1 : n, 1u);
  if (p.qo_indptr == nullptr) {
    r->q0 = b;
    r->q_len = 1;
    return b < p.nnz;
  }
  const int32_t a0 = p.qo_indptr[b], a1 = p.qo_indptr[b + 1];
  r->q0 = static_cast<uint32_t>(a0);
  r->q_len = static_cast<uint32_t>(a1 - a0);
  return a0 >= 0 && a1 >= a0 && static_cast<uint32_t>(a1) <= p.nnz && r->q_len <= p.max_q;
}

// Largest b with f(b) <= x where f does not decrease, plus one; the wave counts
// together, 64 entries a round.
template <class F>
__device__ __forceinline__ uint32_t count_upto(uint32_t n, uint32_t x, F f) {
  uint32_t count = 0;
  for (uint32_t e0 = 0; e0 < n; e0 += 64) {
    const uint32_t e = e0 + threadIdx.x % 64;
    count += __popcll(__ballot(e < n && f(e) <= x));
  }
  return __builtin_amdgcn_readfirstlane(count);
}

template <int D>
__device__ __forceinline__ uint32_t lds_at(uint32_t row, uint32_t c) {
  // 16-byte chunk c of a row.  The xor spreads a column of rows over the banks
  // (256 bytes: two rows of 64 elements, one of 128).
  const uint32_t x = D == 64 ? (row >> 1) & 7u : row & 15u;
  return row * (D * 2) + ((c ^ x) * 16);
}

template <int TYPE>
__device__ __forceinline__ f32x4 mfma(const u32x4& a, const u32x4& b, const f32x4& c) {
  if constexpr (TYPE == PACE_KV_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
}

template <int TYPE>
__device__ __forceinline__ uint32_t pair_of(float a, float b) {
  if constexpr (TYPE == PACE_KV_BF16) {
    const bf16x2 x = {static_cast<__bf16>(a), static_cast<__bf16>(b)};
    return __builtin_bit_cast(uint32_t, x);
  } else {
    const f16x2 x = {static_cast<_Float16>(a), static_cast<_Float16>(b)};
    return __builtin_bit_cast(uint32_t, x);
  }
}

template <int TYPE>
__device__ __forceinline__ float value_of(uint32_t word, int half) {
  const unsigned short h = static_cast<unsigned short>(word >> (16 * half));
  if constexpr (TYPE == PACE_KV_BF16) return __uint_as_float(static_cast<uint32_t>(h) << 16);
  else return static_cast<float>(__builtin_bit_cast(_Float16, h));
}

// Whether either half of a word is an infinity or a NaN.
template <int TYPE>
__device__ __forceinline__ bool odd_word(uint32_t w) {
  constexpr uint32_t kExp = TYPE == PACE_KV_BF16 ? 0x7f80u : 0x7c00u;
  return (w & kExp) == kExp || ((w >> 16) & kExp) == kExp;
}

// TYPE: of queries and output, and what a quantised cache is expanded to.
// R tiles of 16 query rows per wave.  WR = 1: the waves take 32 tokens each of
// a step and join at the end.  WR = 4: each wave takes its own 16 * R rows, and
// all share a tile of 64 tokens.
template <int D, int TYPE, int FORMAT, int R, int WR>
__global__ __launch_bounds__(kThreads) void attention_kernel(const AttnParams p) {
  constexpr int kBits = FORMAT == PACE_KV_PLAIN ? 16 : mx_bits(FORMAT);
  constexpr int kWT = kWaves / WR;
  constexpr uint32_t kTileRows = 16 * R * WR;
  constexpr uint32_t kIdTokens = WR == 1 ? 32 : 64;      // tokens whose pages a wave looks up
  constexpr uint32_t kStep = kIdTokens * kWT;            // tokens of a workgroup's step
  constexpr uint32_t kLoadRows = WR == 1 ? 32 : 16;      // rows that a wave loads
  constexpr uint32_t kPieces = D * kBits / 8 / 16;       // 16-byte pieces of a row
  constexpr uint32_t kLoads = (kLoadRows * kPieces + 63) / 64;
  constexpr uint32_t kLdsRows = WR == 1 ? 128 : 64;
  constexpr int kDT = D / 16, kKS = D / 32;

  __shared__ __attribute__((aligned(16))) char lds[2 * kLdsRows * D * 2];
  __shared__ float lds_ml[kWaves][kTileRows][2];

  const uint32_t lane = threadIdx.x % 64, g = lane / 16, n = lane % 16;
  const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);

  // The heads and row tiles of one item run on one XCD, whose L2 then holds
  // what they share.
  const uint32_t unit = p.heads * p.row_tiles;
  const uint32_t at = blockIdx.x / kXcds, nth = over(p.by_unit, at);
  const uint32_t item = nth * kXcds + blockIdx.x % kXcds;
  if (item >= p.items) return;
  const uint32_t in_unit = at - nth * unit, head = over(p.by_tiles, in_unit), tile = in_unit - head * p.row_tiles;
  const uint32_t count = count_upto(p.batch, item, [&](uint32_t e) { return item_of(p, e, p.kv_indptr[e]); });
  if (count == 0) return;
  Request r;
  const bool valid_request = request_of(p, count - 1, &r);
  r.chunk = item - item_of(p, r.b, r.first_page);
  if (r.chunk >= r.chunks) return;
  if (!valid_request) {
    if (r.chunk == 0 && in_unit == 0 && threadIdx.x == 0 && p.err != nullptr) atomicAdd(p.err, 1);
    return;
  }
  const uint32_t rows = r.q_len * p.group, row0 = tile * kTileRows;
  if (row0 >= rows) return;
  const int32_t base = static_cast<int32_t>(r.kv_len) - static_cast<int32_t>(r.q_len);
  // Without a mask no row of the tile sees past its last query.
  const int32_t first_q = static_cast<int32_t>(over(p.by_group, row0));
  const int32_t last_q = static_cast<int32_t>(over(p.by_group, min(row0 + kTileRows, rows) - 1));
  const int32_t chunk_tokens = static_cast<int32_t>(p.chunk_pages * p.page_size);
  const int32_t t_begin = static_cast<int32_t>(r.chunk) * chunk_tokens;
  int32_t t_end = static_cast<int32_t>(min(static_cast<int64_t>(t_begin) + chunk_tokens, static_cast<int64_t>(r.kv_len)));
  if (p.mask == nullptr) t_end = min(t_end, base + last_q + 1);

  // Query fragments: row n of each tile, eight elements from 32 * ks + 8 * g.
  const uint32_t wave_row0 = row0 + (WR == 1 ? 0 : w * 16 * R);
  u32x4 qf[R][kKS];
  int32_t qi[R];
#pragma unroll
  for (int a = 0; a < R; ++a) {
    const uint32_t row = wave_row0 + a * 16 + n;
    const uint32_t i = over(p.by_group, row);
    qi[a] = static_cast<int32_t>(i);
    const char* src = p.q + static_cast<int64_t>(r.q0 + i) * p.q_stride +
                      (static_cast<int64_t>(head) * p.group + (row - i * p.group)) * (D * 2);
#pragma unroll
    for (int k = 0; k < kKS; ++k) {
      qf[a][k] = u32x4{0, 0, 0, 0};
      if (row < rows) qf[a][k] = *reinterpret_cast<const u32x4*>(src + k * 64 + g * 16);
    }
  }

  f32x4 acc[R][kDT];
  float m[R], l[R];
#pragma unroll
  for (int a = 0; a < R; ++a) {
    m[a] = -INFINITY;
    l[a] = 0.f;
#pragma unroll
    for (int d = 0; d < kDT; ++d) acc[a][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  char* const lds_k = lds;
  char* const lds_v = lds + kLdsRows * D * 2;
  const uint32_t lds_row0 = w * kLoadRows;               // first row that this wave loads

  // A step's loads: page ids (one token per lane), then rows.
  const uint32_t id_lane = lane % kIdTokens;
  int32_t id = 0;
  const auto load_id = [&](int32_t t0) {
    const int32_t t = t0 + static_cast<int32_t>(id_lane);
    id = -1;
    if (t < t_end) id = p.kv_indices[r.first_page + static_cast<int32_t>(over(p.by_page, static_cast<uint32_t>(t)))];
  };
  u32x4 kr[kLoads], vr[kLoads];
  uint64_t ks_byte = 0, vs_byte = 0;                     // the scales of the lane's token
  uint64_t valid = 0;
  const auto load_rows = [&](int32_t t0) {
    const uint32_t t = static_cast<uint32_t>(t0) + id_lane;
    const bool ok = t0 + static_cast<int32_t>(id_lane) < t_end && static_cast<uint32_t>(id) < p.num_pages;
    valid = __ballot(ok);
    if (kIdTokens == 32) valid &= 0xffffffffull;
    const uint32_t slot = t - over(p.by_page, t) * p.page_size;
    const uint32_t off = ok ? static_cast<uint32_t>(id) * p.page16 + slot * p.row16 + head * (D * kBits / 128) : ~0u;
    if constexpr (FORMAT != PACE_KV_PLAIN) {
      ks_byte = vs_byte = 0;
      if (ok && id_lane / kLoadRows == (WR == 1 ? 0 : w)) {
        const char* s = p.cache + static_cast<int64_t>(id) * p.page16 * 16 + p.scale_at +
                        static_cast<int64_t>(slot) * p.scale_row + head * (D / 32);
        const char* sv = s + static_cast<int64_t>(p.half16) * 16;
        if constexpr (D == 64) {
          ks_byte = *reinterpret_cast<const uint16_t*>(s);
          vs_byte = *reinterpret_cast<const uint16_t*>(sv);
        } else if constexpr (D == 128) {
          ks_byte = *reinterpret_cast<const uint32_t*>(s);
          vs_byte = *reinterpret_cast<const uint32_t*>(sv);
        } else {
          ks_byte = *reinterpret_cast<const uint64_t*>(s);
          vs_byte = *reinterpret_cast<const uint64_t*>(sv);
        }
      }
    }
#pragma unroll
    for (uint32_t j = 0; j < kLoads; ++j) {
      const uint32_t piece = j * 64 + lane, row = piece / kPieces, c = piece % kPieces;
      const uint32_t o = __shfl(off, (WR == 1 ? 0 : w * kLoadRows) + row % kLoadRows);
      kr[j] = vr[j] = u32x4{0, 0, 0, 0};
      if (o != ~0u && row < kLoadRows) {
        const char* s = p.cache + (static_cast<int64_t>(o) + c) * 16;
        kr[j] = *reinterpret_cast<const u32x4*>(s);
        vr[j] = *reinterpret_cast<const u32x4*>(s + static_cast<int64_t>(p.half16) * 16);
      }
    }
  };
  const auto store_piece = [&](char* to, uint32_t row, uint32_t c, const u32x4& x, uint64_t bytes) {
    if constexpr (FORMAT == PACE_KV_PLAIN) {
      *reinterpret_cast<u32x4*>(to + lds_at<D>(row, c)) = x;
    } else if constexpr (FORMAT == PACE_KV_MXFP8) {      // 16 elements: half a block
      const float s = scale_of(static_cast<uint32_t>(bytes >> (c / 2 * 8)) & 255u);
      *reinterpret_cast<u32x4*>(to + lds_at<D>(row, 2 * c)) = run_up<TYPE, FORMAT>(u32x2{x[0], x[1]}, s);
      *reinterpret_cast<u32x4*>(to + lds_at<D>(row, 2 * c + 1)) = run_up<TYPE, FORMAT>(u32x2{x[2], x[3]}, s);
    } else {                                             // 32 elements: a block
      const float s = scale_of(static_cast<uint32_t>(bytes >> (c * 8)) & 255u);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        *reinterpret_cast<u32x4*>(to + lds_at<D>(row, 4 * c + k)) = run_up<TYPE, FORMAT>(u32x2{x[k], 0}, s);
    }
  };
  const auto store_rows = [&]() {
#pragma unroll
    for (uint32_t j = 0; j < kLoads; ++j) {
      const uint32_t piece = j * 64 + lane, row = piece / kPieces, c = piece % kPieces;
      uint64_t kb = 0, vb = 0;
      if constexpr (FORMAT != PACE_KV_PLAIN) {
        const uint32_t from = (WR == 1 ? 0 : w * kLoadRows) + row % kLoadRows;
        kb = static_cast<uint32_t>(__shfl(static_cast<uint32_t>(ks_byte), from));
        vb = static_cast<uint32_t>(__shfl(static_cast<uint32_t>(vs_byte), from));
        if constexpr (D == 256) {
          kb |= static_cast<uint64_t>(__shfl(static_cast<uint32_t>(ks_byte >> 32), from)) << 32;
          vb |= static_cast<uint64_t>(__shfl(static_cast<uint32_t>(vs_byte >> 32), from)) << 32;
        }
      }
      if (row < kLoadRows) {
        store_piece(lds_k, lds_row0 + row, c, kr[j], kb);
        store_piece(lds_v, lds_row0 + row, c, vr[j], vb);
      }
    }
  };

  // Which of the 32 tokens from t0 query row a sees (bit i: token t0 + i).
  const auto seen = [&](int32_t t0, int32_t query) -> uint32_t {
    const int32_t d0 = t0 - base;                        // drafted token of bit 0, negative: before them
    if (p.mask == nullptr) {
      const int32_t upto = query - d0 + 1;
      return upto >= 32 ? ~0u : upto <= 0 ? 0u : (1u << upto) - 1u;
    }
    if (d0 <= -32) return ~0u;
    if (query >= static_cast<int32_t>(r.q_len)) return 0u;   // a row of padding
    const uint64_t* bits = p.mask + static_cast<int64_t>(r.q0 + static_cast<uint32_t>(query)) * p.mask_words;
    if (d0 < 0) return static_cast<uint32_t>(bits[0] << -d0) | ((1u << -d0) - 1u);
    const uint32_t word = static_cast<uint32_t>(d0) / 64, sh = static_cast<uint32_t>(d0) % 64;
    uint64_t x = word < p.mask_words ? bits[word] >> sh : 0ull;
    if (sh > 32 && word + 1 < p.mask_words) x |= bits[word + 1] << (64 - sh);
    return static_cast<uint32_t>(x);
  };

  // 32 tokens from t0 whose rows lie at lds_row; `ok`: the tokens that exist.
  const auto attend = [&](int32_t t0, uint32_t lds_row, uint32_t ok) {
    f32x4 s[R][2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int a = 0; a < R; ++a) s[a][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < kKS; ++k) {
        const u32x4 kf = *reinterpret_cast<const u32x4*>(lds_k + lds_at<D>(lds_row + t * 16 + n, k * 4 + g));
#pragma unroll
        for (int a = 0; a < R; ++a) s[a][t] = mfma<TYPE>(kf, qf[a][k], s[a][t]);
      }
    }
    const bool full = ok == ~0u && (t0 + 32 <= base || (p.mask == nullptr && t0 + 31 <= base + first_q));
    bool odd = false;                                    // an infinite or NaN value that some row must not see
    uint32_t sees[R];
    if (!full) {
#pragma unroll
      for (int a = 0; a < R; ++a) sees[a] = seen(t0, qi[a]) & ok;
      bool found = false;
#pragma unroll
      for (uint32_t k = 0; k < 32 * D / 8 / 64; ++k) {
        const uint32_t c = k * 64 + lane;
        const u32x4 x = *reinterpret_cast<const u32x4*>(lds_v + lds_at<D>(lds_row + c / (D / 8), c % (D / 8)));
#pragma unroll
        for (int e = 0; e < 4; ++e) found |= odd_word<TYPE>(x[e]);
      }
      odd = __ballot(found) != 0;
    }
    u32x4 pf[R];
#pragma unroll
    for (int a = 0; a < R; ++a) {
      float x[8];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float y = s[a][t][e] * p.scale_log2;
          // tanh(z) = 1 - 2 / (1 + 2^(2 log2(e) z))
          if (p.cap_log2 > 0.f) y = p.cap_log2 * (1.f - 2.f * __builtin_amdgcn_rcpf(1.f + exp2_of(y)));
          if (!full && !((sees[a] >> (t * 16 + 4 * g + e)) & 1u)) y = -INFINITY;
          x[t * 4 + e] = y;
        }
      float top = x[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) top = fmaxf(top, x[e]);
      top = fmaxf(m[a], across_groups(top, max_of));
      const float from = top == -INFINITY ? 0.f : top;   // nothing seen yet: weights of 2^-inf = 0
      const float shrink = exp2_of(m[a] - from);
      m[a] = top;
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = exp2_of(x[e] - from);
        sum += x[e];
      }
      l[a] = l[a] * shrink + sum;
#pragma unroll
      for (int e = 0; e < 4; ++e) pf[a][e] = pair_of<TYPE>(x[2 * e], x[2 * e + 1]);
      if (__ballot(shrink != 1.f) != 0) {
#pragma unroll
        for (int d = 0; d < kDT; ++d) acc[a][d] *= shrink;
      }
    }
    if (!odd) {
#pragma unroll
      for (int d = 0; d < kDT; ++d) {
        // Lane: row 4 g + n / 4 of each 16 tokens, four columns; transposed over
        // 16 lanes: four tokens of column n.
        const uint32_t row = lds_row + 4 * g + n / 4, c = d * 2 + n % 4 / 2;
        typedef __attribute__((address_space(3))) s16x4* lds_ptr;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_ptr)(lds_v + lds_at<D>(row, c) + n % 2 * 8));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_ptr)(lds_v + lds_at<D>(row + 16, c) + n % 2 * 8));
        const u32x2 lo2 = __builtin_bit_cast(u32x2, lo), hi2 = __builtin_bit_cast(u32x2, hi);
        const u32x4 vf = {lo2[0], lo2[1], hi2[0], hi2[1]};
#pragma unroll
        for (int a = 0; a < R; ++a) acc[a][d] = mfma<TYPE>(vf, pf[a], acc[a][d]);
      }
    } else {
      // A product with weight zero would spread an infinity or a NaN to rows
      // that do not see its token: the same sum, token by token, over those seen.
#pragma unroll
      for (int a = 0; a < R; ++a)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          for (uint32_t go = 0; go < 4; ++go) {
            const uint32_t token = e / 4 * 16 + go * 4 + e % 4;
            const float weight = value_of<TYPE>(__shfl(pf[a][e / 2], go * 16 + n), e % 2);
            if (!((sees[a] >> token) & 1u)) continue;
#pragma unroll
            for (int d = 0; d < kDT; ++d) {
              const u32x2 v = *reinterpret_cast<const u32x2*>(lds_v + lds_at<D>(lds_row + token, d * 2 + g / 2) +
                                                              g % 2 * 8);
#pragma unroll
              for (int c = 0; c < 4; ++c) acc[a][d][c] += weight * value_of<TYPE>(v[c / 2], c % 2);
            }
          }
    }
  };

  const int32_t wave_t0 = t_begin + (WR == 1 ? static_cast<int32_t>(w * kIdTokens) : 0);
  load_id(wave_t0);
  load_rows(wave_t0);
  load_id(wave_t0 + static_cast<int32_t>(kStep));
  for (int32_t t0 = t_begin; t0 < t_end; t0 += static_cast<int32_t>(kStep)) {
    const int32_t tw = t0 + (wave_t0 - t_begin);
    if (WR != 1) __syncthreads();                        // the last step's reads are done
    store_rows();
    const uint64_t ok = valid;
    if (WR != 1) __syncthreads();
    else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    load_rows(tw + static_cast<int32_t>(kStep));
    load_id(tw + 2 * static_cast<int32_t>(kStep));
    __builtin_amdgcn_sched_barrier(0);
    if (WR == 1) {
      if (ok != 0) attend(tw, lds_row0, static_cast<uint32_t>(ok));
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    } else {
      if (static_cast<uint32_t>(ok) != 0) attend(t0, 0, static_cast<uint32_t>(ok));
      if (static_cast<uint32_t>(ok >> 32) != 0) attend(t0 + 32, 32, static_cast<uint32_t>(ok >> 32));
    }
  }
#pragma unroll
  for (int a = 0; a < R; ++a) l[a] = across_groups(l[a], sum_of);

  const bool direct = r.chunks == 1;
  const int64_t part_row0 = (static_cast<int64_t>(item) * unit + in_unit) * kTileRows;
  // Row `in_tile` of the tile: four output columns from d, and its m and l.
  const auto write = [&](uint32_t in_tile, uint32_t d, f32x4 o, float top, float sum, bool first) {
    const uint32_t row = row0 + in_tile;
    if (row >= rows) return;
    if (!direct) {
      *reinterpret_cast<f32x4*>(p.part_o + (part_row0 + in_tile) * D + d) = o;
      if (first) {
        p.part_ml[(part_row0 + in_tile) * 2] = top;
        p.part_ml[(part_row0 + in_tile) * 2 + 1] = sum;
      }
      return;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const uint32_t i = over(p.by_group, row);
    const uint32_t qh = head * p.group + (row - i * p.group);
    const u32x2 x = {pair_of<TYPE>(o[0] * inv, o[1] * inv), pair_of<TYPE>(o[2] * inv, o[3] * inv)};
    *reinterpret_cast<u32x2*>(p.out + static_cast<int64_t>(r.q0 + i) * p.out_stride +
                              (static_cast<int64_t>(qh) * D + d) * 2) = x;
    if (first && p.lse != nullptr)
      p.lse[static_cast<int64_t>(r.q0 + i) * p.heads * p.group + qh] =
          sum == 0.f ? -INFINITY : (top + __log2f(sum)) * 0.69314718055994531f;
  };
  if (WR != 1) {
#pragma unroll
    for (int a = 0; a < R; ++a)
#pragma unroll
      for (int d = 0; d < kDT; ++d) write(w * 16 * R + a * 16 + n, d * 16 + g * 4, acc[a][d], m[a], l[a], d == 0 && g == 0);
    return;
  }
  // The waves' parts of a row join over their common maximum.
  __syncthreads();
  float* part = reinterpret_cast<float*>(lds);           // [wave][row][D], chunks of 4 xored with the row
#pragma unroll
  for (int a = 0; a < R; ++a) {
    const uint32_t row = a * 16 + n;
    if (g == 0) {
      lds_ml[w][row][0] = m[a];
      lds_ml[w][row][1] = l[a];
    }
#pragma unroll
    for (int d = 0; d < kDT; ++d)
      *reinterpret_cast<f32x4*>(part + (w * kTileRows + row) * D + ((d * 4 + g) ^ n) * 4) = acc[a][d];
  }
  __syncthreads();
  for (uint32_t e = threadIdx.x; e < kTileRows * (D / 4); e += kThreads) {
    const uint32_t row = e / (D / 4), c = e % (D / 4);
    float top = -INFINITY;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) top = fmaxf(top, lds_ml[v][row][0]);
    const float from = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int v = 0; v < kWaves; ++v) {
      const float weight = exp2_of(lds_ml[v][row][0] - from);
      sum += weight * lds_ml[v][row][1];
      o += weight * *reinterpret_cast<const f32x4*>(part + (v * kTileRows + row) * D + (c ^ (row & 15u)) * 4);
    }
    write(row, c * 4, o, top, sum, c == 0);
  }
}

// Joins the chunks of each row (token, head): a workgroup per row, its threads
// D / 4 columns of four by as many chunks at a time as fit.
template <int D, int TYPE>
__global__ __launch_bounds__(kThreads) void combine_kernel(const AttnParams p) {
  constexpr uint32_t kCols = D / 4, kGroups = kThreads / kCols;
  __shared__ f32x4 lds_o[kGroups][kCols];
  __shared__ float lds_l[kGroups], lds_m[kGroups];
  const uint32_t all_heads = p.heads * p.group;
  const uint32_t token = blockIdx.x / all_heads, qh = blockIdx.x % all_heads;
  uint32_t b = token;
  if (p.qo_indptr != nullptr) {
    const uint32_t count =
        count_upto(p.batch, token, [&](uint32_t e) { return static_cast<uint32_t>(max(p.qo_indptr[e], 0)); });
    if (count == 0) return;
    b = count - 1;
  }
  if (b >= p.batch) return;
  Request r;
  if (!request_of(p, b, &r) || token < r.q0 || token - r.q0 >= r.q_len || r.chunks == 1) return;
  const uint32_t head = over(p.by_group, qh), row = (token - r.q0) * p.group + (qh - head * p.group);
  const uint32_t tile = row / p.tile_rows;
  const int64_t unit = static_cast<int64_t>(p.heads) * p.row_tiles;
  const int64_t first = (static_cast<int64_t>(item_of(p, b, r.first_page)) * unit +
                         static_cast<int64_t>(head) * p.row_tiles + tile) * p.tile_rows + row % p.tile_rows;
  const int64_t step = unit * p.tile_rows;
  const uint32_t col = threadIdx.x % kCols, part = threadIdx.x / kCols;
  float m = -INFINITY, l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (uint32_t c = part; c < r.chunks; c += kGroups) {
    const int64_t at = first + c * step;
    const float mc = p.part_ml[at * 2], lc = p.part_ml[at * 2 + 1];
    const f32x4 oc = *reinterpret_cast<const f32x4*>(p.part_o + at * D + col * 4);
    const float top = fmaxf(m, mc), from = top == -INFINITY ? 0.f : top;
    const float a = exp2_of(m - from), d = exp2_of(mc - from);
    l = l * a + lc * d;
    o = o * a + oc * d;
    m = top;
  }
  lds_o[part][col] = o;
  if (col == 0) {
    lds_m[part] = m;
    lds_l[part] = l;
  }
  __syncthreads();
  if (part != 0) return;
  float top = -INFINITY;
#pragma unroll
  for (uint32_t v = 0; v < kGroups; ++v) top = fmaxf(top, lds_m[v]);
  const float from = top == -INFINITY ? 0.f : top;
  l = 0.f;
  o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (uint32_t v = 0; v < kGroups; ++v) {
    const float weight = exp2_of(lds_m[v] - from);
    l += weight * lds_l[v];
    o += weight * lds_o[v][col];
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const u32x2 x = {pair_of<TYPE>(o[0] * inv, o[1] * inv), pair_of<TYPE>(o[2] * inv, o[3] * inv)};
  *reinterpret_cast<u32x2*>(p.out + static_cast<int64_t>(token) * p.out_stride +
                            (static_cast<int64_t>(qh) * D + col * 4) * 2) = x;
  if (col == 0 && p.lse != nullptr)
    p.lse[static_cast<int64_t>(token) * all_heads + qh] =
        l == 0.f ? -INFINITY : (top + __log2f(l)) * 0.69314718055994531f;
}

// How a call is cut up.
struct Split {
  uint32_t tile_rows, row_tiles, chunk_pages, items;
  bool by_rows;
  int64_t part_rows() const { return static_cast<int64_t>(items) * row_tiles * tile_rows; }  // times the KV heads
};

constexpr int64_t kTargetGroups = 1024;  // workgroups that a long context is split over
constexpr int64_t kMinChunkTokens = 256;

Split split_of(int64_t batch, int64_t heads, int64_t group, int64_t max_q, int64_t num_indices, int64_t page_size) {
  Split s = {};
  const int64_t rows = max_q * group;
  s.by_rows = rows > 32;
  s.tile_rows = rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : 128;
  s.row_tiles = static_cast<uint32_t>((rows + s.tile_rows - 1) / s.tile_rows);
  const int64_t units = heads * s.row_tiles;
  int64_t chunk = (num_indices * units + kTargetGroups - 1) / kTargetGroups;
  const int64_t least = (kMinChunkTokens + page_size - 1) / page_size;
  if (chunk < least) chunk = least;
  if (chunk > num_indices) chunk = num_indices;
  if (chunk < 1) chunk = 1;
  s.chunk_pages = static_cast<uint32_t>(chunk);
  s.items = static_cast<uint32_t>(num_indices / chunk + batch);
  return s;
}

template <int D, int TYPE, int FORMAT>
const void* pick_rows(const Split& s) {
  switch (s.tile_rows) {
    case 16: return reinterpret_cast<const void*>(&attention_kernel<D, TYPE, FORMAT, 1, 1>);
    case 32: return reinterpret_cast<const void*>(&attention_kernel<D, TYPE, FORMAT, 2, 1>);
    case 64: return reinterpret_cast<const void*>(&attention_kernel<D, TYPE, FORMAT, 1, 4>);
    default: return reinterpret_cast<const void*>(&attention_kernel<D, TYPE, FORMAT, 2, 4>);
  }
}

template <int D, int TYPE>
const void* pick_format(int format, const Split& s) {
  switch (format) {
    case PACE_KV_PLAIN: return pick_rows<D, TYPE, PACE_KV_PLAIN>(s);
    case PACE_KV_MXFP8: return pick_rows<D, TYPE, PACE_KV_MXFP8>(s);
    default: return pick_rows<D, TYPE, PACE_KV_MXFP4>(s);
  }
}

struct Kernels {
  const void* attention;
  const void* combine;
};

template <int D>
Kernels pick(int type, int format, const Split& s) {
  if (type == PACE_KV_BF16)
    return {pick_format<D, PACE_KV_BF16>(format, s), reinterpret_cast<const void*>(&combine_kernel<D, PACE_KV_BF16>)};
  return {pick_format<D, PACE_KV_FP16>(format, s), reinterpret_cast<const void*>(&combine_kernel<D, PACE_KV_FP16>)};
}

int check_sizes(int batch_size, int num_kv_heads, int group, int head_dim, int max_q_len, int64_t num_indices,
                int page_size) {
  if (batch_size < 0 || num_kv_heads <= 0 || group <= 0 || max_q_len <= 0 || num_indices < 0 || page_size <= 0)
    return fail(PACE_KV_EINVAL, "attention: sizes must be positive");
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return fail(PACE_KV_EINVAL, "attention: head_dim must be 64, 128 or 256, got %d", head_dim);
  const int64_t rows = static_cast<int64_t>(max_q_len) * group;
  if (num_indices * page_size > INT32_MAX / 2 || rows > INT32_MAX / 2)
    return fail(PACE_KV_ERANGE, "attention: more than 2^30 tokens or query rows");
  const Split s = split_of(batch_size, num_kv_heads, group, max_q_len, num_indices, page_size);
  if ((static_cast<int64_t>(s.items) + kXcds) * num_kv_heads * s.row_tiles >= (int64_t(1) << 24))
    return fail(PACE_KV_ERANGE, "attention: too many requests, heads or query rows for one call");
  return PACE_KV_OK;
}

int64_t workspace_bytes(const Split& s, int heads, int head_dim, int64_t num_indices) {
  if (s.chunk_pages >= num_indices) return 0;            // no request has more than one chunk
  return s.part_rows() * heads * (head_dim + 2) * 4;
}

}  // namespace
}  // namespace pace_kv

extern "C" {

int pace_kv_attention_workspace(int batch_size, int num_kv_heads, int group, int head_dim, int max_q_len,
                                int64_t num_indices, int page_size, int64_t* bytes) {
  using namespace pace_kv;
  if (!bytes) return fail(PACE_KV_EINVAL, "attention: NULL argument");
  PACE_KV_TRY(check_sizes(batch_size, num_kv_heads, group, head_dim, max_q_len, num_indices, page_size));
  *bytes = workspace_bytes(split_of(batch_size, num_kv_heads, group, max_q_len, num_indices, page_size), num_kv_heads,
                           head_dim, num_indices);
  return PACE_KV_OK;
}

int pace_kv_attention(const void* q, int64_t q_stride_bytes, int elem_type, int64_t nnz, const int32_t* qo_indptr,
                      int batch_size, int num_kv_heads, int group, int head_dim, const void* cache, int format,
                      int64_t num_pages, int page_size, const int32_t* kv_indices, int64_t num_indices,
                      const int32_t* kv_indptr, const int32_t* kv_last_page_len, int max_q_len,
                      const uint64_t* tree_mask, int mask_words, float scale, float soft_cap, void* out,
                      int64_t out_stride_bytes, float* lse, void* workspace, int64_t workspace_size,
                      int32_t* err_count, void* stream) {
  using namespace pace_kv;
  if (nnz < 0) return fail(PACE_KV_EINVAL, "attention: negative size");
  PACE_KV_TRY(check_sizes(batch_size, num_kv_heads, group, head_dim, max_q_len, num_indices, page_size));
  if (elem_type != PACE_KV_BF16 && elem_type != PACE_KV_FP16)
    return fail(PACE_KV_EINVAL, "attention: queries must be bfloat16 or float16");
  if (format != PACE_KV_PLAIN && !is_mx_format(format)) return fail(PACE_KV_EINVAL, "attention: unknown format %d", format);
  if (num_pages < 0 || num_pages > INT32_MAX || nnz > INT32_MAX / 2)
    return fail(PACE_KV_ERANGE, "attention: too many pages or tokens");
  if (!(soft_cap >= 0.f) || !(soft_cap <= 3e38f) || !(scale == scale))
    return fail(PACE_KV_EINVAL, "attention: soft_cap must be finite and >= 0, scale a number");
  if (nnz * num_kv_heads * group >= (int64_t(1) << 24))
    return fail(PACE_KV_ERANGE, "attention: 2^24 query rows or more");
  if (nnz == 0 || batch_size == 0) return PACE_KV_OK;
  if (!q || !cache || !kv_indptr || !kv_last_page_len || !out || (num_indices > 0 && !kv_indices))
    return fail(PACE_KV_EINVAL, "attention: NULL argument");
  if (!qo_indptr && nnz != batch_size)
    return fail(PACE_KV_EINVAL, "attention: without qo_indptr each request has one token");
  if (tree_mask && (mask_words <= 0 || max_q_len > static_cast<int64_t>(mask_words) * 64))
    return fail(PACE_KV_EINVAL, "attention: max_q_len tokens need a mask of ceil(max_q_len / 64) words");
  const int64_t row = static_cast<int64_t>(num_kv_heads) * head_dim, half = page_size * row;
  const int64_t q_row = row * group * 2;
  if (q_stride_bytes < q_row || q_stride_bytes % 16 || out_stride_bytes < q_row || out_stride_bytes % 8)
    return fail(PACE_KV_EINVAL, "attention: token strides must hold a row; q's is a multiple of 16, out's of 8");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(cache)) & 15u ||
      reinterpret_cast<uintptr_t>(out) & 7u || reinterpret_cast<uintptr_t>(tree_mask) & 7u)
    return fail(PACE_KV_EINVAL, "attention: q and cache must be 16-byte aligned, out and mask 8-byte");
  const int bits = format == PACE_KV_PLAIN ? 16 : mx_bits(format);
  const int64_t half_bytes = format == PACE_KV_PLAIN ? half * 2 : mx_half_bytes(half, format);
  if (half_bytes % 16) return fail(PACE_KV_EINVAL, "attention: half a page must be a multiple of 16 bytes");
  if (num_pages * 2 * half_bytes / 16 >= UINT32_MAX)
    return fail(PACE_KV_ERANGE, "attention: a layer's cache must be smaller than 64 GiB");
  const Split s = split_of(batch_size, num_kv_heads, group, max_q_len, num_indices, page_size);
  const int64_t need = workspace_bytes(s, num_kv_heads, head_dim, num_indices);
  if (need > 0 && (!workspace || workspace_size < need || reinterpret_cast<uintptr_t>(workspace) & 15u))
    return fail(PACE_KV_EINVAL, "attention: needs a 16-byte aligned workspace of %lld bytes", (long long)need);
  AttnParams p = {};
  p.q = static_cast<const char*>(q);
  p.q_stride = q_stride_bytes;
  p.qo_indptr = qo_indptr;
  p.cache = static_cast<const char*>(cache);
  p.kv_indices = kv_indices;
  p.kv_indptr = kv_indptr;
  p.kv_last_page_len = kv_last_page_len;
  p.mask = tree_mask;
  p.mask_words = static_cast<uint32_t>(tree_mask ? mask_words : 0);
  p.out = static_cast<char*>(out);
  p.out_stride = out_stride_bytes;
  p.lse = lse;
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = p.part_o + s.part_rows() * num_kv_heads * head_dim;
  p.err = err_count;
  p.num_indices = static_cast<uint32_t>(num_indices);
  p.batch = static_cast<uint32_t>(batch_size);
  p.nnz = static_cast<uint32_t>(nnz);
  p.heads = static_cast<uint32_t>(num_kv_heads);
  p.group = static_cast<uint32_t>(group);
  p.num_pages = static_cast<uint32_t>(num_pages);
  p.page_size = static_cast<uint32_t>(page_size);
  p.max_q = static_cast<uint32_t>(qo_indptr ? max_q_len : 1);
  p.chunk_pages = s.chunk_pages;
  p.items = s.items;
  p.row_tiles = s.row_tiles;
  p.tile_rows = s.tile_rows;
  p.half16 = static_cast<uint32_t>(half_bytes / 16);
  p.page16 = 2 * p.half16;
  p.row16 = static_cast<uint32_t>(row * bits / 128);
  p.scale_at = static_cast<uint32_t>(half * bits / 8);
  p.scale_row = static_cast<uint32_t>(row / kMxBlock);
  p.by_page = fast_div(p.page_size);
  p.by_chunk = fast_div(p.chunk_pages);
  p.by_group = fast_div(p.group);
  p.by_unit = fast_div(p.heads * p.row_tiles);
  p.by_tiles = fast_div(p.row_tiles);
  const float log2e = 1.44269504088896341f;
  p.scale_log2 = soft_cap > 0.f ? scale / soft_cap * (2.f * log2e) : scale * log2e;
  p.cap_log2 = soft_cap * log2e;
  const Kernels k = head_dim == 64    ? pick<64>(elem_type, format, s)
                    : head_dim == 128 ? pick<128>(elem_type, format, s)
                                      : pick<256>(elem_type, format, s);
  const uint32_t items = (s.items + kXcds - 1) / kXcds * kXcds;
  void* args[] = {&p};
  PACE_KV_TRY(hip_status(hipLaunchKernel(k.attention, dim3(items * p.heads * p.row_tiles), dim3(kThreads), args, 0,
                                         static_cast<hipStream_t>(stream)), "attention launch"));
  if (need == 0) return PACE_KV_OK;
  return hip_status(hipLaunchKernel(k.combine, dim3(static_cast<uint32_t>(nnz) * p.heads * p.group), dim3(kThreads),
                                    args, 0, static_cast<hipStream_t>(stream)), "attention combine launch");
}

}  // extern "C"

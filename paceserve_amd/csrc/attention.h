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
// errors that average out over the row); l sums the unrounded weights.  Weights are
// 2^(score - m) of at most 1; in float16 they are of at most 2^15 (m lies 15 below the
// largest score), which leaves those down to 2^-29 of the largest their 2^-11, and the
// least 2^-40 of it: with 1 as the most, a long tail of weights below 2^-14 lost up to
// all of its mass in the output, though not in l.
//
// Work split: a request's pages in chunks of C, the chunks of all requests numbered
// through.  A workgroup finds the request of its number in the tables themselves,
// so a launch needs no plan and a captured one follows them; the grid has room for
// the most chunks there can be, floor(pages / C) + requests.  A request of one chunk
// is written directly; the others leave (o, m, l) in a workspace for the joining
// kernels.  With e its chunks past the first and E those of all requests before it (its
// first item less its number), its parts are 2 E .. 2 E + e: the next split request's E
// is E + e, and 2 e >= e + 1.  A request of n pages has e <= floor(n / C), so
// 2 floor(pages / C) parts are enough, however many requests there are beside the split
// ones, and no search of their own.
//
// Bounds on MI355X (kernel alone): up to 32 rows over a 16-bit cache HBM, 5.3 to 5.7
// TB/s (256 ragged requests of up to 2048 tokens with 8 heads of 128, 8 rows each, 191 to
// 198 us; 12 rows of 32 heads over 32768 tokens 94 to 96 us); less over short ones (33 x
// 2000 tokens 65 us a call for 270 MB), whose chunks do not divide evenly among the CUs.  Over a
// quantised cache, and with more rows, expansion, exponentials and matrix instructions
// take about the same issue time each and overlap only in part: 504 rows over 8 x 4096
// 8-bit tokens 118 us, where the products alone take 27 at the matrix peak (counters:
// matrix instructions 28% of the time, vector ones 59%, LDS 25%).  A single short request
// is a chain of latencies: 13 us over 512 tokens, of which the four steps of a wave take six.
#pragma once

#include <type_traits>

#include "mx.h"

namespace pace_kv {

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
  float* part_o;               // [parts, heads, row_tiles, rows of a tile, D]
  float* part_ml;              // [parts, heads, row_tiles, rows of a tile, 2]
  int32_t* err;
  uint32_t num_indices, batch, nnz, heads, group, num_pages, page_size, max_q, mask_words;
  uint32_t chunk_pages, step_pages, items, parts, row_tiles, tile_rows;
  uint32_t join_turns, token_waves;  // of the joining kernel
  uint32_t page16, half16, row16;  // page, half page and token row, in 16-byte units
  uint32_t scale_at, scale_row;    // scales within a half page, scale bytes of a token
  FastDiv by_page, by_chunk, by_group, by_unit, by_tiles, by_heads, by_token_waves;
  float scale_log2;            // scale * log2(e); with a cap: scale / cap * 2 * log2(e)
  float cap_log2;              // cap * log2(e), or 0
  float uncapped_log2;         // scale * log2(e)
  uint32_t large_cap;          // the cap is past kLargeCap
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

// The larger of three, of the numbers among them where some are NaN.  Plain fmaxf
// quiets its operands first, an instruction each, though no product here is a
// signalling NaN.
__device__ __forceinline__ float max3_of(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// A request and the part of it that a work item covers.
struct Request {
  uint32_t chunk, chunks;
  int32_t first_page;          // in kv_indices
  uint32_t pages;
  uint32_t kv_len;
  uint32_t q0, q_len;
};

// What the tables say of a request.
struct Tables {
  int32_t k0, k1, last, a0, a1;
};

// Where a request stands among the call's: its number, its first work item and, if it is
// split, its first part.
struct Place {
  uint32_t index, item;
  __device__ __forceinline__ uint32_t part() const { return 2 * (item - index); }
};

__device__ __forceinline__ Tables tables_of(const AttnParams& p, uint32_t b) {
  Tables t;
  t.k0 = p.kv_indptr[b];
  t.k1 = p.kv_indptr[b + 1];
  t.last = p.kv_last_page_len[b];
  t.a0 = static_cast<int32_t>(b);
  t.a1 = t.a0 + 1;
  if (p.qo_indptr != nullptr) {
    t.a0 = p.qo_indptr[b];
    t.a1 = p.qo_indptr[b + 1];
  }
  return t;
}

__device__ __forceinline__ uint32_t pages_of(const AttnParams& p, const Tables& t) {
  const uint32_t first = static_cast<uint32_t>(max(t.k0, 0));
  const uint32_t n = t.k1 > t.k0 && t.k1 > 0 ? static_cast<uint32_t>(t.k1) - first : 0u;
  return min(n, p.num_indices - min(first, p.num_indices));
}

// Chunks of a request of n pages; one without pages still has its rows to write.
__device__ __forceinline__ uint32_t chunks_of(const AttnParams& p, uint32_t n) {
  const uint32_t c = over(p.by_chunk, n);
  return max(c * p.chunk_pages < n ? c + 1 : c, 1u);
}

// The sizes of request b; false where its queries are not among nnz or exceed
// max_q.
__device__ __forceinline__ bool request_of(const AttnParams& p, const Tables& t, Request* r) {
  r->first_page = max(t.k0, 0);
  r->pages = pages_of(p, t);
  const int64_t most = static_cast<int64_t>(r->pages) * p.page_size;
  const int64_t len = (most > p.page_size ? most - p.page_size : 0) + t.last;
  r->kv_len = static_cast<uint32_t>(min(max(len, int64_t(0)), most));
  r->chunks = chunks_of(p, r->pages);
  r->q0 = static_cast<uint32_t>(t.a0);
  r->q_len = static_cast<uint32_t>(t.a1 - t.a0);
  return t.a0 >= 0 && t.a1 >= t.a0 && static_cast<uint32_t>(t.a1) <= p.nnz && r->q_len <= p.max_q;
}

// Whether a request's items and parts are among the call's: offsets that run backwards
// can count pages twice.
__device__ __forceinline__ bool has_room(const AttnParams& p, const Request& r, const Place& place) {
  return place.item + r.chunks <= p.items && (r.chunks == 1 || place.part() + r.chunks <= p.parts);
}

// Whether the tables name entries that do not exist, which pages_of and request_of cut off.
__device__ __forceinline__ bool is_cut(const AttnParams& p, const Tables& t, const Request& r) {
  return t.k0 < 0 || (t.k1 > 0 && static_cast<uint32_t>(t.k1) > p.num_indices) ||
         (r.pages > 0 && static_cast<uint32_t>(t.last) > p.page_size);
}

// Sum over the lanes up to this one: within rows of 16 lanes by shifts, then each
// row's total to the rows behind it.
__device__ __forceinline__ uint32_t sum_upto(uint32_t x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2 and 3
  return x;
}

// The last request whose key is at most x, keys not decreasing: what the tables say
// of it, and its place (items: the chunks of the requests before it); false if there
// is none.  The wave looks at 256 requests a round, four neighbours to a
// lane, and holds what it loads of each, so up to 256 cost one load latency.
template <class Key>
__device__ __forceinline__ bool find_request(const AttnParams& p, uint32_t x, Key key, Tables* t, Place* place) {
  const uint32_t lane = threadIdx.x % 64;
  bool found = false;
  uint32_t before = 0;                                   // chunks of the rounds before
  for (uint32_t e0 = 0; e0 < p.batch; e0 += 256) {
    Tables mine[4] = {};
    uint32_t start[4];
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k)
      if (e0 + lane * 4 + k < p.batch) mine[k] = tables_of(p, e0 + lane * 4 + k);
    uint32_t sum = 0;
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) {
      start[k] = sum;
      if (e0 + lane * 4 + k < p.batch) sum += chunks_of(p, pages_of(p, mine[k]));
    }
    const uint32_t upto = sum_upto(sum);                 // over the lanes up to this one
    int best = -1;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      start[k] += before + upto - sum;
      if (e0 + lane * 4 + k < p.batch && key(mine[k], start[k]) <= x) best = k;
    }
    const uint64_t pass = __ballot(best >= 0);
    if (pass != 0) {
      found = true;
      const int at = 63 - __builtin_clzll(pass);
      Tables of = mine[0];
      uint32_t item = start[0];
#pragma unroll
      for (int k = 1; k < 4; ++k)
        if (best == k) {
          of = mine[k];
          item = start[k];
        }
      t->k0 = __builtin_amdgcn_readlane(of.k0, at);
      t->k1 = __builtin_amdgcn_readlane(of.k1, at);
      t->last = __builtin_amdgcn_readlane(of.last, at);
      t->a0 = __builtin_amdgcn_readlane(of.a0, at);
      t->a1 = __builtin_amdgcn_readlane(of.a1, at);
      place->item = __builtin_amdgcn_readlane(item, at);
      place->index = e0 + at * 4 + __builtin_amdgcn_readlane(best, at);
    }
    if (__builtin_amdgcn_readlane(best, 63) != 3) break;
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  return found;
}

// Rows in LDS are padded by 32 bytes, so that 8 rows' 32 bytes of a transposing
// read cover the 256 bytes of all banks once (MI355X, keys and values padded so:
// half the bank conflicts of keys padded by 16).  Unlike a xor of the columns, a
// pad leaves every address one register and an immediate offset.
template <int D>
constexpr uint32_t kStride = D * 2 + 32;

template <int TYPE>
__device__ __forceinline__ f32x4 mfma(const u32x4& a, const u32x4& b, const f32x4& c) {
  if constexpr (TYPE == PACE_KV_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                  0);
}

// log2 of a row's largest weight.
template <int TYPE>
constexpr float kTopWeight = TYPE == PACE_KV_FP16 ? 15.f : 0.f;

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

// Two results.  A weighted mean of finite values is none larger than they are, but
// rounded weights can carry one past float16's largest number by 2^-11 of it.
template <int TYPE>
__device__ __forceinline__ uint32_t result_pair(float a, float b) {
  if constexpr (TYPE == PACE_KV_FP16) {
    constexpr float kMost = 65504.f;
    if (fabsf(a) < INFINITY) a = fminf(fmaxf(a, -kMost), kMost);
    if (fabsf(b) < INFINITY) b = fminf(fmaxf(b, -kMost), kMost);
  }
  return pair_of<TYPE>(a, b);
}

// Natural logarithm of a row's sum of exponentials, l over 2^m.  The 15 that m lies below
// the largest score in float16 go back first: both terms would lose bits to them.
template <int TYPE>
__device__ __forceinline__ float log_sum(float m, float l) {
  constexpr float kTop = kTopWeight<TYPE>, kScale = TYPE == PACE_KV_FP16 ? 0x1p-15f : 1.f;
  return l == 0.f ? -INFINITY : (m + kTop + __log2f(l * kScale)) * 0.69314718055994531f;
}

// Hides where x comes from, so that what a loop derives from it is derived anew
// each time (an add) instead of being held in a register throughout.
__device__ __forceinline__ uint32_t opaque(uint32_t x) {
  asm volatile("" : "+v"(x));
  return x;
}

template <bool HIDE>
__device__ __forceinline__ uint32_t opaque_if(uint32_t x) {
  return HIDE ? opaque(x) : x;
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

// Waves per SIMD that the registers are held to.  Two workgroups a CU fit the
// accumulators and loads of 32 rows of 128 (and of 16 rows of 256, with a few spills
// outside the loops: MI355X, 24 rows over 8 x 4096 bf16 tokens, 93 us against 114
// with one).  A quantised cache, whose loads in flight take fewer registers, leaves room
// for a third: for a decode step its loads count; where a wave takes 32 of 128 rows
// it computes while the others wait (320 rows over 24 x 2000 tokens, 8 bits 177 -> 150 us,
// 4 bits 172 -> 140), if addresses are derived anew in each step.  A 16-bit cache would
// spill there (504 rows over 8 x 4096 tokens 125 -> 161 us, 320 over 24 x 2000 173 -> 166).
constexpr int min_waves(int D, int format, int R, int WR) {
  return D != 256 && format != PACE_KV_PLAIN && (R == 1 ? WR == 1 : WR == 4) ? 3 : 2;
}

// TYPE: of queries and output, and what a quantised cache is expanded to.
// R tiles of 16 query rows per wave.  WR = 1: the waves take 32 tokens each of
// a step for the same rows and join at the end.  WR = 4: each wave takes its own 16 * R rows, and
// all share a tile of 64 tokens.
template <int D, int TYPE, int FORMAT, int R, int WR>
__global__ __launch_bounds__(kThreads, min_waves(D, FORMAT, R, WR)) void attention_kernel(const AttnParams p) {
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
  constexpr bool kTight = R == 2 && WR == 4 && D == 128 && FORMAT != PACE_KV_PLAIN;  // three waves fill the registers
  // Rows that no other workgroup reads are loaded nontemporally, unless two heads
  // share a 128-byte line; with head_dim 256 past 64 rows, whose tiles share them, as
  // well: one kernel serves one tile and several (bf16, 36 to 64 rows over 8 x 4096 to
  // 24 x 2000 tokens 5 to 16% faster so, 128 and 320 rows up to 7% slower; 8 and 4 bits
  // the same within 5%).  MI355X, reading 2 GiB of pages of 8 heads in this pattern:
  // 256-byte rows 6.4 TB/s against 5.8, 128-byte ones 6.3 against 5.6, 64-byte ones
  // 4.8 against 5.9 (and 3.5 with the heads of a page on different XCDs).
  constexpr bool kReadOnce = (WR == 1 || R == 1) && D * kBits / 8 >= 128;

  constexpr uint32_t kRowBytes = WR == 1 ? kStride<D> : 2 * kStride<D>;
  constexpr uint32_t kJoinBytes = WR == 1 ? kWaves * 16 * D * 4 : 0;
  __shared__ __attribute__((aligned(16))) char
      lds[kLdsRows * kRowBytes > kJoinBytes ? kLdsRows * kRowBytes : kJoinBytes];
  __shared__ __attribute__((aligned(16))) char lds_q[WR == 1 ? kTileRows * kStride<D> : 16];
  __shared__ float lds_ml[kWaves][WR == 1 ? kTileRows : 1][2];

  const uint32_t lane = threadIdx.x % 64, g = lane / 16, n = lane % 16;
  const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);

  // The heads and row tiles of one item run on one XCD, whose L2 then holds
  // what they share.
  const uint32_t unit = p.heads * p.row_tiles;
  const uint32_t at = blockIdx.x / kXcds, nth = over(p.by_unit, at);
  const uint32_t item = nth * kXcds + blockIdx.x % kXcds;
  if (item >= p.items) return;
  const uint32_t in_unit = at - nth * unit, head = over(p.by_tiles, in_unit), tile = in_unit - head * p.row_tiles;
  Place place;
  Tables tables;
  if (!find_request(p, item, [](const Tables&, uint32_t start) { return start; }, &tables, &place)) return;
  Request r;
  const bool valid_request = request_of(p, tables, &r) && has_room(p, r, place);
  r.chunk = item - place.item;
  if (r.chunk >= r.chunks) return;
  if (p.err != nullptr && in_unit == 0 && threadIdx.x == 0) {
    if (r.chunk == 0 && (!valid_request || is_cut(p, tables, r))) atomicAdd(p.err, 1);
    // Behind the last item lie requests that no workgroup looks at.
    if (item + 1 == p.items && place.index + 1 < p.batch)
      atomicAdd(p.err, static_cast<int32_t>(p.batch - 1 - place.index));
  }
  if (!valid_request) return;
  const uint32_t rows = r.q_len * p.group, row0 = tile * kTileRows;
  if (row0 >= rows) return;
  const int32_t base = static_cast<int32_t>(r.kv_len) - static_cast<int32_t>(r.q_len);
  // Without a mask no row of the tile sees past its last query.
  const int32_t first_q = static_cast<int32_t>(over(p.by_group, row0));
  const int32_t last_q = static_cast<int32_t>(over(p.by_group, min(row0 + kTileRows, rows) - 1));
  // A request's chunks are of one length, in whole steps and at most chunk_pages, and
  // none is empty: (chunks - 1) * chunk_pages < pages.  A short last one would leave
  // its XCD idle where all requests have as many chunks.
  const uint32_t even = (r.pages + r.chunks - 1) / r.chunks;
  const uint32_t length = min((even + p.step_pages - 1) / p.step_pages * p.step_pages, p.chunk_pages);
  const int32_t chunk_tokens = static_cast<int32_t>(length * p.page_size);
  const int32_t t_begin = static_cast<int32_t>(r.chunk) * chunk_tokens;
  int32_t t_end = static_cast<int32_t>(min(static_cast<int64_t>(t_begin) + chunk_tokens, static_cast<int64_t>(r.kv_len)));
  if (p.mask == nullptr) t_end = min(t_end, base + last_q + 1);
  // Tokens on pages that do not exist are counted by one workgroup of those over a chunk,
  // the last row tile's: it sees all of the chunk.  A look at the pages of its own, that
  // calls without a counter do not take, and no registers in the steps below.
  if (p.err != nullptr && head == 0 && row0 + kTileRows >= rows) {
    const int32_t page = static_cast<int32_t>(p.page_size), first = static_cast<int32_t>(r.chunk * length);
    for (int32_t i = static_cast<int32_t>(threadIdx.x); static_cast<int64_t>(i) * page < t_end - t_begin; i += kThreads)
      if (static_cast<uint32_t>(p.kv_indices[r.first_page + first + i]) >= p.num_pages)
        atomicAdd(p.err, min(page, t_end - t_begin - i * page));
  }

  // Query fragments: row n of each tile, eight elements from 32 * k + 8 * g.  In
  // registers, or (WR = 1, whose registers hold more loads in flight) in LDS.
  const uint32_t wave_row0 = row0 + (WR == 1 ? 0 : w * 16 * R);
  const auto query_at = [&](uint32_t row) {
    const uint32_t i = over(p.by_group, row);
    return p.q + static_cast<int64_t>(r.q0 + i) * p.q_stride +
           (static_cast<int64_t>(head) * p.group + (row - i * p.group)) * (D * 2);
  };
  u32x4 qf[R][kKS];
#pragma unroll
  for (int a = 0; a < R; ++a) {
    const uint32_t row = wave_row0 + a * 16 + n;
    if constexpr (WR != 1) {
#pragma unroll
      for (int k = 0; k < kKS; ++k) {
        qf[a][k] = u32x4{0, 0, 0, 0};
        if (row < rows) qf[a][k] = *reinterpret_cast<const u32x4*>(query_at(row) + k * 64 + g * 16);
      }
    }
  }
  const char* const query = lds_q + n * kStride<D> + g * 16;

  f32x4 acc[R][kDT];
  float m[R], from[R], l[R];
  bool wide[R];                                          // some row's |m| is past 2^20
#pragma unroll
  for (int a = 0; a < R; ++a) {
    wide[a] = false;
    m[a] = -INFINITY;
    from[a] = 0.f;                                       // m, or 0 while nothing is seen: weights of 2^-inf = 0
    l[a] = 0.f;
#pragma unroll
    for (int d = 0; d < kDT; ++d) acc[a][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // WR = 1: a wave's keys, then its values, pass through one region of its own.
  char* const lds_k = WR == 1 ? lds + w * kLoadRows * kStride<D> : lds;
  char* const lds_v = WR == 1 ? lds_k : lds + kLdsRows * kStride<D>;
  const uint32_t lds_row0 = WR == 1 ? 0 : w * kLoadRows;  // first row that this wave loads

  // A step's loads: page ids (one token per lane), then key rows, then value rows.
  const uint32_t id_lane = lane % kIdTokens;
  int32_t id = 0;
  const auto load_id = [&](int32_t t0) {
    const int32_t t = t0 + static_cast<int32_t>(id_lane);
    id = -1;
    if (t < t_end) id = p.kv_indices[r.first_page + static_cast<int32_t>(over(p.by_page, static_cast<uint32_t>(t)))];
  };
  // Load j of a lane: column lane % kPieces of row j * kRowStep + lane / kPieces.
  constexpr uint32_t kRowStep = 64 / kPieces;
  u32x4 kr[kLoads] = {}, vr[kLoads] = {};
  uint32_t row_at = 0;                                   // the lane's token's row, in 16-byte units
  uint64_t k_bytes = 0, v_bytes = 0;                     // the scales of the lane's token
  uint64_t valid = 0;
  const auto fetch = [&](u32x4* to, int64_t from) {
    const uint32_t ln = opaque_if<kTight>(lane), my_row = ln / kPieces, my_col = ln % kPieces;
    const uint32_t first_row = opaque_if<!kTight>((WR == 1 ? 0 : w * kLoadRows) + my_row % kLoadRows);
#pragma unroll
    for (uint32_t j = 0; j < kLoads; ++j) {
      const int64_t at = static_cast<int64_t>(static_cast<uint32_t>(__shfl(row_at, first_row + j * kRowStep))) + from;
      const u32x4* const x = reinterpret_cast<const u32x4*>(p.cache + at * 16) + my_col;
      to[j] = kReadOnce ? __builtin_nontemporal_load(x) : *x;
    }
  };
  const auto load_keys = [&](int32_t t0) {
    const uint32_t t = static_cast<uint32_t>(t0) + id_lane;
    const bool ok = t0 + static_cast<int32_t>(id_lane) < t_end && static_cast<uint32_t>(id) < p.num_pages;
    valid = __ballot(ok);
    if (kIdTokens == 32) valid &= 0xffffffffull;
    if (valid == 0) return;
    const uint32_t slot = t - over(p.by_page, t) * p.page_size;
    // A token that does not exist reads the pool's first row, which is made
    // zeros on its way into LDS: loads without a condition.
    row_at = ok ? static_cast<uint32_t>(id) * p.page16 + slot * p.row16 + head * (D * kBits / 128) : 0u;
    if constexpr (FORMAT != PACE_KV_PLAIN) {
      k_bytes = v_bytes = 0;
      if (ok && id_lane / kLoadRows == (WR == 1 ? 0 : w)) {
        const char* s = p.cache + static_cast<int64_t>(id) * p.page16 * 16 + p.scale_at +
                        static_cast<int64_t>(slot) * p.scale_row + head * (D / 32);
        const char* sv = s + static_cast<int64_t>(p.half16) * 16;
        typedef std::conditional_t<D == 64, uint16_t, std::conditional_t<D == 128, uint32_t, uint64_t>> Scales;
        k_bytes = *reinterpret_cast<const Scales*>(s);
        v_bytes = *reinterpret_cast<const Scales*>(sv);
      }
    }
    fetch(kr, 0);
  };
  const auto load_values = [&]() {
    if (valid != 0) fetch(vr, p.half16);
  };
  // The 16-byte pieces that a lane expands one load to are two (or four) apart from
  // its neighbour's, half the banks: every other group of lanes starts at its second.
  const auto store_piece = [&](char* row, uint32_t c, uint32_t turn, const u32x4& x, uint64_t bytes) {
    u32x4* to = reinterpret_cast<u32x4*>(row);
    if constexpr (FORMAT == PACE_KV_PLAIN) {
      to[c] = x;
    } else if constexpr (FORMAT == PACE_KV_MXFP8) {      // 16 elements: half a block
      const float s = scale_of(static_cast<uint32_t>(bytes >> (c / 2 * 8)) & 255u);
      const u32x2 lo = {x[0], x[1]}, hi = {x[2], x[3]};
      to[2 * c + turn] = run_up<TYPE, FORMAT>(turn ? hi : lo, s);
      to[2 * c + 1 - turn] = run_up<TYPE, FORMAT>(turn ? lo : hi, s);
    } else {                                             // 32 elements: a block
      const float s = scale_of(static_cast<uint32_t>(bytes >> (c * 8)) & 255u);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        to[4 * c + (k + turn) % 4] = run_up<TYPE, FORMAT>(u32x2{turn ? x[(k + 1) % 4] : x[k], 0}, s);
    }
  };
  // Loaded rows into LDS; unless WHOLE, those of tokens outside `exist` as zeros.
  const auto store = [&](auto whole, char* to, u32x4* x, uint64_t bytes, uint64_t exist) {
    const uint32_t ln = opaque_if<kTight>(lane), my_row = ln / kPieces, my_col = ln % kPieces;
    const uint32_t turn = ln >> (FORMAT == PACE_KV_MXFP8 || D == 64 ? 2 : 1) & 1;
    const uint32_t from = opaque_if<!kTight>((WR == 1 ? 0 : w * kLoadRows) + my_row % kLoadRows);
    if constexpr (!decltype(whole)::value) {
#pragma unroll
      for (uint32_t j = 0; j < kLoads; ++j)
        if (!((exist >> (from + j * kRowStep)) & 1)) x[j] = u32x4{0, 0, 0, 0};
    }
    char* const row = to + (lds_row0 + my_row) * kStride<D>;
#pragma unroll
    for (uint32_t j = 0; j < kLoads; ++j) {
      uint64_t b = 0;
      if constexpr (FORMAT != PACE_KV_PLAIN) {
        b = static_cast<uint32_t>(__shfl(static_cast<uint32_t>(bytes), from + j * kRowStep));
        if constexpr (D == 256)
          b |= static_cast<uint64_t>(__shfl(static_cast<uint32_t>(bytes >> 32), from + j * kRowStep)) << 32;
      }
      if (kRowStep <= kLoadRows || my_row < kLoadRows) store_piece(row + j * kRowStep * kStride<D>, my_col, turn, x[j], b);
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

  // The weights of 32 tokens from t0, whose keys lie at lds_row; `ok`: the tokens
  // that exist.
  u32x4 pf[R];
  uint32_t sees[R];
  const float per_score = p.cap_log2 > 0.f || p.scale_log2 == 0.f ? 1.f : fabsf(p.scale_log2);
  const auto weigh = [&](auto full, int32_t t0, uint32_t lds_row, uint32_t ok) {
    const uint32_t ln = opaque_if<kTight>(lane);
    const char* key_at = lds_k + (lds_row + ln % 16) * kStride<D> + ln / 16 * 16;
    f32x4 s[R][2];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int a = 0; a < R; ++a) s[a][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < kKS; ++k) {
      if constexpr (WR == 1) {
#pragma unroll
        for (int a = 0; a < R; ++a)
          qf[a][k] = *reinterpret_cast<const u32x4*>(query + a * 16 * kStride<D> + k * 64);
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const u32x4 kf = *reinterpret_cast<const u32x4*>(key_at + t * 16 * kStride<D> + k * 64);
#pragma unroll
        for (int a = 0; a < R; ++a) s[a][t] = mfma<TYPE>(kf, qf[a][k], s[a][t]);
      }
    }
    // The weights are 2^(per_score * s - m).
    if (p.cap_log2 > 0.f && !p.large_cap) {
      // x = 2 log2(e) z: tanh(z) = 1 - 2 / (1 + 2^x), times the cap: off by 2^-22 of the cap
#pragma unroll
      for (int a = 0; a < R; ++a)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float half = __builtin_amdgcn_rcpf(1.f + exp2_of(s[a][t][e] * p.scale_log2));
            s[a][t][e] = __builtin_fmaf(half, -2.f * p.cap_log2, p.cap_log2);
          }
    } else if (p.cap_log2 > 0.f) {
      // The same where |x| >= 0.8: off by 2^-20 of itself.  Below, the series z (1 - z^2/3 +
      // 2 z^4/15 - 17 z^6/315 + 62 z^8/2835), in x, times the score: off by a few 2^-24 of
      // itself, however large the cap; the next term is below 2^-25.
      constexpr float kSq = 0.12011325f;                 // (ln(2) / 2)^2: z^2 = kSq x^2
      constexpr float c1 = -1.f / 3 * kSq, c2 = 2.f / 15 * kSq * kSq, c3 = -17.f / 315 * kSq * kSq * kSq,
                      c4 = 62.f / 2835 * kSq * kSq * kSq * kSq;
#pragma unroll
      for (int a = 0; a < R; ++a)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = s[a][t][e] * p.scale_log2, x2 = x * x;
            const float half = __builtin_amdgcn_rcpf(1.f + exp2_of(x));
            float f = __builtin_fmaf(x2, c4, c3);
            f = __builtin_fmaf(x2, f, c2);
            f = __builtin_fmaf(x2, f, c1);
            f = __builtin_fmaf(x2, f, 1.f);
            const float near = s[a][t][e] * p.uncapped_log2 * f;
            s[a][t][e] = fabsf(x) < 0.8f ? near : __builtin_fmaf(half, -2.f * p.cap_log2, p.cap_log2);
          }
    } else if (p.scale_log2 <= 0.f) {
      const float sign = p.scale_log2 < 0.f ? -1.f : 0.f;
#pragma unroll
      for (int a = 0; a < R; ++a)
#pragma unroll
        for (int t = 0; t < 2; ++t) s[a][t] *= sign;
    }
    if constexpr (!decltype(full)::value) {
#pragma unroll
      for (int a = 0; a < R; ++a) {
        sees[a] = seen(t0, static_cast<int32_t>(over(p.by_group, wave_row0 + a * 16 + opaque_if<kTight>(n)))) & ok;
        const uint32_t mine = sees[a] >> opaque(4 * g);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!(mine & (1u << (t * 16 + e)))) s[a][t][e] = -INFINITY;
      }
    }
#pragma unroll
    for (int a = 0; a < R; ++a) {
      float top = max3_of(s[a][0][0], s[a][0][1], s[a][0][2]);
      top = max3_of(top, s[a][0][3], s[a][1][0]);
      top = max3_of(top, s[a][1][1], s[a][1][2]);
      top = __builtin_fmaf(max3_of(top, s[a][1][3], s[a][1][3]), per_score, -kTopWeight<TYPE>);
      // m follows the largest score so far exactly: its weight is not rounded, and a
      // weighted value is no larger than the value.  (Raising m only past 2^8 of it spares
      // most steps the joint maximum, MI355X: 3 % over 70 calls, 11 % of 320 rows; but
      // the largest weight is then rounded as the others are, bfloat16 outputs are off by
      // 0.0023 of the values instead of 0.0017, and a value past 2^120 becomes infinite.)
      if (__ballot(top > m[a]) != 0) {
        top = fmaxf(m[a], across_groups(top, max_of));
        from[a] = top == -INFINITY ? 0.f : top;
        const float shrink = exp2_of(m[a] - from[a]);
        m[a] = top;
        wide[a] = __ballot(fabsf(from[a]) > 0x1p20f) != 0;
        l[a] *= shrink;
#pragma unroll
        for (int d = 0; d < kDT; ++d) acc[a][d] *= shrink;
      }
      if (kTight) from[a] = m[a] == -INFINITY ? 0.f : m[a];
      // The fused difference holds what m lost when it was rounded: less than a tenth up
      // to 2^20, but past 2^27 enough to make the largest weight an infinity or a zero.
      if (wide[a]) {
#pragma clang fp contract(off)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float scaled = s[a][t][e] * per_score, x = scaled - from[a];
            s[a][t][e] = x > kTopWeight<TYPE> ? kTopWeight<TYPE> : x;
          }
      } else {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[a][t][e] = __builtin_fmaf(s[a][t][e], per_score, -from[a]);
      }
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const float x = exp2_of(s[a][t][e]), y = exp2_of(s[a][t][e + 1]);
          l[a] += x + y;
          pf[a][t * 2 + e / 2] = pair_of<TYPE>(x, y);
        }
    }
  };
  // Adds the weighted values of those tokens, at lds_row.
  const auto gather = [&](auto full, uint32_t lds_row) {
    const char* value_at = lds_v + lds_row * kStride<D>;
    const uint32_t ln = opaque_if<kTight>(lane);
    bool odd = false;                                    // an infinite or NaN value that some row must not see
    if constexpr (!decltype(full)::value) {
      bool found = false;
#pragma unroll 1
      for (uint32_t c0 = 0; c0 < 32 * D / 8; c0 += 64) {
        const uint32_t c = c0 + lane;
        const u32x4 x = *reinterpret_cast<const u32x4*>(value_at + c / (D / 8) * kStride<D> + c % (D / 8) * 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) found |= odd_word<TYPE>(x[e]);
      }
      odd = __ballot(found) != 0;
    }
#pragma unroll
    for (int d = 0; d < kDT; ++d) {
      // Lane: row 4 g + n / 4 of each 16 tokens, four columns; transposed over
      // 16 lanes: four tokens of column n.
      const char* at = value_at + ln / 4 * kStride<D> + ln % 4 * 8 + d * 32;
      typedef __attribute__((address_space(3))) s16x4* lds_ptr;
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)at);
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(at + 16 * kStride<D>));
      const u32x2 lo2 = __builtin_bit_cast(u32x2, lo), hi2 = __builtin_bit_cast(u32x2, hi);
      u32x4 vf = {lo2[0], lo2[1], hi2[0], hi2[1]};
      if (odd) vf = u32x4{0, 0, 0, 0};
#pragma unroll
      for (int a = 0; a < R; ++a) acc[a][d] = mfma<TYPE>(vf, pf[a], acc[a][d]);
    }
    if constexpr (!decltype(full)::value) if (odd) {
      // A product with weight zero would spread an infinity or a NaN to rows
      // that do not see its token: the same sum, token by token, over those seen.
#pragma unroll
      for (int a = 0; a < R; ++a)
#pragma unroll 1
        for (uint32_t token = 0; token < 32; ++token) {
          const uint32_t word = token / 16 * 2 + token % 4 / 2;
          const uint32_t mine = word == 0 ? pf[a][0] : word == 1 ? pf[a][1] : word == 2 ? pf[a][2] : pf[a][3];
          const float weight = value_of<TYPE>(__shfl(mine, token % 16 / 4 * 16 + n), token % 2);
          if (!((sees[a] >> token) & 1u)) continue;
#pragma unroll
          for (int d = 0; d < kDT; ++d) {
            const u32x2 v = *reinterpret_cast<const u32x2*>(value_at + token * kStride<D> + d * 32 + g * 8);
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[a][d][c] += weight * value_of<TYPE>(v[c / 2], c % 2);
          }
        }
    }
  };
  constexpr uint64_t kAll = kIdTokens == 32 ? 0xffffffffull : ~0ull;
  const int32_t seen_by_all = p.mask == nullptr ? base + first_q + 1 : base;
  // Whether every row sees all the tokens of a wave's step from t0.
  const auto all_seen = [&](int32_t t0) {
    return valid == kAll && t0 + static_cast<int32_t>(kIdTokens) <= seen_by_all;
  };
  const int32_t step = static_cast<int32_t>(kStep);
  int32_t t0 = t_begin + (WR == 1 ? static_cast<int32_t>(w * kIdTokens) : 0);
  const auto one_step = [&](auto full) {
    if constexpr (WR == 1) {
      // No barrier: the region is the wave's own, and its LDS operations run in order.
      const uint64_t ok = valid, bytes = v_bytes;
      store(full, lds_k, kr, k_bytes, ok);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      load_keys(t0 + step);
      load_id(t0 + 2 * step);
      __builtin_amdgcn_sched_barrier(0);
      weigh(full, t0, 0, static_cast<uint32_t>(ok));
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      store(full, lds_v, vr, bytes, ok);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      load_values();
      __builtin_amdgcn_sched_barrier(0);
      gather(full, 0);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    } else {
      // Two tiles in LDS would need one barrier, but cost a third workgroup its
      // place (MI355X, 36 rows over a 4-bit cache: 70 us against 53).
      const uint64_t ok = valid;
      __syncthreads();                                   // the last step's reads are done
      store(full, lds_k, kr, k_bytes, ok);
      store(full, lds_v, vr, v_bytes, ok);
      __syncthreads();
      load_keys(t0 + step);
      load_values();
      load_id(t0 + 2 * step);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll 1
      for (int h = 0; h < 2 && wave_row0 < rows; ++h) {  // a wave of padding only loads
        weigh(full, t0 + 32 * h, 32 * h, static_cast<uint32_t>(ok >> (32 * h)));
        gather(full, 32 * h);
      }
    }
    t0 += step;
  };
  load_id(t0);
  if constexpr (WR == 1) {
#pragma unroll
    for (uint32_t e = threadIdx.x; e < kTileRows * (D / 8); e += kThreads) {
      const uint32_t row = e / (D / 8), c = e % (D / 8);
      u32x4 x = {0, 0, 0, 0};
      if (row0 + row < rows) x = *reinterpret_cast<const u32x4*>(query_at(row0 + row) + c * 16);
      *reinterpret_cast<u32x4*>(lds_q + row * kStride<D> + c * 16) = x;
    }
  }
  load_keys(t0);
  load_values();
  load_id(t0 + step);
  if (WR == 1) __syncthreads();                          // the queries are in LDS
  // The steps whose tokens every row sees, then the others: the first loop is
  // free of masks, and of the registers that they take.
  while (t0 < t_end && all_seen(t0)) one_step(std::true_type{});
#pragma unroll 1
  while (t0 < t_end) one_step(std::false_type{});
#pragma unroll
  for (int a = 0; a < R; ++a) l[a] = across_groups(l[a], sum_of);

  const bool direct = r.chunks == 1;
  const int64_t part_row0 = (static_cast<int64_t>(place.part() + r.chunk) * unit + in_unit) * kTileRows;
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
    const u32x2 x = {result_pair<TYPE>(o[0] * inv, o[1] * inv), result_pair<TYPE>(o[2] * inv, o[3] * inv)};
    *reinterpret_cast<u32x2*>(p.out + static_cast<int64_t>(r.q0 + i) * p.out_stride +
                              (static_cast<int64_t>(qh) * D + d) * 2) = x;
    if (first && p.lse != nullptr)
      p.lse[static_cast<int64_t>(r.q0 + i) * p.heads * p.group + qh] = log_sum<TYPE>(top, sum);
  };
  if (WR != 1) {
#pragma unroll
    for (int a = 0; a < R; ++a)
#pragma unroll
      for (int d = 0; d < kDT; ++d) write(w * 16 * R + a * 16 + n, d * 16 + g * 4, acc[a][d], m[a], l[a], d == 0 && g == 0);
    return;
  }
  // The waves' parts of a row join over their common maximum, 16 rows at a time.
  float* const part = reinterpret_cast<float*>(lds);     // [wave][row][D], chunks of 4 xored with the row
  if (g == 0) {
#pragma unroll
    for (int a = 0; a < R; ++a) {
      lds_ml[w][a * 16 + n][0] = m[a];
      lds_ml[w][a * 16 + n][1] = l[a];
    }
  }
#pragma unroll
  for (int a = 0; a < R; ++a) {
    if (row0 + a * 16 >= rows) break;
    __syncthreads();
#pragma unroll
    for (int d = 0; d < kDT; ++d)
      *reinterpret_cast<f32x4*>(part + (w * 16 + n) * D + ((d * 4 + g) ^ n) * 4) = acc[a][d];
    __syncthreads();
#pragma unroll 1
    for (uint32_t e = threadIdx.x; e < 16 * (D / 4); e += kThreads) {
      const uint32_t row = e / (D / 4), c = e % (D / 4);
      float top = -INFINITY;
#pragma unroll
      for (int v = 0; v < kWaves; ++v) top = fmaxf(top, lds_ml[v][a * 16 + row][0]);
      const float base_m = top == -INFINITY ? 0.f : top;
      float sum = 0.f;
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int v = 0; v < kWaves; ++v) {
        const float weight = exp2_of(lds_ml[v][a * 16 + row][0] - base_m);
        sum += weight * lds_ml[v][a * 16 + row][1];
        o += weight * *reinterpret_cast<const f32x4*>(part + (v * 16 + row) * D + (c ^ row) * 4);
      }
      write(a * 16 + row, c * 4, o, top, sum, c == 0);
    }
  }
}

// Rows that a workgroup takes, of `rows` that a request has for one KV head: up to 32
// the waves split the tokens, past that the rows.  (48 or 64 rows with the tokens
// split fill 256 registers and spill: MI355X, 36 rows over a 4-bit cache, 48 us
// either way.)  Eight waves on 256 rows took 188 us for 252 rows over 32 x 4096 8-bit
// tokens where four on 128 take 203, but up to 60% longer where their workgroups do not
// divide evenly among the CUs.  With head_dim 256 a wave has registers for 16 rows: 320
// rows over 8 x 4096 8-bit tokens 235 us against 561 with 32 (and
// 190 since requests are split evenly).
inline uint32_t tile_rows_of(int head_dim, int64_t rows) {
  if (rows <= 16) return 16;
  if (head_dim == 256) return 64;
  return rows <= 32 ? 32 : rows <= 64 ? 64 : 128;
}

// The kernel for a head_dim and those rows.  One translation unit each.
const void* attention_kernel_d64(int type, int format, uint32_t tile_rows);
const void* attention_kernel_d128(int type, int format, uint32_t tile_rows);
const void* attention_kernel_d256(int type, int format, uint32_t tile_rows);

template <int D, int TYPE, int FORMAT>
const void* pick_rows(uint32_t tile_rows) {
  if (tile_rows == 16) return reinterpret_cast<const void*>(&attention_kernel<D, TYPE, FORMAT, 1, 1>);
  if constexpr (D != 256) {
    if (tile_rows == 32) return reinterpret_cast<const void*>(&attention_kernel<D, TYPE, FORMAT, 2, 1>);
    if (tile_rows == 128) return reinterpret_cast<const void*>(&attention_kernel<D, TYPE, FORMAT, 2, 4>);
  }
  return reinterpret_cast<const void*>(&attention_kernel<D, TYPE, FORMAT, 1, 4>);
}

template <int D, int TYPE>
const void* pick_format(int format, uint32_t tile_rows) {
  switch (format) {
    case PACE_KV_PLAIN: return pick_rows<D, TYPE, PACE_KV_PLAIN>(tile_rows);
    case PACE_KV_MXFP8: return pick_rows<D, TYPE, PACE_KV_MXFP8>(tile_rows);
    default: return pick_rows<D, TYPE, PACE_KV_MXFP4>(tile_rows);
  }
}

template <int D>
const void* pick_attention(int type, int format, uint32_t tile_rows) {
  return type == PACE_KV_BF16 ? pick_format<D, PACE_KV_BF16>(format, tile_rows)
                              : pick_format<D, PACE_KV_FP16>(format, tile_rows);
}

}  // namespace pace_kv

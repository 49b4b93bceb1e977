// Attention of each request's last tokens over a paged cache of latent vectors
// (the absorbed form): one row [c, k] of L + 64 numbers a token, shared by all heads.
//
//   s = scale * (q_l . c + q_r . k);  o = softmax(s) c
//
// with the tables, masks, parts and counting of the attention over a KV cache
// (attention.h): one KV head, whose group are all the query heads.
#include <algorithm>
#include <cmath>

#include "latent.h"

namespace pace_kv {
namespace {

constexpr uint32_t kTile = 32;                           // tokens of a step

// Which of the 32 tokens from t0 query i of request r sees (bit j: token t0 + j).
__device__ __forceinline__ uint32_t seen_of(const AttnParams& p, const Request& r, int32_t base, int32_t t0, int32_t i) {
  const int32_t d0 = t0 - base;                          // drafted token of bit 0, negative: before them
  if (p.mask == nullptr) {
    const int32_t upto = i - d0 + 1;
    return upto >= 32 ? ~0u : upto <= 0 ? 0u : (1u << upto) - 1u;
  }
  if (d0 <= -32) return ~0u;
  if (i >= static_cast<int32_t>(r.q_len)) return 0u;     // a row of padding
  const uint64_t* bits = p.mask + static_cast<int64_t>(r.q0 + static_cast<uint32_t>(i)) * p.mask_words;
  if (d0 < 0) return static_cast<uint32_t>(bits[0] << -d0) | ((1u << -d0) - 1u);
  const uint32_t word = static_cast<uint32_t>(d0) / 64, sh = static_cast<uint32_t>(d0) % 64;
  uint64_t x = word < p.mask_words ? bits[word] >> sh : 0ull;
  if (sh > 32 && word + 1 < p.mask_words) x |= bits[word + 1] << (64 - sh);
  return static_cast<uint32_t>(x);
}

// How far the 16-byte pieces of row r of a tile are xored within 256 bytes.
__device__ __forceinline__ uint32_t swap_of_row(uint32_t r) {
  const uint32_t half = r / 8 % 2;
  return ((r % 8) ^ half * 4) * 2 | half;
}

// The same of the weights' rows of 64 bytes.
__device__ __forceinline__ uint32_t swap_of_weights(uint32_t n) { return (0u - n / 4) & 3u; }

// RT tiles of 16 rows a workgroup, whose four waves sum a quarter of the columns each, of
// all rows.  Up to two tiles every wave makes the weights of all rows for itself.  Of four
// tiles a wave multiplies two by every other 32 columns of the keys, swaps halves of the
// sums with its neighbour, so that each has the scores of one tile, and the waves share the
// weights through LDS: a key that is read from there serves two products.
//
// 32 tokens a step go from memory straight to LDS, into one of two buffers while the
// other is read.  There the latents' 16-byte pieces c of row r lie at c ^ swap(r), within
// each 256 bytes, so that neither 16 rows of one piece (keys) nor 4 rows of two
// (transposed values) meet in a bank.
//
// Bound by memory where a tile is 16 or 32 rows (16 heads read 1152 bytes a token for 35
// thousand operations): the steps read 6.4 TB/s, 128 requests of up to 8192 tokens all in all
// 4.8 in 125 us; the rest is the start, where tables, page ids and rows wait for one another,
// and the last workgroups.  A step of 64 rows takes 5200 to 5500 cycles with two workgroups a
// CU: 2100 to 2500 the scores and the issue of the next rows' loads, 700 the weights, 700 the
// barriers, 1650 to 1800 the values and the products that follow a raised maximum; matrix
// instructions are busy 40 % of it (256 requests of 4096 tokens and 128 heads in 405 us, 720
// TFLOP/s).  128 rows, which would halve the reads of LDS, need more registers than four waves
// have (they spill), or two groups of waves that take turns, which wait for each other (560 us
// where this took 425).
template <int L, int TYPE, int RT>
__global__ __launch_bounds__(kThreads, 2) void latent_kernel(const AttnParams p) {
  constexpr int kW = L + kRope, kKS = L / 32, kCT = L / 64;
  constexpr bool kShare = RT >= 4;
  constexpr int RW = kShare ? 1 : RT;                    // tiles whose weights a wave makes
  constexpr int RQ = kShare ? 2 : RT, kQS = kShare ? kKS / 2 + 1 : kKS + 2;  // tiles and steps of its products
  constexpr uint32_t kRow = L * 2, kRopeAt = kTile * kRow, kBuffer = kRopeAt + kTile * kRope * 2;
  constexpr uint32_t kWeightRow = kTile * 2;
  __shared__ __attribute__((aligned(1024))) char lds[2 * kBuffer];
  // What the waves share, 2 KiB each: first sums for the neighbour, then, in the place of
  // those it has read, a wave's weights, the factors of its rows, whether any is not 1, and
  // in the end their maxima and sums.  (Two workgroups fill a CU's LDS.)
  constexpr uint32_t kShared = 2048, kShrinkAt = 1024, kRaisedAt = 1088, kMlAt = 1152;
  __shared__ __attribute__((aligned(1024))) char lds_p[kShare ? kWaves * kShared : 16];
  const uint32_t lane = threadIdx.x % 64;
  const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t at = blockIdx.x / kXcds, nth = over(p.by_unit, at);
  const uint32_t item = nth * kXcds + blockIdx.x % kXcds;
  if (item >= p.items) return;
  const uint32_t tile = at - nth * p.row_tiles;
  Place place;
  Tables tables;
  if (!find_request(p, item, [](const Tables&, uint32_t start) { return start; }, &tables, &place)) return;
  Request r;
  const bool valid_request = request_of(p, tables, &r) && has_room(p, r, place);
  r.chunk = item - place.item;
  if (r.chunk >= r.chunks) return;
  if (p.err != nullptr && tile == 0 && threadIdx.x == 0) {
    if (r.chunk == 0 && (!valid_request || is_cut(p, tables, r))) atomicAdd(p.err, 1);
    // Behind the last item lie requests that no workgroup looks at.
    if (item + 1 == p.items && place.index + 1 < p.batch)
      atomicAdd(p.err, static_cast<int32_t>(p.batch - 1 - place.index));
  }
  if (!valid_request) return;
  const uint32_t rows = r.q_len * p.group, row0 = tile * (16 * RT);
  if (row0 >= rows) return;
  const int32_t base = static_cast<int32_t>(r.kv_len) - static_cast<int32_t>(r.q_len);
  const int32_t first_q = static_cast<int32_t>(over(p.by_group, row0));
  const int32_t last_q = static_cast<int32_t>(over(p.by_group, min(row0 + 16 * RT, rows) - 1));
  // A request's chunks are of one length, in whole steps, and none is empty.
  const uint32_t even = (r.pages + r.chunks - 1) / r.chunks;
  const uint32_t length = min((even + p.step_pages - 1) / p.step_pages * p.step_pages, p.chunk_pages);
  const int32_t chunk_tokens = static_cast<int32_t>(length * p.page_size);
  const int32_t t_begin = static_cast<int32_t>(r.chunk) * chunk_tokens;
  int32_t t_end = static_cast<int32_t>(min(static_cast<int64_t>(t_begin) + chunk_tokens, static_cast<int64_t>(r.kv_len)));
  if (p.mask == nullptr) t_end = min(t_end, base + last_q + 1);
  // Tokens on pages that do not exist are counted by the last row tile's workgroup.
  if (p.err != nullptr && row0 + 16 * RT >= rows) {
    const int32_t page = static_cast<int32_t>(p.page_size), first = static_cast<int32_t>(r.chunk * length);
    for (int32_t i = static_cast<int32_t>(threadIdx.x); static_cast<int64_t>(i) * page < t_end - t_begin; i += kThreads)
      if (static_cast<uint32_t>(p.kv_indices[r.first_page + first + i]) >= p.num_pages)
        atomicAdd(p.err, min(page, t_end - t_begin - i * page));
  }

  // A step's loads: page ids (a token to a lane, the same in all waves), then rows: each
  // wave brings eight.
  int32_t id = -1;
  uint32_t row_at = 0;                                   // the lane's token's row, in 16-byte units
  uint32_t valid = 0, next_valid = 0;                    // tokens of this step and the next one that exist
  const auto load_id = [&](int32_t t0) {
    const int32_t t = t0 + static_cast<int32_t>(opaque(lane) % kTile);
    id = -1;
    if (t < t_end) id = p.kv_indices[r.first_page + static_cast<int32_t>(over(p.by_page, static_cast<uint32_t>(t)))];
  };
  const auto place_rows = [&](int32_t t0) {
    const uint32_t t = static_cast<uint32_t>(t0) + opaque(lane) % kTile;
    const bool ok = static_cast<uint32_t>(id) < p.num_pages;
    next_valid = static_cast<uint32_t>(__ballot(ok));
    row_at = ok ? static_cast<uint32_t>(id) * p.page16 + (t - over(p.by_page, t) * p.page_size) * (kW / 8) : 0u;
  };
  // The wave's part of a step's rows, 1 KiB at a time: piece i, rows that exist alone unless WHOLE.
  constexpr int kRowsOnce = 1024 / kRow, kPieces = 8 / kRowsOnce + 1;
  const auto load_piece = [&](auto whole, uint32_t ln, int i, uint32_t to) {
    constexpr uint32_t kLanes = 64 / kRowsOnce;
    uint32_t row, from, at, piece;
    if (i < kPieces - 1) {
      row = 8 * w + i * kRowsOnce;
      from = __builtin_amdgcn_readlane(row_at, 8 * w + i * kRowsOnce);
      if constexpr (kRowsOnce == 2) {
        const uint32_t second = __builtin_amdgcn_readlane(row_at, 8 * w + i * kRowsOnce + 1);
        from = ln < kLanes ? from : second;
        row += ln / kLanes;
      }
      at = to + (8 * w + i * kRowsOnce) * kRow;
      piece = (kRowsOnce == 2 ? ln % kLanes : ln) ^ swap_of_row(row);
    } else {
      row = 8 * w + ln / 8;
      from = __shfl(row_at, row);
      at = to + kRopeAt + w * 1024;
      piece = kRow / 16 + ((ln % 8) ^ (row / 2 % 8));
    }
    if (decltype(whole)::value || (next_valid >> row & 1u))
      copy_to_lds(p.cache + static_cast<int64_t>(from) * 16 + piece * 16, at);
    else
      lds_put(at + ln * 16, u32x4{0, 0, 0, 0});
  };

  constexpr int32_t kStep = static_cast<int32_t>(kTile);
  const int32_t seen_by_all = p.mask == nullptr ? base + first_q + 1 : base;
  int32_t t0 = t_begin;
  uint32_t now = lds_offset(lds), other = now + kBuffer;
  const auto load_next = [&](int32_t next, uint32_t to) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      if (next_valid == ~0u) load_piece(std::true_type{}, opaque(lane), i, to);
      else if (next < t_end) load_piece(std::false_type{}, opaque(lane), i, to);
    }
  };
  load_id(t0);

  // Query fragments: row n of each tile, eight elements from 32 k + 8 g, with the scale's
  // sign: what follows takes it as positive.  (A scale of zero makes all scores zero.)  Rows
  // behind the last read it and become zeros: loads under a condition would wait for one
  // another (MI355X: 9 us).
  const uint32_t wave_row0 = row0 + (kShare ? w * 16 : 0), query_row0 = row0 + (kShare ? w / 2 * 32 : 0);
  const uint32_t flip = p.scale_log2 < 0.f ? 0x80008000u : 0u, keep = p.scale_log2 == 0.f ? 0u : ~0u;
  const float per_score = __uint_as_float(
      __builtin_amdgcn_readfirstlane(__float_as_uint(p.scale_log2 == 0.f ? 1.f : fabsf(p.scale_log2))));
  u32x4 qf[RQ][kQS];
#pragma unroll
  for (int a = 0; a < RQ; ++a) {
    const uint32_t row = min(query_row0 + a * 16 + lane % 16, rows - 1), i = over(p.by_group, row);
    const char* const q = p.q + static_cast<int64_t>(r.q0 + i) * p.q_stride + static_cast<int64_t>(row - i * p.group) * (kW * 2);
#pragma unroll
    for (int k = 0; k < kQS; ++k)
      qf[a][k] = *reinterpret_cast<const u32x4*>(q + (kShare ? 2 * k + w % 2 : k) * 64 + lane / 16 * 16);
  }
  // The first rows are on their way before the queries have come.
  place_rows(t0);
  load_next(t0, now);
  load_id(t0 + kStep);
#pragma unroll
  for (int a = 0; a < RQ; ++a) {
    const uint32_t mask = query_row0 + a * 16 + lane % 16 < rows ? keep : 0u;
#pragma unroll
    for (int k = 0; k < kQS; ++k) qf[a][k] = (qf[a][k] ^ flip) & mask;
  }
  f32x4 acc[RT][kCT];
#pragma unroll
  for (int a = 0; a < RT; ++a)
#pragma unroll
    for (int d = 0; d < kCT; ++d) acc[a][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m[RW], l[RW];
  bool wide[RW];                                         // some row's |m| is past 2^20
#pragma unroll
  for (int a = 0; a < RW; ++a) {
    m[a] = kLowest;
    l[a] = 0.f;
    wide[a] = false;
  }

  // Scores of 32 tokens: lane: row n of each tile, tokens 16 t + 4 g + e.
  f32x4 s[RW][2];
  const uint32_t odd_step = kShare ? w % 2 * 64 : 0;
  const uint32_t my_sums = lds_offset(lds_p) + w * kShared, other_sums = lds_offset(lds_p) + (w ^ 1) * kShared;
  const auto score = [&](auto loads, uint32_t from, uint32_t to) {
    const uint32_t ln = opaque(lane), n = ln % 16, g = ln / 16;
    const uint32_t key = from + ((n * kRow + (g ^ swap_of_row(n)) * 16) ^ odd_step);
    const uint32_t rope = from + kRopeAt + ((n * (kRope * 2) + (g ^ (n / 2)) * 16) ^ odd_step);
    constexpr int kMain = kShare ? kKS / 2 : kKS;
    f32x4 x[RQ][2];
#pragma unroll
    for (int a = 0; a < RQ; ++a)
#pragma unroll
      for (int t = 0; t < 2; ++t) x[a][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    const auto read = [&](int i) {
      const int k = i / 2, t = i % 2;
      if (k >= kMain) return lds_get<u32x4>((rope ^ ((k - kMain) * 64)) + t * 16 * (kRope * 2));
      if (kShare) return lds_get<u32x4>((key ^ (k % 2 * 128)) + t * 16 * kRow + k / 2 * 256);
      return lds_get<u32x4>((key ^ (k % 4 * 64)) + t * 16 * kRow + k / 4 * 256);
    };
    // Reads stay kAhead before their products: left to itself the compiler waits for each.
    // (32 rows have no registers for more than one.)
    constexpr int kReads = 2 * kQS, kEach = kReads / kPieces, kAhead = kShare ? 4 : RT == 2 ? 1 : 8;
    u32x4 kf[kReads];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) kf[i] = read(i);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < kReads; ++i) {
      if (i + kAhead < kReads) kf[i + kAhead] = read(i + kAhead);
      if (decltype(loads)::value && i % kEach == 0 && i / kEach < kPieces) load_piece(std::true_type{}, ln, i / kEach, to);
#pragma unroll
      for (int a = 0; a < RQ; ++a) x[a][i % 2] = mfma<TYPE>(kf[i], qf[a][i / 2], x[a][i % 2]);
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (kShare) {
      const bool second = w % 2 != 0;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        lds_put(my_sums + t * 1024 + ln * 16, second ? x[0][t] : x[1][t]);
        s[0][t] = second ? x[1][t] : x[0][t];
      }
      lds_barrier();
#pragma unroll
      for (int t = 0; t < 2; ++t) s[0][t] += lds_get<f32x4>(other_sums + t * 1024 + ln * 16);
    } else {
#pragma unroll
      for (int a = 0; a < RW; ++a)
#pragma unroll
        for (int t = 0; t < 2; ++t) s[a][t] = x[a][t];
    }
  };
  // Weights of those tokens, packed by twos as they lie in s; raises the maximum where a
  // score passes it, for which shrink is the factor of what was summed before.
  u32x4 pf[RW];
  float shrink[RW];
  uint32_t raised = 0;                                   // tiles whose maximum was raised
  const auto weigh = [&](auto full, int32_t t0) {
    if constexpr (!decltype(full)::value) {
      const uint32_t ln = opaque(lane), n = ln % 16, g = ln / 16;
#pragma unroll
      for (int a = 0; a < RW; ++a) {
        const uint32_t sees =
            seen_of(p, r, base, t0, static_cast<int32_t>(over(p.by_group, wave_row0 + a * 16 + n))) & valid;
        const uint32_t mine = sees >> (4 * g);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!(mine & (1u << (t * 16 + e)))) s[a][t][e] = -INFINITY;
      }
    }
    raised = 0;
    settle(s);
#pragma unroll
    for (int a = 0; a < RW; ++a) {
      float top = max3_of(s[a][0][0], s[a][0][1], s[a][0][2]);
      top = max3_of(top, s[a][0][3], s[a][1][0]);
      top = max3_of(top, s[a][1][1], s[a][1][2]);
      top = scaled(max3_of(top, s[a][1][3], s[a][1][3]), per_score);
      shrink[a] = 1.f;
      if (__ballot(top > m[a]) != 0) {
        raised |= 1u << a;
        top = across_groups(top, max_of);
        const float next = top > m[a] ? top : m[a];
        shrink[a] = exp2_of(m[a] - next);
        m[a] = next;
        l[a] *= shrink[a];
        wide[a] = __ballot(fabsf(next) > 0x1p20f && next != kLowest) != 0;
      }
      // The fused difference holds what m lost when it was rounded: less than a tenth up
      // to 2^20, but past 2^27 enough to make the largest weight an infinity or a zero.
      if (wide[a]) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[a][t][e] = unfused(scaled(s[a][t][e], per_score), m[a]) + kUnit<TYPE>;
      } else {
        const float offset = kUnit<TYPE> - m[a];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[a][t][e] = __builtin_fmaf(s[a][t][e], per_score, offset);
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

  // Takes infinities and NaN out of the wave's columns of a buffer: a product with weight
  // zero would spread them to rows that do not see their token.
  bool odd = false;
  const auto clean = [&](uint32_t from) {
    bool found = false;
#pragma unroll 1
    for (uint32_t c = lane; c < kTile * kCT * 2; c += 64) {
      const uint32_t row = c / (kCT * 2), piece = (w * kCT * 2 + c % (kCT * 2)) ^ swap_of_row(row);
      u32x4 x = lds_get<u32x4>(from + row * kRow + piece * 16);
      bool here = false;
#pragma unroll
      for (int e = 0; e < 4; ++e) here |= odd_word<TYPE>(x[e]);
      if (here) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = finite_halves<TYPE>(x[e]);
        lds_put(from + row * kRow + piece * 16, x);
        found = true;
      }
    }
    odd |= __ballot(found) != 0;
  };

  // Adds the weighted values of the tokens in a buffer.  For weights in registers the
  // tokens of a lane's group of 16 are 4 g .. 4 g + 3 and the same behind 16; through LDS
  // they are 8 g .. 8 g + 7.
  const auto gather = [&](uint32_t from) {
    const uint32_t ln = opaque(lane), n = ln % 16, g = ln / 16;
    const uint32_t v_row = kShare ? 8 * g + n / 4 : 4 * g + n / 4;
    const uint32_t v = from + v_row * kRow + ((w * kCT * 2 + n % 4 / 2) ^ swap_of_row(v_row)) * 16 + n % 2 * 8;
    const uint32_t p_at = lds_offset(lds_p) + n * kWeightRow + (g ^ swap_of_weights(n)) * 16;  // tile a's are at (a ^ 1) * kShared
    u32x4 weight[RT];
#pragma unroll
    for (int a = 0; a < RT; ++a) {
      if constexpr (kShare) weight[a] = lds_get<u32x4>(p_at + (a ^ 1) * kShared);
      else weight[a] = pf[a];
    }
    const auto read = [&](int d) {
      const u32x2 lo = lds_transposed(v ^ (d * 32));
      const u32x2 hi = lds_transposed(kShare ? (v ^ (d * 32 ^ 128)) + 4 * kRow : (v ^ (d * 32)) + 16 * kRow);
      return u32x4{lo[0], lo[1], hi[0], hi[1]};
    };
    constexpr int kAhead = RT == 2 ? 1 : 3;
    u32x4 vf[kCT];
#pragma unroll
    for (int d = 0; d < kAhead; ++d) vf[d] = read(d);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int d = 0; d < kCT; ++d) {
      if (d + kAhead < kCT) vf[d + kAhead] = read(d + kAhead);
#pragma unroll
      for (int a = 0; a < RT; ++a) acc[a][d] = mfma<TYPE>(vf[d], weight[a], acc[a][d]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  const auto one_step = [&](auto full) {
    valid = next_valid;
    place_rows(t0 + kStep);
    rows_barrier();                                      // this step's rows are in LDS, the other buffer's readers done
    // The next step's rows are asked for between the products.
    if (next_valid == ~0u) {
      score(std::true_type{}, now, other);
    } else {
      load_next(t0 + kStep, other);
      score(std::false_type{}, now, other);
    }
    load_id(t0 + 2 * kStep);
    weigh(full, t0);
    if constexpr (kShare) {
      const uint32_t ln = opaque(lane), n = ln % 16, g = ln / 16;
#pragma unroll
      for (int t = 0; t < 2; ++t)
        lds_put(other_sums + n * kWeightRow + ((2 * t + g / 2) ^ swap_of_weights(n)) * 16 + g % 2 * 8,
                u32x2{pf[0][2 * t], pf[0][2 * t + 1]});
      if (g == 0) lds_put(other_sums + kShrinkAt + n * 4, shrink[0]);
      if (ln == 0) lds_put(other_sums + kRaisedAt, raised);
    }
    if (kShare || !decltype(full)::value) lds_barrier();
    if constexpr (!decltype(full)::value) clean(now);
    if constexpr (kShare) {
      const uint32_t ln = opaque(lane), n = ln % 16;
      const uint32_t any = lds_get<uint32_t>(lds_offset(lds_p) + ln % kWaves * kShared + kRaisedAt);
      const uint64_t which = __ballot(any != 0);         // bit a: tile a ^ 1
      if (which != 0) {
#pragma unroll
        for (int a = 0; a < RT; ++a)
          if (which >> (a ^ 1) & 1u) {
            const float by = lds_get<float>(lds_offset(lds_p) + (a ^ 1) * kShared + kShrinkAt + n * 4);
#pragma unroll
            for (int d = 0; d < kCT; ++d) acc[a][d] *= by;
          }
      }
    } else {
#pragma unroll
      for (int a = 0; a < RT; ++a)
        if (raised & (1u << a)) {
#pragma unroll
          for (int d = 0; d < kCT; ++d) acc[a][d] *= shrink[a];
        }
    }
    gather(now);
    const uint32_t x = now;
    now = other;
    other = x;
    t0 += kStep;
  };
  // The steps whose tokens every row sees, then the others.
  while (t0 + kStep <= seen_by_all && next_valid == ~0u) one_step(std::true_type{});
  const int32_t t_masked = t0;
#pragma unroll 1
  while (t0 < t_end) one_step(std::false_type{});
  const uint32_t ln = opaque(lane), n = ln % 16, g = ln / 16;
#pragma unroll
  for (int a = 0; a < RW; ++a) {
    l[a] = across_groups(l[a], sum_of);
    if constexpr (kShare)
      if (g == 0) lds_put(other_sums + kMlAt + n * 8, f32x2{m[a], l[a]});
  }
  if (kShare) __syncthreads();
  const bool direct = r.chunks == 1;
  const int64_t part_row0 = (static_cast<int64_t>(place.part() + r.chunk) * p.row_tiles + tile) * (16 * RT);
  const auto out_at = [&](uint32_t row) {
    const uint32_t i = over(p.by_group, row);
    return p.out + static_cast<int64_t>(r.q0 + i) * p.out_stride + static_cast<int64_t>(row - i * p.group) * (L * 2);
  };
  const uint32_t col0 = w * kCT * 16 + g * 4;
#pragma unroll
  for (int a = 0; a < RT; ++a) {
    const uint32_t in_tile = a * 16 + n, row = row0 + in_tile;
    if (row >= rows) continue;
    float top, sum;
    if constexpr (kShare) {
      const f32x2 ml = lds_get<f32x2>(lds_offset(lds_p) + (a ^ 1) * kShared + kMlAt + n * 8);
      top = ml[0];
      sum = ml[1];
    } else {
      top = m[a];
      sum = l[a];
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    char* const out = out_at(row);
#pragma unroll
    for (int d = 0; d < kCT; ++d) {
      const f32x4 o = acc[a][d];
      if (!direct) {
        *reinterpret_cast<f32x4*>(p.part_o + (part_row0 + in_tile) * L + col0 + d * 16) = o;
      } else {
        const u32x2 x = {result_pair<TYPE>(o[0] * inv, o[1] * inv), result_pair<TYPE>(o[2] * inv, o[3] * inv)};
        *reinterpret_cast<u32x2*>(out + (col0 + d * 16) * 2) = x;
      }
    }
    if (w == 0 && g == 0) {
      if (!direct) {
        p.part_ml[(part_row0 + in_tile) * 2] = top;
        p.part_ml[(part_row0 + in_tile) * 2 + 1] = sum;
      } else if (p.lse != nullptr) {
        const uint32_t i = over(p.by_group, row);
        p.lse[static_cast<int64_t>(r.q0 + i) * p.group + (row - i * p.group)] = log_total<TYPE>(top, sum);
      }
    }
  }
  if (!odd) return;
  // An infinity or a NaN in a latent that a row sees is in its score too: either the row
  // has no sum (NaN), or the token's weight is zero, and zero times it makes its column NaN.
#pragma unroll 1
  for (uint32_t a = 0; a < RT; ++a) {
    const uint32_t in_tile = a * 16 + n, row = row0 + in_tile;
    if (row >= rows) continue;
    char* const out = out_at(row);
#pragma unroll 1
    for (int32_t t = t_masked; t < t_end; ++t) {
      const uint32_t page = over(p.by_page, static_cast<uint32_t>(t));
      const uint32_t of = static_cast<uint32_t>(p.kv_indices[r.first_page + static_cast<int32_t>(page)]);
      if (of >= p.num_pages || !(seen_of(p, r, base, t, static_cast<int32_t>(over(p.by_group, row))) & 1u)) continue;
      const char* const x = p.cache + (static_cast<int64_t>(of) * p.page_size + (static_cast<uint32_t>(t) - page * p.page_size)) *
                                          (kW * 2) + col0 * 2;
#pragma unroll 1
      for (uint32_t c = 0; c < kCT * 4; ++c) {
        const uint32_t col = c / 4 * 16 + c % 4;
        if (!odd_word<TYPE>(*reinterpret_cast<const uint16_t*>(x + col * 2))) continue;
        if (!direct) p.part_o[(part_row0 + in_tile) * L + col0 + col] = NAN;
        else *reinterpret_cast<uint16_t*>(out + (col0 + col) * 2) = 0x7fffu;
      }
    }
  }
}

// Joins the parts of split requests' rows, WAVES waves a row (four where the rows alone do
// not fill the GPU): the chunks' maxima and sums come first, 64 at a time, so that the loads
// of their outputs do not wait for one another.
template <int L, int TYPE, uint32_t WAVES>
__global__ __launch_bounds__(kThreads) void latent_join_kernel(const AttnParams p) {
  constexpr uint32_t kVec = L / 64;                      // columns of a lane
  typedef float vec __attribute__((ext_vector_type(kVec)));
  __shared__ vec lds_o[WAVES == 1 ? 1 : WAVES][WAVES == 1 ? 1 : 64];
  const uint32_t lane = threadIdx.x % 64, w = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t id = WAVES == 1 ? blockIdx.x * kWaves + w : blockIdx.x;
  const uint32_t token = over(p.by_heads, id), head = id - token * p.group, part = WAVES == 1 ? 0 : w;
  if (token >= p.nnz) return;
  Tables t;
  Place place;
  if (!find_request(p, token, [](const Tables& x, uint32_t) { return static_cast<uint32_t>(max(x.a0, 0)); }, &t, &place))
    return;
  Request r;
  if (!(request_of(p, t, &r) && token >= r.q0 && token - r.q0 < r.q_len && r.chunks > 1 && has_room(p, r, place))) return;
  const uint32_t row = (token - r.q0) * p.group + head, tile = row / p.tile_rows;
  const int64_t first = (static_cast<int64_t>(place.part()) * p.row_tiles + tile) * p.tile_rows + row % p.tile_rows;
  const int64_t step = static_cast<int64_t>(p.row_tiles) * p.tile_rows;
  // A wave's parts of 64 chunks; the first ones are asked for before their weights are known.
  constexpr uint32_t kParts = 4;
  vec x[kParts];
  const auto load = [&](uint32_t c0) {
#pragma unroll
    for (uint32_t j = 0; j < kParts; ++j)
      x[j] = *reinterpret_cast<const vec*>(p.part_o + (first + min(c0 + part + j * WAVES, r.chunks - 1) * step) * L + lane * kVec);
  };
  load(0);
  // The maximum over all chunks, which every wave finds for itself.
  float m = -INFINITY;
  for (uint32_t c = lane; c < r.chunks; c += 64) m = fmaxf(m, p.part_ml[(first + c * step) * 2]);
#pragma unroll
  for (int k = 1; k < 64; k *= 2) m = fmaxf(m, __shfl_xor(m, k));
  const float from = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  vec o = {};
  for (uint32_t c0 = 0; c0 < r.chunks; c0 += 64) {
    float weight = 0.f;
    if (c0 + lane < r.chunks) {
      const int64_t at = (first + (c0 + lane) * step) * 2;
      weight = exp2_of(p.part_ml[at] - from);
      l += weight * p.part_ml[at + 1];
    }
    const uint32_t n = min(r.chunks - c0, 64u);
    for (uint32_t c = part; c < n;) {
#pragma unroll
      for (uint32_t j = 0; j < kParts; ++j, c += WAVES)
        if (c < n) o += __shfl(weight, c) * x[j];
      const uint32_t after = c < n ? c0 + c - part : c0 + 64;
      if (after < r.chunks) load(after);
    }
  }
#pragma unroll
  for (int k = 1; k < 64; k *= 2) l += __shfl_xor(l, k);
  if constexpr (WAVES > 1) {
    if (w != 0) lds_o[w][lane] = o;
    __syncthreads();
    if (w != 0) return;
#pragma unroll
    for (uint32_t v = 1; v < WAVES; ++v) o += lds_o[v][lane];
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  char* const out = p.out + static_cast<int64_t>(token) * p.out_stride + (static_cast<int64_t>(head) * L + lane * kVec) * 2;
#pragma unroll
  for (uint32_t k = 0; k < kVec; k += 2)
    *reinterpret_cast<uint32_t*>(out + k * 2) = result_pair<TYPE>(o[k] * inv, o[k + 1] * inv);
  if (lane == 0 && p.lse != nullptr) p.lse[static_cast<int64_t>(token) * p.group + head] = log_total<TYPE>(m, l);
}

struct Split {
  uint32_t tile_rows, row_tiles, chunk_pages, step_pages, items, parts;
  int64_t part_rows() const { return static_cast<int64_t>(parts) * row_tiles * tile_rows; }
};

// A call's contexts are cut so that the CUs' places for workgroups (two a CU, or three of 256
// columns: 128 requests of up to 8192 tokens and 16 heads then take 86 us instead of 94) are
// filled evenly.  With w workgroups of n steps on P places a call takes about
// ceil(w / P) (n + kStart) steps, and, where requests are cut, the joining kernel: its launch,
// and the parts written and read.  Of the requests' lengths the host knows only the sum: w is
// taken as the mean of what equal lengths give and what lengths spread evenly give, whose last
// chunks are half empty.
constexpr int64_t kStart = 3, kJoin = 2, kPartBytes = int64_t(8) << 20;

Split split_of(int64_t batch, int64_t rows, int latent_dim, int64_t num_indices, int64_t page_size) {
  Split s = {};
  s.tile_rows = rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
  s.row_tiles = static_cast<uint32_t>((rows + s.tile_rows - 1) / s.tile_rows);
  s.step_pages = static_cast<uint32_t>(kTile % page_size ? 1 : kTile / page_size);
  const int64_t requests = std::max<int64_t>(batch, 1), pages = std::max<int64_t>((num_indices + requests - 1) / requests, 1);
  const auto steps_of = [&](int64_t chunk) { return (chunk * page_size + kTile - 1) / kTile; };
  const int64_t places = latent_dim == 256 ? 768 : 512;
  const auto turns_of = [&](int64_t items) { return (items * s.row_tiles + places - 1) / places; };
  const int64_t part_bytes = requests * rows * latent_dim * 8;
  int64_t chunk = pages, best = INT64_MAX, before = 0;
  const int64_t most = std::min<int64_t>(std::max<int64_t>(steps_of(pages), 1), 256);
  for (int64_t k = 1; k <= most; ++k) {
    const int64_t length = ((pages + k - 1) / k + s.step_pages - 1) / s.step_pages * s.step_pages;
    if (length == before) continue;
    before = length;
    const int64_t even = requests * ((pages + length - 1) / length);
    const int64_t spread = batch > 1 ? num_indices / length + requests / 2 : even;
    const int64_t join = k == 1 ? 0 : 2 * kJoin + 2 * part_bytes * k / kPartBytes;
    const int64_t cost = (turns_of(even) + turns_of(spread)) * (steps_of(length) + kStart) + join;
    if (cost < best) {
      best = cost;
      chunk = length;
    }
  }
  chunk = std::max<int64_t>(std::min(chunk, num_indices), 1);
  s.chunk_pages = static_cast<uint32_t>(chunk);
  s.items = static_cast<uint32_t>(num_indices / chunk + batch);
  s.parts = chunk >= num_indices ? 0 : batch == 1 ? s.items : static_cast<uint32_t>(2 * (num_indices / chunk));
  return s;
}

// Workgroups of a launch, whose threads are counted in 32 bits.
constexpr int64_t kMostGroups = int64_t(1) << 24;

int check_sizes(int batch_size, int heads, int latent_dim, int max_q_len, int64_t num_indices, int page_size) {
  if (batch_size < 0 || heads <= 0 || max_q_len <= 0 || num_indices < 0 || page_size <= 0)
    return fail(PACE_KV_EINVAL, "latent attention: sizes must be positive");
  if (latent_dim != 256 && latent_dim != 512)
    return fail(PACE_KV_EINVAL, "latent attention: latent_dim must be 256 or 512, got %d", latent_dim);
  const int64_t rows = static_cast<int64_t>(max_q_len) * heads;
  if (num_indices > INT32_MAX / 2 / page_size || rows > INT32_MAX / 2)
    return fail(PACE_KV_ERANGE, "latent attention: more than 2^30 tokens or query rows");
  bool fits = batch_size < kMostGroups;
  if (fits) {
    const Split s = split_of(batch_size, rows, latent_dim, num_indices, page_size);
    fits = s.row_tiles < kMostGroups && (static_cast<int64_t>(s.items) + kXcds) * s.row_tiles < kMostGroups;
  }
  if (!fits) return fail(PACE_KV_ERANGE, "latent attention: too many requests, heads or query rows for one call");
  return PACE_KV_OK;
}

int64_t workspace_bytes(const Split& s, int latent_dim) { return s.part_rows() * (latent_dim + 2) * 4; }

template <int L, int TYPE>
const void* pick_latent(uint32_t tile_rows) {
  switch (tile_rows) {
    case 16: return reinterpret_cast<const void*>(&latent_kernel<L, TYPE, 1>);
    case 32: return reinterpret_cast<const void*>(&latent_kernel<L, TYPE, 2>);
    default: return reinterpret_cast<const void*>(&latent_kernel<L, TYPE, 4>);
  }
}

template <int L>
const void* pick_latent(int type, uint32_t tile_rows) {
  return type == PACE_KV_BF16 ? pick_latent<L, PACE_KV_BF16>(tile_rows) : pick_latent<L, PACE_KV_FP16>(tile_rows);
}

// Rows of a call from which on a wave joins one by itself.  (MI355X, calls with four waves a
// row and with one: 16 rows of 63 parts 16 us and 21, 4096 rows 84 and 79, 12800 124 and 104.)
constexpr int64_t kManyRows = 4096;

template <int L, int TYPE>
const void* pick_join(bool many) {
  return many ? reinterpret_cast<const void*>(&latent_join_kernel<L, TYPE, 1>)
              : reinterpret_cast<const void*>(&latent_join_kernel<L, TYPE, kWaves>);
}

template <int L>
const void* pick_join(int type, bool many) {
  return type == PACE_KV_BF16 ? pick_join<L, PACE_KV_BF16>(many) : pick_join<L, PACE_KV_FP16>(many);
}

}  // namespace
}  // namespace pace_kv

extern "C" {

int pace_kv_latent_attention_workspace(int batch_size, int num_heads, int latent_dim, int max_q_len, int64_t num_indices,
                                       int page_size, int64_t* bytes) {
  using namespace pace_kv;
  if (!bytes) return fail(PACE_KV_EINVAL, "latent attention: NULL argument");
  PACE_KV_TRY(check_sizes(batch_size, num_heads, latent_dim, max_q_len, num_indices, page_size));
  *bytes = workspace_bytes(split_of(batch_size, static_cast<int64_t>(max_q_len) * num_heads, latent_dim, num_indices, page_size),
                           latent_dim);
  return PACE_KV_OK;
}

int pace_kv_latent_attention(const void* q, int64_t q_stride_bytes, int elem_type, int64_t nnz, const int32_t* qo_indptr,
                             int batch_size, int num_heads, int latent_dim, const void* cache, int64_t num_pages,
                             int page_size, const int32_t* kv_indices, int64_t num_indices, const int32_t* kv_indptr,
                             const int32_t* kv_last_page_len, int max_q_len, const uint64_t* tree_mask, int mask_words,
                             float scale, void* out, int64_t out_stride_bytes, float* lse, void* workspace,
                             int64_t workspace_size, int32_t* err_count, void* stream) {
  using namespace pace_kv;
  if (nnz < 0) return fail(PACE_KV_EINVAL, "latent attention: negative size");
  PACE_KV_TRY(check_sizes(batch_size, num_heads, latent_dim, max_q_len, num_indices, page_size));
  if (elem_type != PACE_KV_BF16 && elem_type != PACE_KV_FP16)
    return fail(PACE_KV_EINVAL, "latent attention: queries must be bfloat16 or float16");
  if (num_pages < 0 || num_pages > INT32_MAX || nnz > INT32_MAX / 2)
    return fail(PACE_KV_ERANGE, "latent attention: too many pages or tokens");
  const float scale_log2 = scale * 1.44269504088896341f;
  if (!std::isfinite(scale_log2)) return fail(PACE_KV_EINVAL, "latent attention: scale must be within float's range");
  if (nnz * num_heads >= (int64_t(1) << 24)) return fail(PACE_KV_ERANGE, "latent attention: 2^24 query rows or more");
  if (nnz == 0 || batch_size == 0) return PACE_KV_OK;
  if (!q || (num_pages > 0 && !cache) || !kv_indptr || !kv_last_page_len || !out || (num_indices > 0 && !kv_indices))
    return fail(PACE_KV_EINVAL, "latent attention: NULL argument");
  if (!qo_indptr && nnz != batch_size)
    return fail(PACE_KV_EINVAL, "latent attention: without qo_indptr each request has one token");
  if (tree_mask && (mask_words <= 0 || max_q_len > static_cast<int64_t>(mask_words) * 64))
    return fail(PACE_KV_EINVAL, "latent attention: max_q_len tokens need a mask of ceil(max_q_len / 64) words");
  const int64_t width = latent_dim + kRope, q_row = width * num_heads * 2, out_row = int64_t(2) * latent_dim * num_heads;
  if (q_stride_bytes < q_row || q_stride_bytes % 16 || out_stride_bytes < out_row || out_stride_bytes % 16)
    return fail(PACE_KV_EINVAL, "latent attention: token strides must hold a row and be multiples of 16");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(cache) | reinterpret_cast<uintptr_t>(out)) & 15u ||
      reinterpret_cast<uintptr_t>(tree_mask) & 7u)
    return fail(PACE_KV_EINVAL, "latent attention: q, cache and out must be 16-byte aligned, mask 8-byte");
  if (page_size > (INT64_C(1) << 36) / (width * 2) || num_pages * (page_size * width / 8) >= UINT32_MAX)
    return fail(PACE_KV_ERANGE, "latent attention: a layer's cache must be smaller than 64 GiB");
  const Split s = split_of(batch_size, static_cast<int64_t>(max_q_len) * num_heads, latent_dim, num_indices, page_size);
  const int64_t need = workspace_bytes(s, latent_dim);
  if (need > 0 && (!workspace || workspace_size < need || reinterpret_cast<uintptr_t>(workspace) & 15u))
    return fail(PACE_KV_EINVAL, "latent attention: needs a 16-byte aligned workspace of %lld bytes", (long long)need);
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
  p.part_ml = p.part_o + s.part_rows() * latent_dim;
  p.err = err_count;
  p.num_indices = static_cast<uint32_t>(num_indices);
  p.batch = static_cast<uint32_t>(batch_size);
  p.nnz = static_cast<uint32_t>(nnz);
  p.heads = 1;
  p.group = static_cast<uint32_t>(num_heads);
  p.num_pages = static_cast<uint32_t>(num_pages);
  p.page_size = static_cast<uint32_t>(page_size);
  p.max_q = static_cast<uint32_t>(qo_indptr ? max_q_len : 1);
  p.chunk_pages = s.chunk_pages;
  p.step_pages = s.step_pages;
  p.items = s.items;
  p.parts = s.parts;
  p.row_tiles = s.row_tiles;
  p.tile_rows = s.tile_rows;
  p.page16 = static_cast<uint32_t>(page_size * width / 8);
  p.by_page = fast_div(p.page_size);
  p.by_chunk = fast_div(p.chunk_pages);
  p.by_group = fast_div(p.group);
  p.by_heads = fast_div(p.group);
  p.by_unit = fast_div(p.row_tiles);
  p.scale_log2 = scale_log2;
  const uint32_t items = (s.items + kXcds - 1) / kXcds * kXcds;
  void* args[] = {&p};
  PACE_KV_TRY(hip_status(hipLaunchKernel(latent_dim == 512 ? pick_latent<512>(elem_type, s.tile_rows)
                                                           : pick_latent<256>(elem_type, s.tile_rows),
                                         dim3(items * p.row_tiles), dim3(kThreads), args, 0,
                                         static_cast<hipStream_t>(stream)), "latent attention launch"));
  if (need == 0) return PACE_KV_OK;
  const int64_t out_rows = nnz * num_heads;
  const bool many = out_rows >= kManyRows;
  return hip_status(hipLaunchKernel(latent_dim == 512 ? pick_join<512>(elem_type, many) : pick_join<256>(elem_type, many),
                                    dim3(static_cast<uint32_t>(many ? (out_rows + kWaves - 1) / kWaves : out_rows)),
                                    dim3(kThreads), args, 0, static_cast<hipStream_t>(stream)),
                    "latent attention join launch");
}

}  // extern "C"

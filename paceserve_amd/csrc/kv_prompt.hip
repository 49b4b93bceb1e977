// Attention of prompts over keys and values that are expanded from latent vectors:
// each head has Dn columns of keys and of values of its own, and all heads share a
// token's 64 rotated columns.
//
//   s_h = scale * (q_h . k_h + q_r . k_r);  o_h = softmax(s_h) v_h
//
// Request b's queries are rows qo_indptr[b] .. qo_indptr[b + 1], its keys
// kv_indptr[b] .. kv_indptr[b + 1]; causal: query i of q_len sees the keys up to
// kv_len - q_len + i.
#include <algorithm>
#include <cmath>

#include "latent.h"

namespace pace_kv {
namespace {

constexpr uint32_t kTile = 32;                           // keys of a step
constexpr uint32_t kLoadRows = kTile / kWaves;           // of which a wave loads so many
constexpr int kRT = 2;                                   // tiles of 16 query rows of a wave
constexpr uint32_t kRows = 16 * kRT * kWaves;            // query rows of a workgroup

struct PromptParams {
  const char* q;
  const char* key;
  const char* rope_key;
  const char* value;
  char* out;
  float* lse;                  // [nnz, heads], or nullptr
  const int32_t* qo_indptr;
  const int32_t* kv_indptr;
  int32_t* err;
  float* part_o;               // [parts, nnz, heads, DN], of more than one
  float* part_ml;              // [parts, nnz, heads, 2]
  int64_t q_token, q_head, k_token, k_head, r_token, v_token, v_head, o_token, o_head;  // strides in bytes
  uint32_t batch, nnz, keys, heads, max_q, tiles, parts;
  float scale_log2;
  uint32_t causal;
};

struct PromptRequest {
  uint32_t tile;
  int32_t q0, q1, k0, k1;      // its rows of queries and keys
};

// Whether a request's queries are among the rows, and not too many.
__device__ __forceinline__ bool has_rows(const PromptParams& p, int32_t q0, int32_t q1) {
  return q0 >= 0 && q1 > q0 && static_cast<uint32_t>(q1) <= p.nnz && static_cast<uint32_t>(q1 - q0) <= p.max_q;
}

__device__ __forceinline__ uint32_t tiles_of(int32_t q0, int32_t q1) {
  return (static_cast<uint32_t>(q1 - q0) + kRows - 1) / kRows;
}

// Row tile x of a call and its request; false past the last.  A request's tiles that see the
// most keys come first, and of up to 64 requests, a lane each, the one with the most: a long
// tile that starts last would keep the call waiting.  (MI355X, 16 heads of 8 requests of up
// to 2000 tokens in order 130 us, so 110; all tiles by their keys 109, but 4 requests of
// 128 heads, whose keys then share the caches, 826 and 998.)
__device__ __forceinline__ bool find_tile(const PromptParams& p, uint32_t x, PromptRequest* r) {
  const uint32_t lane = threadIdx.x % 64;
  const auto load = [&](uint32_t b) {
    PromptRequest mine = {0, 0, 0, 0, 0};
    if (b < p.batch) {
      mine.q0 = p.qo_indptr[b];
      mine.q1 = p.qo_indptr[b + 1];
      mine.k0 = p.kv_indptr[b];
      mine.k1 = p.kv_indptr[b + 1];
    }
    return mine;
  };
  const auto take = [&](const PromptRequest& of, int at, uint32_t tile) {
    r->q0 = __builtin_amdgcn_readlane(of.q0, at);
    r->q1 = __builtin_amdgcn_readlane(of.q1, at);
    r->k0 = min(max(__builtin_amdgcn_readlane(of.k0, at), 0), static_cast<int32_t>(p.keys));
    r->k1 = min(max(__builtin_amdgcn_readlane(of.k1, at), r->k0), static_cast<int32_t>(p.keys));
    r->tile = tile;
    return true;
  };
  const auto total_of = [](uint32_t v) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(sum_upto(v), 63)); };
  PromptRequest mine = load(lane);
  uint32_t n = has_rows(p, mine.q0, mine.q1) ? tiles_of(mine.q0, mine.q1) : 0u;
  const uint32_t total = total_of(n);
  if (p.batch <= 64 && total <= p.tiles) {
    if (x >= total) return false;
    const int64_t most = n > 0 ? max(static_cast<int64_t>(mine.k1) - mine.k0, int64_t(0)) : -1;
    const int32_t key = static_cast<int32_t>(min(most, int64_t(INT32_MAX)));
    uint32_t first = 0;                                  // tiles of the requests before the lane's
    for (uint32_t j = 0; j < p.batch; ++j) {
      const int32_t other = __builtin_amdgcn_readlane(key, j);
      const uint32_t tiles = __builtin_amdgcn_readlane(n, j);
      if (other > key || (other == key && j < lane)) first += tiles;
    }
    const uint64_t here = __ballot(x >= first && x - first < n);
    const int at = here != 0 ? __builtin_ctzll(here) : 0;
    return take(mine, at, __builtin_amdgcn_readlane(n, at) - 1 - (x - __builtin_amdgcn_readlane(first, at)));
  }
  const uint32_t y = p.tiles - 1 - x;
  uint32_t done = 0;
  for (uint32_t b0 = 0; b0 < p.batch; b0 += 64) {
    if (b0 != 0) {
      mine = load(b0 + lane);
      n = has_rows(p, mine.q0, mine.q1) ? tiles_of(mine.q0, mine.q1) : 0u;
    }
    const uint32_t upto = done + sum_upto(n);
    const uint64_t past = __ballot(y < upto);
    if (past != 0) {
      const int at = __builtin_ctzll(past);
      return take(mine, at, y - (__builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(n, at)));
    }
    done = __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

// Counts the requests that are skipped or cut; by one wave.
__device__ __forceinline__ void count_bad(const PromptParams& p) {
  const uint32_t lane = threadIdx.x % 64;
  uint32_t before = 0;
  for (uint32_t b0 = 0; b0 < p.batch; b0 += 64) {
    const uint32_t b = b0 + lane;
    uint32_t n = 0;
    bool fine = true;
    if (b < p.batch) {
      const int32_t q0 = p.qo_indptr[b], q1 = p.qo_indptr[b + 1], k0 = p.kv_indptr[b], k1 = p.kv_indptr[b + 1];
      const bool rows = has_rows(p, q0, q1);
      n = rows ? tiles_of(q0, q1) : 0u;
      fine = (rows || q0 == q1) && q0 >= 0 && static_cast<uint32_t>(q1) <= p.nnz && k0 >= 0 && k1 >= k0 &&
             static_cast<uint32_t>(k1) <= p.keys;
    }
    const uint32_t upto = before + sum_upto(n);
    if (upto > p.tiles && n > 0) fine = false;           // offsets that overlap: more tiles than nnz rows have
    if (!fine) atomicAdd(p.err, 1);
    before = __builtin_amdgcn_readlane(upto, 63);
  }
}

// How far the 16-byte pieces of row r of a tile are xored, within 256 bytes (rows of 128
// columns) or 128 (of 64, two rows to 256): neither 16 rows of one piece (keys) nor 4 rows
// of two (transposed values) meet in a bank.
template <int D>
__device__ __forceinline__ uint32_t swap_of(uint32_t r) {
  const uint32_t half = r / 8 % 2;
  return D == 128 ? ((r % 8) ^ half * 4) * 2 | half : ((r / 2 % 4) ^ half * 2) * 2 | half;
}

// A workgroup takes 128 query rows of a head, 32 a wave, and passes over the keys they see,
// 32 at a time: rows go from memory straight to LDS, into one of two buffers while the
// other is read.  With 128 columns the buffers take 40 KiB, so that three workgroups fit a CU
// and one's softmax may lie under another's products.
//
// Bound by the SIMDs' issue: of 1390 cycles that a wave's step takes of one, matrix
// instructions are 640 and vector ones about 720, 256 of them exponentials and some 80 the
// products that follow a raised maximum; LDS is busy a quarter of the time, without conflicts
// (MI355X, 4096 queries of 32 heads behind 4096 keys in 499 us, 1033 TFLOP/s; 8192 alone in
// 628, 1095).  Every instruction less shows: lanes'
// places in memory kept in registers were 6 %, a finite lowest maximum 3.  Two workgroups
// with 64 keys a step took 743 us where three with 32 took 693.  Waves of long tiles at a
// higher priority: no change.
template <int DN, int TYPE>
__global__ __launch_bounds__(kThreads, 3) void prompt_kernel(const PromptParams p) {
  constexpr int kNS = DN / 32, kCT = DN / 16;
  constexpr uint32_t kRow = DN * 2, kRopeRow = kRope * 2;
  constexpr uint32_t kRopeAt = kTile * kRow, kValueAt = kRopeAt + kTile * kRopeRow, kBuffer = kValueAt + kTile * kRow;
  __shared__ __attribute__((aligned(1024))) char lds[2 * kBuffer];
  const uint32_t lane = threadIdx.x % 64, g = lane / 16, n = lane % 16;
  const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t head = blockIdx.x;
  if (p.err != nullptr && blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0 && w == 0) count_bad(p);
  PromptRequest r;
  if (!find_tile(p, blockIdx.y, &r)) return;
  const int32_t k0 = r.k0, q_len = r.q1 - r.q0, kv_len = r.k1 - r.k0, base = kv_len - q_len;
  const int32_t row0 = static_cast<int32_t>(r.tile * kRows), wave_row0 = row0 + static_cast<int32_t>(w * 16 * kRT);
  int32_t t_end = kv_len;
  if (p.causal) t_end = min(t_end, base + min(row0 + static_cast<int32_t>(kRows), q_len));
  // The keys that the tile sees are dealt to its workgroups in whole steps.
  int32_t t_begin = 0;
  if (p.parts > 1) {
    const uint32_t steps = (static_cast<uint32_t>(max(t_end, 0)) + kTile - 1) / kTile;
    const uint32_t each = (steps + p.parts - 1) / p.parts * kTile;
    t_begin = static_cast<int32_t>(blockIdx.z * each);
    t_end = min(t_end, t_begin + static_cast<int32_t>(each));
  }
  // Keys that a row sees: those before `seen_by`.
  const auto seen_by = [&](int32_t row) { return p.causal ? base + row + 1 : kv_len; };

  // A step's loads: kLoadRows rows of keys, rotated parts and values a wave, 1 KiB an instruction.
  const char* const key0 = p.key + k0 * p.k_token + head * p.k_head;
  const char* const value0 = p.value + k0 * p.v_token + head * p.v_head;
  const char* const rope0 = p.rope_key + k0 * p.r_token;
  // A lane's place in them: the row within an instruction's, and the piece that belongs at its
  // place in LDS; four rows further on that is the piece eight away.  Held in registers over
  // the steps that have no masks (8192 tokens of 32 heads 719 us, so 690), else derived anew.
  struct Places {
    uint32_t key, rope, value, four_on;
  };
  const auto place_of = [&](uint32_t ln, auto dim, int64_t stride) {
    constexpr uint32_t kD = decltype(dim)::value, kLanes = kD / 8;
    const uint32_t in = ln / kLanes;
    return in * static_cast<uint32_t>(stride) + ((ln % kLanes) ^ swap_of<kD>(w * kLoadRows + in)) * 16;
  };
  const auto places_of = [&](uint32_t ln) {
    return Places{place_of(ln, std::integral_constant<int, DN>{}, p.k_token),
                  place_of(ln, std::integral_constant<int, kRope>{}, p.r_token),
                  place_of(ln, std::integral_constant<int, DN>{}, p.v_token),
                  (ln ^ swap_of<DN>(w * kLoadRows + ln / 16)) & 8u ? 0u - 128u : 128u};
  };
  const auto load_part = [&](auto whole, auto dim, const char* from, int64_t stride, uint32_t place, uint32_t four_on,
                             int32_t t0, uint32_t to) {
    constexpr uint32_t kD = decltype(dim)::value, kLanes = kD / 8, kAtOnce = 64 / kLanes;
#pragma unroll
    for (uint32_t i = 0; i < kLoadRows; i += kAtOnce) {
      const uint32_t row = w * kLoadRows + i, at = to + row * (kD * 2);
      const char* const rows = from + (static_cast<int64_t>(t0) + row) * stride;
      const char* const x = rows + static_cast<uint64_t>(i == 0 ? place : place + four_on);
      const uint32_t ln = decltype(whole)::value ? 0u : opaque(lane);
      if (decltype(whole)::value || t0 + static_cast<int32_t>(row + ln / kLanes) < t_end) copy_to_lds(x, at);
      else lds_put(at + ln * 16, u32x4{0, 0, 0, 0});
    }
  };
  const auto load_step = [&](auto whole, const Places& at, int32_t t0, uint32_t to) {
    load_part(whole, std::integral_constant<int, DN>{}, key0, p.k_token, at.key, at.four_on, t0, to);
    load_part(whole, std::integral_constant<int, kRope>{}, rope0, p.r_token, at.rope, 0u, t0, to + kRopeAt);
    load_part(whole, std::integral_constant<int, DN>{}, value0, p.v_token, at.value, at.four_on, t0, to + kValueAt);
  };
  const auto load_next = [&](int32_t t0, uint32_t to) {
    if (t0 >= t_end) return;
    const Places at = places_of(opaque(lane));
    if (t0 + static_cast<int32_t>(kTile) <= t_end) load_step(std::true_type{}, at, t0, to);
    else load_step(std::false_type{}, at, t0, to);
  };

  constexpr int32_t kStep = static_cast<int32_t>(kTile);
  uint32_t now = lds_offset(lds), other = now + kBuffer;
  int32_t t0 = t_begin;
  load_next(t0, now);

  // Query fragments with the scale's sign: what follows takes it as positive.  (A scale
  // of zero makes all scores zero.)  Rows behind the last read it and become zeros: loads
  // under a condition would wait for one another (MI355X: 6 us).
  const uint32_t flip = p.scale_log2 < 0.f ? 0x80008000u : 0u, keep = p.scale_log2 == 0.f ? 0u : ~0u;
  const float per_score = __uint_as_float(
      __builtin_amdgcn_readfirstlane(__float_as_uint(p.scale_log2 == 0.f ? 1.f : fabsf(p.scale_log2))));
  u32x4 qf[kRT][kNS + 2];
#pragma unroll
  for (int a = 0; a < kRT; ++a) {
    const int32_t row = min(wave_row0 + a * 16 + static_cast<int32_t>(n), q_len - 1);
    const char* const q = p.q + static_cast<int64_t>(r.q0 + row) * p.q_token + head * p.q_head;
#pragma unroll
    for (int k = 0; k < kNS + 2; ++k) qf[a][k] = *reinterpret_cast<const u32x4*>(q + k * 64 + g * 16);
  }
#pragma unroll
  for (int a = 0; a < kRT; ++a) {
    const uint32_t mask = wave_row0 + a * 16 + static_cast<int32_t>(n) < q_len ? keep : 0u;
#pragma unroll
    for (int k = 0; k < kNS + 2; ++k) qf[a][k] = (qf[a][k] ^ flip) & mask;
  }
  f32x4 acc[kRT][kCT];
  float m[kRT], l[kRT];
  bool wide[kRT];                                        // some row's |m| is past 2^20
#pragma unroll
  for (int a = 0; a < kRT; ++a) {
    m[a] = kLowest;
    l[a] = 0.f;
    wide[a] = false;
#pragma unroll
    for (int d = 0; d < kCT; ++d) acc[a][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // Scores of a buffer's keys: lane: row n of each tile, keys 16 t + 4 g + e.
  f32x4 s[kRT][2];
  const uint32_t key_at = n * kRow + (g ^ swap_of<DN>(n)) * 16, rope_at = kRopeAt + n * kRopeRow + (g ^ swap_of<kRope>(n)) * 16;
  const auto score = [&](uint32_t from) {
    const uint32_t key = opaque(key_at) + from, rope = opaque(rope_at) + from;
#pragma unroll
    for (int a = 0; a < kRT; ++a)
#pragma unroll
      for (int t = 0; t < 2; ++t) s[a][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    const auto read = [&](int i) {
      const int k = i / 2, t = i % 2;
      return lds_get<u32x4>(k < kNS ? (key ^ (k * 64)) + t * 16 * kRow : (rope ^ ((k - kNS) * 64)) + t * 16 * kRopeRow);
    };
    // Reads stay two before their products (8192 tokens of 32 heads 640 us to 631; four before,
    // registers spill).
    constexpr int kReads = 2 * (kNS + 2), kAhead = 2;
    u32x4 kf[kReads];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) kf[i] = read(i);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < kReads; ++i) {
      if (i + kAhead < kReads) kf[i + kAhead] = read(i + kAhead);
#pragma unroll
      for (int a = 0; a < kRT; ++a) s[a][i % 2] = mfma<TYPE>(kf[i], qf[a][i / 2], s[a][i % 2]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // Weights of those keys, the first of which is t0, packed by twos as they lie in s.
  u32x4 pf[kRT];
  const auto weigh = [&](auto full) {
    if constexpr (!decltype(full)::value) {
#pragma unroll
      for (int a = 0; a < kRT; ++a) {
        const int32_t upto = min(seen_by(wave_row0 + a * 16 + static_cast<int32_t>(n)), t_end) - t0 - 4 * static_cast<int32_t>(g);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (t * 16 + e >= upto) s[a][t][e] = -INFINITY;
      }
    }
    settle(s);
#pragma unroll
    for (int a = 0; a < kRT; ++a) {
      float top = max3_of(s[a][0][0], s[a][0][1], s[a][0][2]);
      top = max3_of(top, s[a][0][3], s[a][1][0]);
      top = max3_of(top, s[a][1][1], s[a][1][2]);
      top = scaled(max3_of(top, s[a][1][3], s[a][1][3]), per_score);
      if (__ballot(top > m[a]) != 0) {
        top = across_groups(top, max_of);
        const float next = top > m[a] ? top : m[a];
        const float shrink = exp2_of(m[a] - next);
        m[a] = next;
        l[a] *= shrink;
        wide[a] = __ballot(fabsf(next) > 0x1p20f && next != kLowest) != 0;
#pragma unroll
        for (int d = 0; d < kCT; ++d) acc[a][d] *= shrink;
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
  // Adds the weighted values of those keys: a lane's group holds those of rows 4 g .. 4 g + 3
  // and the same behind 16.
  const uint32_t v_row = 4 * g + n / 4;
  const uint32_t v_at = kValueAt + v_row * kRow + (n % 4 / 2 ^ swap_of<DN>(v_row)) * 16 + n % 2 * 8;
  const auto gather = [&](uint32_t from) {
    const uint32_t v = opaque(v_at) + from;
    const auto read = [&](int d) {
      const uint32_t x = v ^ (d * 32);
      const u32x2 lo = lds_transposed(x), hi = lds_transposed(x + 16 * kRow);
      return u32x4{lo[0], lo[1], hi[0], hi[1]};
    };
    constexpr int kAhead = 2;
    u32x4 vf[kCT];
#pragma unroll
    for (int d = 0; d < kAhead; ++d) vf[d] = read(d);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int d = 0; d < kCT; ++d) {
      if (d + kAhead < kCT) vf[d + kAhead] = read(d + kAhead);
#pragma unroll
      for (int a = 0; a < kRT; ++a) acc[a][d] = mfma<TYPE>(vf[d], pf[a], acc[a][d]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // Takes infinities and NaN out of the values that the wave loaded: a product with weight
  // zero would spread them to rows that do not see their key.
  bool odd = false;
  const auto clean = [&](uint32_t from) {
    bool found = false;
#pragma unroll 1
    for (uint32_t c = lane; c < kLoadRows * DN / 8; c += 64) {
      const uint32_t at = from + kValueAt + w * kLoadRows * kRow + c * 16;
      u32x4 x = lds_get<u32x4>(at);
      bool here = false;
#pragma unroll
      for (int e = 0; e < 4; ++e) here |= odd_word<TYPE>(x[e]);
      if (here) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = finite_halves<TYPE>(x[e]);
        lds_put(at, x);
        found = true;
      }
    }
    odd |= found;
  };

  const Places held = places_of(lane);
  const auto one_step = [&](auto full) {
    rows_barrier();                                      // this step's rows are in LDS, the other buffer's readers done
    if constexpr (decltype(full)::value) load_step(std::true_type{}, held, t0 + kStep, other);
    else load_next(t0 + kStep, other);
    if constexpr (!decltype(full)::value) {
      clean(now);
      lds_barrier();
    }
    // Steps of which no row of the wave sees any are passed over.
    if (decltype(full)::value || t0 < seen_by(wave_row0 + 16 * kRT - 1)) {
      score(now);
      weigh(full);
      gather(now);
    }
    const uint32_t x = now;
    now = other;
    other = x;
    t0 += kStep;
  };
  // The steps whose keys every row sees, if a whole one follows, then the others.
  const int32_t last_full = min(min(seen_by(row0), t_end) - kStep, t_end - 2 * kStep);
  while (t0 <= last_full) one_step(std::true_type{});
  const int32_t t_masked = t0;
#pragma unroll 1
  while (t0 < t_end) one_step(std::false_type{});
  const auto part_at = [&](int32_t row) {
    return (static_cast<int64_t>(blockIdx.z) * p.nnz + static_cast<uint32_t>(r.q0 + row)) * p.heads + head;
  };
#pragma unroll
  for (int a = 0; a < kRT; ++a) {
    l[a] = across_groups(l[a], sum_of);
    const int32_t row = wave_row0 + a * 16 + static_cast<int32_t>(n);
    if (row >= q_len) continue;
    const float inv = l[a] == 0.f ? 0.f : 1.f / l[a];
    if (p.parts > 1) {
      const int64_t at = part_at(row);
#pragma unroll
      for (int d = 0; d < kCT; ++d) *reinterpret_cast<f32x4*>(p.part_o + at * DN + d * 16 + g * 4) = acc[a][d];
      if (g == 0) *reinterpret_cast<f32x2*>(p.part_ml + at * 2) = f32x2{m[a], l[a]};
      continue;
    }
    char* const out = p.out + static_cast<int64_t>(r.q0 + row) * p.o_token + head * p.o_head;
#pragma unroll
    for (int d = 0; d < kCT; ++d) {
      const u32x2 x = {result_pair<TYPE>(acc[a][d][0] * inv, acc[a][d][1] * inv),
                       result_pair<TYPE>(acc[a][d][2] * inv, acc[a][d][3] * inv)};
      *reinterpret_cast<u32x2*>(out + (d * 16 + g * 4) * 2) = x;
    }
    if (g == 0 && p.lse != nullptr) p.lse[static_cast<int64_t>(r.q0 + row) * p.heads + head] = log_total<TYPE>(m[a], l[a]);
  }
  if (t_masked >= t_end) return;
  // What any wave took out reaches the rows that see it.  The buffers, which nobody reads any
  // more, hold who found something.
  __syncthreads();
  const bool found = __ballot(odd) != 0;
  if (lane == 0) lds_put(lds_offset(lds) + w * 4, found ? 1u : 0u);
  __syncthreads();
  const u32x4 any = lds_get<u32x4>(lds_offset(lds));
  if ((any[0] | any[1] | any[2] | any[3]) == 0) return;
#pragma unroll 1
  for (int a = 0; a < kRT; ++a) {
    const int32_t row = wave_row0 + a * 16 + static_cast<int32_t>(n);
    if (row >= q_len) continue;
    char* const out = p.out + static_cast<int64_t>(r.q0 + row) * p.o_token + head * p.o_head;
#pragma unroll 1
    for (int32_t t = t_masked; t < min(seen_by(row), t_end); ++t) {
      const char* const x = value0 + static_cast<int64_t>(t) * p.v_token;
#pragma unroll 1
      for (uint32_t c = 0; c < kCT * 4; ++c) {
        const uint32_t at = (c / 4 * 16 + g * 4 + c % 4) * 2;
        const uint32_t v = *reinterpret_cast<const uint16_t*>(x + at);
        if (!odd_word<TYPE>(v)) continue;
        if (p.parts > 1) {
          p.part_o[part_at(row) * DN + at / 2] += value_of<TYPE>(v, 0);
          continue;
        }
        uint16_t* const o = reinterpret_cast<uint16_t*>(out + at);
        *o = static_cast<uint16_t>(pair_of<TYPE>(value_of<TYPE>(*o, 0) + value_of<TYPE>(v, 0), 0.f));
      }
    }
  }
}

// Joins the parts of a tile's rows, as many at a time as DN / 4 lanes a row leave room for:
// a lane takes four columns.
template <int DN, int TYPE>
__global__ __launch_bounds__(kThreads) void prompt_join_kernel(const PromptParams p) {
  constexpr uint32_t kLanes = DN / 4, kAtOnce = kThreads / kLanes;
  const uint32_t head = blockIdx.x, col = threadIdx.x % kLanes * 4;
  PromptRequest r;
  if (!find_tile(p, blockIdx.y, &r)) return;
  const int32_t token = r.q0 + static_cast<int32_t>(r.tile * kRows + blockIdx.z * kAtOnce + threadIdx.x / kLanes);
  if (token < r.q1) {
    const int64_t at = static_cast<int64_t>(token) * p.heads + head, step = static_cast<int64_t>(p.nnz) * p.heads;
    float m = -INFINITY, l = 0.f;
#pragma unroll 4
    for (uint32_t k = 0; k < p.parts; ++k) m = fmaxf(m, p.part_ml[(at + k * step) * 2]);
    const float from = m == -INFINITY ? 0.f : m;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (uint32_t k = 0; k < p.parts; ++k) {
      const f32x2 ml = *reinterpret_cast<const f32x2*>(p.part_ml + (at + k * step) * 2);
      const float weight = exp2_of(ml[0] - from);
      l += weight * ml[1];
      o += weight * *reinterpret_cast<const f32x4*>(p.part_o + (at + k * step) * DN + col);
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const u32x2 x = {result_pair<TYPE>(o[0] * inv, o[1] * inv), result_pair<TYPE>(o[2] * inv, o[3] * inv)};
    *reinterpret_cast<u32x2*>(p.out + static_cast<int64_t>(token) * p.o_token + head * p.o_head + col * 2) = x;
    if (col == 0 && p.lse != nullptr) p.lse[at] = log_total<TYPE>(m, l);
  }
}

template <int DN>
const void* pick_join(int type) {
  return type == PACE_KV_BF16 ? reinterpret_cast<const void*>(&prompt_join_kernel<DN, PACE_KV_BF16>)
                              : reinterpret_cast<const void*>(&prompt_join_kernel<DN, PACE_KV_FP16>);
}

// Workgroups that a call's row tiles and heads can be, a short last tile for each request.
int64_t tiles_of_call(int64_t nnz, int64_t batch) { return std::min<int64_t>(nnz, nnz / kRows + batch); }

// What they come to if every other request's last tile is half empty.
int64_t likely_tiles(int64_t nnz, int64_t batch) { return (nnz + kRows - 1) / kRows + (batch - 1) / 2; }

// Parts that the keys of each row tile are cut into.  The CUs have 768 places for workgroups
// (three a CU); a call takes as long as its longest workgroup, or as all of them dealt to the
// places, kStart steps more each; the joining kernel costs kJoin steps and what it reads.
// The host knows the mean lengths alone.
constexpr int64_t kPlaces = 768, kStart = 4, kJoin = 4, kMostParts = 32, kStepBytes = int64_t(4) << 20;

int64_t parts_of_call(int64_t nnz, int64_t keys, int64_t batch, int64_t heads, int64_t head_dim, bool causal) {
  if (batch == 0 || nnz == 0) return 1;
  const int64_t groups = likely_tiles(nnz, batch) * heads;
  const int64_t longest = (keys / batch + kTile - 1) / kTile;
  const int64_t mean = causal ? std::max<int64_t>(longest - nnz / batch / 2 / kTile, 1) : longest;
  int64_t best = INT64_MAX, parts = 1;
  for (int64_t k = 1; k <= std::min(kMostParts, std::max<int64_t>(longest, 1)); ++k) {
    const int64_t each = (longest + k - 1) / k;
    const int64_t dealt = (groups * (mean + k * kStart) + kPlaces - 1) / kPlaces + each / 2;
    const int64_t join = k == 1 ? 0 : kJoin + 2 * k * nnz * heads * head_dim * 4 / kStepBytes;
    const int64_t cost = std::max(each + kStart, dealt) + join;
    if (cost < best) {
      best = cost;
      parts = k;
    }
  }
  return parts;
}

// LDS that a workgroup asks for beyond its own, so that two fit a CU instead of three: the
// last turn of few workgroups a CU costs more than three at a time gain.  One, two and three
// workgroups a CU take about 10, 11 and 15 for the same keys (MI355X, 8192 tokens of 32 heads
// of 128 columns: 536, 993 and 1060 TFLOP/s): four a CU take 22 by twos and 25 by threes.
uint32_t spare_lds(int64_t groups, int head_dim) {
  constexpr int64_t kCus = 256, kTime[4] = {0, 10, 11, 15};
  const int64_t each = (groups + kCus - 1) / kCus;
  const auto time_of = [&](int64_t at_once) { return each / at_once * kTime[at_once] + kTime[each % at_once]; };
  if (time_of(3) <= time_of(2)) return 0;
  const uint32_t own = 2 * kTile * (2 * head_dim + kRope) * 2;
  return (uint32_t(56) << 10) - own;                     // 160 KiB a CU
}

int64_t workspace_of_call(int64_t parts, int64_t nnz, int64_t heads, int64_t head_dim) {
  return parts == 1 ? 0 : parts * nnz * heads * (head_dim + 2) * 4;
}

int check_sizes(int64_t nnz, int64_t num_keys, int batch_size, int num_heads, int head_dim) {
  if (nnz < 0 || num_keys < 0 || batch_size < 0 || num_heads <= 0)
    return fail(PACE_KV_EINVAL, "prompt attention: sizes must be positive");
  if (head_dim != 64 && head_dim != 128)
    return fail(PACE_KV_EINVAL, "prompt attention: head_dim must be 64 or 128, got %d", head_dim);
  if (nnz > INT32_MAX / 2 || num_keys > INT32_MAX / 2)
    return fail(PACE_KV_ERANGE, "prompt attention: more than 2^30 queries or keys");
  const int64_t tiles = tiles_of_call(nnz, batch_size);
  if (tiles > 65535 || num_heads > (1 << 20) || tiles * num_heads >= (int64_t(1) << 24))
    return fail(PACE_KV_ERANGE, "prompt attention: too many requests, heads or queries for one call");
  return PACE_KV_OK;
}

template <int DN>
const void* pick_prompt(int type) {
  return type == PACE_KV_BF16 ? reinterpret_cast<const void*>(&prompt_kernel<DN, PACE_KV_BF16>)
                              : reinterpret_cast<const void*>(&prompt_kernel<DN, PACE_KV_FP16>);
}

}  // namespace
}  // namespace pace_kv

extern "C" {

int pace_kv_prompt_attention_workspace(int64_t nnz, int64_t num_keys, int batch_size, int num_heads, int head_dim,
                                       int causal, int64_t* bytes) {
  using namespace pace_kv;
  if (!bytes) return fail(PACE_KV_EINVAL, "prompt attention: NULL argument");
  PACE_KV_TRY(check_sizes(nnz, num_keys, batch_size, num_heads, head_dim));
  *bytes = workspace_of_call(parts_of_call(nnz, num_keys, batch_size, num_heads, head_dim, causal != 0), nnz, num_heads,
                             head_dim);
  return PACE_KV_OK;
}

int pace_kv_prompt_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* key,
                             int64_t k_token_stride, int64_t k_head_stride, const void* rope_key,
                             int64_t rope_token_stride, const void* value, int64_t v_token_stride, int64_t v_head_stride,
                             int elem_type, int num_heads, int head_dim, int64_t nnz, int64_t num_keys,
                             const int32_t* qo_indptr, const int32_t* kv_indptr, int batch_size, int max_q_len,
                             float scale, int causal, void* out, int64_t out_token_stride, int64_t out_head_stride,
                             float* lse, void* workspace, int64_t workspace_size, int32_t* err_count, void* stream) {
  using namespace pace_kv;
  PACE_KV_TRY(check_sizes(nnz, num_keys, batch_size, num_heads, head_dim));
  if (max_q_len <= 0) return fail(PACE_KV_EINVAL, "prompt attention: sizes must be positive");
  if (elem_type != PACE_KV_BF16 && elem_type != PACE_KV_FP16)
    return fail(PACE_KV_EINVAL, "prompt attention: queries must be bfloat16 or float16");
  const float scale_log2 = scale * 1.44269504088896341f;
  if (!std::isfinite(scale_log2)) return fail(PACE_KV_EINVAL, "prompt attention: scale must be within float's range");
  if (nnz == 0 || batch_size == 0) return PACE_KV_OK;
  if (!q || !qo_indptr || !kv_indptr || !out || (num_keys > 0 && (!key || !rope_key || !value)))
    return fail(PACE_KV_EINVAL, "prompt attention: NULL argument");
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(key) | reinterpret_cast<uintptr_t>(rope_key) |
       reinterpret_cast<uintptr_t>(value) | reinterpret_cast<uintptr_t>(out) |
       static_cast<uintptr_t>(q_token_stride | q_head_stride | k_token_stride | k_head_stride | rope_token_stride |
                              v_token_stride | v_head_stride | out_token_stride | out_head_stride)) & 15u)
    return fail(PACE_KV_EINVAL, "prompt attention: rows and strides must be multiples of 16 bytes");
  if (rows_overlap(nnz, out_token_stride, num_heads, out_head_stride, int64_t(2) * head_dim))
    return fail(PACE_KV_EINVAL, "prompt attention: output rows overlap");
  const int64_t longest = std::max({k_token_stride, rope_token_stride, v_token_stride});
  if (longest >= int64_t(1) << 26 || std::min({k_token_stride, rope_token_stride, v_token_stride}) < 0)
    return fail(PACE_KV_EINVAL, "prompt attention: token strides of keys and values must be in [0, 2^26)");
  const int64_t parts = parts_of_call(nnz, num_keys, batch_size, num_heads, head_dim, causal != 0);
  const int64_t need = workspace_of_call(parts, nnz, num_heads, head_dim);
  if (need > 0 && (!workspace || workspace_size < need || reinterpret_cast<uintptr_t>(workspace) & 15u))
    return fail(PACE_KV_EINVAL, "prompt attention: needs a 16-byte aligned workspace of %lld bytes", (long long)need);
  PromptParams p = {};
  p.q = static_cast<const char*>(q);
  p.key = static_cast<const char*>(key);
  p.rope_key = static_cast<const char*>(rope_key);
  p.value = static_cast<const char*>(value);
  p.out = static_cast<char*>(out);
  p.lse = lse;
  p.qo_indptr = qo_indptr;
  p.kv_indptr = kv_indptr;
  p.err = err_count;
  p.q_token = q_token_stride, p.q_head = q_head_stride;
  p.k_token = k_token_stride, p.k_head = k_head_stride;
  p.r_token = rope_token_stride;
  p.v_token = v_token_stride, p.v_head = v_head_stride;
  p.o_token = out_token_stride, p.o_head = out_head_stride;
  p.batch = static_cast<uint32_t>(batch_size);
  p.nnz = static_cast<uint32_t>(nnz);
  p.keys = static_cast<uint32_t>(num_keys);
  p.heads = static_cast<uint32_t>(num_heads);
  p.max_q = static_cast<uint32_t>(max_q_len);
  p.tiles = static_cast<uint32_t>(tiles_of_call(nnz, batch_size));
  p.parts = static_cast<uint32_t>(parts);
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = p.part_o + parts * nnz * num_heads * head_dim;
  p.scale_log2 = scale_log2;
  p.causal = causal != 0;
  void* args[] = {&p};
  PACE_KV_TRY(hip_status(hipLaunchKernel(head_dim == 128 ? pick_prompt<128>(elem_type) : pick_prompt<64>(elem_type),
                                         dim3(p.heads, p.tiles, p.parts), dim3(kThreads), args,
                                         spare_lds(likely_tiles(nnz, batch_size) * num_heads * parts, head_dim),
                                         static_cast<hipStream_t>(stream)), "prompt attention launch"));
  if (parts == 1) return PACE_KV_OK;
  return hip_status(hipLaunchKernel(head_dim == 128 ? pick_join<128>(elem_type) : pick_join<64>(elem_type),
                                    dim3(p.heads, p.tiles, kRows * head_dim / 4 / kThreads), dim3(kThreads), args, 0,
                                    static_cast<hipStream_t>(stream)), "prompt attention join launch");
}

}  // extern "C"

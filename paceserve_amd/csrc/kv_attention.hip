// Attention over a paged cache: how a call is cut up, the kernel that joins the
// parts, and the entry points.  The attention itself: attention.h.
#include <algorithm>
#include <cmath>

#include "attention.h"

namespace pace_kv {
namespace {

// A row (query head qh of a token) whose chunks are joined: where its parts are.
struct Parts {
  int64_t first, step;
  uint32_t chunks;
};

// The parts of rows of `token`; false where its request is not split.
__device__ __forceinline__ bool parts_of(const AttnParams& p, uint32_t token, Request* r, uint32_t* first_part) {
  Tables t;
  Place place;
  if (!find_request(p, token, [](const Tables& x, uint32_t) { return static_cast<uint32_t>(max(x.a0, 0)); }, &t, &place))
    return false;
  *first_part = place.part();
  return request_of(p, t, r) && token >= r->q0 && token - r->q0 < r->q_len && r->chunks > 1 && has_room(p, *r, place);
}

__device__ __forceinline__ Parts parts_of_row(const AttnParams& p, const Request& r, uint32_t first_part, uint32_t token,
                                              uint32_t qh) {
  const uint32_t head = over(p.by_group, qh), row = (token - r.q0) * p.group + (qh - head * p.group);
  const uint32_t tile = row / p.tile_rows;
  const int64_t unit = static_cast<int64_t>(p.heads) * p.row_tiles;
  return {(static_cast<int64_t>(first_part) * unit + static_cast<int64_t>(head) * p.row_tiles + tile) * p.tile_rows +
              row % p.tile_rows,
          unit * p.tile_rows, r.chunks};
}

// Four columns of a row, of its weighted sum o and the sum l of weights over 2^m.
template <int TYPE>
__device__ __forceinline__ void write_row(const AttnParams& p, uint32_t token, uint32_t qh, int D, uint32_t col, f32x4 o,
                                          float m, float l) {
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const u32x2 x = {result_pair<TYPE>(o[0] * inv, o[1] * inv), result_pair<TYPE>(o[2] * inv, o[3] * inv)};
  *reinterpret_cast<u32x2*>(p.out + static_cast<int64_t>(token) * p.out_stride +
                            (static_cast<int64_t>(qh) * D + col * 4) * 2) = x;
  if (col == 0 && p.lse != nullptr)
    p.lse[static_cast<int64_t>(token) * (p.heads * p.group) + qh] = log_sum<TYPE>(m, l);
}

// Few rows of many chunks: a workgroup joins a row.  D / 4 lanes take four columns
// each of a chunk, a wave as many chunks at a time as fit, and the waves a quarter of
// the chunks each.  The chunks' weights come first, 64 at a time, so that the loads
// of their outputs do not wait for one another.
template <int D, int TYPE>
__global__ __launch_bounds__(kThreads) void combine_few_kernel(const AttnParams p) {
  constexpr uint32_t kCols = D / 4, kGroups = 64 / kCols;
  __shared__ f32x4 lds_o[kWaves][kCols];
  __shared__ float lds_m[kWaves], lds_l[kWaves];
  const uint32_t lane = threadIdx.x % 64, w = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t token = over(p.by_heads, blockIdx.x), qh = blockIdx.x - token * p.heads * p.group;
  Request r;
  uint32_t first_part;
  if (!parts_of(p, token, &r, &first_part)) return;
  const auto [first, step, chunks] = parts_of_row(p, r, first_part, token, qh);
  const uint32_t col = lane % kCols, group = lane / kCols;
  // The wave's part of the chunks.
  const uint32_t per_wave = (chunks + kWaves - 1) / kWaves;
  const uint32_t c_begin = w * per_wave, c_end = min(c_begin + per_wave, chunks);
  float m = -INFINITY, l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
  for (uint32_t c0 = c_begin; c0 < c_end; c0 += 64) {
    float mc = -INFINITY, lc = 0.f;
    if (c0 + lane < c_end) {
      const int64_t at = first + (c0 + lane) * step;
      mc = p.part_ml[at * 2];
      lc = p.part_ml[at * 2 + 1];
    }
    float top = mc;
#pragma unroll
    for (int k = 1; k < 64; k *= 2) top = fmaxf(top, __shfl_xor(top, k));
    top = fmaxf(m, top);
    const float from = top == -INFINITY ? 0.f : top, shrink = exp2_of(m - from);
    const float weight = exp2_of(mc - from);
    float sum = weight * lc;
#pragma unroll
    for (int k = 1; k < 64; k *= 2) sum += __shfl_xor(sum, k);
    l = l * shrink + sum;
    o *= shrink;
    m = top;
    const uint32_t n = min(c_end - c0, 64u);
    // Every lane takes part in every turn: a lane that had left would hand no weight
    // to the others.
#pragma unroll 8
    for (uint32_t c = 0; c < n; c += kGroups) {
      const float mine = __shfl(weight, c + group);      // 0 past the last chunk
      if (c + group < n)
        o += mine * *reinterpret_cast<const f32x4*>(p.part_o + (first + (c0 + c + group) * step) * D + col * 4);
    }
  }
#pragma unroll
  for (int k = kCols; k < 64; k *= 2)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], k);
  if (group == 0) lds_o[w][col] = o;
  if (lane == 0) {
    lds_m[w] = m;
    lds_l[w] = l;
  }
  __syncthreads();
  if (w != 0) return;
  m = -INFINITY;
#pragma unroll
  for (int v = 0; v < kWaves; ++v) m = fmaxf(m, lds_m[v]);
  const float from = m == -INFINITY ? 0.f : m;
  l = 0.f;
  o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int v = 0; v < kWaves; ++v) {
    const float weight = exp2_of(lds_m[v] - from);
    l += weight * lds_l[v];
    o += weight * lds_o[v][col];
  }
  if (group == 0) write_row<TYPE>(p, token, qh, D, col, o, m, l);
}

// Many rows of few chunks: D / 4 lanes join a row by themselves, and a wave takes
// p.join_turns times as many rows of a token as fit into it; finding the token's
// request costs as much as joining a row.  MI355X, 32256 rows of two chunks: 13 us,
// where a wave per row takes 23 and four rows a wave 19.
template <int D, int TYPE>
__global__ __launch_bounds__(kThreads) void combine_many_kernel(const AttnParams p) {
  constexpr uint32_t kCols = D / 4, kGroups = 64 / kCols;
  const uint32_t lane = threadIdx.x % 64, w = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t wave = blockIdx.x * kWaves + w;
  const uint32_t token = over(p.by_token_waves, wave);
  if (token >= p.nnz) return;
  Request r;
  uint32_t first_part;
  if (!parts_of(p, token, &r, &first_part)) return;
  const uint32_t col = lane % kCols, heads = p.heads * p.group;
  const uint32_t qh0 = (wave - token * p.token_waves) * p.join_turns * kGroups + lane / kCols;
  for (uint32_t turn = 0; turn < p.join_turns; ++turn) {
    const uint32_t qh = qh0 + turn * kGroups;
    if (qh >= heads) return;
    const auto [first, step, chunks] = parts_of_row(p, r, first_part, token, qh);
    float m = -INFINITY;
#pragma unroll 4
    for (uint32_t c = 0; c < chunks; ++c) m = fmaxf(m, p.part_ml[(first + c * step) * 2]);
    const float from = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (uint32_t c = 0; c < chunks; ++c) {
      const int64_t at = first + c * step;
      const float weight = exp2_of(p.part_ml[at * 2] - from);
      l += weight * p.part_ml[at * 2 + 1];
      o += weight * *reinterpret_cast<const f32x4*>(p.part_o + at * D + col * 4);
    }
    write_row<TYPE>(p, token, qh, D, col, o, m, l);
  }
}

// How a call is cut up.
struct Split {
  uint32_t tile_rows, row_tiles, chunk_pages, step_pages, items, parts;
  int64_t part_rows() const { return static_cast<int64_t>(parts) * row_tiles * tile_rows; }  // times the KV heads
};

// A call's contexts are split so that every CU gets as many workgroups of about one
// length: a request's work items go round the XCDs, and an item's heads and row tiles
// to the CUs of its XCD.  With w workgroups for the fullest CU, of n tokens, the call
// takes about (w + idle) * (n + start): `start` is what a workgroup's start and the
// joining of its part cost, in tokens, and `idle` what a CU loses while it holds too
// few waves to hide its loads: two thirds and a third of a workgroup with one and two
// of those that fit it by threes, half of one alone of others.  The fewest turns win; of the
// requests' lengths the host knows only the sum, so they are taken as equal.
// MI355X, against 768 (512 of 128 rows) workgroups whatever the sizes: 144 calls of 1
// to 112 rows 4 % faster as a whole, 126 calls of 72 to 504 rows 11 %; 504 rows over
// 3 x 9000 bf16 tokens 131 -> 98 us, 1 row of 32 heads over 5 x 20000 300 -> 262 us.
constexpr int64_t kXcdCus = 32, kMostTurns = 6;

Split split_of(int64_t batch, int64_t heads, int64_t group, int head_dim, int64_t max_q, int64_t num_indices,
               int64_t page_size, bool quantised) {
  Split s = {};
  const int64_t rows = max_q * group;
  s.tile_rows = tile_rows_of(head_dim, rows);
  s.row_tiles = static_cast<uint32_t>((rows + s.tile_rows - 1) / s.tile_rows);
  const bool by_tokens = s.tile_rows <= 32;
  const bool three = by_tokens || (head_dim != 256 && (quantised || (head_dim == 64 && s.tile_rows == 128)));
  // A chunk is whole steps of a wave, and long enough to be worth a part: MI355X, 4
  // rows over 512 tokens, 13 us in one launch, 7 + 4 in two, which take the host 3 more.
  const int64_t step = by_tokens ? 32 : 64, start = by_tokens ? 128 : 512, least = by_tokens ? 512 : 128;
  s.step_pages = static_cast<uint32_t>(step % page_size ? 1 : step / page_size);
  const int64_t unit = heads * s.row_tiles, requests = std::max<int64_t>(batch, 1);
  const int64_t pages = std::max<int64_t>((num_indices + requests - 1) / requests, 1);
  const int64_t most_chunks = std::max<int64_t>(pages * page_size / least, 1);
  int64_t chunk = pages, best = INT64_MAX;
  for (int64_t turns = 0; turns <= kMostTurns; ++turns) {
    // The most chunks a request that keep to so many turns; first of all one.
    const int64_t k = turns == 0 ? 1 : std::min(kXcds * (kXcdCus * turns / unit) / requests, most_chunks);
    if (k < 1) continue;
    const int64_t length = ((pages + k - 1) / k + s.step_pages - 1) / s.step_pages * s.step_pages;
    const int64_t groups = (requests * k + kXcds - 1) / kXcds * unit, each = (groups + kXcdCus - 1) / kXcdCus;
    const int64_t idle = three ? std::max<int64_t>(6 - 2 * each, 0) : each == 1 ? 3 : 0;   // in sixths
    const int64_t cost = (6 * each + idle) * (length * page_size + start);
    if (cost < best) {
      best = cost;
      chunk = length;
    }
  }
  // Without a split only requests far longer than the others are cut: past the length
  // that would give 768 workgroups, which for large tiles is at least the mean.  (200
  // ragged requests of 56 rows: 47 us, 54 with those past the mean cut.)
  if (chunk >= pages) chunk = std::max((num_indices * unit + 767) / 768, by_tokens ? 1 : pages);
  const int64_t least_pages = (least + page_size - 1) / page_size;
  chunk = std::max(chunk, least_pages);
  if (num_indices <= least_pages + least_pages / 2) chunk = num_indices;  // no short second chunk
  chunk = std::max<int64_t>(std::min(chunk, num_indices), 1);
  s.chunk_pages = static_cast<uint32_t>(chunk);
  s.items = static_cast<uint32_t>(num_indices / chunk + batch);
  s.parts = chunk >= num_indices ? 0 : batch == 1 ? s.items : static_cast<uint32_t>(2 * (num_indices / chunk));
  return s;
}

// Rows of a call from which on they are joined several to a wave.
constexpr int64_t kManyRows = 2048;
// Waves that the GPU holds at once: 256 CUs, eight waves on each of their four SIMDs.
constexpr int64_t kWavesHeld = 8192;

template <int D, int TYPE>
const void* pick_combine(bool many) {
  return many ? reinterpret_cast<const void*>(&combine_many_kernel<D, TYPE>)
              : reinterpret_cast<const void*>(&combine_few_kernel<D, TYPE>);
}

template <int D>
const void* pick_combine(int type, bool many) {
  return type == PACE_KV_BF16 ? pick_combine<D, PACE_KV_BF16>(many) : pick_combine<D, PACE_KV_FP16>(many);
}

// Caps past this one are applied so that scores far below them keep their accuracy:
// up to it the simple form is off by 2^-16 at most, a 128th of what a weight loses when
// it is rounded to bfloat16.  MI355X, cap 30: 36 rows over 16 ragged requests of up to
// 4000 4-bit tokens 37 us, 39 with the other form; 504 over 8 x 4096 bf16 tokens 144, 159.
constexpr float kLargeCap = 64.f;

// LDS that a workgroup asks for beyond its own.  16 rows of 128 columns over a 16-bit
// cache fit a CU by threes, which long contexts read more slowly than by twos: MI355X,
// ragged requests of up to 4096 tokens, 64 of 32 heads 402 us by threes, 393 by twos, up
// to 2048 tokens, 256 of 8 heads 207 and 200, up to 1500, 100 of 32 heads 230 and 227; but
// up to 1000, 256 of 32 heads 361 and 373, up to 300, 300 of 32 heads 158 and 191.  (Half
// of those lengths on the mean.)
uint32_t spare_lds(int head_dim, uint32_t tile_rows, bool quantised, int64_t batch, int64_t num_indices,
                   int64_t page_size) {
  const bool by_twos = head_dim == 128 && tile_rows == 16 && !quantised && num_indices * page_size >= 768 * batch;
  return by_twos ? 14 << 10 : 0;                         // 41 KiB of its own; 160 KiB a CU
}

// Workgroups of a launch, whose threads are counted in 32 bits.
constexpr int64_t kMostGroups = int64_t(1) << 24;

int check_sizes(int batch_size, int num_kv_heads, int group, int head_dim, int max_q_len, int64_t num_indices,
                int page_size) {
  if (batch_size < 0 || num_kv_heads <= 0 || group <= 0 || max_q_len <= 0 || num_indices < 0 || page_size <= 0)
    return fail(PACE_KV_EINVAL, "attention: sizes must be positive");
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return fail(PACE_KV_EINVAL, "attention: head_dim must be 64, 128 or 256, got %d", head_dim);
  const int64_t rows = static_cast<int64_t>(max_q_len) * group;
  if (num_indices > INT32_MAX / 2 / page_size || rows > INT32_MAX / 2)
    return fail(PACE_KV_ERANGE, "attention: more than 2^30 tokens or query rows");
  // No product below passes 64 bits, and no divisor of the kernel 32: each factor is
  // bounded before it is multiplied.
  const int64_t tile = tile_rows_of(head_dim, rows), unit = num_kv_heads * ((rows + tile - 1) / tile);
  bool fits = batch_size < kMostGroups && unit < kMostGroups && (batch_size + kXcds) * unit < kMostGroups;
  for (bool quantised : {false, true}) {
    if (!fits) break;
    const Split s = split_of(batch_size, num_kv_heads, group, head_dim, max_q_len, num_indices, page_size, quantised);
    fits = (static_cast<int64_t>(s.items) + kXcds) * unit < kMostGroups;
  }
  if (!fits) return fail(PACE_KV_ERANGE, "attention: too many requests, heads or query rows for one call");
  return PACE_KV_OK;
}

int64_t workspace_bytes(const Split& s, int heads, int head_dim) {
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
  *bytes = 0;                                            // of either kind of cache
  for (bool quantised : {false, true})
    *bytes = std::max(*bytes, workspace_bytes(split_of(batch_size, num_kv_heads, group, head_dim, max_q_len, num_indices,
                                                       page_size, quantised), num_kv_heads, head_dim));
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
  const float log2e = 1.44269504088896341f;
  const float scale_log2 = soft_cap > 0.f ? scale / soft_cap * (2.f * log2e) : scale * log2e;
  if (!(soft_cap >= 0.f) || !std::isfinite(soft_cap * log2e) || !std::isfinite(scale_log2) ||
      !std::isfinite(scale * log2e))
    return fail(PACE_KV_EINVAL, "attention: soft_cap must be >= 0, and it, scale and scale / soft_cap within float's range");
  if (nnz * num_kv_heads * group >= (int64_t(1) << 24))
    return fail(PACE_KV_ERANGE, "attention: 2^24 query rows or more");
  if (nnz == 0 || batch_size == 0) return PACE_KV_OK;
  // A pool without pages has no memory, and none of its pages is read.
  if (!q || (num_pages > 0 && !cache) || !kv_indptr || !kv_last_page_len || !out || (num_indices > 0 && !kv_indices))
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
  if (half_bytes >= int64_t(1) << 36 || num_pages * (2 * half_bytes / 16) >= UINT32_MAX)
    return fail(PACE_KV_ERANGE, "attention: a layer's cache must be smaller than 64 GiB");
  const Split s = split_of(batch_size, num_kv_heads, group, head_dim, max_q_len, num_indices, page_size,
                           format != PACE_KV_PLAIN);
  const int64_t need = workspace_bytes(s, num_kv_heads, head_dim);
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
  p.step_pages = s.step_pages;
  p.items = s.items;
  p.parts = s.parts;
  p.row_tiles = s.row_tiles;
  p.tile_rows = s.tile_rows;
  p.half16 = static_cast<uint32_t>(half_bytes / 16);
  p.page16 = 2 * p.half16;
  p.row16 = static_cast<uint32_t>(row * bits / 128);
  p.scale_at = static_cast<uint32_t>(half * bits / 8);
  p.scale_row = static_cast<uint32_t>(row / kMxBlock);
  const int64_t out_rows = nnz * num_kv_heads * group;
  const bool many = out_rows >= kManyRows;
  // Rows that one turn of a wave joins, turns so that the GPU holds all waves, and
  // waves that a token's rows take.
  const int64_t turn_rows = 256 / head_dim, token_rows = static_cast<int64_t>(num_kv_heads) * group;
  const int64_t turns = std::min((out_rows + turn_rows * kWavesHeld - 1) / (turn_rows * kWavesHeld),
                                 (token_rows + turn_rows - 1) / turn_rows);
  p.join_turns = static_cast<uint32_t>(turns);
  p.token_waves = static_cast<uint32_t>((token_rows + turn_rows * turns - 1) / (turn_rows * turns));
  p.by_token_waves = fast_div(p.token_waves);
  p.by_page = fast_div(p.page_size);
  p.by_chunk = fast_div(p.chunk_pages);
  p.by_group = fast_div(p.group);
  p.by_heads = fast_div(p.heads * p.group);
  p.by_unit = fast_div(p.heads * p.row_tiles);
  p.by_tiles = fast_div(p.row_tiles);
  p.scale_log2 = scale_log2;
  p.cap_log2 = soft_cap * log2e;
  p.uncapped_log2 = scale * log2e;
  p.large_cap = soft_cap > kLargeCap;
  const void* attention = head_dim == 64    ? attention_kernel_d64(elem_type, format, s.tile_rows)
                          : head_dim == 128 ? attention_kernel_d128(elem_type, format, s.tile_rows)
                                            : attention_kernel_d256(elem_type, format, s.tile_rows);
  const void* combine = head_dim == 64    ? pick_combine<64>(elem_type, many)
                        : head_dim == 128 ? pick_combine<128>(elem_type, many)
                                          : pick_combine<256>(elem_type, many);
  const uint32_t items = (s.items + kXcds - 1) / kXcds * kXcds;
  void* args[] = {&p};
  PACE_KV_TRY(hip_status(hipLaunchKernel(attention, dim3(items * p.heads * p.row_tiles), dim3(kThreads), args,
                                         spare_lds(head_dim, s.tile_rows, format != PACE_KV_PLAIN, batch_size,
                                                   num_indices, page_size),
                                         static_cast<hipStream_t>(stream)), "attention launch"));
  if (need == 0) return PACE_KV_OK;
  const uint32_t groups = static_cast<uint32_t>(many ? (nnz * p.token_waves + kWaves - 1) / kWaves : out_rows);
  return hip_status(hipLaunchKernel(combine, dim3(groups), dim3(kThreads), args, 0, static_cast<hipStream_t>(stream)),
                    "attention combine launch");
}

}  // extern "C"

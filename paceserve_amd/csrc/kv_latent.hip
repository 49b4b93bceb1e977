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

// A workgroup takes 16 rows and a chunk of tokens, 32 at a time through LDS.  Each of its
// four waves makes the weights of all rows for itself and sums a quarter of the columns.
template <int L, int TYPE>
__global__ __launch_bounds__(kThreads, 1) void latent_kernel(const AttnParams p) {
  constexpr int kW = L + kRope, kKS = kW / 32, kCT = L / 64;
  constexpr uint32_t kRow = kStride<kW>, kPieces = kW / 8;
  __shared__ __attribute__((aligned(16))) char lds[kTile * kRow];
  const uint32_t lane = threadIdx.x % 64, g = lane / 16, n = lane % 16;
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
    if (item + 1 == p.items && place.index + 1 < p.batch)
      atomicAdd(p.err, static_cast<int32_t>(p.batch - 1 - place.index));
  }
  if (!valid_request) return;
  const uint32_t rows = r.q_len * p.group, row0 = tile * 16;
  if (row0 >= rows) return;
  const int32_t base = static_cast<int32_t>(r.kv_len) - static_cast<int32_t>(r.q_len);
  const int32_t last_q = static_cast<int32_t>(over(p.by_group, min(row0 + 16, rows) - 1));
  const uint32_t even = (r.pages + r.chunks - 1) / r.chunks;
  const uint32_t length = min((even + p.step_pages - 1) / p.step_pages * p.step_pages, p.chunk_pages);
  const int32_t chunk_tokens = static_cast<int32_t>(length * p.page_size);
  const int32_t t_begin = static_cast<int32_t>(r.chunk) * chunk_tokens;
  int32_t t_end = static_cast<int32_t>(min(static_cast<int64_t>(t_begin) + chunk_tokens, static_cast<int64_t>(r.kv_len)));
  if (p.mask == nullptr) t_end = min(t_end, base + last_q + 1);
  if (p.err != nullptr && row0 + 16 >= rows) {
    const int32_t page = static_cast<int32_t>(p.page_size), first = static_cast<int32_t>(r.chunk * length);
    for (int32_t i = static_cast<int32_t>(threadIdx.x); static_cast<int64_t>(i) * page < t_end - t_begin; i += kThreads)
      if (static_cast<uint32_t>(p.kv_indices[r.first_page + first + i]) >= p.num_pages)
        atomicAdd(p.err, min(page, t_end - t_begin - i * page));
  }
  const uint32_t my_row = row0 + n, my_query = over(p.by_group, my_row);
  u32x4 qf[kKS];
#pragma unroll
  for (int k = 0; k < kKS; ++k) {
    qf[k] = u32x4{0, 0, 0, 0};
    if (my_row < rows)
      qf[k] = *reinterpret_cast<const u32x4*>(p.q + static_cast<int64_t>(r.q0 + my_query) * p.q_stride +
                                              static_cast<int64_t>(my_row - my_query * p.group) * (kW * 2) + k * 64 + g * 16);
  }
  f32x4 acc[kCT];
#pragma unroll
  for (int d = 0; d < kCT; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  for (int32_t t0 = t_begin; t0 < t_end; t0 += kTile) {
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < kTile * kPieces; e += kThreads) {
      const uint32_t row = e / kPieces, c = e % kPieces;
      const int32_t t = t0 + static_cast<int32_t>(row);
      u32x4 x = {0, 0, 0, 0};
      if (t < t_end) {
        const uint32_t pg = over(p.by_page, static_cast<uint32_t>(t));
        const uint32_t id = static_cast<uint32_t>(p.kv_indices[r.first_page + static_cast<int32_t>(pg)]);
        if (id < p.num_pages)
          x = *reinterpret_cast<const u32x4*>(
              p.cache + (static_cast<int64_t>(id) * p.page_size + (static_cast<uint32_t>(t) - pg * p.page_size)) * (kW * 2) +
              c * 16);
      }
      *reinterpret_cast<u32x4*>(lds + row * kRow + c * 16) = x;
    }
    uint32_t ok = 0;
    {
      const int32_t t = t0 + static_cast<int32_t>(lane % 32);
      bool exists = t < t_end;
      if (exists)
        exists = static_cast<uint32_t>(p.kv_indices[r.first_page + static_cast<int32_t>(over(p.by_page, static_cast<uint32_t>(t)))]) <
                 p.num_pages;
      ok = static_cast<uint32_t>(__ballot(exists));
    }
    __syncthreads();
    f32x4 s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int k = 0; k < kKS; ++k)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const u32x4 kf = *reinterpret_cast<const u32x4*>(lds + (t * 16 + n) * kRow + k * 64 + g * 16);
        s[t] = mfma<TYPE>(kf, qf[k], s[t]);
      }
    const uint32_t sees = seen_of(p, r, base, t0, static_cast<int32_t>(my_query)) & ok, mine = sees >> (4 * g);
    float top = -INFINITY;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[t][e] = (mine & (1u << (t * 16 + e))) ? scaled(s[t][e], p.scale_log2) : -INFINITY;
        top = fmaxf(top, s[t][e]);
      }
    top = fmaxf(m, across_groups(top, max_of));
    const float from = top == -INFINITY ? 0.f : top, shrink = exp2_of(m - from);
    m = top;
    l *= shrink;
#pragma unroll
    for (int d = 0; d < kCT; ++d) acc[d] *= shrink;
    u32x4 pf;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int e = 0; e < 4; e += 2) {
        const float x = weight_of<TYPE>(s[t][e], from), y = weight_of<TYPE>(s[t][e + 1], from);
        l += x + y;
        pf[t * 2 + e / 2] = pair_of<TYPE>(x, y);
      }
    const bool full = __ballot(sees == ~0u) == ~0ull;
    bool odd = false;
    if (!full) {
      bool found = false;
      for (uint32_t c = lane; c < kTile * L / 8; c += 64) {
        const u32x4 x = *reinterpret_cast<const u32x4*>(lds + c / (L / 8) * kRow + c % (L / 8) * 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) found |= odd_word<TYPE>(x[e]);
      }
      odd = __ballot(found) != 0;
    }
#pragma unroll
    for (int d = 0; d < kCT; ++d) {
      const char* v = lds + lane / 4 * kRow + (w * kCT + d) * 32 + lane % 4 * 8;
      typedef __attribute__((address_space(3))) s16x4* lds_ptr;
      const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)v));
      const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(v + 16 * kRow)));
      if (!odd) acc[d] = mfma<TYPE>(u32x4{lo[0], lo[1], hi[0], hi[1]}, pf, acc[d]);
    }
    if (odd) {
#pragma unroll 1
      for (uint32_t token = 0; token < kTile; ++token) {
        const uint32_t word = token / 16 * 2 + token % 4 / 2;
        const uint32_t of = word == 0 ? pf[0] : word == 1 ? pf[1] : word == 2 ? pf[2] : pf[3];
        const float weight = value_of<TYPE>(__shfl(of, token % 16 / 4 * 16 + n), token % 2);
        if (!((sees >> token) & 1u)) continue;
#pragma unroll
        for (int d = 0; d < kCT; ++d) {
          const u32x2 v = *reinterpret_cast<const u32x2*>(lds + token * kRow + (w * kCT + d) * 32 + g * 8);
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[d][c] += weight * value_of<TYPE>(v[c / 2], c % 2);
        }
      }
    }
  }
  l = across_groups(l, sum_of);
  if (my_row >= rows) return;
  const bool direct = r.chunks == 1;
  const int64_t part_row = (static_cast<int64_t>(place.part() + r.chunk) * p.row_tiles + tile) * 16 + n;
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int d = 0; d < kCT; ++d) {
    const uint32_t col = (w * kCT + d) * 16 + g * 4;
    if (!direct) {
      *reinterpret_cast<f32x4*>(p.part_o + part_row * L + col) = acc[d];
    } else {
      const u32x2 x = {result_pair<TYPE>(acc[d][0] * inv, acc[d][1] * inv),
                       result_pair<TYPE>(acc[d][2] * inv, acc[d][3] * inv)};
      *reinterpret_cast<u32x2*>(p.out + static_cast<int64_t>(r.q0 + my_query) * p.out_stride +
                                (static_cast<int64_t>(my_row - my_query * p.group) * L + col) * 2) = x;
    }
  }
  if (w == 0 && g == 0) {
    if (!direct) {
      p.part_ml[part_row * 2] = m;
      p.part_ml[part_row * 2 + 1] = l;
    } else if (p.lse != nullptr) {
      p.lse[static_cast<int64_t>(r.q0 + my_query) * p.group + (my_row - my_query * p.group)] = log_total<TYPE>(m, l);
    }
  }
}

// Joins the parts of split requests' rows, a wave a row.
template <int L, int TYPE>
__global__ __launch_bounds__(kThreads) void latent_join_kernel(const AttnParams p) {
  constexpr uint32_t kVec = L / 64;                      // columns of a lane
  typedef float vec __attribute__((ext_vector_type(kVec)));
  const uint32_t lane = threadIdx.x % 64, w = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t id = blockIdx.x * kWaves + w, token = over(p.by_heads, id), head = id - token * p.group;
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
  float m = -INFINITY;
  for (uint32_t c = 0; c < r.chunks; ++c) m = fmaxf(m, p.part_ml[(first + c * step) * 2]);
  const float from = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  vec o = {};
  for (uint32_t c = 0; c < r.chunks; ++c) {
    const int64_t at = first + c * step;
    const float weight = exp2_of(p.part_ml[at * 2] - from);
    l += weight * p.part_ml[at * 2 + 1];
    o += weight * *reinterpret_cast<const vec*>(p.part_o + at * L + lane * kVec);
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

Split split_of(int64_t batch, int64_t rows, int64_t num_indices, int64_t page_size) {
  Split s = {};
  s.tile_rows = 16;
  s.row_tiles = static_cast<uint32_t>((rows + s.tile_rows - 1) / s.tile_rows);
  s.step_pages = static_cast<uint32_t>(kTile % page_size ? 1 : kTile / page_size);
  const int64_t requests = std::max<int64_t>(batch, 1), pages = std::max<int64_t>((num_indices + requests - 1) / requests, 1);
  const int64_t least = 256;
  const int64_t k = std::max<int64_t>(std::min<int64_t>(512 / (requests * s.row_tiles), pages * page_size / least), 1);
  int64_t chunk = ((pages + k - 1) / k + s.step_pages - 1) / s.step_pages * s.step_pages;
  chunk = std::max<int64_t>(chunk, (least + page_size - 1) / page_size);
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
    const Split s = split_of(batch_size, rows, num_indices, page_size);
    fits = s.row_tiles < kMostGroups && (static_cast<int64_t>(s.items) + kXcds) * s.row_tiles < kMostGroups;
  }
  if (!fits) return fail(PACE_KV_ERANGE, "latent attention: too many requests, heads or query rows for one call");
  return PACE_KV_OK;
}

int64_t workspace_bytes(const Split& s, int latent_dim) { return s.part_rows() * (latent_dim + 2) * 4; }

template <int L>
const void* pick_latent(int type) {
  return type == PACE_KV_BF16 ? reinterpret_cast<const void*>(&latent_kernel<L, PACE_KV_BF16>)
                              : reinterpret_cast<const void*>(&latent_kernel<L, PACE_KV_FP16>);
}

template <int L>
const void* pick_join(int type) {
  return type == PACE_KV_BF16 ? reinterpret_cast<const void*>(&latent_join_kernel<L, PACE_KV_BF16>)
                              : reinterpret_cast<const void*>(&latent_join_kernel<L, PACE_KV_FP16>);
}

}  // namespace
}  // namespace pace_kv

extern "C" {

int pace_kv_latent_attention_workspace(int batch_size, int num_heads, int latent_dim, int max_q_len, int64_t num_indices,
                                       int page_size, int64_t* bytes) {
  using namespace pace_kv;
  if (!bytes) return fail(PACE_KV_EINVAL, "latent attention: NULL argument");
  PACE_KV_TRY(check_sizes(batch_size, num_heads, latent_dim, max_q_len, num_indices, page_size));
  *bytes = workspace_bytes(split_of(batch_size, static_cast<int64_t>(max_q_len) * num_heads, num_indices, page_size),
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
  const Split s = split_of(batch_size, static_cast<int64_t>(max_q_len) * num_heads, num_indices, page_size);
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
  p.by_page = fast_div(p.page_size);
  p.by_chunk = fast_div(p.chunk_pages);
  p.by_group = fast_div(p.group);
  p.by_heads = fast_div(p.group);
  p.by_unit = fast_div(p.row_tiles);
  p.scale_log2 = scale_log2;
  const uint32_t items = (s.items + kXcds - 1) / kXcds * kXcds;
  void* args[] = {&p};
  PACE_KV_TRY(hip_status(hipLaunchKernel(latent_dim == 512 ? pick_latent<512>(elem_type) : pick_latent<256>(elem_type),
                                         dim3(items * p.row_tiles), dim3(kThreads), args, 0,
                                         static_cast<hipStream_t>(stream)), "latent attention launch"));
  if (need == 0) return PACE_KV_OK;
  return hip_status(hipLaunchKernel(latent_dim == 512 ? pick_join<512>(elem_type) : pick_join<256>(elem_type),
                                    dim3(static_cast<uint32_t>((nnz * num_heads + kWaves - 1) / kWaves)), dim3(kThreads),
                                    args, 0, static_cast<hipStream_t>(stream)), "latent attention join launch");
}

}  // extern "C"

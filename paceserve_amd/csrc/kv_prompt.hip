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
constexpr uint32_t kRows = 64;                           // query rows of a workgroup

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
  int64_t q_token, q_head, k_token, k_head, r_token, v_token, v_head, o_token, o_head;  // strides in bytes
  uint32_t batch, nnz, keys, heads, max_q, tiles;
  float scale_log2;
  uint32_t causal;
};

struct PromptRequest {
  uint32_t index, tile;        // the request, and the tile of it
  int32_t q0, q1, k0, k1;
};

// The request whose row tiles (ceil(q_len / kRows) each) hold number x; false past the
// last.  The wave looks at 64 requests a round.
__device__ __forceinline__ bool find_tile(const PromptParams& p, uint32_t x, PromptRequest* r) {
  const uint32_t lane = threadIdx.x % 64;
  uint32_t before = 0;
  for (uint32_t b0 = 0; b0 < p.batch; b0 += 64) {
    const uint32_t b = b0 + lane;
    int32_t q0 = 0, q1 = 0;
    if (b < p.batch) {
      q0 = p.qo_indptr[b];
      q1 = p.qo_indptr[b + 1];
    }
    // Offsets outside the rows leave the request without tiles.
    const bool fine = q0 >= 0 && q1 > q0 && static_cast<uint32_t>(q1) <= p.nnz && static_cast<uint32_t>(q1 - q0) <= p.max_q;
    const uint32_t n = fine ? (static_cast<uint32_t>(q1 - q0) + kRows - 1) / kRows : 0u;
    const uint32_t upto = before + sum_upto(n);
    const uint64_t mine = __ballot(x < upto);
    if (mine != 0) {
      const int at = __builtin_ctzll(mine);
      r->index = b0 + at;
      r->tile = x - (__builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(n, at));
      r->q0 = __builtin_amdgcn_readlane(q0, at);
      r->q1 = __builtin_amdgcn_readlane(q1, at);
      return true;
    }
    before = __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

template <int DN, int TYPE>
__global__ __launch_bounds__(kThreads, 1) void prompt_kernel(const PromptParams p) {
  constexpr int kW = DN + kRope, kKS = kW / 32, kCT = DN / 16;
  constexpr uint32_t kKeyRow = kStride<kW>, kValRow = kStride<DN>;
  __shared__ __attribute__((aligned(16))) char lds_k[kTile * kKeyRow];
  __shared__ __attribute__((aligned(16))) char lds_v[kTile * kValRow];
  const uint32_t lane = threadIdx.x % 64, g = lane / 16, n = lane % 16;
  const uint32_t w = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t head = blockIdx.x;
  // One workgroup counts the requests that are cut or skipped.
  if (p.err != nullptr && blockIdx.x == 0 && blockIdx.y == 0) {
    for (uint32_t b = threadIdx.x; b < p.batch; b += kThreads) {
      const int32_t q0 = p.qo_indptr[b], q1 = p.qo_indptr[b + 1], k0 = p.kv_indptr[b], k1 = p.kv_indptr[b + 1];
      const bool fine = q0 >= 0 && q1 >= q0 && static_cast<uint32_t>(q1) <= p.nnz &&
                        static_cast<uint32_t>(q1 - q0) <= p.max_q && k0 >= 0 && k1 >= k0 &&
                        static_cast<uint32_t>(k1) <= p.keys;
      if (!fine) atomicAdd(p.err, 1);
    }
  }
  PromptRequest r;
  if (!find_tile(p, blockIdx.y, &r)) return;
  const int32_t k0 = min(max(p.kv_indptr[r.index], 0), static_cast<int32_t>(p.keys));
  const int32_t k1 = min(max(p.kv_indptr[r.index + 1], k0), static_cast<int32_t>(p.keys));
  const int32_t q_len = r.q1 - r.q0, kv_len = k1 - k0, base = kv_len - q_len;
  const int32_t row0 = static_cast<int32_t>(r.tile * kRows), my_row = row0 + static_cast<int32_t>(w * 16 + n);
  int32_t t_end = kv_len;
  if (p.causal) t_end = min(t_end, base + min(row0 + static_cast<int32_t>(kRows), q_len));
  u32x4 qf[kKS];
#pragma unroll
  for (int k = 0; k < kKS; ++k) {
    qf[k] = u32x4{0, 0, 0, 0};
    if (my_row < q_len)
      qf[k] = *reinterpret_cast<const u32x4*>(p.q + static_cast<int64_t>(r.q0 + my_row) * p.q_token + head * p.q_head +
                                              k * 64 + g * 16);
  }
  f32x4 acc[kCT];
#pragma unroll
  for (int d = 0; d < kCT; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  for (int32_t t0 = 0; t0 < t_end; t0 += kTile) {
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < kTile * (kW / 8); e += kThreads) {
      const uint32_t row = e / (kW / 8), c = e % (kW / 8);
      const int64_t t = k0 + t0 + static_cast<int64_t>(row);
      u32x4 x = {0, 0, 0, 0};
      if (t0 + static_cast<int32_t>(row) < t_end)
        x = c < DN / 8 ? *reinterpret_cast<const u32x4*>(p.key + t * p.k_token + head * p.k_head + c * 16)
                       : *reinterpret_cast<const u32x4*>(p.rope_key + t * p.r_token + (c - DN / 8) * 16);
      *reinterpret_cast<u32x4*>(lds_k + row * kKeyRow + c * 16) = x;
    }
    for (uint32_t e = threadIdx.x; e < kTile * (DN / 8); e += kThreads) {
      const uint32_t row = e / (DN / 8), c = e % (DN / 8);
      const int64_t t = k0 + t0 + static_cast<int64_t>(row);
      u32x4 x = {0, 0, 0, 0};
      if (t0 + static_cast<int32_t>(row) < t_end)
        x = *reinterpret_cast<const u32x4*>(p.value + t * p.v_token + head * p.v_head + c * 16);
      *reinterpret_cast<u32x4*>(lds_v + row * kValRow + c * 16) = x;
    }
    __syncthreads();
    f32x4 s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int k = 0; k < kKS; ++k)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const u32x4 kf = *reinterpret_cast<const u32x4*>(lds_k + (t * 16 + n) * kKeyRow + k * 64 + g * 16);
        s[t] = mfma<TYPE>(kf, qf[k], s[t]);
      }
    const int32_t upto = min((p.causal ? base + my_row + 1 : kv_len) - t0, t_end - t0);
    const uint32_t sees = upto >= 32 ? ~0u : upto <= 0 ? 0u : (1u << upto) - 1u, mine = sees >> (4 * g);
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
    bool odd = false;
    if (__ballot(sees == ~0u) != ~0ull) {
      bool found = false;
      for (uint32_t c = lane; c < kTile * DN / 8; c += 64) {
        const u32x4 x = *reinterpret_cast<const u32x4*>(lds_v + c / (DN / 8) * kValRow + c % (DN / 8) * 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) found |= odd_word<TYPE>(x[e]);
      }
      odd = __ballot(found) != 0;
    }
#pragma unroll
    for (int d = 0; d < kCT; ++d) {
      const char* v = lds_v + lane / 4 * kValRow + d * 32 + lane % 4 * 8;
      typedef __attribute__((address_space(3))) s16x4* lds_ptr;
      const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)v));
      const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(v + 16 * kValRow)));
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
          const u32x2 v = *reinterpret_cast<const u32x2*>(lds_v + token * kValRow + d * 32 + g * 8);
#pragma unroll
          for (int c = 0; c < 4; ++c) acc[d][c] += weight * value_of<TYPE>(v[c / 2], c % 2);
        }
      }
    }
  }
  l = across_groups(l, sum_of);
  if (my_row >= q_len) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int d = 0; d < kCT; ++d) {
    const u32x2 x = {result_pair<TYPE>(acc[d][0] * inv, acc[d][1] * inv),
                     result_pair<TYPE>(acc[d][2] * inv, acc[d][3] * inv)};
    *reinterpret_cast<u32x2*>(p.out + static_cast<int64_t>(r.q0 + my_row) * p.o_token + head * p.o_head +
                              (d * 16 + g * 4) * 2) = x;
  }
  if (g == 0 && p.lse != nullptr) p.lse[static_cast<int64_t>(r.q0 + my_row) * p.heads + head] = log_total<TYPE>(m, l);
}

template <int DN>
const void* pick_prompt(int type) {
  return type == PACE_KV_BF16 ? reinterpret_cast<const void*>(&prompt_kernel<DN, PACE_KV_BF16>)
                              : reinterpret_cast<const void*>(&prompt_kernel<DN, PACE_KV_FP16>);
}

}  // namespace
}  // namespace pace_kv

extern "C" {

int pace_kv_prompt_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, const void* key,
                             int64_t k_token_stride, int64_t k_head_stride, const void* rope_key,
                             int64_t rope_token_stride, const void* value, int64_t v_token_stride, int64_t v_head_stride,
                             int elem_type, int num_heads, int head_dim, int64_t nnz, int64_t num_keys,
                             const int32_t* qo_indptr, const int32_t* kv_indptr, int batch_size, int max_q_len,
                             float scale, int causal, void* out, int64_t out_token_stride, int64_t out_head_stride,
                             float* lse, int32_t* err_count, void* stream) {
  using namespace pace_kv;
  if (nnz < 0 || num_keys < 0 || batch_size < 0 || num_heads <= 0 || max_q_len <= 0)
    return fail(PACE_KV_EINVAL, "prompt attention: sizes must be positive");
  if (head_dim != 64 && head_dim != 128)
    return fail(PACE_KV_EINVAL, "prompt attention: head_dim must be 64 or 128, got %d", head_dim);
  if (elem_type != PACE_KV_BF16 && elem_type != PACE_KV_FP16)
    return fail(PACE_KV_EINVAL, "prompt attention: queries must be bfloat16 or float16");
  if (nnz > INT32_MAX / 2 || num_keys > INT32_MAX / 2)
    return fail(PACE_KV_ERANGE, "prompt attention: more than 2^30 queries or keys");
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
  // As many tiles as there can be: a short last one for each request.
  const int64_t tiles = std::min<int64_t>(nnz, nnz / kRows + batch_size);
  if (tiles > 65535 || num_heads > (1 << 20) || tiles * num_heads >= (int64_t(1) << 24))
    return fail(PACE_KV_ERANGE, "prompt attention: too many requests, heads or queries for one call");
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
  p.tiles = static_cast<uint32_t>(tiles);
  p.scale_log2 = scale_log2;
  p.causal = causal != 0;
  void* args[] = {&p};
  return hip_status(hipLaunchKernel(head_dim == 128 ? pick_prompt<128>(elem_type) : pick_prompt<64>(elem_type),
                                    dim3(p.heads, p.tiles), dim3(kThreads), args, 0, static_cast<hipStream_t>(stream)),
                    "prompt attention launch");
}

}  // extern "C"

// The tables of a batch from its lengths: page lists end to end, positions and
// cache slots of the tokens that the step appends.
//
//   pages[b]  = ceil(seq_lens[b] / P);  kv_indptr = their running sum
//   kv_indices[kv_indptr[b] + i] = page_table[b][i]
//   token j of request b's n: pos = seq_lens[b] - n + j,
//   slot = page_table[b][pos / P] * P + pos % P
//
// Bound by latency: a decode step's tables are a few KiB, those of hundreds of
// long requests some MB.  So one launch: a workgroup takes a request (or a share
// of a long one), adds up the pages of the requests before it by itself (all
// lengths are a few loads a lane, from L2 after the first workgroup), and writes
// its part of every output.
#include "internal.h"

namespace pace_kv {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
// Entries (page ids, tokens) that a workgroup takes before a request gets
// another one, and the most workgroups that the longest lists are spread over.
constexpr int64_t kEntries = 1024, kMostShares = 64, kMostGroups = 2048;

struct TableParams {
  const int32_t* page_table;
  int64_t table_stride;        // entries between requests
  const int32_t* seq_lens;
  const int32_t* append_indptr;  // batch + 1 entries, or nullptr: one token per request
  int32_t* kv_indices;
  int32_t* kv_indptr;
  int32_t* kv_last_page_len;
  int32_t* positions;
  int64_t* slots;
  int32_t* err;
  uint32_t batch, width, page_size, nnz, num_indices, shares;
  FastDiv by_page;
};

__device__ __forceinline__ uint32_t pages_for(const TableParams& p, int32_t len) {
  const uint32_t n = static_cast<uint32_t>(max(len, 0));
  const uint32_t whole = over(p.by_page, n);
  return min(whole + (whole * p.page_size < n ? 1u : 0u), p.width);
}

__device__ __forceinline__ uint32_t wave_sum(uint32_t x) {
#pragma unroll
  for (int k = 1; k < 64; k *= 2) x += __shfl_xor(x, k);
  return x;
}

__global__ __launch_bounds__(kThreads) void tables_kernel(const TableParams p) {
  __shared__ uint32_t lds_before[kWaves], lds_all[kWaves];
  const uint32_t b = blockIdx.x, share = blockIdx.y, tid = threadIdx.x;
  const uint32_t step = p.shares * kThreads, first = share * kThreads + tid;
  // What the request is, before the sums that all of its entries wait for.
  const int32_t len = p.seq_lens[b];
  int32_t a0 = static_cast<int32_t>(b), a1 = a0 + 1, tokens_end = static_cast<int32_t>(p.batch), tokens_first = 0;
  if (p.append_indptr != nullptr) {
    a0 = p.append_indptr[b];
    a1 = p.append_indptr[b + 1];
    tokens_first = p.append_indptr[0];
    tokens_end = p.append_indptr[p.batch];
  }
  uint32_t before = 0, all = 0;
  for (uint32_t i = tid; i < p.batch; i += kThreads) {
    const uint32_t n = pages_for(p, p.seq_lens[i]);
    all += n;
    if (i < b) before += n;
  }
  before = wave_sum(before);
  all = wave_sum(all);
  if (tid % 64 == 0) {
    lds_before[tid / 64] = before;
    lds_all[tid / 64] = all;
  }
  __syncthreads();
  before = all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    before += lds_before[w];
    all += lds_all[w];
  }
  const uint32_t pages = pages_for(p, len);
  const int64_t room = static_cast<int64_t>(p.width) * p.page_size;
  const int32_t kept = static_cast<int32_t>(min(static_cast<int64_t>(max(len, 0)), room));
  const int64_t lo = min(max(static_cast<int64_t>(a0), int64_t(0)), static_cast<int64_t>(p.nnz));
  const int64_t hi = min(max(static_cast<int64_t>(a1), lo), static_cast<int64_t>(p.nnz));
  if (share == 0 && tid == 0) {
    p.kv_indptr[b] = static_cast<int32_t>(before);
    if (b + 1 == p.batch) p.kv_indptr[p.batch] = static_cast<int32_t>(all);
    p.kv_last_page_len[b] = pages == 0 ? 0 : kept - static_cast<int32_t>((pages - 1) * p.page_size);
    // A request of no tokens without offsets is a place of a fixed batch that nobody holds.
    const bool idle = p.append_indptr == nullptr && len == 0;
    const bool cut = len != kept || lo != a0 || hi != a1 || (hi - lo > len && !idle) || before + pages > p.num_indices;
    if (p.err != nullptr && cut) atomicAdd(p.err, 1);
  }
  const int32_t* const row = p.page_table + static_cast<int64_t>(b) * p.table_stride;
  for (uint32_t i = first; i < pages; i += step)
    if (before + i < p.num_indices) p.kv_indices[before + i] = row[i];
  const int64_t base = static_cast<int64_t>(len) - (hi - lo);
  for (int64_t j = first; j < hi - lo; j += step) {
    const int64_t pos = base + j;
    int64_t slot = -1;
    if (pos >= 0 && pos < kept) {
      const uint32_t at = over(p.by_page, static_cast<uint32_t>(pos));
      const int32_t page = row[at];
      if (page >= 0) slot = static_cast<int64_t>(page) * p.page_size + (pos - static_cast<int64_t>(at) * p.page_size);
    }
    p.positions[lo + j] = static_cast<int32_t>(max(pos, int64_t(-1)));
    p.slots[lo + j] = slot;
  }
  // Entries behind the last request, and tokens outside every request, by all workgroups.
  const uint64_t groups = static_cast<uint64_t>(p.batch) * p.shares * kThreads;
  const uint64_t mine = (static_cast<uint64_t>(b) * p.shares + share) * kThreads + tid;
  for (uint64_t i = all + mine; i < p.num_indices; i += groups) p.kv_indices[i] = -1;
  const uint64_t tail = static_cast<uint64_t>(max(tokens_end, 0));
  for (uint64_t i = tail + mine; i < p.nnz; i += groups) {
    p.positions[i] = -1;
    p.slots[i] = -1;
  }
  const uint64_t head = min(static_cast<uint64_t>(max(tokens_first, 0)), static_cast<uint64_t>(p.nnz));
  for (uint64_t i = mine; i < head; i += groups) {
    p.positions[i] = -1;
    p.slots[i] = -1;
  }
}

// The tables of a batch of no requests.
__global__ __launch_bounds__(kThreads) void no_tables_kernel(const TableParams p) {
  const uint64_t groups = static_cast<uint64_t>(gridDim.x) * kThreads;
  const uint64_t mine = static_cast<uint64_t>(blockIdx.x) * kThreads + threadIdx.x;
  if (mine == 0) p.kv_indptr[0] = 0;
  for (uint64_t i = mine; i < p.num_indices; i += groups) p.kv_indices[i] = -1;
  for (uint64_t i = mine; i < p.nnz; i += groups) {
    p.positions[i] = -1;
    p.slots[i] = -1;
  }
}

}  // namespace
}  // namespace pace_kv

extern "C" {

int pace_kv_build_tables(const int32_t* page_table, int64_t table_stride, int width, const int32_t* seq_lens,
                         int batch_size, int page_size, const int32_t* append_indptr, int64_t nnz, int32_t* kv_indices,
                         int64_t num_indices, int32_t* kv_indptr, int32_t* kv_last_page_len, int32_t* positions,
                         int64_t* slot_mapping, int32_t* err_count, void* stream) {
  using namespace pace_kv;
  if (batch_size < 0 || width < 0 || nnz < 0 || num_indices < 0 || page_size <= 0)
    return fail(PACE_KV_EINVAL, "tables: negative size, or pages of no tokens");
  if (nnz > INT32_MAX || num_indices > INT32_MAX || static_cast<int64_t>(batch_size) * width > INT32_MAX)
    return fail(PACE_KV_ERANGE, "tables: more than 2^31 - 1 tokens or table entries");
  if (!kv_indptr || (batch_size > 0 && (!seq_lens || !kv_last_page_len || (width > 0 && !page_table))) ||
      (num_indices > 0 && !kv_indices) || (nnz > 0 && (!positions || !slot_mapping)))
    return fail(PACE_KV_EINVAL, "tables: NULL argument");
  if (width > 0 && batch_size > 1 && table_stride < width)
    return fail(PACE_KV_EINVAL, "tables: rows of the page table overlap");
  if (!append_indptr && nnz < batch_size)
    return fail(PACE_KV_EINVAL, "tables: without append_indptr each request has one token");
  TableParams p = {};
  p.page_table = page_table;
  p.table_stride = table_stride;
  p.seq_lens = seq_lens;
  p.append_indptr = append_indptr;
  p.kv_indices = kv_indices;
  p.kv_indptr = kv_indptr;
  p.kv_last_page_len = kv_last_page_len;
  p.positions = positions;
  p.slots = slot_mapping;
  p.err = err_count;
  p.batch = static_cast<uint32_t>(batch_size);
  p.width = static_cast<uint32_t>(width);
  p.page_size = static_cast<uint32_t>(page_size);
  p.nnz = static_cast<uint32_t>(nnz);
  p.num_indices = static_cast<uint32_t>(num_indices);
  p.by_page = fast_div(p.page_size);
  const int64_t entries = nnz > num_indices ? nnz : num_indices;
  void* args[] = {&p};
  if (batch_size == 0) {
    const int64_t groups = entries / kEntries + 1;
    return hip_status(hipLaunchKernel(reinterpret_cast<const void*>(&no_tables_kernel),
                                      dim3(static_cast<uint32_t>(groups < kMostGroups ? groups : kMostGroups)),
                                      dim3(kThreads), args, 0, static_cast<hipStream_t>(stream)), "tables launch");
  }
  int64_t shares = (entries + kEntries * batch_size - 1) / (kEntries * batch_size);
  if (shares > kMostShares) shares = kMostShares;
  if (shares * batch_size > kMostGroups) shares = kMostGroups / batch_size;
  p.shares = static_cast<uint32_t>(shares > 1 ? shares : 1);
  return hip_status(hipLaunchKernel(reinterpret_cast<const void*>(&tables_kernel), dim3(p.batch, p.shares),
                                    dim3(kThreads), args, 0, static_cast<hipStream_t>(stream)), "tables launch");
}

}  // extern "C"

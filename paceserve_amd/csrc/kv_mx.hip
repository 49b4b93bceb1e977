// Pages between a pool of 16- or 32-bit elements and a quantised one (format:
// mx.h), all layers in one call:
//   quantize:   dst[l][dst_ids[j]] = elements and scales of src[l][src_ids[j]]
//   dequantize: dst[l][dst_ids[j]] = values of src[l][src_ids[j]]
//
// A page half is one run of N = page_size * H * D elements on either side, so a
// wave takes kRuns * 512 consecutive elements of one half.  Bound by HBM: what is
// done to a value is half an instruction of conversion and less than one of
// finding its block's largest magnitude.  Rows and elements stream through: stored
// and, on the way down, loaded nontemporally.  MI355X, bytes read and written:
//   256 pages of 64 KiB, 32 layers, bf16 to 8 bits    127 us (6.4 TB/s), 144 with plain accesses
//   the same back                                     133 us (6.1 TB/s), 141
//   2048 pages of 8 KiB, 64 layers, to 8 bits         256 us (6.4 TB/s), 292
//   63 pages of 256 KiB, 32 layers, fp16 to 4 bits    107 us (6.2 TB/s), 121; back 110, 126
//   32 pages of 64 KiB, 32 layers, to 8 bits          17.5 us (5.8 TB/s), 17.4
// Two or eight runs a lane measured within 3% of four.  A float32 lane that wrote two
// vectors 32 bytes apart took 208 us for 256 pages of 128 KiB, 16 layers, nontemporally.
#include "mx.h"

namespace pace_kv {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kRuns = 4;                              // runs of 8 elements that a lane carries
constexpr int64_t kTileElems = 64 * kLaneElems * kRuns;
constexpr int64_t kMaxItems = int64_t(1) << 30;       // waves of one launch

struct PagesParams {
  const char* src[PACE_KV_MAX_LAYERS_PER_LAUNCH];
  char* dst[PACE_KV_MAX_LAYERS_PER_LAUNCH];
  const int32_t* src_ids;
  const int32_t* dst_ids;
  uint32_t src_pool, dst_pool;
  int32_t* err;
  int64_t half_elems;
  int64_t mx_half;         // bytes of a quantised half page
  uint32_t tiles;          // per half page
  uint32_t n_pages;
  uint32_t items;          // layers * pages * 2 * tiles
  uint32_t first_page;     // of this launch, among the call's
  FastDiv by_tiles, by_pages;
};

// Source and destination of one wave's tile.
struct Tile {
  uint32_t layer, half;
  int64_t first;           // element of the half
  uint32_t src_page, dst_page;
};

__device__ __forceinline__ bool locate_tile(const PagesParams& p, Tile* t) {
  const uint32_t item = __builtin_amdgcn_readfirstlane(blockIdx.x * kWaves + threadIdx.x / 64);
  if (item >= p.items) return false;
  const uint32_t side = over(p.by_tiles, item);       // (layer * n_pages + j) * 2 + half
  const uint32_t tile = item - side * p.tiles;
  t->half = side & 1;
  t->layer = over(p.by_pages, side >> 1);
  const uint32_t j = (side >> 1) - t->layer * p.n_pages;
  t->first = tile * kTileElems;
  t->src_page = static_cast<uint32_t>(p.src_ids[p.first_page + j]);
  t->dst_page = static_cast<uint32_t>(p.dst_ids[p.first_page + j]);
  if (t->src_page < p.src_pool && t->dst_page < p.dst_pool) return true;
  if (tile == 0 && t->half == 0 && threadIdx.x % 64 == 0 && p.err != nullptr) atomicAdd(p.err, 1);
  return false;
}

template <int TYPE, int FORMAT>
__global__ __launch_bounds__(kThreads) void quantize_pages_kernel(const PagesParams p) {
  Tile t;
  if (!locate_tile(p, &t)) return;
  constexpr int kElem = elem_bytes(TYPE);
  const char* src = p.src[t.layer] + (2 * static_cast<int64_t>(t.src_page) + t.half) * p.half_elems * kElem;
  char* dst = p.dst[t.layer] + (2 * static_cast<int64_t>(t.dst_page) + t.half) * p.mx_half;
  char* scales = dst + p.half_elems * mx_bits(FORMAT) / 8;
  const int64_t at = t.first + threadIdx.x % 64 * kLaneElems;
  Run<TYPE> r[kRuns];
#pragma unroll
  for (int k = 0; k < kRuns; ++k) {
    const int64_t e = at + k * 64 * kLaneElems;
    if (e < p.half_elems) r[k] = load_run<TYPE, true>(src + e * kElem);
  }
#pragma unroll
  for (int k = 0; k < kRuns; ++k) {
    const int64_t e = at + k * 64 * kLaneElems;
    if (e >= p.half_elems) break;                     // whole blocks: half_elems is a multiple of 32
    store_run<TYPE, FORMAT, true>(r[k], scale_byte<FORMAT>(block_amax<TYPE>(r[k])), dst + e * mx_bits(FORMAT) / 8,
                            scales + e / kMxBlock);
  }
}

template <int TYPE, int FORMAT>
__global__ __launch_bounds__(kThreads) void dequantize_pages_kernel(const PagesParams p) {
  Tile t;
  if (!locate_tile(p, &t)) return;
  constexpr int kElem = elem_bytes(TYPE);
  const char* src = p.src[t.layer] + (2 * static_cast<int64_t>(t.src_page) + t.half) * p.mx_half;
  const char* scales = src + p.half_elems * mx_bits(FORMAT) / 8;
  char* dst = p.dst[t.layer] + (2 * static_cast<int64_t>(t.dst_page) + t.half) * p.half_elems * kElem;
  // A lane writes 16 bytes at a time, next to its neighbours': eight 16-bit values,
  // or four of 32 bits.
  constexpr int kElems = 16 / kElem, kSteps = kTileElems / (64 * kElems);
  const int64_t at = t.first + threadIdx.x % 64 * kElems;
  u32x2 q[kSteps];
  uint32_t byte[kSteps];
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    const int64_t e = at + k * 64 * kElems;
    if (e >= p.half_elems) break;
    constexpr int kBytes = kElems * mx_bits(FORMAT) / 8;
    const char* const from = src + e * mx_bits(FORMAT) / 8;
    if constexpr (kBytes == 8) q[k] = *reinterpret_cast<const u32x2*>(from);
    else if constexpr (kBytes == 4) q[k] = u32x2{*reinterpret_cast<const uint32_t*>(from), 0};
    else q[k] = u32x2{*reinterpret_cast<const uint16_t*>(from), 0};
    byte[k] = *reinterpret_cast<const uint8_t*>(scales + e / kMxBlock);
  }
#pragma unroll
  for (int k = 0; k < kSteps; ++k) {
    const int64_t e = at + k * 64 * kElems;
    if (e >= p.half_elems) break;
    const float s = scale_of(byte[k]);
    u32x4* const to = reinterpret_cast<u32x4*>(dst + e * kElem);
    if constexpr (TYPE == PACE_KV_FP32) {
      const f32x2 x = pair_up_f32<FORMAT, 0>(q[k][0], s), y = pair_up_f32<FORMAT, 1>(q[k][0], s);
      put<true>(to, u32x4{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(y[0]), __float_as_uint(y[1])});
    } else {
      put<true>(to, run_up<TYPE, FORMAT>(q[k], s));
    }
  }
}

template <int FORMAT>
const void* pick(bool down, int type) {
  switch (type) {
    case PACE_KV_BF16:
      return down ? reinterpret_cast<const void*>(&quantize_pages_kernel<PACE_KV_BF16, FORMAT>)
                  : reinterpret_cast<const void*>(&dequantize_pages_kernel<PACE_KV_BF16, FORMAT>);
    case PACE_KV_FP16:
      return down ? reinterpret_cast<const void*>(&quantize_pages_kernel<PACE_KV_FP16, FORMAT>)
                  : reinterpret_cast<const void*>(&dequantize_pages_kernel<PACE_KV_FP16, FORMAT>);
    default:
      return down ? reinterpret_cast<const void*>(&quantize_pages_kernel<PACE_KV_FP32, FORMAT>)
                  : reinterpret_cast<const void*>(&dequantize_pages_kernel<PACE_KV_FP32, FORMAT>);
  }
}

// Checks the arguments both directions share and launches, at most
// PACE_KV_MAX_LAYERS_PER_LAUNCH layers and kMaxItems waves at a time.
int convert_pages(const char* what, bool down, const void* const* src_layers, int64_t src_pool, const int32_t* src_ids,
                  void* const* dst_layers, int64_t dst_pool, const int32_t* dst_ids, int type, int format,
                  int num_layers, int64_t n_pages, int64_t half_elems, int32_t* err, hipStream_t stream) {
  if (num_layers < 0 || n_pages < 0 || src_pool < 0 || dst_pool < 0)
    return fail(PACE_KV_EINVAL, "%s: negative size", what);
  if (!is_elem_type(type)) return fail(PACE_KV_EINVAL, "%s: unknown element type %d", what, type);
  if (!is_mx_format(format)) return fail(PACE_KV_EINVAL, "%s: unknown format %d", what, format);
  if (num_layers == 0 || n_pages == 0) return PACE_KV_OK;
  if (!src_layers || !dst_layers || !src_ids || !dst_ids) return fail(PACE_KV_EINVAL, "%s: NULL argument", what);
  if (half_elems <= 0 || half_elems % kMxBlock != 0 || mx_half_bytes(half_elems, format) % 16 != 0)
    return fail(PACE_KV_EINVAL, "%s: half a page (page_size * H * D elements) must be whole blocks of 32 and, "
                "quantised, a multiple of 16 bytes", what);
  if ((reinterpret_cast<uintptr_t>(src_ids) | reinterpret_cast<uintptr_t>(dst_ids)) & 3u)
    return fail(PACE_KV_EINVAL, "%s: page ids must be 4-byte aligned", what);
  if (src_pool > INT32_MAX || dst_pool > INT32_MAX || n_pages > INT32_MAX)
    return fail(PACE_KV_ERANGE, "%s: too many pages", what);
  for (int l = 0; l < num_layers; ++l) {
    if (!src_layers[l] || !dst_layers[l]) return fail(PACE_KV_EINVAL, "%s: layer %d is NULL", what, l);
    if ((reinterpret_cast<uintptr_t>(src_layers[l]) | reinterpret_cast<uintptr_t>(dst_layers[l])) & 15u)
      return fail(PACE_KV_EINVAL, "%s: layer %d must be 16-byte aligned", what, l);
  }
  const int64_t tiles = (half_elems + kTileElems - 1) / kTileElems;
  if (2 * tiles > kMaxItems) return fail(PACE_KV_ERANGE, "%s: page too large", what);
  PagesParams p = {};
  p.src_ids = src_ids;
  p.dst_ids = dst_ids;
  p.src_pool = static_cast<uint32_t>(src_pool);
  p.dst_pool = static_cast<uint32_t>(dst_pool);
  p.err = err;
  p.half_elems = half_elems;
  p.mx_half = mx_half_bytes(half_elems, format);
  p.tiles = static_cast<uint32_t>(tiles);
  p.by_tiles = fast_div(p.tiles);
  const void* fn = format == PACE_KV_MXFP8 ? pick<PACE_KV_MXFP8>(down, type) : pick<PACE_KV_MXFP4>(down, type);
  const int64_t max_sides = kMaxItems / (2 * tiles);  // layer pages of one launch, at least one
  for (int l0 = 0; l0 < num_layers;) {
    int64_t layers = num_layers - l0 < PACE_KV_MAX_LAYERS_PER_LAUNCH ? num_layers - l0 : PACE_KV_MAX_LAYERS_PER_LAUNCH;
    const int64_t pages = n_pages < max_sides ? n_pages : max_sides;
    if (layers * pages > max_sides) layers = max_sides / pages;
    for (int l = 0; l < layers; ++l) {
      p.src[l] = static_cast<const char*>(src_layers[l0 + l]);
      p.dst[l] = static_cast<char*>(dst_layers[l0 + l]);
    }
    for (int64_t j0 = 0; j0 < n_pages; j0 += pages) {
      const int64_t n = n_pages - j0 < pages ? n_pages - j0 : pages;
      p.first_page = static_cast<uint32_t>(j0);
      p.n_pages = static_cast<uint32_t>(n);
      p.by_pages = fast_div(p.n_pages);
      p.items = static_cast<uint32_t>(layers * n * 2 * tiles);
      void* args[] = {&p};
      PACE_KV_TRY(hip_status(hipLaunchKernel(fn, dim3((p.items + kWaves - 1) / kWaves), dim3(kThreads), args, 0,
                                             stream), what));
    }
    l0 += static_cast<int>(layers);
  }
  return PACE_KV_OK;
}

}  // namespace
}  // namespace pace_kv

extern "C" {

int pace_kv_quantize_pages(const void* const* src_layers, int64_t src_pool_pages, const int32_t* src_ids,
                           int elem_type, void* const* dst_layers, int64_t dst_pool_pages, const int32_t* dst_ids,
                           int format, int num_layers, int64_t n_pages, int64_t half_elems, int32_t* err_count,
                           void* stream) {
  return pace_kv::convert_pages("quantize_pages", true, src_layers, src_pool_pages, src_ids, dst_layers,
                                dst_pool_pages, dst_ids, elem_type, format, num_layers, n_pages, half_elems, err_count,
                                static_cast<hipStream_t>(stream));
}

int pace_kv_dequantize_pages(const void* const* src_layers, int64_t src_pool_pages, const int32_t* src_ids, int format,
                             void* const* dst_layers, int64_t dst_pool_pages, const int32_t* dst_ids, int elem_type,
                             int num_layers, int64_t n_pages, int64_t half_elems, int32_t* err_count, void* stream) {
  return pace_kv::convert_pages("dequantize_pages", false, src_layers, src_pool_pages, src_ids, dst_layers,
                                dst_pool_pages, dst_ids, elem_type, format, num_layers, n_pages, half_elems, err_count,
                                static_cast<hipStream_t>(stream));
}

}  // extern "C"

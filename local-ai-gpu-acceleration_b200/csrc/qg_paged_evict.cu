// qg_paged_evict.cu -- qg_kv_evict: sequences of a paged key-value cache cut back to a budget
// of slots by the attention weight that their slots received (declared in
// include/qgemv_b200.h).  Two launches:
//
//  * evict_select_kernel, one CTA per (kv head, sequence): the need-th largest weight of the
//    slots between the first `sink` and the last `recent` by radix selection (11 + 11 + 10
//    bits of an order-preserving integer image of the weights, histograms in shared memory),
//    then the kept slots in ascending order: every warp counts its stretch of the slots, one
//    scan over the warps, every warp writes its stretch.  Weights equal to the threshold are
//    taken from the lowest slot on.
//  * evict_move_kernel: rows kept[i] -> i.  kept[] ascends and kept[i] >= i, so in place a CTA
//    that walks i upwards, reading a chunk of rows before it writes it, never overwrites a
//    row that is still to be read; a row's columns are independent, so (K, V) x (64-byte
//    column slices) walk side by side.  Into other pages there is no such order and the rows
//    are split over CTAs as well.
//
// Bound by memory: the weights once, the kept rows once in and once out.
#include <algorithm>

#include <mutex>
#include <set>

#include "qg_paged.cuh"

namespace qg {
namespace {

constexpr uint32_t kSelectThreads = 1024;
constexpr uint32_t kSelectWarps = kSelectThreads / 32;
constexpr uint32_t kBins = 2048;
constexpr uint32_t kCachedKeys = 48u * 1024u;  // slots whose keys fit in shared memory (192 KB)

struct EvictArgs {
  const int32_t* lens;
  int32_t* lens_out;
  const float* weight;
  float* weight_out;
  int32_t* kept;
  const int32_t* to_table;
  uint32_t to_stride;
  uint32_t max_len, weight_stride, budget, sink, recent;
  uint32_t slices, parts;
  bool in_place;
};

// An integer that orders like the weight: NaN lowest, -0 equal to +0.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (isnan(w)) return 0u;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) != 0u ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(const PagedView c, const EvictArgs a,
                                                                      bool cached) {
  extern __shared__ uint32_t keys[];
  __shared__ uint32_t bins[kBins];
  __shared__ uint32_t warp_a[kSelectWarps], warp_b[kSelectWarps];
  __shared__ uint32_t found_bin, found_left;
  const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  const uint32_t kv = blockIdx.x, b = blockIdx.y;
  pdl_wait();
  pdl_trigger();
  const uint32_t n = paged_len(a.lens[b], min(a.max_len, c.capacity));
  const float* w = a.weight + (static_cast<size_t>(b) * c.n_kv + kv) * a.weight_stride;
  int32_t* kept = a.kept + (static_cast<size_t>(b) * c.n_kv + kv) * a.budget;
  if (n <= a.budget) {
    for (uint32_t i = tid; i < a.budget; i += kSelectThreads) kept[i] = i < n ? static_cast<int32_t>(i) : -1;
    return;
  }
  const uint32_t lo = a.sink, hi = n - a.recent;  // the slots that are chosen from
  uint32_t left = a.budget - a.sink - a.recent;   // how many of them stay
  auto key_at = [&](uint32_t i) { return cached ? keys[i] : weight_key(w[i]); };
  if (cached) {
    for (uint32_t i = lo + tid; i < hi; i += kSelectThreads) keys[i] = weight_key(w[i]);
  }
  // ---- the threshold: the left-th largest key, and how many equal to it stay
  uint32_t prefix = 0u, mask = 0u;
  if (left != 0u) {
    for (uint32_t pass = 0; pass < 3u; ++pass) {
      const uint32_t shift = pass == 0u ? 21u : pass == 1u ? 10u : 0u;
      const uint32_t width = pass == 2u ? 1024u : 2048u;
      for (uint32_t i = tid; i < kBins; i += kSelectThreads) bins[i] = 0u;
      __syncthreads();
      for (uint32_t i0 = lo; i0 < hi; i0 += kSelectThreads) {
        const uint32_t i = i0 + tid;
        const uint32_t key = i < hi ? key_at(i) : 0u;
        const bool counts = i < hi && (key & mask) == prefix;
        const uint32_t bin = (key >> shift) & (width - 1u);
        // one addition where a whole warp falls into one bin (weights that are all alike)
        const uint32_t live = __ballot_sync(0xffffffffu, counts);
        if (live == 0u) continue;
        const uint32_t lead = __ffs(live) - 1u;
        const uint32_t lead_bin = __shfl_sync(0xffffffffu, bin, lead);
        const uint32_t same = __ballot_sync(0xffffffffu, counts && bin == lead_bin);
        if (same == live) {
          if (lane == lead) atomicAdd(&bins[bin], static_cast<uint32_t>(__popc(live)));
        } else if (counts) {
          atomicAdd(&bins[bin], 1u);
        }
      }
      __syncthreads();
      // thread t holds bins 2 t and 2 t + 1; above = keys in higher bins
      const uint32_t b0 = bins[2u * tid], b1 = bins[2u * tid + 1u];
      uint32_t upto = b0 + b1;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const uint32_t o = __shfl_down_sync(0xffffffffu, upto, off);
        if (lane + off < 32u) upto += o;
      }
      if (lane == 0u) warp_a[warp] = upto;
      __syncthreads();
      for (uint32_t x = warp + 1u; x < kSelectWarps; ++x) upto += warp_a[x];
      const uint32_t above1 = upto - b0 - b1, above0 = upto - b0;
      if (above1 < left && left <= above1 + b1) {
        found_bin = 2u * tid + 1u;
        found_left = left - above1;
      } else if (above0 < left && left <= above0 + b0) {
        found_bin = 2u * tid;
        found_left = left - above0;
      }
      __syncthreads();
      prefix |= found_bin << shift;
      mask |= (width - 1u) << shift;
      left = found_left;
    }
  } else {
    prefix = 0xffffffffu;  // above every key
    __syncthreads();
  }
  // ---- the kept slots in ascending order
  const uint32_t per = ((n + kSelectWarps - 1u) / kSelectWarps + 31u) & ~31u;
  const uint32_t from = min(warp * per, n), to = min(from + per, n);
  uint32_t more = 0, ties = 0;
  for (uint32_t i0 = from; i0 < to; i0 += 32u) {
    const uint32_t i = i0 + lane;
    const bool always = i < lo || (i >= hi && i < to);
    const uint32_t key = i >= lo && i < min(hi, to) ? key_at(i) : 0u;
    const bool inside = i >= lo && i < min(hi, to);
    more += __popc(__ballot_sync(0xffffffffu, (always && i < to) || (inside && key > prefix)));
    ties += __popc(__ballot_sync(0xffffffffu, inside && key == prefix));
  }
  if (lane == 0u) {
    warp_a[warp] = more;
    warp_b[warp] = ties;
  }
  __syncthreads();
  more = ties = 0;
  for (uint32_t x = 0; x < warp; ++x) {
    more += warp_a[x];
    ties += warp_b[x];
  }
  const uint32_t below = (1u << lane) - 1u;
  for (uint32_t i0 = from; i0 < to; i0 += 32u) {
    const uint32_t i = i0 + lane;
    const bool always = i < lo || (i >= hi && i < to);
    const bool inside = i >= lo && i < min(hi, to);
    const uint32_t key = inside ? key_at(i) : 0u;
    const uint32_t mb = __ballot_sync(0xffffffffu, (always && i < to) || (inside && key > prefix));
    const uint32_t tb = __ballot_sync(0xffffffffu, inside && key == prefix);
    const uint32_t m = more + __popc(mb & below), t = ties + __popc(tb & below);
    const bool stays = (mb >> lane & 1u) != 0u || ((tb >> lane & 1u) != 0u && t < left);
    if (stays) kept[m + min(t, left)] = static_cast<int32_t>(i);
    more += __popc(mb);
    ties += __popc(tb);
  }
}

constexpr uint32_t kMoveThreads = 256;
constexpr uint32_t kMoveDepth = 8;                      // pieces in flight per thread
constexpr uint32_t kSliceLanes = 4;                     // 16-byte pieces of a column slice
constexpr uint32_t kMoveRows = kMoveThreads / kSliceLanes * kMoveDepth;  // rows of a chunk

// blockIdx.x: the weights (0), then (plane, slice, part).
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const PagedView c, const EvictArgs a) {
  const uint32_t tid = threadIdx.x, kv = blockIdx.y, b = blockIdx.z;
  pdl_wait();
  pdl_trigger();
  // lens may be lens_out: the old and the new length give the same count
  const uint32_t n = min(paged_len(a.lens[b], min(a.max_len, c.capacity)), a.budget);
  const size_t row = static_cast<size_t>(b) * c.n_kv + kv;
  const int32_t* kept = a.kept + row * a.budget;
  if (blockIdx.x == 0u) {
    const float* from = a.weight + row * a.weight_stride;
    float* to = a.weight_out + row * a.weight_stride;
    constexpr uint32_t kChunk = kMoveThreads * kMoveDepth;
    for (uint32_t i0 = 0; i0 < n; i0 += kChunk) {
      float v[kMoveDepth];
#pragma unroll
      for (uint32_t u = 0; u < kMoveDepth; ++u) {
        const uint32_t i = i0 + u * kMoveThreads + tid;
        if (i < n) v[u] = from[kept[i]];
      }
      __syncthreads();  // a chunk is read before it is written
#pragma unroll
      for (uint32_t u = 0; u < kMoveDepth; ++u) {
        const uint32_t i = i0 + u * kMoveThreads + tid;
        if (i < n) to[i] = v[u];
      }
    }
    for (uint32_t i = n + tid; i < a.max_len; i += kMoveThreads) to[i] = 0.f;
    if (kv == 0u && tid == 0u) a.lens_out[b] = static_cast<int32_t>(n);
    return;
  }
  const uint32_t x = blockIdx.x - 1u;
  const uint32_t part = x % a.parts, slice = x / a.parts % a.slices, plane = x / a.parts / a.slices;
  const uint32_t piece = slice * kSliceLanes + tid % kSliceLanes;
  const bool active = piece * 8u < c.dim;
  uint8_t* const pool = (plane == 0u ? c.k : c.v) + piece * 16u;
  const int32_t* from_pages = c.table + static_cast<size_t>(b) * c.table_stride;
  const int32_t* to_pages = a.to_table + static_cast<size_t>(b) * a.to_stride;
  const uint32_t first = tid / kSliceLanes;
  for (uint32_t i0 = part * kMoveRows; i0 < n; i0 += a.parts * kMoveRows) {
    if (a.in_place) {  // rows that stay where they are come before the first that moves
      const uint32_t last = min(i0 + kMoveRows, n) - 1u;
      if (kept[last] == static_cast<int32_t>(last)) continue;
    }
    uint4 v[kMoveDepth];
#pragma unroll
    for (uint32_t u = 0; u < kMoveDepth; ++u) {
      const uint32_t i = i0 + u * (kMoveThreads / kSliceLanes) + first;
      v[u] = make_uint4(0u, 0u, 0u, 0u);
      if (i < n && active) {
        const uint64_t at = paged_row(c, from_pages, static_cast<uint32_t>(kept[i]), kv);
        if (at != kNoRow) v[u] = *reinterpret_cast<const uint4*>(pool + at);
      }
    }
    if (a.in_place) __syncthreads();  // a chunk is read before it is written
#pragma unroll
    for (uint32_t u = 0; u < kMoveDepth; ++u) {
      const uint32_t i = i0 + u * (kMoveThreads / kSliceLanes) + first;
      if (i < n && active) {
        const uint64_t at = paged_row(c, to_pages, i, kv);
        if (at != kNoRow) *reinterpret_cast<uint4*>(pool + at) = v[u];
      }
    }
  }
}

cudaError_t select_smem_attr() {
  static std::mutex mu;
  static std::set<int> done;
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lock(mu);
  if (done.count(dev) != 0u) return cudaSuccess;
  const cudaError_t e =
      cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kCachedKeys * 4u);
  if (e == cudaSuccess) done.insert(dev);
  return e;
}

}  // namespace
}  // namespace qg

extern "C" cudaError_t qg_kv_evict(const qg_kv_pages* cache, const qg_evict* e, cudaStream_t stream) {
  using namespace qg;
  PagedView c;
  if (!paged_view(cache, &c) || e == nullptr) return cudaErrorInvalidValue;
  if (e->lens == nullptr || e->lens_out == nullptr || e->weight == nullptr || e->weight_out == nullptr ||
      e->kept == nullptr || e->max_len == 0u || e->max_len > 0x7fffffffu || e->weight_stride < e->max_len ||
      e->budget == 0u || e->budget > 0x7fffffffu ||
      static_cast<uint64_t>(e->sink) + e->recent > e->budget) {
    return cudaErrorInvalidValue;
  }
  const uint32_t most = std::min(std::min(e->budget, e->max_len), c.capacity);  // rows that can move
  const uint64_t room = static_cast<uint64_t>(e->new_table_pages) * cache->page_size;
  if (e->new_table != nullptr && (room < most || e->new_table_stride < e->new_table_pages)) {
    return cudaErrorInvalidValue;
  }
  EvictArgs a{};
  a.lens = e->lens;
  a.lens_out = e->lens_out;
  a.weight = e->weight;
  a.weight_out = e->weight_out;
  a.kept = e->kept;
  a.in_place = e->new_table == nullptr;
  a.to_table = a.in_place ? c.table : e->new_table;
  a.to_stride = a.in_place ? c.table_stride : e->new_table_stride;
  a.max_len = e->max_len;
  a.weight_stride = e->weight_stride;
  a.budget = e->budget;
  a.sink = e->sink;
  a.recent = e->recent;
  a.slices = (c.dim + kSliceLanes * 8u - 1u) / (kSliceLanes * 8u);
  a.parts = a.in_place ? 1u : (most + kMoveRows - 1u) / kMoveRows;
  cudaError_t err = select_smem_attr();
  if (err != cudaSuccess) return err;
  const bool cached = e->max_len <= kCachedKeys;
  err = launch_k(evict_select_kernel, dim3(c.n_kv, c.batch), kSelectThreads, cached ? e->max_len * 4u : 0u,
                 stream, c, a, cached);
  if (err != cudaSuccess) return err;
  return launch_k(evict_move_kernel, dim3(1u + 2u * a.slices * a.parts, c.n_kv, c.batch), kMoveThreads, 0,
                  stream, c, a);
}

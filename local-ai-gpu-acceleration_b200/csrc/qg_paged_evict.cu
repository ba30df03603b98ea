// qg_paged_evict.cu -- qg_kv_evict: sequences of a paged key-value cache cut back to a budget
// of slots by the attention weight that their slots received (declared in
// include/qgemv_b200.h).  Two launches:
//
//  * evict_select_kernel, one CTA per (kv head, sequence): the budget-th largest key by radix
//    selection (11 + 11 + 10 bits of an order-preserving integer image of the weights, the
//    slots that always stay above every weight; histograms in shared memory), then the kept
//    slots in ascending order: every warp counts its stretch of the slots, one scan over the
//    warps, every warp writes its stretch.  Keys equal to the threshold are taken from the
//    lowest slot on.  After the first pass the keys of the threshold's bin, where they fit,
//    are listed and the other passes read the list alone.  Bound by instruction issue (one
//    SM works for each (head, sequence)), so a lane takes 4 slots at a time.
//  * evict_move_kernel: rows kept[i] -> i, K and V of a row with one look-up; a lane looks up
//    one row's places and the warp moves 32 rows through them.  In place a CTA walks i
//    upwards and reads a chunk of rows before it writes it: kept[] ascends and
//    kept[i] >= i, so no row is overwritten that is still to be read.  A row's columns are
//    independent, so 64-byte column slices walk side by side.  Into other pages there is no
//    such order: whole rows, split over CTAs.  Bound by memory: the kept rows once in and
//    once out.
#include <algorithm>

#include <mutex>
#include <set>

#include "qg_paged.cuh"

namespace qg {
namespace {

constexpr uint32_t kSelectThreads = 1024;
constexpr uint32_t kSelectWarps = kSelectThreads / 32;
constexpr uint32_t kBins = 2048;
constexpr uint32_t kListed = 4096;             // keys of one bin that fit the list
constexpr uint32_t kCachedKeys = 48u * 1024u;  // slots whose keys fit in shared memory (192 KB)
constexpr uint32_t kStays = 0xffffffffu;       // key of a slot that always stays

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
  bool same_pages;
};

// An integer that orders like the weight: NaN lowest, -0 equal to +0.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (isnan(w)) return 0u;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) != 0u ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(const PagedView c, const EvictArgs a,
                                                                      bool cached) {
  extern __shared__ uint4 keys4[];  // cached: the keys of all slots, then zeros to a multiple of 4
  __shared__ uint32_t bins[kBins], list[kListed];
  __shared__ uint32_t warp_a[kSelectWarps], warp_b[kSelectWarps];
  __shared__ uint32_t found_bin, found_left, found_count, listed;
  const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  const uint32_t kv = blockIdx.x, b = blockIdx.y;
  uint32_t* const keys = reinterpret_cast<uint32_t*>(keys4);
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
  auto slot_key = [&](uint32_t i) { return i < lo || i >= hi ? kStays : weight_key(w[i]); };
  if (tid == 0u) listed = 0u;

  // One histogram step: a warp's keys that count go to bins[]; the first one's bin in one
  // addition, so weights that are all alike do not queue up.
  auto count_keys = [&](uint32_t bin, bool counts) {
    const uint32_t live = __ballot_sync(0xffffffffu, counts);
    if (live == 0u) return;
    const uint32_t lead = __ffs(live) - 1u;
    const uint32_t lead_bin = __shfl_sync(0xffffffffu, bin, lead);
    const uint32_t same = __ballot_sync(0xffffffffu, counts && bin == lead_bin);
    if (lane == lead) {
      atomicAdd(&bins[bin], static_cast<uint32_t>(__popc(same)));
    } else if (counts && bin != lead_bin) {
      atomicAdd(&bins[bin], 1u);
    }
  };
  uint32_t left = a.budget;  // of the keys that match the prefix, how many stay
  // The bin of the left-th largest counted key, with how many of its keys stay.
  auto find_bin = [&]() {
    __syncthreads();
    // thread t holds bins 2 t and 2 t + 1; upto: keys in them and in higher bins
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
      found_bin = 2u * tid + 1u, found_left = left - above1, found_count = b1;
    } else if (above0 < left && left <= above0 + b0) {
      found_bin = 2u * tid, found_left = left - above0, found_count = b0;
    }
    __syncthreads();
    left = found_left;
  };
  auto clear_bins = [&]() {
    __syncthreads();
    for (uint32_t i = tid; i < kBins; i += kSelectThreads) bins[i] = 0u;
    __syncthreads();
  };

  // ---- the threshold: bits 31-21 over all slots, then 20-10 and 9-0 over those that match
  clear_bins();
  for (uint32_t i0 = 0; i0 < n; i0 += 4u * kSelectThreads) {
    uint32_t key[4];
#pragma unroll
    for (uint32_t u = 0; u < 4u; ++u) {
      const uint32_t i = i0 + u * kSelectThreads + tid;
      key[u] = i < n ? slot_key(i) : 0u;
    }
#pragma unroll
    for (uint32_t u = 0; u < 4u; ++u) {
      const uint32_t i = i0 + u * kSelectThreads + tid;
      if (cached && i < ((n + 3u) & ~3u)) keys[i] = key[u];
      count_keys(key[u] >> 21, i < n);
    }
  }
  find_bin();
  uint32_t threshold = found_bin << 21;
  const bool short_list = found_count <= kListed;
  // four slots' keys from slot i (a multiple of 4); slots past n are 0 and never asked for
  auto four_keys = [&](uint32_t i) {
    if (cached) return keys4[i / 4u];
    uint4 k;
    k.x = i < n ? slot_key(i) : 0u;
    k.y = i + 1u < n ? slot_key(i + 1u) : 0u;
    k.z = i + 2u < n ? slot_key(i + 2u) : 0u;
    k.w = i + 3u < n ? slot_key(i + 3u) : 0u;
    return k;
  };
  if (short_list) {
    for (uint32_t i = 4u * tid; i < n; i += 4u * kSelectThreads) {
      const uint4 k = four_keys(i);
      const uint32_t key[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
      for (uint32_t u = 0; u < 4u; ++u) {
        if (i + u < n && key[u] >> 21 == found_bin) list[atomicAdd(&listed, 1u)] = key[u];
      }
    }
  }
#pragma unroll
  for (uint32_t pass = 0; pass < 2u; ++pass) {
    const uint32_t shift = pass == 0u ? 10u : 0u, width = pass == 0u ? 2048u : 1024u;
    const uint32_t above = pass == 0u ? 21u : 10u;  // bits from here on are settled
    clear_bins();
    const uint32_t m = short_list ? listed : n;
    for (uint32_t i0 = 0; i0 < m; i0 += kSelectThreads) {
      const uint32_t i = i0 + tid;
      const uint32_t key = i >= m ? 0u : short_list ? list[i] : cached ? keys[i] : slot_key(i);
      count_keys((key >> shift) & (width - 1u), i < m && (key ^ threshold) >> above == 0u);
    }
    find_bin();
    threshold |= found_bin << shift;
  }

  // ---- the kept slots in ascending order: larger keys, and the first `left` equal ones
  const uint32_t per = ((n + kSelectWarps - 1u) / kSelectWarps + 127u) & ~127u;
  const uint32_t from = min(warp * per, n), to = min(from + per, n);
  uint32_t more = 0, ties = 0;
  for (uint32_t i = from + 4u * lane; i < to; i += 128u) {
    const uint4 k = four_keys(i);
    const uint32_t key[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
    for (uint32_t u = 0; u < 4u; ++u) {
      more += i + u < n && key[u] > threshold;
      ties += i + u < n && key[u] == threshold;
    }
  }
  more = __reduce_add_sync(0xffffffffu, more);
  ties = __reduce_add_sync(0xffffffffu, ties);
  __syncthreads();
  if (lane == 0u) warp_a[warp] = more, warp_b[warp] = ties;
  __syncthreads();
  more = ties = 0;
  for (uint32_t x = 0; x < warp; ++x) {
    more += warp_a[x];
    ties += warp_b[x];
  }
  for (uint32_t i0 = from; i0 < to; i0 += 128u) {
    const uint32_t i = i0 + 4u * lane;
    const uint4 k = i < to ? four_keys(i) : make_uint4(0u, 0u, 0u, 0u);
    const uint32_t key[4] = {k.x, k.y, k.z, k.w};
    uint32_t mine = 0;  // larger keys in the low half, equal ones in the high half
#pragma unroll
    for (uint32_t u = 0; u < 4u; ++u) {
      if (i + u < to) mine += key[u] > threshold ? 1u : key[u] == threshold ? 0x10000u : 0u;
    }
    uint32_t before = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const uint32_t o = __shfl_up_sync(0xffffffffu, before, off);
      if (lane >= static_cast<uint32_t>(off)) before += o;
    }
    const uint32_t all = __shfl_sync(0xffffffffu, before, 31);
    before -= mine;
    uint32_t m = more + (before & 0xffffu), t = ties + (before >> 16);
#pragma unroll
    for (uint32_t u = 0; u < 4u; ++u) {
      if (i + u >= to) break;
      if (key[u] > threshold) {
        kept[m + min(t, left)] = static_cast<int32_t>(i + u);
        ++m;
      } else if (key[u] == threshold) {
        if (t < left) kept[m + t] = static_cast<int32_t>(i + u);
        ++t;
      }
    }
    more += all & 0xffffu;
    ties += all >> 16;
  }
}

constexpr uint32_t kMoveThreads = 256;
constexpr uint32_t kMoveDepth = 4;               // rows in flight per lane, K and V
constexpr uint32_t kSliceLanes = 4;              // 16-byte pieces of an ordered walk's column slice
constexpr uint32_t kMoveRows = kMoveThreads;     // rows of a chunk: 32 a warp

__device__ __forceinline__ uint64_t shfl64(uint64_t v, uint32_t from) {
  return __shfl_sync(0xffffffffu, v, from);
}

// ORDERED: one CTA walks all rows of a column slice of LANES pieces, a chunk at a time.
// Otherwise LANES lanes hold a whole row and blockIdx.x is the chunk.
template <bool ORDERED, int LANES>
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const PagedView c, const EvictArgs a) {
  static_assert(!ORDERED || LANES == kMoveDepth, "an ordered chunk is read whole before it is written");
  const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  const uint32_t kv = blockIdx.y, b = blockIdx.z;
  const uint32_t part = ORDERED ? 0u : blockIdx.x, slice = ORDERED ? blockIdx.x : 0u;
  pdl_wait();
  pdl_trigger();
  // lens may be lens_out: the old and the new length give the same count
  const uint32_t n = min(paged_len(a.lens[b], min(a.max_len, c.capacity)), a.budget);
  const size_t line = static_cast<size_t>(b) * c.n_kv + kv;
  const int32_t* kept = a.kept + line * a.budget;
  const float* weight = a.weight + line * a.weight_stride;
  float* weight_out = a.weight_out + line * a.weight_stride;
  const int32_t* from_pages = c.table + static_cast<size_t>(b) * c.table_stride;
  const int32_t* to_pages = a.to_table + static_cast<size_t>(b) * a.to_stride;
  const uint32_t piece = slice * LANES + lane % LANES;
  const bool active = piece * 8u < c.dim;
  const uint32_t chunk_step = ORDERED ? kMoveRows : a.parts * kMoveRows;

  uint32_t c0 = part * kMoveRows;
  if (ORDERED && a.same_pages && a.weight_out == a.weight) {
    // rows that stay where they are come before the first that moves
    while (c0 + kMoveRows <= n && kept[c0 + kMoveRows - 1u] == static_cast<int32_t>(c0 + kMoveRows - 1u)) {
      c0 += kMoveRows;
    }
  }
  // this lane's row of a chunk: where from, where to, its weight
  uint64_t src = kNoRow, dst = kNoRow;
  float w = 0.f;
  auto look_up = [&](uint32_t at) {
    const uint32_t i = at + warp * 32u + lane;
    src = dst = kNoRow;
    if (i < n) {
      const uint32_t k = static_cast<uint32_t>(kept[i]);
      if (slice == 0u) w = weight[k];
      src = paged_row(c, from_pages, k, kv);
      dst = paged_row(c, to_pages, i, kv);
    }
  };
  look_up(c0);
  for (; c0 < n; c0 += chunk_step) {
    const uint32_t i = c0 + warp * 32u + lane;
#pragma unroll
    for (uint32_t g = 0; g < LANES; g += kMoveDepth) {
      uint4 k[kMoveDepth], v[kMoveDepth];
      uint64_t to[kMoveDepth];
#pragma unroll
      for (uint32_t u = 0; u < kMoveDepth; ++u) {
        const uint32_t r = (g + u) * (32u / LANES) + lane / LANES;
        const uint64_t at = shfl64(src, r);
        to[u] = shfl64(dst, r);
        k[u] = v[u] = make_uint4(0u, 0u, 0u, 0u);
        if (at != kNoRow && active) {
          k[u] = *reinterpret_cast<const uint4*>(c.k + at + piece * 16u);
          v[u] = *reinterpret_cast<const uint4*>(c.v + at + piece * 16u);
        }
      }
      if (ORDERED) {
        const float w_now = w;
        look_up(c0 + chunk_step);  // rows further up: nothing that this chunk writes
        __syncthreads();           // a chunk is read before it is written
        if (slice == 0u && i < n) weight_out[i] = w_now;
      } else if (g == 0u && i < n) {
        weight_out[i] = w;
      }
#pragma unroll
      for (uint32_t u = 0; u < kMoveDepth; ++u) {
        if (to[u] != kNoRow && active) {
          *reinterpret_cast<uint4*>(c.k + to[u] + piece * 16u) = k[u];
          *reinterpret_cast<uint4*>(c.v + to[u] + piece * 16u) = v[u];
        }
      }
    }
    if (!ORDERED && c0 + chunk_step < n) look_up(c0 + chunk_step);
  }
  if (slice == 0u) {
    // the tail of the weights; in an ordered walk its old values have all been read
    for (uint32_t i = n + part * kMoveThreads + tid; i < a.max_len; i += (ORDERED ? 1u : a.parts) * kMoveThreads) {
      weight_out[i] = 0.f;
    }
    if (part == 0u && kv == 0u && tid == 0u) a.lens_out[b] = static_cast<int32_t>(n);
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
  a.same_pages = e->new_table == nullptr;
  a.to_table = a.same_pages ? c.table : e->new_table;
  a.to_stride = a.same_pages ? c.table_stride : e->new_table_stride;
  a.max_len = e->max_len;
  a.weight_stride = e->weight_stride;
  a.budget = e->budget;
  a.sink = e->sink;
  a.recent = e->recent;
  // rows or weights that move where they are have to move in order
  const bool ordered = a.same_pages || e->weight_out == e->weight;
  a.slices = ordered ? (c.dim + kSliceLanes * 8u - 1u) / (kSliceLanes * 8u) : 1u;
  a.parts = ordered ? 1u : (most + kMoveRows - 1u) / kMoveRows;
  cudaError_t err = select_smem_attr();
  if (err != cudaSuccess) return err;
  const bool cached = e->max_len <= kCachedKeys;
  err = launch_k(evict_select_kernel, dim3(c.n_kv, c.batch), kSelectThreads,
                 cached ? (e->max_len + 3u) / 4u * 16u : 0u, stream, c, a, cached);
  if (err != cudaSuccess) return err;
  const dim3 grid(a.slices * a.parts, c.n_kv, c.batch);
  if (ordered) return launch_k(evict_move_kernel<true, kSliceLanes>, grid, kMoveThreads, 0, stream, c, a);
  if (c.dim <= 64u) return launch_k(evict_move_kernel<false, 8>, grid, kMoveThreads, 0, stream, c, a);
  if (c.dim <= 128u) return launch_k(evict_move_kernel<false, 16>, grid, kMoveThreads, 0, stream, c, a);
  return launch_k(evict_move_kernel<false, 32>, grid, kMoveThreads, 0, stream, c, a);
}

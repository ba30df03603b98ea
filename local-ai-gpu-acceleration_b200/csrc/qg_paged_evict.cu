// qg_paged_evict.cu -- qg_kv_evict: sequences of a paged key-value cache cut back to a budget
// of slots by the attention weight that their slots received (declared in
// include/qgemv_b200.h).  Two launches:
//
//  * evict_select_kernel, a cluster of 1 to 8 CTAs per (kv head, sequence), each with a
//    stretch of the slots: the budget-th largest key by radix selection (11 + 11 + 10 bits of
//    an order-preserving integer image of the weights, the slots that always stay above every
//    weight; histograms in shared memory, added over the cluster through distributed shared
//    memory), then the kept slots in ascending order: every warp counts its stretch, one scan
//    over the warps and CTAs, every warp writes its stretch.  Keys equal to the threshold are
//    taken from the lowest slot on.  Bound by instruction issue: some 100 instructions a warp
//    for each 32 slots, which is why the cluster grows while SMs are free.
//  * evict_move_kernel: rows kept[i] -> i, K and V of a row with one look-up; a lane looks up
//    one row's places and the warp moves 32 rows through them.  In place a CTA walks i
//    upwards and reads a chunk of rows before it writes it: kept[] ascends and
//    kept[i] >= i, so no row is overwritten that is still to be read.  A row's columns are
//    independent, so 64-byte column slices walk side by side.  Into other pages there is no
//    such order: whole rows, split over CTAs.  Bound by memory: the kept rows once in and
//    once out.
//
// Measured (B200, time on the GPU, floor = weights in, kept rows in and out at 6.46 TB/s), into
// other pages and in place:
// 8 x 32768 slots to 8192, 8 heads x 128 fp16: 113 and 147 us (floor 86; selection 22, move 90);
// 16 x 700..9001 to 1500, 8 heads x 80 bf16: 42 and 43 us (18; selection 18, latency of its 12
// barriers); 1 x 2500 to 2048: 12.5 and 21 us; 1 x 131072 to 65536, 8 heads x 128: 119 and 506 us
// (85): in place it is 32 CTAs, one for each head and 64-byte slice, whatever the length.
#include <cooperative_groups.h>

#include <algorithm>

#include "qg_paged.cuh"

namespace qg {
namespace {

// Threads of a selecting CTA: few for short sequences, so that four CTAs share an SM and a
// barrier waits for 8 warps; the rule is in qg_kv_evict.
constexpr uint32_t kManyThreads = 1024, kFewThreads = 256;
constexpr uint32_t kShort = 1024;              // slots: below this a sequence is short
constexpr uint32_t kBins = 2048;
constexpr uint32_t kCachedKeys = 48u * 1024u;  // keys that fit in a CTA's shared memory (192 KB)
constexpr uint32_t kMaxCluster = 8;            // CTAs of a cluster on every device
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
  const uint32_t u = __float_as_uint(w + 0.f);
  const uint32_t key = u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
  return isnan(w) ? 0u : key;
}
constexpr uint32_t kZeroKey = 0x80000000u;     // of weight 0, the one that many slots share

// blockIdx.x: rank in the cluster.  A CTA's stretch is a multiple of 32 slots a warp.
__host__ __device__ constexpr uint32_t stretch(uint32_t n, uint32_t ctas, uint32_t threads) {
  return ((n + ctas - 1u) / ctas + threads - 1u) / threads * threads;
}

template <uint32_t kSelectThreads>
__global__ void __launch_bounds__(kSelectThreads, kManyThreads / kSelectThreads)
    evict_select_kernel(const PagedView c, const EvictArgs a, bool cached) {
  constexpr uint32_t kSelectWarps = kSelectThreads / 32, kMine = kBins / kSelectThreads;
  extern __shared__ uint32_t keys[];  // cached: the keys of this CTA's stretch
  __shared__ uint32_t bins[kBins];
  __shared__ uint32_t warp_a[kSelectWarps], warp_b[kSelectWarps];
  __shared__ uint32_t found_bin, found_left, totals[2];
  auto cluster = cooperative_groups::this_cluster();
  const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  const uint32_t kv = blockIdx.y, b = blockIdx.z, rank = blockIdx.x, ctas = gridDim.x;
  auto sync_all = [&]() {
    if (ctas == 1u) {
      __syncthreads();
    } else {
      cluster.sync();
    }
  };
  pdl_wait();
  pdl_trigger();
  const uint32_t n = paged_len(a.lens[b], min(a.max_len, c.capacity));
  const float* w = a.weight + (static_cast<size_t>(b) * c.n_kv + kv) * a.weight_stride;
  int32_t* kept = a.kept + (static_cast<size_t>(b) * c.n_kv + kv) * a.budget;
  if (n <= a.budget) {
    for (uint32_t i = rank * kSelectThreads + tid; i < a.budget; i += ctas * kSelectThreads) {
      kept[i] = i < n ? static_cast<int32_t>(i) : -1;
    }
    return;
  }
  const uint32_t lo = a.sink, hi = n - a.recent;  // the slots that are chosen from
  const uint32_t share = stretch(n, ctas, kSelectThreads);
  const uint32_t s0 = min(rank * share, n), s1 = min(s0 + share, n);
  auto slot_key = [&](uint32_t i) { return i < lo || i >= hi ? kStays : weight_key(w[i]); };
  auto key_at = [&](uint32_t i) { return cached ? keys[i - s0] : slot_key(i); };

  // Histograms count one key at a time, but for slots that never had weight: those are
  // counted in a register and added once a warp, so they do not queue up at one bin.
  uint32_t zeros = 0;
  auto count_key = [&](uint32_t key, uint32_t bin) {
    if (key == kZeroKey) {
      ++zeros;
    } else {
      atomicAdd(&bins[bin], 1u);
    }
  };
  uint32_t left = a.budget;  // of the keys that match the prefix, how many stay
  // Adds the warps' zeros, then finds the bin of the left-th largest key that was counted.
  auto find_bin = [&](uint32_t zero_bin) {
    zeros = __reduce_add_sync(0xffffffffu, zeros);
    if (lane == 0u && zeros != 0u) atomicAdd(&bins[zero_bin], zeros);
    zeros = 0u;
    sync_all();
    // thread t holds bins kMine t and on; upto: keys in them and in higher bins
    uint32_t bin[kMine] = {};
    for (uint32_t r = 0; r < ctas; ++r) {
      const uint32_t* of = ctas == 1u ? bins : cluster.map_shared_rank(bins, r);
#pragma unroll
      for (uint32_t i = 0; i < kMine; i += 2u) {
        const uint2 x = *reinterpret_cast<const uint2*>(of + kMine * tid + i);
        bin[i] += x.x;
        bin[i + 1u] += x.y;
      }
    }
    uint32_t upto = 0;
#pragma unroll
    for (uint32_t i = 0; i < kMine; ++i) upto += bin[i];
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const uint32_t o = __shfl_down_sync(0xffffffffu, upto, off);
      if (lane + off < 32u) upto += o;
    }
    if (lane == 0u) warp_a[warp] = upto;
    __syncthreads();
    upto += __reduce_add_sync(0xffffffffu, lane > warp && lane < kSelectWarps ? warp_a[lane] : 0u);
#pragma unroll
    for (uint32_t i = 0; i < kMine; ++i) {
      const uint32_t above = upto - bin[i];  // keys in higher bins
      if (above < left && left <= upto) found_bin = kMine * tid + i, found_left = left - above;
      if (i + 1u < kMine) upto = upto - bin[i];
    }
    sync_all();  // every CTA has read the bins
    left = found_left;
  };
  auto clear_bins = [&]() {
#pragma unroll
    for (uint32_t i = 0; i < kMine; ++i) bins[i * kSelectThreads + tid] = 0u;
    __syncthreads();
  };

  // ---- the threshold: bits 31-21 over all slots, then 20-10 and 9-0 over those that match
  clear_bins();
  constexpr uint32_t kAhead = 8;  // weights in flight per thread
  for (uint32_t i0 = s0; i0 < s1; i0 += kAhead * kSelectThreads) {
    uint32_t key[kAhead];
#pragma unroll
    for (uint32_t u = 0; u < kAhead; ++u) {
      const uint32_t i = i0 + u * kSelectThreads + tid;
      if (i < s1) key[u] = slot_key(i);
    }
#pragma unroll
    for (uint32_t u = 0; u < kAhead; ++u) {
      const uint32_t i = i0 + u * kSelectThreads + tid;
      if (i < s1) {
        if (cached) keys[i - s0] = key[u];
        count_key(key[u], key[u] >> 21);
      }
    }
  }
  find_bin(kZeroKey >> 21);
  uint32_t threshold = found_bin << 21;
#pragma unroll
  for (uint32_t pass = 0; pass < 2u; ++pass) {
    const uint32_t shift = pass == 0u ? 10u : 0u, width = pass == 0u ? 2048u : 1024u;
    const uint32_t settled = pass == 0u ? 21u : 10u;  // bits from here on match
    clear_bins();
    for (uint32_t i = s0 + tid; i < s1; i += kSelectThreads) {
      const uint32_t key = key_at(i);
      if ((key ^ threshold) >> settled == 0u) count_key(key, (key >> shift) & (width - 1u));
    }
    find_bin((kZeroKey >> shift) & (width - 1u));
    threshold |= found_bin << shift;
  }

  // ---- the kept slots in ascending order: larger keys, and the first `left` equal ones
  const uint32_t per = share / kSelectWarps;
  const uint32_t from = min(s0 + warp * per, s1), to = min(from + per, s1);
  uint32_t more = 0, ties = 0;
  for (uint32_t i = from + lane; i < to; i += 32u) {
    const uint32_t key = key_at(i);
    more += key > threshold;
    ties += key == threshold;
  }
  more = __reduce_add_sync(0xffffffffu, more);
  ties = __reduce_add_sync(0xffffffffu, ties);
  if (lane == 0u) warp_a[warp] = more, warp_b[warp] = ties;
  __syncthreads();
  const uint32_t in_a = lane < kSelectWarps ? warp_a[lane] : 0u, in_b = lane < kSelectWarps ? warp_b[lane] : 0u;
  if (warp == 0u) {
    const uint32_t all_a = __reduce_add_sync(0xffffffffu, in_a), all_b = __reduce_add_sync(0xffffffffu, in_b);
    if (lane == 0u) totals[0] = all_a, totals[1] = all_b;
  }
  more = __reduce_add_sync(0xffffffffu, lane < warp ? in_a : 0u);
  ties = __reduce_add_sync(0xffffffffu, lane < warp ? in_b : 0u);
  sync_all();
  for (uint32_t r = 0; r < rank; ++r) {
    const uint32_t* t = cluster.map_shared_rank(totals, r);
    more += t[0];
    ties += t[1];
  }
  const uint32_t below = (1u << lane) - 1u;
  for (uint32_t i0 = from; i0 < to; i0 += 32u) {
    const uint32_t i = i0 + lane;
    const uint32_t key = i < to ? key_at(i) : 0u;
    const uint32_t mb = __ballot_sync(0xffffffffu, i < to && key > threshold);
    const uint32_t tb = __ballot_sync(0xffffffffu, i < to && key == threshold);
    const uint32_t m = more + __popc(mb & below), t = ties + __popc(tb & below);
    const bool stays = ((mb | (t < left ? tb : 0u)) >> lane & 1u) != 0u;
    if (stays) kept[m + min(t, left)] = static_cast<int32_t>(i);
    more += __popc(mb);
    ties += __popc(tb);
  }
  sync_all();  // no CTA leaves while another may read its totals
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
__global__ void __launch_bounds__(kMoveThreads, 3) evict_move_kernel(const PagedView c, const EvictArgs a) {
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
  static SmemAttr select_attr;
  cudaError_t err =
      select_attr.set(reinterpret_cast<const void*>(evict_select_kernel<kManyThreads>), kCachedKeys * 4u);
  if (err != cudaSuccess) return err;
  const uint64_t lines = static_cast<uint64_t>(c.n_kv) * c.batch, sms = static_cast<uint64_t>(paged_sm_count());
  // The lengths are on the device, so max_len stands for them.  Few threads for short lines, and up
  // to twice that where the lines do not fit on the SMs at once.  Whole call with 1024 and 256
  // threads, max_len the longest length, head size 128 (112 in the first), us: 37 x 26..45
  // slots of 16 heads 27.8 and 11.7, of 8 heads: 16 x 1000 20.7 and 15.4, 64 x 2048 75.2 and 61.1,
  // 1 x 1000 11.5 and 11.8.  Past the rule: 1 x 2000 12.5 and 17.0, 20 x 3096..4096 35 and 39,
  // 40 x 100..8000 44 and 61; only where all are long and many it would gain (64 x 4096 82 and 70).
  // A max_len far above the lengths costs the form for long lines and their tail of zeros: in
  // place with 131072 in the place of the longest, 64 x 576 to 512 130 us (59), 1 x 2500 37 (21).
  const bool few = e->max_len < kShort || (e->max_len <= 2u * kShort && lines > sms);
  const uint32_t threads = few ? kFewThreads : kManyThreads;
  // CTAs of a selection: while SMs are free and a stretch keeps two slots a thread
  uint32_t ctas = 1;
  while (ctas < kMaxCluster && lines * ctas * 2u <= sms && e->max_len >= ctas * 2u * 2u * threads) ctas *= 2u;
  const uint32_t slots = stretch(e->max_len, ctas, threads);
  const bool cached = slots <= kCachedKeys;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas, c.n_kv, c.batch);
  cfg.blockDim = threads;
  cfg.dynamicSmemBytes = cached ? slots * 4u : 0u;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  err = few ? cudaLaunchKernelEx(&cfg, evict_select_kernel<kFewThreads>, c, a, cached)
            : cudaLaunchKernelEx(&cfg, evict_select_kernel<kManyThreads>, c, a, cached);
  if (err != cudaSuccess) return err;
  const dim3 grid(a.slices * a.parts, c.n_kv, c.batch);
  if (ordered) return launch_k(evict_move_kernel<true, kSliceLanes>, grid, kMoveThreads, 0, stream, c, a);
  if (c.dim <= 64u) return launch_k(evict_move_kernel<false, 8>, grid, kMoveThreads, 0, stream, c, a);
  if (c.dim <= 128u) return launch_k(evict_move_kernel<false, 16>, grid, kMoveThreads, 0, stream, c, a);
  return launch_k(evict_move_kernel<false, 32>, grid, kMoveThreads, 0, stream, c, a);
}

// qg_paged8_attn.cu -- qg_paged_attn8: attention of new tokens, one or many a sequence, over an
// 8-bit paged key-value cache (declared in include/qgemv_b200.h); this file holds the entry
// point, the list of tiles and the kernel for few rows and for fp32 queries.
//
// Mathematics.  One pass over a segment's slots, cut anywhere and joined by the softmax's rule, as
// in qg_paged_attn.cu.  With key codes c, scales ks and vs of a slot's block, in log2 units,
//   s = (q . c) * scale * ks * log2 e,  y = s + log2 vs,
// the probability that multiplies the value's codes is 2^(y - M), M the running maximum of y:
// the block's scale costs one addition a score and none a value.  The softmax's sum takes
// 2^(y - M) / vs, one multiplication for 16 slots: probabilities in fp16 are weighed by what they add
// to the row.  Two scales can lie 120 powers apart, and a slot of the smaller one weighs as much in the
// sum as one of the larger, so fp32 does not hold the sum's terms as they are: small powers of slots
// with small scales are raised (kRaise) for the sum, and a sum is scaled by the root of a factor, twice.
//
// Bound by memory for few rows: a slot's K and V codes are read once for all rows of a tile, and there
// is half as much of them as in 16 bits, so a byte carries twice the arithmetic.  Codes become fp16
// pairs in registers (exact, one cvt for two) on their way from shared memory to mma.sync: a code
// of every 4 bytes that ldmatrix gives a lane.  For K the four are dims 4 t .. 4 t + 3 of a slot; the
// products do not mind the order of dims, so the queries take the same one.  For V, transposed by
// ldmatrix as 16-bit pairs, they are two slots x two dims; one byte permutation makes them pairs
// of slots of even and of odd dims, and a lane's sums become four dims in a row.
//
// Work.  Segments, blocks of 256 slots (128 at head size 256), ranges of equal length for every CTA, four
// tiles of a block for the four warps, records and joins as in qg_paged_attn.cu; a tile's rows may be
// several tokens', with a mask for each where the tile touches the end of what any row sees.  A
// ragged call's tiles are listed by a small kernel before (one CTA; it costs 2 to 3 us), a call of one row
// a sequence counts them in every CTA.  Where segments are many and short every warp takes whole ones alone.
// A warp fetches its K and V tiles through its own ring, once a tile; places and scales of the next 32
// 16-slot steps are looked up a lane each, a set ahead, and wait in shared memory.
//
// Measured (B200, 6.56 TB/s for a plain copy; time on the GPU, floor = bytes that have to move at that rate):
// 16 x 32768 slots, 64/8 heads x 128: 179 us (floor 164); 1 x 131072: 56 us (41; 37 CTAs a head leave
// records that are joined at the end); 64 x ..4097, 16/16 heads x 64, window 2000, rows 1024 bytes apart:
// 85 us (34); 256 x 300, 32/8 heads: 50 us (25); 1 x 511: 12.6 us, all latency.  Two warps a scheduler (255 registers) issue in 40% of the
// cycles; the rest is the latency of their chains.
//
// Rows.  fp32 queries, and any in a call without offsets of at most 8 query heads a kv head or with offsets of
// at most 8 rows for a kv head in all: eight rows fill rows 0-7 of the A operand and their fp16 errors rows
// 8-15 (22 bits), probabilities alike.  Other calls with 16-bit queries: 16 rows whole, probabilities rounded
// to fp16 once (11 bits, the output's own precision).
#include <math_constants.h>

#include <algorithm>

#include "qg_mma.cuh"
#include "qg_paged8_attn.cuh"

namespace qg {
namespace {

constexpr uint32_t kWarps = 4;
constexpr uint32_t kAttnThreads = kWarps * 32;
// Slots of one warp's tile: as many as 255 registers hold.  At head size 128 tiles of 32 slots took 236 us for
// 16 x 32768, of 64 208: a tile's sums and bookkeeping cost the same whatever its slots.
constexpr uint32_t log_tile8(uint32_t dp, uint32_t rs, uint32_t terms) {
  return dp == 256u || (dp == 128u && rs * terms == 4u) ? 5u : 6u;
}
constexpr uint32_t kMaxCtas = 512;
constexpr uint32_t kJoinAll = 48;             // records of a tile that are joined at once
constexpr uint32_t kJoin = 16;                // records of a group where there are more
constexpr uint32_t kInFlight = 16;            // records whose sums are asked for together
constexpr uint32_t kEntries = 64;             // 16-slot steps whose places and scales a warp keeps
static_assert(2u * kMaxCtas * 4u <= QG_PAGED_ATTN_ZEROED, "two counters per CTA");
static_assert(kMaxCtas / kJoin <= 64u && kJoinAll <= 64u, "two records a lane");
constexpr float kShare = 14.f;                // log2 of the factor that fp16 probabilities carry
// exp2 gives zero below 2^-126.  Where a lane's four powers of a 16-slot step are all below 2^kRaiseBelow (zero in
// fp16 either way) and the step's value scale below 2^kLowScale, they are computed 2^kRaise times as large.  So what a
// sum loses has at most 2^(60 - kLowScale - 126) = 2^-42 of the heaviest slot's weight, or 2^-24 of that of one of
// the four, or, raised, 2^(120 - 126 - kRaise).  Without raising it was 2^-20 (kShare counted): 65520 such slots
// beside 16 of the largest scale came out 2^-8 too light.
constexpr float kLowScale = -24.f, kRaiseBelow = -102.f, kRaise = 64.f, kLower = 0x1p-64f;

struct AttnMaps8 {
  CUtensorMap k, v;
};

// The power p with top in [2^p, 2^(p + 1)), kept where both 2^p and 2^-p are normal numbers.
__device__ __forceinline__ int power_of8(float top) {
  return top == 0.f ? 0 : max(-126, min(126, static_cast<int>(__float_as_uint(top) >> 23) - 127));
}

// As mma() without `volatile`: the products of a tile may be put in any order, between the loads.
__device__ __forceinline__ void mma8(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// DP: head_dim rounded up to 64, 128 or 256.  RS: rows of a lane (8 RS rows a tile).  TERMS: fp16
// terms of a query and of a probability.
template <int DP, int RS, int TERMS>
struct Attn8Shape {
  static_assert(TERMS == 2 || RS == 2, "one term: 16 rows");
  static constexpr uint32_t kRows = 8u * RS;
  static constexpr uint32_t kLogTile = log_tile8(DP, RS, TERMS), kTile = 1u << kLogTile, kLogBlock = kLogTile + 2u;
  static constexpr uint32_t kUnit = kTile * DP;             // a warp's K or V tile
  static constexpr int kCtasPerSm = DP == 64 && RS == 1 ? 3 : 2;
  // K and V tiles of a warp's ring: V of the tile in work, K of the next one too, more where they fit
  static constexpr uint32_t kUnits = (kCtasPerSm == 3 ? 64u : 96u) * 1024u / (kWarps * kUnit);
  static constexpr uint32_t kK = kUnits >= 6u ? 4u : 2u, kV = kUnits >= 4u ? 2u : 1u;
  static constexpr uint32_t kSmem = kWarps * (kK + kV) * kUnit + 1024u;  // the ring starts on 1024 bytes
  static constexpr uint32_t kRowBytes = DP == 64 ? 64u : 128u;        // of a box
  static constexpr uint32_t kPanels = DP / kRowBytes;
  static constexpr uint32_t kRecord = kRows * (DP + 2u);    // m[], l[], o[][]
  // What a segment costs beside its blocks, in blocks; us with 0, 1, 2 and 4: head size 64, 100 x 10..2000 (16/16
  // heads) 66, 56, 55 and 61; 128, the same of 32/8 64, 55, 51 and 57, 2 x 30000 49, 45, 43 and 43; 256, 32 x
  // ..8191 (8/2) 43, 43, 37 and 37.
  static constexpr uint32_t kHeader = 2;
  static_assert(8u * DP * 4u <= kUnit, "the sums of eight rows join in a free unit");
};

template <int DP, int RS, int TERMS>
__global__ void __launch_bounds__(kAttnThreads, Attn8Shape<DP, RS, TERMS>::kCtasPerSm)
    paged_attn8_kernel(const Paged8View cache, const Attn8Args a, const __grid_constant__ AttnMaps8 maps) {
  using Shape = Attn8Shape<DP, RS, TERMS>;
  constexpr uint32_t kUnit = Shape::kUnit, kRows = Shape::kRows, kK = Shape::kK, kV = Shape::kV;
  constexpr uint32_t kLogTile = Shape::kLogTile, kTile = Shape::kTile, kLogBlock = Shape::kLogBlock;
  constexpr uint32_t kRowBytes = Shape::kRowBytes, kPanels = Shape::kPanels, kPanel = kTile * kRowBytes;
  constexpr uint32_t kPieces = kRowBytes / 16u;             // 16-byte pieces of a row of a panel
  constexpr int kMma = TERMS == 2 ? RS : 1;                 // products for a tile
  constexpr int kSteps = kTile / 16;                        // 16-slot steps
  constexpr uint32_t kChunks = DP / 16;                     // 16-dim chunks
  constexpr uint32_t kSet = 32u / kSteps;                   // tiles looked up together
  const PagedView& c = cache.c;
  extern __shared__ uint8_t smem_raw[];
  __shared__ float join_m[kWarps][kRows], join_l[kWarps][kRows];
  __shared__ __align__(8) uint64_t full_k[kWarps][kK], full_v[kWarps][kV];
  // of the steps of a warp's next tiles: {page, place, head}; key scale, log2 of the value scale, its reciprocal
  __shared__ int4 where[kWarps][kEntries];
  __shared__ __align__(16) float ks_of[kWarps][kEntries], lg_of[kWarps][kEntries], inv_of[kWarps][kEntries];
  __shared__ uint64_t sum64[kWarps];
  __shared__ uint32_t most_of[kWarps];
  __shared__ uint32_t first_at[3];
  __shared__ uint32_t is_last;
  __shared__ float share[kRows][64];

  const uint32_t tid = threadIdx.x, lane = tid & 31u, g = lane >> 2, t4 = lane & 3u;
  const uint32_t warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  uint8_t* const smem = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
  uint8_t* const ring = smem + warp * ((kK + kV) * kUnit);   // kK tiles of K, kV of V
  const uint32_t ring_at = smem_addr(ring);
  if (lane == 0u) {
    for (uint32_t i = 0; i < kK; ++i) mbar_init(&full_k[warp][i], 1u);
    for (uint32_t i = 0; i < kV; ++i) mbar_init(&full_v[warp][i], 1u);
    fence_mbar_init();
  }
  if (tid < 2u) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(tid == 0u ? &maps.k : &maps.v)) : "memory");
  }
  pdl_wait();
  pdl_trigger();

  const bool ragged = a.items != nullptr;
  const uint32_t lines = ragged ? c.n_kv : c.n_kv * a.tiles;  // segments of an item (a tile, a sequence)
  // the segment (s.item, s.line) in steps of 2^log slots; `fresh`: the item is another one than before
  auto make = [&](Segment8& s, bool fresh, uint32_t log) {
    if (ragged) {
      take_item8(a, s, fresh, log);
      return;
    }
    if (fresh) {
      s.b = s.token = s.item;
      s.p0 = static_cast<int32_t>(paged_len(a.lens[s.b], c.capacity)) - 1;
    }
    s.kv = s.line / a.tiles;
    s.sub = (s.line - s.kv * a.tiles) * kRows;
    s.rows = min(kRows, a.group.d - s.sub);
    s.bounds(a, log);
    s.j = 0u;
  };

  // ---- this CTA's range [r0, r1) of the line of units: the blocks of all segments, and headers
  // before each segment's; or, where segments are short and many, whole segments for every warp
  uint64_t total = 0, ctas = 0, r0 = 0, r1 = 0;
  uint32_t header = 0;
  bool solo = false;
  auto cut = [&](uint64_t blocks, uint64_t segments, uint32_t most) {  // false where nothing is left for this CTA
    // Time in 1500 cycles: a tile (a block of a CTA) takes 3, a segment 4 in a warp and 5 in a CTA.  With every
    // segment taken for the longest, a segment a warp has to be the faster way.
    const uint64_t busy = min(static_cast<uint64_t>(gridDim.x), blocks);
    const uint64_t rounds = (segments + gridDim.x * kWarps - 1u) / (gridDim.x * kWarps);
    solo = rounds * (most * 3ull + 4u) * busy <= blocks * 3u + segments * 5u;
    if (solo) return true;
    // fewer blocks than CTAs: a block each; otherwise segments cost more than their blocks
    if (blocks > gridDim.x) header = Shape::kHeader;
    total = blocks + header * segments;
    ctas = min(static_cast<uint64_t>(gridDim.x), total);
    if (blockIdx.x >= ctas) return false;
    r0 = blockIdx.x * total / ctas;
    r1 = (blockIdx.x + 1u) * total / ctas;
    return true;
  };
  Segment8 use;
  uint32_t in_segment = 0, segments = 0;  // units of the first segment before the range
  if (ragged) {
    const uint32_t n = a.item_count[0];
    if (n == 0u) return;
    segments = n * lines;
    if (!cut(a.item_blocks[n] * lines, segments, a.item_count[1])) return;
    if (!solo) find_unit8(a, n, lines, header, r0, use.item, use.line, in_segment);
  } else {
    uint32_t most = 0;
    auto blocks_of = [&](uint32_t b) {
      Segment8 s;
      s.item = b;
      s.line = 0u;
      make(s, true, kLogTile);
      most = max(most, s.j1);
      s.bounds(a, kLogBlock);
      return s.j1;
    };
    uint64_t blocks = 0;  // of one line of every sequence
    for (uint32_t b = tid; b < a.tokens; b += kAttnThreads) blocks += blocks_of(b);
    const uint64_t mine = blocks;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) blocks += __shfl_xor_sync(0xffffffffu, blocks, off);
    most = __reduce_max_sync(0xffffffffu, most);
    if (lane == 0u) sum64[warp] = blocks, most_of[warp] = most;
    __syncthreads();
    blocks = 0;
#pragma unroll
    for (uint32_t w = 0; w < kWarps; ++w) {
      blocks += sum64[w];
      most = max(most, most_of[w]);
    }
    segments = a.tokens * lines;
    if (!cut(blocks * lines, segments, most)) return;
    for (uint64_t base = 0, b0 = 0; !solo && b0 < a.tokens; b0 += kAttnThreads) {
      const uint32_t b = static_cast<uint32_t>(b0) + tid;
      const uint64_t n = b < a.tokens ? (a.tokens <= kAttnThreads ? mine : blocks_of(b)) : 0u;
      uint64_t upto = n;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const uint64_t o = __shfl_up_sync(0xffffffffu, upto, off);
        if (lane >= static_cast<uint32_t>(off)) upto += o;
      }
      __syncthreads();
      if (lane == 31u) sum64[warp] = upto;
      __syncthreads();
      uint64_t all = 0;
#pragma unroll
      for (uint32_t w = 0; w < kWarps; ++w) {
        if (w < warp) upto += sum64[w];
        all += sum64[w];
      }
      const uint64_t units = n + header;
      upto += base + static_cast<uint64_t>(header) * (b + 1u);
      if (n != 0u && r0 >= (upto - units) * lines && r0 < upto * lines) {
        const uint64_t in = r0 - (upto - units) * lines;
        first_at[0] = b;
        first_at[1] = static_cast<uint32_t>(in / units);
        first_at[2] = static_cast<uint32_t>(in % units);
      }
      base += all;
      if ((base + static_cast<uint64_t>(header) * (b0 + kAttnThreads)) * lines > r0) break;
    }
    __syncthreads();
    if (!solo) {
      use.item = first_at[0];
      use.line = first_at[1];
      in_segment = first_at[2];
    }
  }
  const uint32_t log_step = solo ? kLogTile : kLogBlock, warp_slot = solo ? 0u : warp * kTile;
  uint32_t left;  // units of the range, or steps of the segment, from use.j on (below 2^31)
  uint32_t index = warp * gridDim.x + blockIdx.x;  // of a lone warp's segment
  auto skip_header = [&](uint32_t& units, uint32_t done) { units -= min(units, header - min(done, header)); };
  // segment `at` of the line for a lone warp
  auto take = [&](Segment8& s, uint32_t at, uint32_t& units) {
    units = 0u;
    if (at >= segments) return;
    s.item = at / lines;
    s.line = at - s.item * lines;
    make(s, true, kLogTile);
    units = s.j1;
  };
  // the segment after one that is done
  auto advance = [&](Segment8& s, uint32_t& at, uint32_t& units) {
    if (solo) {
      at += gridDim.x * kWarps;
      take(s, at, units);
      return;
    }
    skip_header(units, 0u);
    if (units == 0u) return;
    const bool fresh = ++s.line == lines;
    if (fresh) s.line = 0u, ++s.item;
    make(s, fresh, kLogBlock);
  };
  if (solo) {
    take(use, index, left);
  } else {
    make(use, true, kLogBlock);
    left = static_cast<uint32_t>(r1 - r0);
    skip_header(left, in_segment);
    use.j = in_segment - min(in_segment, header);
  }

  // ---- fetching.  The page ids of the next 32 steps of this warp's tiles are asked for a set ahead, a step
  // a lane; a set that is settled has its places in `where` and asks for its scales, which go to
  // shared memory with the next set, or when the first of its tiles needs them.
  const uint64_t policy = l2_evict_first_policy();
  const uint32_t boxes = 1u << a.log_boxes;
  Segment8 ahead = use;
  uint32_t ahead_left = left, ahead_index = index;
  int32_t ask_page = 0, ask_place = 0, ask_head = 0;
  bool ask_scales = false;
  uint32_t ask_tiles = 0, settled = 0, scaled = 0;          // tiles asked for; with places; with scales
  float wait_ks = 0.f, wait_vs = 1.f;                        // of tiles [scaled, settled)
  auto ask = [&]() {
    ask_tiles = 0u;
    if (ahead_left == 0u) return;
    ask_tiles = min(min(kSet, ahead.j1 - ahead.j), ahead_left);
    const uint32_t step = min(lane / kSteps, ask_tiles - 1u);
    const uint32_t slot = (ahead.block(ahead.j + step) << log_step) + warp_slot + lane % kSteps * 16u;
    const uint32_t at = div_by(slot, c.page), box = kTile >> a.log_boxes;
    ask_page = static_cast<int32_t>(c.num_pages);  // past the pool: a box of zeros
    ask_place = static_cast<int32_t>(slot - at * c.page.d);
    ask_head = static_cast<int32_t>(ahead.kv);
    ask_scales = false;
    if (ahead.some_see(slot & ~(box - 1u), box)) {
      const uint32_t id = static_cast<uint32_t>(c.table[static_cast<size_t>(ahead.b) * c.table_stride + at]);
      if (id < c.num_pages) {
        ask_page = static_cast<int32_t>(id);
        ask_scales = ahead.some_see(slot, 16u);
      } else {
        atomicOr(&g_error_word, QG_ERR_PAGE);
      }
    }
    ahead.j += ask_tiles;
    ahead_left -= ask_tiles;
    if (ahead.j == ahead.j1) advance(ahead, ahead_index, ahead_left);
  };
  auto flush = [&]() {  // the scales that have been waited for
    if (lane / kSteps < settled - scaled) {
      const uint32_t at = (scaled * kSteps + lane) % kEntries;
      const float vs = fminf(fmaxf(wait_vs, 0x1p-60f), 0x1p60f);
      ks_of[warp][at] = wait_ks;
      lg_of[warp][at] = log2f(vs);
      inv_of[warp][at] = 1.f / vs;
    }
    scaled = settled;
    __syncwarp();
  };
  auto settle = [&]() {
    flush();
    if (lane / kSteps < ask_tiles) {
      where[warp][(settled * kSteps + lane) % kEntries] = make_int4(ask_page, ask_place, ask_head, 0);
      wait_ks = 0.f;
      wait_vs = 1.f;
      if (ask_scales) {
        const uint64_t s = static_cast<uint32_t>(ask_page) * cache.scale_page + static_cast<uint32_t>(ask_head) * cache.scale_head +
                           (static_cast<uint32_t>(ask_place) >> cache.log_block);
        wait_ks = cache.ks[s];
        wait_vs = cache.vs[s];
      }
    }
    settled += ask_tiles;
    __syncwarp();
    ask();
  };
  auto fetch = [&](const CUtensorMap* map, uint64_t* bar, uint32_t to, uint32_t tile) {
    const bool leads = elect_one();
    if (leads) mbar_arrive_expect_tx(bar, kUnit);
#pragma unroll 1
    for (uint32_t i = 0; i < boxes; ++i) {
      const int4 at = where[warp][(tile * kSteps + (i * kSteps >> a.log_boxes)) % kEntries];
      if (leads) {
#pragma unroll
        for (uint32_t p = 0; p < kPanels; ++p) {
          tma_load_4d(to + p * kPanel + (i * kTile >> a.log_boxes) * kRowBytes, map, static_cast<int32_t>(p * kRowBytes),
                      a.heads_inside ? at.z : at.y, a.heads_inside ? at.y : at.z, at.x, smem_addr(bar), policy);
        }
      }
    }
  };
  uint32_t tile = 0, next_k = 0, next_v = 0;                 // this warp's tile in work; the next ones to fetch
  auto refill = [&]() {  // what tile `tile` and the ring leave room for
    while (next_k < tile + kK) {
      if (next_k == settled) {
        if (ask_tiles == 0u) break;
        settle();
      }
      fetch(&maps.k, &full_k[warp][next_k % kK], ring_at + next_k % kK * kUnit, next_k);
      ++next_k;
    }
    while (next_v < min(tile + kV, settled)) {
      fetch(&maps.v, &full_v[warp][next_v % kV], ring_at + (kK + next_v % kV) * kUnit, next_v);
      ++next_v;
    }
  };
  ask();

  // ldmatrix rows and 16-byte pieces of this lane (K: 8 slots x 2 pieces x 2; V, transposed:
  // 16 slots x 2 pieces); pieces 2 n and 2 n + 1 of a panel are at lane_at ^ (n << 5)
  auto swizzled = [](uint32_t r, uint32_t piece) {
    return r * kRowBytes + ((piece ^ (kRowBytes == 64u ? (r >> 1) & 3u : r & 7u)) << 4);
  };
  const uint32_t k_lane = swizzled((lane & 7u) + ((lane >> 4) << 3), (lane >> 3) & 1u);
  const uint32_t v_lane = swizzled((lane & 7u) + ((lane >> 3) & 1u) * 8u, lane >> 4);
  constexpr uint32_t kPairs = kPieces / 2u;                 // pairs of pieces of a panel

  uint32_t qa[kMma][kChunks][4];
  float o[RS][DP / 8][2], m[RS], l[RS], mult[RS];
  int32_t p_row[RS];                                        // slot of the row's token
  bool arrives = true, written = false;  // written: by this warp, where a tile will land
  auto await = [&](uint64_t* bar, uint32_t parity) {
    if (!__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) {
      arrives = arrives && __all_sync(0xffffffffu, mbar_wait_bounded(bar, parity));
    }
  };

  auto go_on = [&]() {  // what has been used is fetched into
    if (written) fence_proxy_async_smem();
    __syncwarp();
    written = false;
    if (arrives) refill();
  };

  while (left != 0u) {
    go_on();
    const uint32_t from_j = use.j, to_j = min(use.j1, use.j + left);
    // ---- the queries, as the A operand takes them: of chunk k this lane has dims 16 k + 4 t4 to
    // + 3 of its rows
#pragma unroll
    for (int i = 0; i < RS; ++i) {
      const uint32_t r = i * 8u + g;
      const bool has = r < use.rows;
      const uint32_t at = use.sub + (has ? r : 0u), down = div_by(at, a.group);
      p_row[i] = has ? use.p0 + static_cast<int32_t>(down) : use.p1;
      const uint64_t from = (use.token + down) * a.q_stride +
                            static_cast<uint64_t>(use.kv * a.group.d + (at - down * a.group.d)) * c.dim + 4u * t4;
      float4 x[kChunks];
      float top = 0.f;
#pragma unroll
      for (uint32_t k = 0; k < kChunks; ++k) {
        x[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (has && k * 16u < c.dim) {
          if (TERMS == 2 && a.dtype == QG_F32) {
            x[k] = *reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + from + k * 16u);
          } else {
            const uint2 w = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.q) + from + k * 16u);
            const float2 u = a.dtype == QG_F16 ? unpack2(w.x, __half()) : unpack2(w.x, __nv_bfloat16());
            const float2 v = a.dtype == QG_F16 ? unpack2(w.y, __half()) : unpack2(w.y, __nv_bfloat16());
            x[k] = make_float4(u.x, u.y, v.x, v.y);
          }
        }
        top = fmaxf(fmaxf(top, fmaxf(fabsf(x[k].x), fabsf(x[k].y))), fmaxf(fabsf(x[k].z), fabsf(x[k].w)));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int power = power_of8(top);
      const float down2 = power_of_two(-power);
      mult[i] = a.scale_log2 * power_of_two(power);
#pragma unroll
      for (uint32_t k = 0; k < kChunks; ++k) {
        if constexpr (TERMS == 2) {
          uint32_t lo[2], hi[2];
          split_terms<__half>(x[k].x * down2, x[k].y * down2, lo);
          split_terms<__half>(x[k].z * down2, x[k].w * down2, hi);
          qa[i][k][0] = lo[0], qa[i][k][1] = lo[1], qa[i][k][2] = hi[0], qa[i][k][3] = hi[1];
        } else {
          qa[0][k][i] = pack2(x[k].x * down2, x[k].y * down2, __half());
          qa[0][k][2 + i] = pack2(x[k].z * down2, x[k].w * down2, __half());
        }
      }
      m[i] = -CUDART_INF_F;
      l[i] = 0.f;
#pragma unroll
      for (uint32_t n = 0; n < DP / 8; ++n) o[i][n][0] = o[i][n][1] = 0.f;
    }


    while (true) {
      const uint32_t slot0 = (use.block(use.j) << log_step) + warp_slot;
      const bool whole = use.all_see(a, slot0, kTile);
      const bool seen = use.some_see(slot0, kTile);
      if (tile == scaled) flush();
      const uint32_t scales = tile * kSteps % kEntries;
      // ---- scores
      uint32_t p[kMma][kSteps][2][2];  // probabilities: [16-slot step][8-slot half][term or row]
      float fade[RS];
      await(&full_k[warp][tile % kK], tile / kK & 1u);
      if (seen && arrives) {
        float s[kMma][2 * kSteps][4];
#pragma unroll
        for (int i = 0; i < kMma; ++i) {
#pragma unroll
          for (int n = 0; n < 2 * kSteps; ++n) {
#pragma unroll
            for (int e = 0; e < 4; ++e) s[i][n][e] = 0.f;
          }
        }
        const uint32_t k_at = ring_at + tile % kK * kUnit;
        uint32_t kb[2][kSteps][4];  // the next pair of chunks is loaded while this one is multiplied
        auto load_k = [&](uint32_t kk) {
#pragma unroll
          for (int st = 0; st < kSteps; ++st) {
            ldsm_x4(kb[kk & 1u][st], k_at + (k_lane ^ ((kk % kPairs) << 5)) + kk / kPairs * kPanel + st * 16u * kRowBytes);
          }
        };
        load_k(0u);
#pragma unroll
        for (uint32_t kk = 0; kk < kChunks / 2u; ++kk) {
          if (kk + 1u < kChunks / 2u) load_k(kk + 1u);
#pragma unroll
          for (int f = 0; f < 2; ++f) {          // chunk 2 kk + f
#pragma unroll
            for (int st = 0; st < kSteps; ++st) {
#pragma unroll
              for (int e = 0; e < 2; ++e) {      // slots 8 e of the step
                uint32_t lo, hi;
                codes_to_half(kb[kk & 1u][st][2 * e + f], lo, hi);
#pragma unroll
                for (int i = 0; i < kMma; ++i) mma8(s[i][2 * st + e], qa[i][2 * kk + f], lo, hi);
              }
            }
          }
        }
        // ---- probabilities: this lane's slots are 8 n + 2 t4 and one more
#pragma unroll
        for (int i = 0; i < RS; ++i) {
          float by[kSteps], lg[kSteps], inv[kSteps];
#pragma unroll
          for (int st = 0; st < kSteps; ++st) {
            by[st] = mult[i] * ks_of[warp][scales + st];
            lg[st] = lg_of[warp][scales + st];
            inv[st] = inv_of[warp][scales + st];
          }
          float x[2 * kSteps][2];
          float top = -CUDART_INF_F;
#pragma unroll
          for (int n = 0; n < 2 * kSteps; ++n) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float dot = TERMS == 2 ? s[i * (TERMS - 1)][n][e] + s[i * (TERMS - 1)][n][e + 2] : s[0][n][2 * i + e];
              x[n][e] = fmaf(dot, by[n / 2], lg[n / 2]);
              if (!whole && !sees(a, p_row[i], slot0 + n * 8u + 2u * t4 + e)) x[n][e] = -CUDART_INF_F;
            }
            top = fmaxf(top, fmaxf(x[n][0], x[n][1]));
          }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const float now = fmaxf(m[i], top);
          const float from = now == -CUDART_INF_F ? 0.f : now;
          const float root = exp2_fast(0.5f * (m[i] - from));
          fade[i] = root * root;
          m[i] = now;
          const float base = kShare - from;
          float sum[kSteps] = {}, plus[kSteps], all = 0.f;
#pragma unroll
          for (int st = 0; st < kSteps; ++st) {
            plus[st] = base;
            if (__builtin_expect(lg[st] < kLowScale, 0)) {  // the same for the whole warp
              const float most = fmaxf(fmaxf(x[2 * st][0], x[2 * st][1]), fmaxf(x[2 * st + 1][0], x[2 * st + 1][1]));
              if (most + base < kRaiseBelow) plus[st] += kRaise, inv[st] *= kLower;
            }
          }
#pragma unroll
          for (int n = 0; n < 2 * kSteps; ++n) {
            x[n][0] = exp2_fast(x[n][0] + plus[n / 2]);
            x[n][1] = exp2_fast(x[n][1] + plus[n / 2]);
            sum[n / 2] += x[n][0] + x[n][1];
            if constexpr (TERMS == 2) {
              split_terms<__half>(x[n][0], x[n][1], p[i][n / 2][n % 2]);
            } else {
              p[0][n / 2][n % 2][i] = pack2(x[n][0], x[n][1], __half());
            }
          }
#pragma unroll
          for (int st = 0; st < kSteps; ++st) all = fmaf(sum[st], inv[st], all);
          l[i] = fmaf(l[i] * root, root, all);
        }
      }

      // ---- weighted values
      await(&full_v[warp][tile % kV], tile / kV & 1u);
      if (seen && arrives) {
        uint8_t* const v_mem = ring + (kK + tile % kV) * kUnit;
        if (!whole) {  // 0 x NaN must not reach the sums: what no row sees is cleared
          written = true;
          bool odd = false;  // a NaN that some rows see and some do not
          for (uint32_t i = lane; i < kTile * DP / 16u; i += 32u) {
            const uint32_t slot = slot0 + i / kPieces % kTile;
            uint4* const at = reinterpret_cast<uint4*>(v_mem) + i;
            if (!use.some_see(slot, 1u)) {
              *at = make_uint4(0u, 0u, 0u, 0u);
            } else if (!use.all_see(a, slot, 1u)) {
              const uint4 w = *at;
              auto nan = [](uint32_t u) { return ((u & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; };
              odd = odd || (nan(w.x) | nan(w.y) | nan(w.z) | nan(w.w)) != 0u;
            }
          }
          __syncwarp();
          if (__any_sync(0xffffffffu, odd)) {
            // the columns of the rows that see one become NaN by hand, the codes zeros
            for (uint32_t sl = 0; sl < kTile; ++sl) {
              if (use.all_see(a, slot0 + sl, 1u) || !use.some_see(slot0 + sl, 1u)) continue;
#pragma unroll
              for (uint32_t k = 0; k < kChunks; ++k) {
                uint32_t* const at = reinterpret_cast<uint32_t*>(
                    v_mem + k / kPieces * kPanel + swizzled(sl, k % kPieces) + t4 * 4u);
                const uint32_t w = *at;
                __syncwarp();
                uint32_t clean = w;
#pragma unroll
                for (uint32_t e = 0; e < 4; ++e) {
                  if ((w >> (8u * e) & 0x7fu) != 0x7fu) continue;
                  clean &= ~(0xffu << (8u * e));
#pragma unroll
                  for (int i = 0; i < RS; ++i) {
                    if (sees(a, p_row[i], slot0 + sl)) o[i][2 * k + e % 2][e / 2] = CUDART_NAN_F;
                  }
                }
                if (clean != w && g == 0u) *at = clean;  // the lanes of a column share the word
              }
            }
            __syncwarp();
          }
        }
        const uint32_t v_at = ring_at + (kK + tile % kV) * kUnit;
        uint32_t vw[2][kSteps][4];
        auto load_v = [&](uint32_t n) {
#pragma unroll
          for (int st = 0; st < kSteps; ++st) {
            ldsm_x4_trans(vw[n & 1u][st], v_at + (v_lane ^ ((n % kPairs) << 5)) + n / kPairs * kPanel + st * 16u * kRowBytes);
          }
        };
        load_v(0u);
#pragma unroll
        for (uint32_t n = 0; n < kChunks / 2u; ++n) {
          if (n + 1u < kChunks / 2u) load_v(n + 1u);
          uint32_t (&vb)[kSteps][4] = vw[n & 1u];
#pragma unroll
          for (int st = 0; st < kSteps; ++st) {
#pragma unroll
            for (int e = 0; e < 4; ++e) vb[st][e] = __byte_perm(vb[st][e], 0u, 0x3120u);
          }
#pragma unroll
          for (uint32_t e = 0; e < 2; ++e) {    // 16-dim chunk 2 n + e
            uint32_t b[kSteps][2][2];           // [step][even, odd dims][8-slot half]
#pragma unroll
            for (int st = 0; st < kSteps; ++st) {
              codes_to_half(vb[st][2 * e], b[st][0][0], b[st][1][0]);
              codes_to_half(vb[st][2 * e + 1], b[st][0][1], b[st][1][1]);
            }
#pragma unroll
            for (int i = 0; i < kMma; ++i) {
#pragma unroll
              for (uint32_t f = 0; f < 2; ++f) {
                float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int st = 0; st < kSteps; ++st) {
                  const uint32_t ps[4] = {p[i][st][0][0], p[i][st][0][1], p[i][st][1][0], p[i][st][1][1]};
                  mma8(d, ps, b[st][f][0], b[st][f][1]);
                }
                const uint32_t at = 2u * (2u * n + e) + f;
                if constexpr (TERMS == 2) {
                  o[i][at][0] = fmaf(o[i][at][0], fade[i], d[0] + d[2]);
                  o[i][at][1] = fmaf(o[i][at][1], fade[i], d[1] + d[3]);
                } else {
                  o[0][at][0] = fmaf(o[0][at][0], fade[0], d[0]);
                  o[0][at][1] = fmaf(o[0][at][1], fade[0], d[1]);
                  o[1][at][0] = fmaf(o[1][at][0], fade[1], d[2]);
                  o[1][at][1] = fmaf(o[1][at][1], fade[1], d[3]);
                }
              }
            }
          }
        }
      }
      __syncwarp();
      if (++use.j == to_j) break;
      ++tile;
      go_on();
    }
    left -= to_j - from_j;

    // ---- the end of the segment, or of the range inside it
    const bool mine = solo || (from_j == 0u && to_j == use.j1);
    // each warp's sums over the tile it has just used, rows 0-7 over V, 8-15 over K, pieces swizzled by row
    const uint32_t at0 = (kK + tile % kV) * kUnit, at1 = tile % kK * kUnit;
#pragma unroll
    for (int i = 0; i < RS; ++i) {
      float sum = l[i];
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      if (t4 == 0u) {
        join_m[warp][i * 8 + g] = m[i];
        join_l[warp][i * 8 + g] = sum;
      }
      float4* to = reinterpret_cast<float4*>(ring + (i == 0 ? at0 : at1)) + g * (DP / 4u);
#pragma unroll
      for (uint32_t k = 0; k < kChunks; ++k) {
        to[(k * 4u + t4) ^ ((g & 1u) << 2)] = make_float4(o[i][2 * k][0], o[i][2 * k + 1][0], o[i][2 * k][1], o[i][2 * k + 1][1]);
      }
    }
    written = true;
    ++tile;
    // a lone warp joins nothing but its own; the others' lie where its own do, they have gone as many tiles
    const uint32_t w0 = solo ? warp : 0u, w1 = solo ? warp + 1u : kWarps;
    if (solo) {
      __syncwarp();
    } else {
      __syncthreads();
    }
    float* record = a.records + (static_cast<size_t>(blockIdx.x) * 2u + (from_j == 0u ? 1u : 0u)) * Shape::kRecord;
    auto finish = [&](uint32_t r, uint32_t ch, float top, float sum, float4 v) {
      const uint32_t at = use.sub + r, down = div_by(at, a.group);
      const uint32_t h = use.kv * a.group.d + (at - down * a.group.d), token = use.token + down;
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      v.x *= inv, v.y *= inv, v.z *= inv, v.w *= inv;
      const size_t to = token * a.out_stride + static_cast<size_t>(h) * c.dim + ch * 4u;
      if (ch * 4u < c.dim) {
        if (a.dtype == QG_F32) {
          *reinterpret_cast<float4*>(static_cast<float*>(a.out) + to) = v;
        } else if (a.dtype == QG_F16) {
          *reinterpret_cast<uint2*>(static_cast<__half*>(a.out) + to) =
              make_uint2(pack2(v.x, v.y, __half()), pack2(v.z, v.w, __half()));
        } else {
          *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + to) =
              make_uint2(pack2(v.x, v.y, __nv_bfloat16()), pack2(v.z, v.w, __nv_bfloat16()));
        }
      }
      if (ch == 0u && a.lse != nullptr) {
        a.lse[static_cast<size_t>(token) * a.n_q + h] =
            sum == 0.f ? -CUDART_INF_F : (top + log2f(sum) - kShare) * 0.69314718055994530942f;
      }
    };
#pragma unroll 1
    for (uint32_t i = solo ? lane : tid; i < use.rows * (DP / 4u); i += solo ? 32u : kAttnThreads) {
      const uint32_t r = i / (DP / 4u), ch = i % (DP / 4u);
      float top = -CUDART_INF_F;
      for (uint32_t w = w0; w < w1; ++w) top = fmaxf(top, join_m[w][r]);
      const float from = top == -CUDART_INF_F ? 0.f : top;
      float sum = 0.f;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      for (uint32_t w = w0; w < w1; ++w) {
        const float root = exp2_fast(0.5f * (join_m[w][r] - from)), f = root * root;
        const float4 x = reinterpret_cast<const float4*>(smem + w * ((kK + kV) * kUnit) + (r < 8u ? at0 : at1))
            [(r & 7u) * (DP / 4u) + (ch ^ ((r & 1u) << 2))];
        sum = fmaf(join_l[w][r] * root, root, sum);
        v.x = fmaf(x.x, f, v.x), v.y = fmaf(x.y, f, v.y);
        v.z = fmaf(x.z, f, v.z), v.w = fmaf(x.w, f, v.w);
      }
      if (mine) {
        finish(r, ch, top, sum, v);
      } else {
        if (ch == 0u) {
          record[r] = top;
          record[kRows + r] = sum;
        }
        reinterpret_cast<float4*>(record + 2u * kRows)[r * (DP / 4u) + ch] = v;
      }
    }
    if (!mine) {
      // the CTAs that share this segment own its first to its last block, in order
      const uint64_t seg0 = r1 - left - to_j, seg1 = seg0 + use.j1;
      const uint32_t c0 = static_cast<uint32_t>(((seg0 + 1u) * ctas - 1u) / total);
      const uint32_t count = static_cast<uint32_t>((seg1 * ctas - 1u) / total) - c0 + 1u;
      const uint32_t per = count <= kJoinAll ? count : kJoin;
      const uint32_t index = blockIdx.x - c0, group = index / per;
      const uint32_t groups = (count + per - 1u) / per, members = min(per, count - group * per);
      auto record_of = [&](uint32_t cta) {
        return a.records + (static_cast<size_t>(cta) * 2u + (cta == c0 ? 1u : 0u)) * Shape::kRecord;
      };
      // whether this CTA is the last of `n` to arrive; the others' records can then be read
      auto last_of = [&](uint32_t* counter, uint32_t n) {
        __syncthreads();
        if (tid == 0u) {
          __threadfence();  // this CTA's records, ordered before by the barrier, are out
          is_last = atomicAdd(counter, 1u) == n - 1u;
          if (is_last != 0u) *counter = 0u;
          __threadfence();
        }
        __syncthreads();
        return is_last != 0u;
      };
      // joins the n <= 64 records of CTAs first, first + step, ..; put(row, piece, m, l, o)
      auto join_records = [&](uint32_t first, uint32_t step, uint32_t n, auto put) {
        constexpr uint32_t kItems = kRows * (DP / 4u) / kAttnThreads;       // float4 pieces of a thread
        constexpr uint32_t kOnce = kItems < 2u ? 1u : 2u;                   // .. that it works on together
        float4 x[kOnce][kInFlight];
        auto ask = [&](uint32_t i0, uint32_t q0) {
#pragma unroll
          for (uint32_t q = 0; q < kInFlight; ++q) {
            const float4* rec = reinterpret_cast<const float4*>(record_of(first + (q0 + q) * step) + 2u * kRows);
#pragma unroll
            for (uint32_t e = 0; e < kOnce; ++e) {
              const uint32_t i = (i0 + e) * kAttnThreads + tid;
              x[e][q] = make_float4(0.f, 0.f, 0.f, 0.f);
              if (q0 + q < n && i < use.rows * (DP / 4u)) x[e][q] = __ldcg(rec + i);
            }
          }
        };
        ask(0u, 0u);
        constexpr uint32_t kRowsPerWarp = kRows / kWarps;
        float pm[kRowsPerWarp][2], pl[kRowsPerWarp][2];  // two records a lane
#pragma unroll
        for (uint32_t e = 0; e < 2; ++e) {
          const uint32_t q = lane + 32u * e;
          const float* rec = record_of(first + min(q, n - 1u) * step);
#pragma unroll
          for (uint32_t i = 0; i < kRowsPerWarp; ++i) {
            const uint32_t r = warp + i * kWarps;
            pm[i][e] = q < n && r < use.rows ? __ldcg(rec + r) : -CUDART_INF_F;
            pl[i][e] = q < n && r < use.rows ? __ldcg(rec + kRows + r) : 0.f;
          }
        }
#pragma unroll
        for (uint32_t i = 0; i < kRowsPerWarp; ++i) {
          const uint32_t r = warp + i * kWarps;
          float top = fmaxf(pm[i][0], pm[i][1]);
#pragma unroll
          for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
          const float from = top == -CUDART_INF_F ? 0.f : top;
          const float r0 = exp2_fast(0.5f * (pm[i][0] - from)), r1 = exp2_fast(0.5f * (pm[i][1] - from));
          float all = fmaf(pl[i][0] * r0, r0, pl[i][1] * r1 * r1);
#pragma unroll
          for (int off = 16; off > 0; off >>= 1) all += __shfl_xor_sync(0xffffffffu, all, off);
          share[r][lane] = r0 * r0;
          share[r][lane + 32u] = r1 * r1;
          if (lane == 0u) join_m[0][r] = top, join_l[0][r] = all;
        }
        __syncthreads();
#pragma unroll
        for (uint32_t i0 = 0; i0 < kItems; i0 += kOnce) {
          float4 v[kOnce];
#pragma unroll
          for (uint32_t e = 0; e < kOnce; ++e) v[e] = make_float4(0.f, 0.f, 0.f, 0.f);
          for (uint32_t q0 = 0; q0 < n; q0 += kInFlight) {
            if (i0 + q0 != 0u) ask(i0, q0);
#pragma unroll
            for (uint32_t q = 0; q < kInFlight; ++q) {
#pragma unroll
              for (uint32_t e = 0; e < kOnce; ++e) {
                const float f = share[((i0 + e) * kAttnThreads + tid) / (DP / 4u)][q0 + q];
                v[e].x = fmaf(x[e][q].x, f, v[e].x), v[e].y = fmaf(x[e][q].y, f, v[e].y);
                v[e].z = fmaf(x[e][q].z, f, v[e].z), v[e].w = fmaf(x[e][q].w, f, v[e].w);
              }
            }
          }
#pragma unroll
          for (uint32_t e = 0; e < kOnce; ++e) {
            const uint32_t i = (i0 + e) * kAttnThreads + tid, r = i / (DP / 4u);
            if (r < use.rows) put(r, i % (DP / 4u), join_m[0][r], join_l[0][r], v[e]);
          }
        }
      };
      auto to_record = [&](float* rec) {
        return [=](uint32_t r, uint32_t ch, float top, float sum, float4 v) {
          if (ch == 0u) rec[r] = top, rec[kRows + r] = sum;
          reinterpret_cast<float4*>(rec + 2u * kRows)[r * (DP / 4u) + ch] = v;
        };
      };
      // few records are joined at once, many in groups, then the groups' records
      const uint32_t g0 = c0 + group * per;
      if (members == 1u || last_of(a.arrived + g0, members)) {
        if (groups == 1u) {
          join_records(g0, 1u, members, finish);
        } else {
          if (members > 1u) join_records(g0, 1u, members, to_record(record_of(g0)));
          if (last_of(a.arrived + kMaxCtas + c0, groups)) join_records(c0, per, groups, finish);
        }
      }
    }
    // the units and the joins are free again
    if (solo) {
      __syncwarp();
    } else {
      __syncthreads();
    }
    if (use.j == use.j1) advance(use, index, left);
  }
  if (!arrives) {  // a wait ran out (QG_ERR_WAIT_TIMEOUT is set): let what is in flight land
    for (uint32_t i = next_k > kK ? next_k - kK : 0u; i < next_k; ++i) mbar_wait_bounded(&full_k[warp][i % kK], i / kK & 1u);
    for (uint32_t i = next_v > kV ? next_v - kV : 0u; i < next_v; ++i) mbar_wait_bounded(&full_v[warp][i % kV], i / kV & 1u);
  }
}

// ---- the tiles of a ragged call

constexpr uint32_t kPlanThreads = 1024;

// Sums of a value over the threads before this one and over all; all threads take part.
__device__ __forceinline__ uint64_t plan_scan(uint64_t v, uint64_t& all) {
  __shared__ uint64_t sums[kPlanThreads / 32u];
  const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
  uint64_t upto = v;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const uint64_t o = __shfl_up_sync(0xffffffffu, upto, off);
    if (lane >= static_cast<uint32_t>(off)) upto += o;
  }
  __syncthreads();
  if (lane == 31u) sums[warp] = upto;
  __syncthreads();
  uint64_t before = 0;
  all = 0;
  for (uint32_t w = 0; w < kPlanThreads / 32u; ++w) {
    if (w < warp) before += sums[w];
    all += sums[w];
  }
  return before + upto - v;
}

// log: of a block; log_tile: of the steps of a lone warp
__global__ void __launch_bounds__(kPlanThreads) plan8_kernel(const Paged8View cache, const Attn8Args a, uint32_t rows,
                                                             uint32_t log, uint32_t log_tile) {
  __shared__ uint32_t longest;
  pdl_wait();
  pdl_trigger();
  const PagedView& c = cache.c;
  const uint32_t tid = threadIdx.x;
  uint64_t tiles = 0;
  for (uint32_t b0 = 0; b0 < c.batch; b0 += kPlanThreads) {
    const uint32_t b = b0 + tid;
    uint64_t n = 0, all;
    if (b < c.batch) n = (static_cast<uint64_t>(rows_of(c, a.lens, a.offsets, a.tokens, b).n) * a.group.d + rows - 1u) / rows;
    const uint64_t at = tiles + plan_scan(n, all);
    tiles += all;
    if (b < c.batch) a.seq_tiles[b] = static_cast<uint32_t>(min(at, static_cast<uint64_t>(a.max_items)));
  }
  // offsets that overlap could name more rows than there are
  const uint32_t items = static_cast<uint32_t>(min(tiles, static_cast<uint64_t>(a.max_items)));
  if (tid == 0u) {
    a.seq_tiles[c.batch] = items;
    a.item_count[0] = items;
    longest = 0u;
    if (items < tiles) atomicOr(&g_error_word, QG_ERR_PAGE);
  }
  __syncthreads();
  uint64_t blocks = 0;
  for (uint32_t i0 = 0; i0 < items; i0 += kPlanThreads) {
    const uint32_t i = i0 + tid;
    uint64_t n = 0, all;
    if (i < items) {
      uint32_t lo = 0, hi = c.batch;  // the last sequence whose tiles begin at or before i
      while (hi - lo > 1u) {
        const uint32_t mid = (lo + hi) / 2u;
        if (a.seq_tiles[mid] <= i) {
          lo = mid;
        } else {
          hi = mid;
        }
      }
      const Rows8 r = rows_of(c, a.lens, a.offsets, a.tokens, lo);
      const uint64_t row = static_cast<uint64_t>(i - a.seq_tiles[lo]) * rows, most = static_cast<uint64_t>(r.n) * a.group.d;
      const uint32_t down = static_cast<uint32_t>(row / a.group.d);
      Segment8 s;
      s.sub = static_cast<uint32_t>(row - static_cast<uint64_t>(down) * a.group.d);
      s.rows = static_cast<uint32_t>(min(static_cast<uint64_t>(rows), most - row));
      // no slots: rows of a sequence that holds nothing, or does not fit
      s.p0 = r.len == 0u ? INT32_MIN / 2 : static_cast<int32_t>(r.len - r.n + down);
      s.bounds(a, log_tile);
      atomicMax(&longest, s.j1);
      s.bounds(a, log);
      n = s.j1;
      a.items[i] = make_uint4(lo, r.first + down, static_cast<uint32_t>(s.p0), s.sub | (s.rows << 16));
    }
    const uint64_t at = blocks + plan_scan(n, all);
    blocks += all;
    if (i < items) a.item_blocks[i] = at;
  }
  __syncthreads();
  if (tid == 0u) {
    a.item_blocks[items] = blocks;
    a.item_count[1] = longest;
  }
}

// ---- host side

constexpr size_t round_up8(size_t v) { return (v + 255u) & ~static_cast<size_t>(255u); }

struct Plan8 {
  uint32_t dp, rs;
  size_t records_at, count_at, items_at, blocks_at, seqs_at, prompt_at, bytes;
  uint32_t max_items;
};

// Rows of a tile: 8 where that is all that a kv head has.
bool plan_attn8(const Paged8View& c, uint32_t n_q, uint32_t tokens, Plan8* p) {
  if (n_q == 0u || n_q > 65535u || n_q % c.c.n_kv != 0u || tokens > 0x7fffffffu) return false;
  const uint32_t group = n_q / c.c.n_kv;
  p->dp = c.c.dim <= 64u ? 64u : c.c.dim <= 128u ? 128u : 256u;
  const uint64_t items = most_tiles(tokens, c.c.batch, group, 8u);
  if (items > 0x7fffffffull) return false;
  p->max_items = static_cast<uint32_t>(items);
  p->records_at = QG_PAGED_ATTN_ZEROED;
  p->count_at = round_up8(p->records_at + static_cast<size_t>(kMaxCtas) * 2u * 16u * (p->dp + 2u) * 4u);
  p->items_at = p->count_at + 256u;
  p->blocks_at = round_up8(p->items_at + items * 16u);
  p->seqs_at = round_up8(p->blocks_at + (items + 1u) * 8u);
  p->prompt_at = round_up8(p->seqs_at + (c.c.batch + 1u) * 4u);
  p->bytes = p->prompt_at + (prompt8_fits(p->dp, tokens, c.c.batch, group) ? prompt8_bytes(p->dp) : 0u);
  return true;
}

// As in qg_paged_attn.cu: strides of a tensor map nest.
struct PoolStrides8 {
  uint64_t inner, outer, page;
  bool heads_inside;
};
bool pool_strides8(const qg_kv_pages8* cache, PoolStrides8* s) {
  uint64_t head = cache->head_stride, slot = cache->slot_stride;
  const uint64_t row = cache->head_dim;
  s->heads_inside = cache->n_kv_heads != 1u && head < slot;
  if (cache->n_kv_heads == 1u) head = slot;
  s->inner = s->heads_inside ? head : slot;
  s->outer = s->heads_inside ? slot : head;
  s->page = cache->num_pages == 1u ? s->outer : cache->page_stride;
  return s->inner >= row && s->inner % 16u == 0u && s->outer >= s->inner && s->outer % s->inner == 0u &&
         s->page >= s->outer && s->page % s->outer == 0u && s->page < (1ull << 40);
}

bool encode_pool8(CUtensorMap* map, void* pool, const qg_kv_pages8* cache, const PoolStrides8& s, uint32_t box_slots,
                  uint32_t dp) {
  const auto encode = tensor_map_encoder();
  if (encode == nullptr) return false;
  const uint32_t inner = s.heads_inside ? cache->n_kv_heads : cache->page_size;
  const uint32_t outer = s.heads_inside ? cache->page_size : cache->n_kv_heads;
  const cuuint64_t dims[4] = {cache->head_dim, inner, outer, cache->num_pages};
  const cuuint64_t strides[3] = {s.inner, s.outer, s.page};
  const cuuint32_t box[4] = {dp == 64u ? 64u : 128u, s.heads_inside ? 1u : box_slots, s.heads_inside ? box_slots : 1u, 1u};
  const cuuint32_t step[4] = {1u, 1u, 1u, 1u};
  // Where a row's neighbours in memory are other heads' rows, no more than the row is brought to L2: 16 x 32768 in
  // that order 287 us with 256 bytes a request, 217 with 128; 64 x ..4097 of 64-byte rows 115 and, with 64, 100 us.
  const auto promotion = !s.heads_inside ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B
                         : dp == 64u     ? CU_TENSOR_MAP_L2_PROMOTION_L2_64B
                                         : CU_TENSOR_MAP_L2_PROMOTION_L2_128B;
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, pool, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                dp == 64u ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, promotion,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DP, int RS, int TERMS>
cudaError_t launch_attn8(const Paged8View& c, const Attn8Args& args, const AttnMaps8& maps, cudaStream_t stream) {
  using Shape = Attn8Shape<DP, RS, TERMS>;
  const auto kernel = paged_attn8_kernel<DP, RS, TERMS>;
  static SmemAttr attr;
  cudaError_t e = attr.set(reinterpret_cast<const void*>(kernel), Shape::kSmem);
  if (e != cudaSuccess) return e;
  Attn8Args a = args;
  a.tiles = (a.group.d + Shape::kRows - 1u) / Shape::kRows;
  const uint64_t tiles = a.offsets != nullptr ? most_tiles(a.tokens, c.c.batch, a.group.d, Shape::kRows)
                                              : static_cast<uint64_t>(a.tokens) * a.tiles;
  const uint64_t blocks = tiles * c.c.n_kv * ((c.c.capacity + (1u << Shape::kLogBlock) - 1u) >> Shape::kLogBlock);
  const uint64_t fit = static_cast<uint64_t>(paged_sm_count()) * Shape::kCtasPerSm;
  const uint32_t grid = static_cast<uint32_t>(std::min<uint64_t>(std::min<uint64_t>(blocks, fit), kMaxCtas));
  // a CTA counts its units in 32 bits, segments are numbered in 32
  if (blocks / grid >= (1ull << 29) || tiles * c.c.n_kv >= (1ull << 32)) return cudaErrorInvalidValue;
  if (a.offsets != nullptr) {
    e = launch_plan8(c, a, Shape::kRows, Shape::kLogBlock, Shape::kLogTile, stream);
    if (e != cudaSuccess) return e;
  }
  return launch_k(kernel, grid, kAttnThreads, Shape::kSmem, stream, c, a, maps);
}

}  // namespace

cudaError_t launch_plan8(const Paged8View& c, const Attn8Args& a, uint32_t rows, uint32_t log, uint32_t log_tile,
                         cudaStream_t stream) {
  return launch_k(plan8_kernel, 1u, kPlanThreads, 0, stream, c, a, rows, log, log_tile);
}

}  // namespace qg

extern "C" cudaError_t qg_paged_attn8_workspace_bytes(const qg_kv_pages8* cache, uint32_t n_q_heads, uint32_t tokens,
                                                      size_t* bytes) {
  using namespace qg;
  Paged8View c;
  Plan8 p;
  if (bytes == nullptr || !paged8_view(cache, &c) || !plan_attn8(c, n_q_heads, tokens, &p)) return cudaErrorInvalidValue;
  *bytes = p.bytes;
  return cudaSuccess;
}

extern "C" cudaError_t qg_paged_attn8(const qg_kv_pages8* cache, const qg_attn8* p, void* workspace,
                                      cudaStream_t stream) {
  using namespace qg;
  Paged8View c;
  Plan8 plan;
  if (!paged8_view(cache, &c) || p == nullptr || !dtype_ok(p->dtype) || !plan_attn8(c, p->n_q_heads, p->tokens, &plan)) {
    return cudaErrorInvalidValue;
  }
  if (p->tokens == 0u) return cudaSuccess;
  const uint64_t piece = 16u / dtype_bytes(p->dtype);
  if (p->q == nullptr || p->out == nullptr || p->lens == nullptr || workspace == nullptr || p->q_stride % piece != 0u ||
      p->out_stride % piece != 0u || !aligned16(p->q) || !aligned16(p->out) ||
      (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0u || (p->offsets == nullptr && p->tokens > cache->batch)) {
    return cudaErrorInvalidValue;
  }
  PoolStrides8 strides;
  if (!pool_strides8(cache, &strides)) return cudaErrorInvalidValue;
  // rows of a kv head: a call of one row a sequence has its group; of a ragged call only the sum is known here
  const uint32_t group = p->n_q_heads / c.c.n_kv;
  const bool few = (p->offsets == nullptr ? 1ull : p->tokens) * group <= 8u, wide = p->dtype == QG_F32;
  const uint32_t rs = few || (wide && plan.dp == 256u) ? 1u : 2u, terms = few || wide ? 2u : 1u;
  // a box is part of one tile and page
  const uint32_t log_tile = log_tile8(plan.dp, rs, terms);
  const uint32_t log_box = std::min<uint32_t>(log_tile, __builtin_ctz(cache->page_size));
  AttnMaps8 maps;
  if (!encode_pool8(&maps.k, cache->k, cache, strides, 1u << log_box, plan.dp) ||
      !encode_pool8(&maps.v, cache->v, cache, strides, 1u << log_box, plan.dp)) {
    return cudaErrorNotSupported;
  }
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  Attn8Args a{};
  a.q = p->q;
  a.out = p->out;
  a.dtype = p->dtype;
  a.q_stride = p->q_stride;
  a.out_stride = p->out_stride;
  a.lens = p->lens;
  a.offsets = p->offsets;
  a.tokens = p->tokens;
  a.window = p->window;
  a.sink = p->sink;
  a.n_q = p->n_q_heads;
  a.group = fast_div(group);
  a.scale_log2 = p->scale * 1.44269504088896340736f;
  a.lse = p->lse;
  a.arrived = reinterpret_cast<uint32_t*>(ws);
  a.records = reinterpret_cast<float*>(ws + plan.records_at);
  if (p->offsets != nullptr) {
    a.item_count = reinterpret_cast<uint32_t*>(ws + plan.count_at);
    a.items = reinterpret_cast<uint4*>(ws + plan.items_at);
    a.item_blocks = reinterpret_cast<uint64_t*>(ws + plan.blocks_at);
    a.seq_tiles = reinterpret_cast<uint32_t*>(ws + plan.seqs_at);
    a.max_items = plan.max_items;
  }
  a.log_boxes = log_tile - log_box;
  a.heads_inside = strides.heads_inside;
  if (p->offsets != nullptr && p->dtype != QG_F32 && prompt8_fits(plan.dp, p->tokens, cache->batch, a.group.d)) {
    a.records = reinterpret_cast<float*>(ws + plan.prompt_at);
    return launch_prompt8(c, a, plan.dp, stream);
  }
  if (plan.dp == 64u) {
    if (rs == 1u) return launch_attn8<64, 1, 2>(c, a, maps, stream);
    return terms == 2u ? launch_attn8<64, 2, 2>(c, a, maps, stream) : launch_attn8<64, 2, 1>(c, a, maps, stream);
  }
  if (plan.dp == 128u) {
    if (rs == 1u) return launch_attn8<128, 1, 2>(c, a, maps, stream);
    return terms == 2u ? launch_attn8<128, 2, 2>(c, a, maps, stream) : launch_attn8<128, 2, 1>(c, a, maps, stream);
  }
  return rs == 1u ? launch_attn8<256, 1, 2>(c, a, maps, stream) : launch_attn8<256, 2, 1>(c, a, maps, stream);
}

// qg_paged_attn.cu -- qg_paged_attn: attention of one new token per sequence over a paged
// key-value cache (declared in include/qgemv_b200.h).
//
// Mathematics.  One pass over a sequence's slots with the running maximum m, sum l and
// weighted value sum o of a softmax, in log2 units: s = (q . k) * scale * log2 e,
//   m' = max(m, s),  l' = l 2^(m - m') + 2^(s - m'),  o' = o 2^(m - m') + 2^(s - m') v;
// two passes over disjoint slots join by the same rule, so a sequence is cut anywhere.
//
// Bound by memory: a slot's K and V rows are read once for every 8 or 16 query heads of their kv
// head (16 where more than 8 share it: at head size 64, and at 128 but for fp32 queries over
// bf16), at half a multiply-add a byte for one query head, 8 for 16.  The dot products still go to the matrix pipe, because on
// the CUDA cores a group of 8 heads would need 8 fp32 FMAs and conversions for every 2 bytes.
// mma.sync (m16n8k16) keeps scores, probabilities and sums in the registers of the warp that
// loads the slots; its rate is far above the few per cent that the memory can feed, so
// tcgen05 with its trip through tensor memory has nothing to win here.
//
// Work.  The unit is a block of 128 slots (64 at head size 256) of one (sequence, kv head, head
// tile).  All blocks of the batch, whatever the lengths, form one line that is cut into equal
// ranges, one a CTA, two or three CTAs an SM; a segment of the line (one sequence, head and
// tile) counts kHeader blocks more than it has, because its queries and sums cost about that.
// In a range, warp w owns a quarter of every block, a tile, and runs on its own: it fetches its K
// and V tiles in turn through its own ring and keeps its own (m, l, o).  Tiles arrive as TMA
// boxes of gcd(tile, page_size) slots x 64 values, swizzled for ldmatrix, so no box crosses a
// page, whatever the page size, and values past head_dim, slots of no page and slots past the
// sequence's last box are the tensor map's zeros; page ids are read 32 boxes at a time, ahead of
// their use.  Only rows that share a box with the sequence's ends can hold what is not the
// sequence's: their V rows are cleared in shared memory, their scores are masked.  Where a
// segment ends inside the range the four warps join through shared memory; where the range cuts
// it, the CTA leaves a record.  The CTA that arrives last joins a head's records (more than 48 in
// groups of 16 first, each by its last CTA), always in CTA order, so results do not depend on
// timing.  Where segments are many and short (the rule is in the kernel, on the lengths) a CTA
// would spend its time between them, 4.4 us each; there every warp takes whole segments alone,
// with no barrier and no record.  98 sequences of 16/16 heads x 112 that see one slot: 26 us by
// CTAs, 14 by warps; 256 x 300 slots, 32/8 heads x 128: 65 and 61 us; 89 x 1..2 slots, 40/8 heads
// x 112: 17 and 9 us.
//
// Measured (B200, 6.46 TB/s for a plain copy; time on the GPU, floor = bytes that have to move
// at that rate): 16 x 32768 slots, 64/8 heads x 128 fp16: 338 us (floor 332); 1 x 131072: 94 us
// (83; the join of 37 records a head is 7 of them); 32 x 1..8191 bf16 with weights: 36 us (21);
// 64 x ..4097, 16/16 heads x 64, window 2000, pages of 24: 79 us (70); 1 x 511: 10 us, all
// latency.  Per-lane asynchronous copies in the place of TMA boxes took 439 us for the first,
// one 16-slot tile at a time 384 us.
//
// Matrix fragments.  Rows of the A operand are query heads.  Eight heads fill rows 0-7 and
// the rounding errors of their values rows 8-15: q = hi + lo in the cache's type, so one mma
// gives (hi + lo) . k, fp16 pairs carrying 22 bits and bf16 pairs 16.  (A fp32 q with a bf16
// cache takes a third term, 24 bits, in a second mma.)  q is first scaled by a power of two
// per head to a largest value in [1, 2), so neither term leaves fp16's range, or in
// [2^-10, 2^-9) over bf16, so 256 products with its largest keys stay within fp32's.  The scores'
// accumulators are laid out like the A operand of the next product, so probabilities go back
// in without a shuffle, again as hi + lo; in fp16 they carry a factor 2^14 (removed with l), which
// keeps probabilities down to 2^-38 exact enough when a million slots share the sum.  bf16 has
// fp32's exponents: it needs no factor, and values above 2^114 could not bear one.
// Each tile's P V is accumulated from zero and added to o in fp32 on the CUDA cores: o lives for
// thousands of tiles, and how the matrix pipe rounds a running sum is not specified.
#include <math_constants.h>

#include <algorithm>

#include "qg_mma.cuh"

namespace qg {
namespace {

constexpr uint32_t kWarps = 4;
constexpr uint32_t kAttnThreads = kWarps * 32;
// Slots of one warp's tile: 8 KB of K at head sizes 128 and 256, 4 KB at 64.
constexpr uint32_t log_tile(uint32_t dp) { return dp == 256u ? 4u : 5u; }
constexpr uint32_t block_slots(uint32_t dp) { return kWarps << log_tile(dp); }
constexpr uint32_t kMaxCtas = 512;
constexpr uint32_t kJoinAll = 48;             // records of a head that are joined at once
constexpr uint32_t kJoin = 16;                // records of a group where there are more
constexpr uint32_t kInFlight = 16;            // records whose sums are asked for together
static_assert(2u * kMaxCtas * 4u <= QG_PAGED_ATTN_ZEROED, "two counters per CTA");
static_assert(kMaxCtas / kJoin <= 64u && kJoinAll <= 64u, "two records a lane");
// log2 of the factor that probabilities carry in the cache's type
template <typename T>
constexpr float kShareBits = std::is_same<T, __half>::value ? 14.f : 0.f;

struct AttnArgs {
  const void* q;
  void* out;
  int dtype;
  uint64_t q_stride, out_stride;
  const int32_t* lens;
  uint32_t max_len, window;
  uint32_t n_q, group, tiles;  // query heads, per kv head, head tiles per kv head
  float scale_log2;
  float* lse;
  uint32_t* arrived;           // [2][kMaxCtas], zero between calls
  float* records;              // [cta][2] partial results
  float* scores;               // [batch][n_q][score_stride], log2 units, or NULL
  float* norm;                 // [batch][n_q]: log2 of the full sum, with scores
  uint32_t score_stride;
  uint32_t log_boxes;          // log2 of the boxes of a tile
  bool heads_inside;           // a page's heads lie inside its slots ([place][head][dim])
};

// K and V pools as [page][.][.][dim] tensors; the middle two in the order of their strides.
struct AttnMaps {
  CUtensorMap k, v;
};

// The power p with top in [2^p, 2^(p + 1)), kept where both 2^p and 2^-p are normal numbers.  For
// bf16 it is 10 more, less where that would pass 116 (the scale times 2^p has to stay finite).
template <typename T>
__device__ __forceinline__ int power_of(float top) {
  constexpr int kRoom = std::is_same<T, __half>::value ? 0 : 10;
  const int p = max(-126, min(126, static_cast<int>(__float_as_uint(top) >> 23) - 127));
  return top == 0.f ? 0 : min(p + kRoom, max(p, 126 - kRoom));
}
// One (sequence, kv head x head tile) of the line: its seen slots [start, len) are steps
// [j0, j1) of 2^log slots; j is the next one.
struct Segment {
  uint32_t b, h, j, j0, j1, start, len;

  __device__ __forceinline__ void bounds(const PagedView& c, const AttnArgs& a, uint32_t log) {
    len = paged_len(a.lens[b], min(a.max_len, c.capacity));
    start = a.window != 0u && len > a.window ? len - a.window : 0u;
    j0 = start >> log;
    j1 = max(((len - 1u) >> log) + 1u, j0 + 1u);  // an empty sequence has one empty step
    if (len == 0u) j1 = j0 + 1u;
  }
};

// T: cache type.  DP: head_dim rounded up to 64, 128 or 256.  MT: tiles of 8 heads.
// EXTRA: third terms of q and of the probabilities (fp32 queries over a bf16 cache).
template <typename T, int DP, int MT, bool EXTRA>
struct AttnShape {
  static constexpr uint32_t kTile = 1u << log_tile(DP);
  static constexpr uint32_t kBlock = block_slots(DP);
  static constexpr uint32_t kHeads = 8u * MT;
  static constexpr uint32_t kUnit = kTile * DP * 2u;        // a warp's K or V tile
  // CTAs an SM.  Small heads do the most work a byte and fit three in registers: 64 x ..4097
  // (16/16 heads x 64) 84 us with two, 79 with three.  At 128 three CTAs of 168 registers are
  // 2-7% faster where many segments run (256 x 300: 65 and 60 us) and 5-15% slower where few
  // do (1 x 8192: 17.7 and 20.3, 1 x 131072: 92.6 and 97.1 us), so it keeps two.  Both sizes then
  // hold a head tile without spills.  The wider forms do spill, bytes of stores: two tiles at 128
  // 364; 256 104; fp32 over bf16 64 (64), two tiles at 64 216, 128 180, 256 482.  8 x 16384 slots,
  // us (floor): 64/4 heads x 128 64 (42), 32/4 x 256 fp16 98 (83), fp32 over bf16 108 (83).
  static constexpr int kCtasPerSm = DP == 64 && MT == 1 ? 3 : 2;
  static constexpr uint32_t kUnits = DP != 64 ? 3 : kCtasPerSm == 3 ? 4 : 6;  // of its ring
  static constexpr uint32_t kRing = kWarps * kUnits * kUnit;
  static constexpr uint32_t kQRows = MT * (EXTRA ? 24u : 16u);
  static constexpr uint32_t kQBytes = kQRows * DP * 2u;
  static constexpr uint32_t kSmem = kRing + kQBytes + 1024u;  // the ring starts on 1024 bytes
  static constexpr uint32_t kPanels = DP / 64u;             // 128-byte column panels of a row
  static constexpr uint32_t kRecord = kHeads * (DP + 2u);   // m[], l[], o[][]
  // What a segment costs beside its blocks, in blocks: queries in, sums out, joins.  No value is
  // the best for all lengths; us at
  //   head size 64, 1 to 4: 64 x ..4097 (16/16 heads, window 2000) 78.9, 79.5, 80.8 and 78.2;
  //     100 x 10..2000 (32/8) 27.0, 26.7, 27.5 and 28.4; 32 x 100..8191 34.3, 33.6, 32.5 and 31.3;
  //   128, 1 to 4: 32 x ..8191 (32/8) 35.3, 33.2, 32.0 and 32.3; 100 x 10..2000 38.4, 39.7, 42.9
  //     and 46.0; 48 x 200..6000 (40/8) 64.6, 64.4, 64.1 and 63.9;
  //   256, 0 to 3: 62 x ..752 (16/4) 21.0, 19.1, 20.0 and 19.3; 32 x ..8191 (16/2) 33.3, 28.3, 27.5
  //     and 26.7; 100 x 10..2000 (8/2) 30.8, 26.6, 25.5 and 25.0.
  static constexpr uint32_t kHeader = DP == 64 ? 2 : DP == 128 ? 3 : 1;
  // Whether a lone warp may take whole segments (below): where the code for it costs the rest
  // little (1%).  At head size 256 and with two tiles of heads it cost 5-10%, at 64, whose three
  // CTAs an SM change segments faster, 2-4% (64 x ..4097: 79.2 and 81.1 us).
  static constexpr bool kSolo = DP == 128 && MT == 1;
  static_assert(kHeads * DP * 4u <= kUnit, "a warp's sums join in a free unit");
};

template <typename T, int DP, int MT, bool EXTRA>
__global__ void __launch_bounds__(kAttnThreads, AttnShape<T, DP, MT, EXTRA>::kCtasPerSm)
    paged_attn_kernel(const PagedView c, const AttnArgs a, const __grid_constant__ AttnMaps maps) {
  using Shape = AttnShape<T, DP, MT, EXTRA>;
  constexpr uint32_t kTile = Shape::kTile, kLogTile = log_tile(DP), kLogBlock = kLogTile + 2u;
  static_assert(kWarps == 4u, "a block is four tiles");
  constexpr uint32_t kUnits = Shape::kUnits, kUnit = Shape::kUnit, kHeads = Shape::kHeads;
  constexpr int kTerms = EXTRA ? 3 : 2;
  constexpr int kSteps = kTile / 16;    // 16-slot steps of a product over slots
  constexpr uint32_t kPanels = Shape::kPanels, kPanel = kTile * 128u;
  extern __shared__ uint8_t smem_raw[];
  __shared__ float join_m[kWarps][kHeads], join_l[kWarps][kHeads], q_mult[kHeads];
  __shared__ __align__(8) uint64_t full[kWarps][kUnits];
  __shared__ uint64_t sum64[kWarps];
  __shared__ uint32_t most_of[kWarps];
  __shared__ uint32_t first_at[3];
  __shared__ uint32_t is_last;
  __shared__ float share[kHeads][64];

  const uint32_t tid = threadIdx.x, lane = tid & 31u, g = lane >> 2, t4 = lane & 3u;
  const uint32_t warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // the same in every lane, and known to be
  uint8_t* const smem = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
  uint8_t* const ring = smem + warp * (kUnits * kUnit);
  const uint32_t ring_at = smem_addr(ring), q_at = smem_addr(smem + Shape::kRing);
  if (lane == 0u) {
    for (uint32_t i = 0; i < kUnits; ++i) mbar_init(&full[warp][i], 1u);
    fence_mbar_init();
  }
  if (tid < 2u) {  // the tensor maps are kernel parameters: nothing to wait for
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(tid == 0u ? &maps.k : &maps.v)) : "memory");
  }

  pdl_wait();
  pdl_trigger();

  // ---- this CTA's range [r0, r1) of the line of units (blocks, and headers before each
  // segment's), or, where segments are short and many, a whole segment for every warp
  const uint32_t lines = c.n_kv * a.tiles;
  auto blocks_of = [&](uint32_t b, uint32_t& most) {
    Segment s;
    s.b = b;
    s.bounds(c, a, kLogTile);
    most = max(most, s.j1 - s.j0);
    s.bounds(c, a, kLogBlock);
    return s.j1 - s.j0;
  };
  uint64_t total = 0;  // blocks of one line of every sequence, then units of all lines
  uint32_t most = 0;   // tiles of the longest
  if (c.batch > kAttnThreads) {
    for (uint32_t b = tid; b < c.batch; b += kAttnThreads) total += blocks_of(b, most);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) total += __shfl_xor_sync(0xffffffffu, total, off);
    if (lane == 0u) sum64[warp] = total;
    __syncthreads();
    total = 0;
#pragma unroll
    for (uint32_t w = 0; w < kWarps; ++w) total += sum64[w];
  }
  uint64_t ctas = 0, r0 = 0, r1 = 0;
  const uint32_t segments = c.batch * lines;  // below 2^32: both are below 2^16
  bool solo_now = false;
  uint32_t header = 0;  // units of a segment that stand for its cost beside its blocks
  for (uint64_t base = 0, b0 = 0; b0 < c.batch; b0 += kAttnThreads) {
    const uint32_t b = static_cast<uint32_t>(b0) + tid;
    const uint64_t n = b < c.batch ? blocks_of(b, most) : 0u;
    uint64_t upto = n;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const uint64_t o = __shfl_up_sync(0xffffffffu, upto, off);
      if (lane >= static_cast<uint32_t>(off)) upto += o;
    }
    most = __reduce_max_sync(0xffffffffu, most);
    __syncthreads();
    if (lane == 31u) sum64[warp] = upto, most_of[warp] = most;
    __syncthreads();
    uint64_t all = 0;
#pragma unroll
    for (uint32_t w = 0; w < kWarps; ++w) {
      if (w < warp) upto += sum64[w];
      all += sum64[w];
    }
    if (b0 == 0u) {
      if (c.batch <= kAttnThreads) total = all;
#pragma unroll
      for (uint32_t w = 0; w < kWarps; ++w) most = max(most, most_of[w]);
      const uint64_t blocks = total * lines;
      if constexpr (Shape::kSolo) {
        // Time in fifths of a microsecond: a tile takes 12 in a warp, a block 12 in a CTA, a
        // segment 5 more in a warp and 10 in a CTA.  With every segment taken for the longest, a
        // segment a warp has to be the faster way.
        const uint64_t busy = min(static_cast<uint64_t>(gridDim.x), blocks);
        const uint64_t rounds = (segments + gridDim.x * kWarps - 1u) / (gridDim.x * kWarps);
        solo_now = rounds * (most * 12ull + 5u) * busy <= blocks * 12u + segments * 10ull;
        if (solo_now) break;
      }
      // fewer blocks than CTAs: a block each; otherwise segments cost more than their blocks
      if (blocks > gridDim.x) header = Shape::kHeader;
      total = blocks + static_cast<uint64_t>(header) * segments;
      ctas = min(static_cast<uint64_t>(gridDim.x), total);
      if (blockIdx.x >= ctas) return;
      r0 = blockIdx.x * total / ctas;
      r1 = (blockIdx.x + 1u) * total / ctas;
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
  const bool solo = Shape::kSolo && solo_now;
  const uint32_t log_step = solo ? kLogTile : kLogBlock, warp_slot = solo ? 0u : warp * kTile;
  Segment use;
  uint32_t use_index = 0, left = 0;  // left: units of the range, or steps of the segment, from use.j on
  auto skip_header = [&](uint32_t& units, uint32_t done) { units -= min(units, header - min(done, header)); };
  // segment `index` of the line for a lone warp
  auto take = [&](Segment& s, uint32_t index, uint32_t& steps) {
    steps = 0u;
    if (index >= segments) return;
    s.b = index / lines;
    s.h = index - s.b * lines;
    s.bounds(c, a, log_step);
    s.j = s.j0;
    steps = s.j1 - s.j0;
  };
  // the segment after one that is done
  auto advance = [&](Segment& s, uint32_t& index, uint32_t& steps) {
    if (solo) {
      index += gridDim.x * kWarps;
      take(s, index, steps);
    } else {
      skip_header(steps, 0u);
      if (++s.h == lines) {
        s.h = 0;
        ++s.b;
        if (steps != 0u) s.bounds(c, a, log_step);
      }
      s.j = s.j0;
    }
  };
  if (solo) {
    use_index = warp * gridDim.x + blockIdx.x;
    take(use, use_index, left);
  } else {
    use.b = first_at[0];
    use.h = first_at[1];
    use.bounds(c, a, log_step);
    left = static_cast<uint32_t>(r1 - r0);  // below 2^31
    skip_header(left, first_at[2]);
    use.j = use.j0 + (first_at[2] - min(first_at[2], header));
  }

  // A segment's queries as this lane of a CTA splits them: rows warp, warp + 4, .. of its head tile
  constexpr uint32_t kPer = DP / 32, kQRowsPerWarp = kHeads / kWarps;
  uint32_t q_raw[kQRowsPerWarp][kPer];  // fp32 words, or pairs of 16-bit values in the first half
  auto load_queries = [&](const Segment& s) {
    const uint32_t kv = s.h / a.tiles, ht = s.h - kv * a.tiles;
    const uint32_t heads = a.group - ht * kHeads;  // or more than the tile has
    const uint32_t bytes = a.dtype == QG_F32 ? 4u : 2u;
#pragma unroll
    for (uint32_t i = 0; i < kQRowsPerWarp; ++i) {
      const uint32_t r = warp + i * kWarps;
      const uint64_t row = s.b * a.q_stride + static_cast<uint64_t>(kv * a.group + ht * kHeads + r) * c.dim;
      const uint32_t* at = reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.q) +
                                                             (row + lane * kPer) * bytes);
      const bool has = r < heads && lane * kPer < c.dim;  // dim is a multiple of 8, kPer divides it
#pragma unroll
      for (uint32_t e = 0; e < kPer; ++e) {
        q_raw[i][e] = 0u;
        if (has && (e < kPer / 2u || a.dtype == QG_F32)) q_raw[i][e] = at[e];
      }
    }
  };
  if (!solo && left != 0u) load_queries(use);

  // ---- fetching.  A set of page ids covers the next 32 boxes of this warp's tiles, a box a
  // lane; the set after it is read while this one is used.
  const uint64_t policy = l2_evict_first_policy();
  const uint32_t boxes = 1u << a.log_boxes, log_box = kLogTile - a.log_boxes;
  Segment ahead = use;
  uint32_t ahead_index = use_index, ahead_left = left;
  int32_t page = 0, place = 0, head = 0, next_page = 0, next_place = 0, next_head = 0;
  uint32_t at_tile = 0, tiles = 0, next_tiles = 0;  // of the set
  auto look_up = [&]() {
    next_tiles = 0u;
    if (ahead_left == 0u) return;
    next_tiles = min(min(32u >> a.log_boxes, ahead.j1 - ahead.j), ahead_left);
    const uint32_t t = lane >> a.log_boxes;
    const uint32_t slot = ((ahead.j + t) << log_step) + warp_slot + ((lane & (boxes - 1u)) << log_box);
    const uint32_t at = div_by(slot, c.page);
    next_page = static_cast<int32_t>(c.num_pages);  // past the pool: a box of zeros
    next_place = static_cast<int32_t>(slot - at * c.page.d);
    next_head = static_cast<int32_t>(ahead.h / a.tiles);
    if (t < next_tiles && slot < ahead.len && slot + (1u << log_box) > ahead.start) {
      const uint32_t id = static_cast<uint32_t>(c.table[static_cast<size_t>(ahead.b) * c.table_stride + at]);
      if (id < c.num_pages) {
        next_page = static_cast<int32_t>(id);
      } else {
        atomicOr(&g_error_word, QG_ERR_PAGE);
      }
    }
    ahead.j += next_tiles;
    ahead_left -= next_tiles;
    if (ahead.j == ahead.j1) advance(ahead, ahead_index, ahead_left);
  };
  auto next_set = [&]() {
    page = next_page;
    place = next_place;
    head = next_head;
    tiles = next_tiles;
    at_tile = 0;
    look_up();
  };
  // the K (before its V) or V tile of the next block into unit u
  auto fetch = [&](uint32_t u, bool is_v) {
    if (!is_v && at_tile == tiles) next_set();
    if (at_tile == tiles) return;  // the range is fetched
    const uint32_t to = ring_at + u * kUnit, bar = smem_addr(&full[warp][u]);
    const CUtensorMap* map = is_v ? &maps.v : &maps.k;
    const bool leads = elect_one();
    if (leads) mbar_arrive_expect_tx(&full[warp][u], kUnit);
    for (uint32_t i = 0; i < boxes; ++i) {  // one lane asks: a copy takes warp-uniform operands
      const uint32_t from = ((at_tile << a.log_boxes) + i) & 31u;
      const int32_t pg = __shfl_sync(0xffffffffu, page, from), pl = __shfl_sync(0xffffffffu, place, from);
      if (leads) {
#pragma unroll
        for (uint32_t p = 0; p < kPanels; ++p) {
          tma_load_4d(to + p * kPanel + (i << log_box) * 128u, map, static_cast<int32_t>(p * 64u),
                      a.heads_inside ? head : pl, a.heads_inside ? pl : head, pg, bar, policy);
        }
      }
    }
    if (is_v) ++at_tile;
  };
  look_up();
#pragma unroll
  for (uint32_t u = 0; u < kUnits; ++u) fetch(u, (u & 1u) != 0u);
  bool fetch_v = (kUnits & 1u) != 0u;  // what the next free unit receives

  // ldmatrix rows and 16-byte pieces of this lane (K: 8 slots x 2 pieces x 2; V, transposed:
  // 16 slots x 2 pieces); piece 2 n of a panel is at lane_at ^ (n << 5)
  const uint32_t kr = (lane & 7u) + ((lane >> 4) << 3), vr = (lane & 7u) + ((lane >> 3) & 1u) * 8u;
  const uint32_t k_lane = kr * 128u + ((((lane >> 3) & 1u) ^ (kr & 7u)) << 4);
  const uint32_t v_lane = vr * 128u + (((lane >> 4) ^ (vr & 7u)) << 4);

  uint32_t qa[MT][DP / 16][4], qx[MT][EXTRA ? DP / 16 : 1][2];
  float o[MT][DP / 8][2], m[MT], l[MT], mult[MT];
  uint32_t unit = 0, parity = 0;
  bool arrives = true;
  auto await_unit = [&]() {
    if (!__all_sync(0xffffffffu, mbar_try_wait(&full[warp][unit], parity))) {
      arrives = arrives && __all_sync(0xffffffffu, mbar_wait_bounded(&full[warp][unit], parity));
    }
  };
  auto release_unit = [&](bool written) {
    if (written) fence_proxy_async_smem();
    __syncwarp();
    if (arrives) fetch(unit, fetch_v);
    fetch_v = !fetch_v;
    if (++unit == kUnits) {
      unit = 0;
      parity ^= 1u;
    }
  };

  while (left != 0u) {
    const uint32_t kv = use.h / a.tiles, ht = use.h - kv * a.tiles;
    const uint32_t heads = min(kHeads, a.group - ht * kHeads);
    const uint32_t head0 = kv * a.group + ht * kHeads;
    const uint32_t from_j = use.j, to_j = min(use.j1, use.j + left);
    // log-sum-exp of a finished head
    auto put_stats = [&](uint32_t h, float top, float sum) {
      const size_t at = static_cast<size_t>(use.b) * a.n_q + h;
      const float full_sum = sum == 0.f ? -CUDART_INF_F : top + log2f(sum) - kShareBits<T>;
      if (a.lse != nullptr) a.lse[at] = full_sum * 0.69314718055994530942f;
      if (a.norm != nullptr) a.norm[at] = full_sum;
    };

    // ---- the queries
    if (solo) {
      // A lone warp takes them as the A operand does: this lane has values 16 k + 2 t4, + 1, + 8
      // and + 9 of head g of every tile of 8.
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        constexpr uint32_t kK = DP / 16;
        const uint64_t at = use.b * a.q_stride + static_cast<uint64_t>(head0 + i * 8u + g) * c.dim + 2u * t4;
        float2 x[kK][2];
        float top = 0.f;
#pragma unroll
        for (uint32_t k = 0; k < kK; ++k) {
#pragma unroll
          for (uint32_t e = 0; e < 2; ++e) {
            const uint32_t d = 16u * k + 8u * e;
            x[k][e] = make_float2(0.f, 0.f);
            if (i * 8u + g < heads && d < c.dim) {
              if (a.dtype == QG_F32) {
                x[k][e] = *reinterpret_cast<const float2*>(static_cast<const float*>(a.q) + at + d);
              } else {
                const uint32_t w = *reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(a.q) + at + d);
                x[k][e] = a.dtype == QG_F16 ? unpack2(w, __half()) : unpack2(w, __nv_bfloat16());
              }
            }
            top = fmaxf(top, fmaxf(fabsf(x[k][e].x), fabsf(x[k][e].y)));
          }
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int power = power_of<T>(top);
        const float down = power_of_two(-power);
        mult[i] = a.scale_log2 * power_of_two(power);
#pragma unroll
        for (uint32_t k = 0; k < kK; ++k) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            uint32_t term[kTerms];
            split_terms<T>(x[k][e].x * down, x[k][e].y * down, term);
            qa[i][k][2 * e] = term[0];
            qa[i][k][2 * e + 1] = term[1];
            if constexpr (EXTRA) qx[i][k][e] = term[2];
          }
        }
      }
    } else {
#pragma unroll
      for (uint32_t row = 0; row < kQRowsPerWarp; ++row) {
        const uint32_t r = warp + row * kWarps;
        float x[kPer];
        if (a.dtype == QG_F32) {
#pragma unroll
          for (uint32_t e = 0; e < kPer; ++e) x[e] = __uint_as_float(q_raw[row][e]);
        } else {
#pragma unroll
          for (uint32_t e = 0; e < kPer / 2u; ++e) {
            const float2 f = a.dtype == QG_F16 ? unpack2(q_raw[row][e], __half()) : unpack2(q_raw[row][e], __nv_bfloat16());
            x[2u * e] = f.x;
            x[2u * e + 1u] = f.y;
          }
        }
        float top = 0.f;
#pragma unroll
        for (uint32_t e = 0; e < kPer; ++e) top = fmaxf(top, fabsf(x[e]));
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        const int power = power_of<T>(top);
        const float down = power_of_two(-power);
        if (lane == 0u) q_mult[r] = a.scale_log2 * power_of_two(power);
#pragma unroll
        for (uint32_t e = 0; e < kPer; e += 2) {
          uint32_t term[kTerms];
          split_terms<T>(x[e] * down, x[e + 1] * down, term);
          const uint32_t d = lane * kPer + e;
#pragma unroll
          for (int i = 0; i < kTerms; ++i) {
            const uint32_t qr = (r / 8u) * (EXTRA ? 24u : 16u) + i * 8u + (r & 7u);
            *reinterpret_cast<uint32_t*>(smem + Shape::kRing + qr * (DP * 2u) + (((d / 8u) ^ (qr & 7u)) << 4) +
                                         (d & 7u) * 2u) = term[i];
          }
        }
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const uint32_t r0q = i * (EXTRA ? 24u : 16u);
#pragma unroll
        for (uint32_t kk = 0; kk < DP / 16; ++kk) {
          const uint32_t r = r0q + (lane & 7u) + ((lane >> 3) & 1u) * 8u, ch = 2u * kk + (lane >> 4);
          ldsm_x4(qa[i][kk], q_at + r * (DP * 2u) + ((ch ^ (r & 7u)) << 4));
          if constexpr (EXTRA) {
            const uint32_t rx = r0q + 16u + g;
#pragma unroll
            for (uint32_t e = 0; e < 2; ++e) {
              qx[i][kk][e] = *reinterpret_cast<const uint32_t*>(smem + Shape::kRing + rx * (DP * 2u) +
                                                                (((2u * kk + e) ^ (rx & 7u)) << 4) + t4 * 4u);
            }
          }
        }
        mult[i] = q_mult[i * 8 + g];
      }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      m[i] = -CUDART_INF_F;
      l[i] = 0.f;
#pragma unroll
      for (uint32_t n = 0; n < DP / 8; ++n) o[i][n][0] = o[i][n][1] = 0.f;
    }

    for (; use.j < to_j; ++use.j) {
      const uint32_t slot0 = (use.j << log_step) + warp_slot;
      const bool whole = slot0 >= use.start && slot0 + kTile <= use.len;
      const bool seen = slot0 < use.len && slot0 + kTile > use.start;
      // ---- scores
      uint32_t p[MT][kSteps][2][kTerms];  // probabilities: [16-slot step][8-slot half][term]
      float fade[MT];
      await_unit();
      if (seen && arrives) {
        float s[MT][2 * kSteps][4], sx[MT][2 * kSteps][EXTRA ? 4 : 1];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
#pragma unroll
          for (int n = 0; n < 2 * kSteps; ++n) {
#pragma unroll
            for (int e = 0; e < 4; ++e) s[i][n][e] = 0.f;
#pragma unroll
            for (int e = 0; e < (EXTRA ? 4 : 1); ++e) sx[i][n][e] = 0.f;
          }
        }
        const uint32_t k_at = ring_at + unit * kUnit;
#pragma unroll
        for (uint32_t kk = 0; kk < DP / 16; ++kk) {
#pragma unroll
          for (int st = 0; st < kSteps; ++st) {
            uint32_t kb[4];
            ldsm_x4(kb, k_at + (k_lane ^ ((kk & 3u) << 5)) + kk / 4u * kPanel + st * 2048u);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              const uint32_t* q = qa[i][kk];
              mma(s[i][2 * st], q[0], q[1], q[2], q[3], kb[0], kb[1], T());
              mma(s[i][2 * st + 1], q[0], q[1], q[2], q[3], kb[2], kb[3], T());
              if constexpr (EXTRA) {
                mma(sx[i][2 * st], qx[i][kk][0], 0u, qx[i][kk][1], 0u, kb[0], kb[1], T());
                mma(sx[i][2 * st + 1], qx[i][kk][0], 0u, qx[i][kk][1], 0u, kb[2], kb[3], T());
              }
            }
          }
        }
        // ---- probabilities: this thread's head is 8 i + g, its slots 8 n + 2 t4 and one more
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          float x[2 * kSteps][2];
          float top = -CUDART_INF_F;
#pragma unroll
          for (int n = 0; n < 2 * kSteps; ++n) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float hi = s[i][n][e];
              float lo = s[i][n][e + 2];
              if constexpr (EXTRA) lo += sx[i][n][e];
              // an infinite key: the errors' products are not numbers, the first term's sum is right
              x[n][e] = (fabsf(hi) == CUDART_INF_F ? hi : hi + lo) * mult[i];
              const uint32_t slot = slot0 + n * 8u + 2u * t4 + e;
              if (!whole && (slot < use.start || slot >= use.len)) x[n][e] = -CUDART_INF_F;
            }
            if (a.scores != nullptr && i * 8u + g < heads) {
              const size_t row = static_cast<size_t>(use.b) * a.n_q + head0 + i * 8u + g;
              *reinterpret_cast<float2*>(a.scores + row * a.score_stride + slot0 + n * 8u + 2u * t4) =
                  make_float2(x[n][0], x[n][1]);
            }
            top = fmaxf(top, fmaxf(x[n][0], x[n][1]));
          }
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const float now = fmaxf(m[i], top);
          const float from = now == -CUDART_INF_F ? 0.f : now;
          fade[i] = exp2_fast(m[i] - from);
          m[i] = now;
          const float base = kShareBits<T> - from;
          float sum = 0.f;
#pragma unroll
          for (int n = 0; n < 2 * kSteps; ++n) {
            x[n][0] = exp2_fast(x[n][0] + base);
            x[n][1] = exp2_fast(x[n][1] + base);
            sum += x[n][0] + x[n][1];
            split_terms<T>(x[n][0], x[n][1], p[i][n / 2][n % 2]);
          }
          l[i] = fmaf(l[i], fade[i], sum);
        }
      }
      release_unit(false);

      // ---- weighted values
      await_unit();
      bool written = false;  // by this warp, where the next box will land
      if (seen && arrives) {
        if (!whole) {  // V rows beside the sequence's ends: 0 x NaN must not reach the sums
          written = true;
          for (uint32_t i = lane; i < kTile * DP / 8u; i += 32u) {
            const uint32_t slot = slot0 + i / 8u % kTile;
            if (slot < use.start || slot >= use.len) {
              reinterpret_cast<uint4*>(ring + unit * kUnit)[i] = make_uint4(0u, 0u, 0u, 0u);
            }
          }
          __syncwarp();
        }
        const uint32_t v_at = ring_at + unit * kUnit;
#pragma unroll
        for (uint32_t n = 0; n < DP / 16; ++n) {
          uint32_t vb[kSteps][4];
#pragma unroll
          for (int st = 0; st < kSteps; ++st) {
            ldsm_x4_trans(vb[st], v_at + (v_lane ^ ((n & 3u) << 5)) + n / 4u * kPanel + st * 2048u);
          }
#pragma unroll
          for (int i = 0; i < MT; ++i) {
#pragma unroll
            for (uint32_t e = 0; e < 2; ++e) {
              float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int st = 0; st < kSteps; ++st) {
                const auto& ps = p[i][st];
                mma(d, ps[0][0], ps[0][1], ps[1][0], ps[1][1], vb[st][2 * e], vb[st][2 * e + 1], T());
                if constexpr (EXTRA) {
                  mma(d, ps[0][kTerms - 1], 0u, ps[1][kTerms - 1], 0u, vb[st][2 * e], vb[st][2 * e + 1], T());
                }
              }
              o[i][2 * n + e][0] = fmaf(o[i][2 * n + e][0], fade[i], d[0] + d[2]);
              o[i][2 * n + e][1] = fmaf(o[i][2 * n + e][1], fade[i], d[1] + d[3]);
            }
          }
        }
      }
      __syncwarp();
      if (use.j + 1u < to_j) release_unit(written);  // the last one is where the warp joins
    }
    left -= to_j - from_j;

    // ---- the end of the segment, or of the range inside it
    Segment after = use;
    const uint64_t here = r1 - left;  // the unit after this segment's part
    if (use.j == use.j1) advance(after, use_index, left);
    if (!solo && left != 0u) load_queries(after);  // on their way while this segment joins
    if (solo) {
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const uint32_t h = i * 8u + g;
        float sum = l[i];
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        if (h >= heads) continue;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        const size_t at = use.b * a.out_stride + static_cast<size_t>(head0 + h) * c.dim + 2u * t4;
#pragma unroll
        for (uint32_t n = 0; n < DP / 8; ++n) {
          if (n * 8u >= c.dim) break;
          const float u = o[i][n][0] * inv, v = o[i][n][1] * inv;
          if (a.dtype == QG_F32) {
            *reinterpret_cast<float2*>(static_cast<float*>(a.out) + at + n * 8u) = make_float2(u, v);
          } else {
            *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + at + n * 8u) =
                a.dtype == QG_F16 ? pack2(u, v, __half()) : pack2(u, v, __nv_bfloat16());
          }
        }
        if (t4 == 0u) put_stats(head0 + h, m[i], sum);
      }
    } else {
      const bool mine = from_j == use.j0 && to_j == use.j1;
      // each warp's sums into the unit it has just used, float4 pieces swizzled by head
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        float sum = l[i];
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        if (t4 == 0u) {
          join_m[warp][i * 8 + g] = m[i];
          join_l[warp][i * 8 + g] = sum;
        }
        float2* to = reinterpret_cast<float2*>(ring + unit * kUnit) + (i * 8u + g) * (DP / 2u);
#pragma unroll
        for (uint32_t n = 0; n < DP / 8; ++n) {
          to[(n * 4u + t4) ^ ((g & 3u) << 2)] = make_float2(o[i][n][0], o[i][n][1]);
        }
      }
      __syncthreads();
      float* record = a.records + (static_cast<size_t>(blockIdx.x) * 2u + (from_j == use.j0 ? 1u : 0u)) * Shape::kRecord;
      auto finish = [&](uint32_t h, uint32_t ch, float top, float sum, float4 v) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        v.x *= inv, v.y *= inv, v.z *= inv, v.w *= inv;
        const size_t at = use.b * a.out_stride + static_cast<size_t>(head0 + h) * c.dim + ch * 4u;
        if (ch * 4u < c.dim) {
          if (a.dtype == QG_F32) {
            *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = v;
          } else if (a.dtype == QG_F16) {
            *reinterpret_cast<uint2*>(static_cast<__half*>(a.out) + at) =
                make_uint2(pack2(v.x, v.y, __half()), pack2(v.z, v.w, __half()));
          } else {
            *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + at) =
                make_uint2(pack2(v.x, v.y, __nv_bfloat16()), pack2(v.z, v.w, __nv_bfloat16()));
          }
        }
        if (ch == 0u) put_stats(head0 + h, top, sum);
      };
      for (uint32_t i = tid; i < heads * (DP / 4u); i += kAttnThreads) {
        const uint32_t h = i / (DP / 4u), ch = i % (DP / 4u);
        float top = join_m[0][h];
#pragma unroll
        for (uint32_t w = 1; w < kWarps; ++w) top = fmaxf(top, join_m[w][h]);
        const float from = top == -CUDART_INF_F ? 0.f : top;
        float sum = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (uint32_t w = 0; w < kWarps; ++w) {
          const float f = exp2_fast(join_m[w][h] - from);
          const float4 x = reinterpret_cast<const float4*>(smem + (w * kUnits + unit) * kUnit)
              [h * (DP / 4u) + (ch ^ ((h & 3u) << 1))];
          sum = fmaf(join_l[w][h], f, sum);
          v.x = fmaf(x.x, f, v.x), v.y = fmaf(x.y, f, v.y);
          v.z = fmaf(x.z, f, v.z), v.w = fmaf(x.w, f, v.w);
        }
        if (mine) {
          finish(h, ch, top, sum, v);
        } else {
          if (ch == 0u) {
            record[h] = top;
            record[kHeads + h] = sum;
          }
          reinterpret_cast<float4*>(record + 2u * kHeads)[h * (DP / 4u) + ch] = v;
        }
      }
      if (!mine) {
        // the CTAs that share this head own its first to its last block, in order
        const uint64_t seg0 = here - (to_j - use.j0), seg1 = seg0 + (use.j1 - use.j0);
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
        // joins the n <= 64 records of CTAs first, first + step, ..; put(head, piece, m, l, o)
        auto join_records = [&](uint32_t first, uint32_t step, uint32_t n, auto put) {
          constexpr uint32_t kItems = kHeads * (DP / 4u) / kAttnThreads;      // float4 pieces of a thread
          constexpr uint32_t kOnce = kItems < 2u ? 1u : 2u;                   // .. that it works on together
          float4 x[kOnce][kInFlight];
          auto ask = [&](uint32_t i0, uint32_t q0) {
#pragma unroll
            for (uint32_t q = 0; q < kInFlight; ++q) {
              const float4* rec = reinterpret_cast<const float4*>(record_of(first + (q0 + q) * step) + 2u * kHeads);
#pragma unroll
              for (uint32_t e = 0; e < kOnce; ++e) {
                const uint32_t i = (i0 + e) * kAttnThreads + tid;
                x[e][q] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (q0 + q < n && i < heads * (DP / 4u)) x[e][q] = __ldcg(rec + i);
              }
            }
          };
          ask(0u, 0u);
          constexpr uint32_t kHeadsPerWarp = kHeads / kWarps;
          float pm[kHeadsPerWarp][2], pl[kHeadsPerWarp][2];  // two records a lane
#pragma unroll
          for (uint32_t e = 0; e < 2; ++e) {
            const uint32_t q = lane + 32u * e;
            const float* rec = record_of(first + min(q, n - 1u) * step);
#pragma unroll
            for (uint32_t i = 0; i < kHeadsPerWarp; ++i) {
              const uint32_t h = warp + i * kWarps;
              pm[i][e] = q < n && h < heads ? __ldcg(rec + h) : -CUDART_INF_F;
              pl[i][e] = q < n && h < heads ? __ldcg(rec + kHeads + h) : 0.f;
            }
          }
#pragma unroll
          for (uint32_t i = 0; i < kHeadsPerWarp; ++i) {
            const uint32_t h = warp + i * kWarps;
            float top = fmaxf(pm[i][0], pm[i][1]);
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
            const float from = top == -CUDART_INF_F ? 0.f : top;
            const float f0 = exp2_fast(pm[i][0] - from), f1 = exp2_fast(pm[i][1] - from);
            float all = fmaf(pl[i][0], f0, pl[i][1] * f1);
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) all += __shfl_xor_sync(0xffffffffu, all, off);
            share[h][lane] = f0;
            share[h][lane + 32u] = f1;
            if (lane == 0u) join_m[0][h] = top, join_l[0][h] = all;
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
              const uint32_t i = (i0 + e) * kAttnThreads + tid, h = i / (DP / 4u);
              if (h < heads) put(h, i % (DP / 4u), join_m[0][h], join_l[0][h], v[e]);
            }
          }
        };
        auto to_record = [&](float* rec) {
          return [=](uint32_t h, uint32_t ch, float top, float sum, float4 v) {
            if (ch == 0u) rec[h] = top, rec[kHeads + h] = sum;
            reinterpret_cast<float4*>(rec + 2u * kHeads)[h * (DP / 4u) + ch] = v;
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
      __syncthreads();  // the units, the joins and the queries are free again
    }
    release_unit(true);
    use = after;
  }
  if (!arrives) {  // a wait ran out (QG_ERR_WAIT_TIMEOUT is set): let what is in flight land
    for (uint32_t i = 0; i < kUnits; ++i) {
      const uint32_t u = unit + i < kUnits ? unit + i : unit + i - kUnits;
      mbar_wait_bounded(&full[warp][u], unit + i < kUnits ? parity : parity ^ 1u);
    }
  }
}

// weight_out = weight_in + the slot's shares summed over the heads of its kv head.
constexpr uint32_t kWeightThreads = 128, kWeightSlots = 4;  // of a thread, a block's width apart

__global__ void __launch_bounds__(kWeightThreads) attn_weight_kernel(const PagedView c, const AttnArgs a,
                                                                     const float* weight_in, float* weight_out,
                                                                     uint32_t weight_stride) {
  pdl_wait();
  pdl_trigger();
  const uint32_t kv = blockIdx.y, b = blockIdx.z, j0 = blockIdx.x * (kWeightThreads * kWeightSlots) + threadIdx.x;
  const uint32_t len = paged_len(a.lens[b], min(a.max_len, c.capacity));
  if (j0 - threadIdx.x >= len) return;
  const uint32_t start = a.window != 0u && len > a.window ? len - a.window : 0u;
  const size_t head = static_cast<size_t>(b) * a.n_q + kv * a.group;
  const size_t row = (static_cast<size_t>(b) * c.n_kv + kv) * weight_stride;
  float old[kWeightSlots], sum[kWeightSlots];
#pragma unroll
  for (uint32_t u = 0; u < kWeightSlots; ++u) {
    const uint32_t j = j0 + u * kWeightThreads;
    old[u] = weight_in != nullptr && j < len ? weight_in[row + j] : 0.f;
    sum[u] = 0.f;
  }
#pragma unroll 2
  for (uint32_t h = 0; h < a.group; ++h) {
    // minus infinity: no seen score of the head is above it, so its output is zero and so are its shares
    const float norm = a.norm[head + h], full = norm == -CUDART_INF_F ? 0.f : norm;
    const float* scores = a.scores + (head + h) * a.score_stride;
#pragma unroll
    for (uint32_t u = 0; u < kWeightSlots; ++u) {
      const uint32_t j = j0 + u * kWeightThreads;
      if (j >= start && j < len) sum[u] += exp2_fast(scores[j] - full);
    }
  }
#pragma unroll
  for (uint32_t u = 0; u < kWeightSlots; ++u) {
    const uint32_t j = j0 + u * kWeightThreads;
    if (j < len) weight_out[row + j] = old[u] + sum[u];
  }
}

// ---- host side

struct AttnPlan {
  uint32_t dp, mt, tiles, record, score_stride;
  size_t records_at, scores_at, norm_at, bytes;
};

constexpr size_t round_up(size_t v) { return (v + 255u) & ~static_cast<size_t>(255u); }

bool plan_attn(const PagedView& c, uint32_t n_q, uint32_t max_len, bool weights,
               bool extra, AttnPlan* p) {
  if (n_q == 0u || n_q > 65535u || n_q % c.n_kv != 0u || max_len == 0u || max_len > 0x7fffffffu) return false;
  const uint32_t group = n_q / c.n_kv;
  p->dp = c.dim <= 64u ? 64u : c.dim <= 128u ? 128u : 256u;
  // two tiles of 8 heads share a pass over the slots where their registers allow it
  p->mt = group > 8u && (p->dp == 64u || (p->dp == 128u && !extra)) ? 2u : 1u;
  p->tiles = (group + 8u * p->mt - 1u) / (8u * p->mt);
  p->record = 8u * p->mt * (p->dp + 2u);
  p->records_at = QG_PAGED_ATTN_ZEROED;
  p->scores_at = round_up(p->records_at + static_cast<size_t>(kMaxCtas) * 2u * p->record * 4u);
  const uint32_t block = block_slots(p->dp);
  const size_t stride = (max_len + block - 1u) / block * block;
  p->score_stride = static_cast<uint32_t>(stride);
  p->norm_at = round_up(p->scores_at + (weights ? static_cast<size_t>(c.batch) * n_q * stride * 4u : 0u));
  p->bytes = round_up(p->norm_at + (weights ? static_cast<size_t>(c.batch) * n_q * 4u : 0u));
  return true;
}

// Strides of a tensor map nest: each is a multiple of the one inside it (a dimension of one
// entry takes whatever fits).  False where the pools' do not.
struct PoolStrides {
  uint64_t inner, outer, page;  // bytes
  bool heads_inside;
};
bool pool_strides(const qg_kv_pages* cache, PoolStrides* s) {
  uint64_t head = cache->head_stride * 2u, slot = cache->slot_stride * 2u;
  const uint64_t row = cache->head_dim * 2u;
  s->heads_inside = cache->n_kv_heads != 1u && (cache->page_size == 1u || head < slot);
  if (cache->n_kv_heads == 1u) head = cache->page_size == 1u ? row : slot;
  if (cache->page_size == 1u) slot = head;
  s->inner = s->heads_inside ? head : slot;
  s->outer = s->heads_inside ? slot : head;
  s->page = cache->num_pages == 1u ? s->outer : cache->page_stride * 2u;
  return s->inner >= row && s->inner % 16u == 0u && s->outer >= s->inner && s->outer % s->inner == 0u &&
         s->page >= s->outer && s->page % s->outer == 0u && s->page < (1ull << 40);
}

bool encode_pool(CUtensorMap* map, void* pool, const qg_kv_pages* cache, const PoolStrides& s, uint32_t box_slots) {
  const auto encode = tensor_map_encoder();
  if (encode == nullptr) return false;
  const uint32_t inner = s.heads_inside ? cache->n_kv_heads : cache->page_size;
  const uint32_t outer = s.heads_inside ? cache->page_size : cache->n_kv_heads;
  const cuuint64_t dims[4] = {cache->head_dim, inner, outer, cache->num_pages};
  const cuuint64_t strides[3] = {s.inner, s.outer, s.page};
  const cuuint32_t box[4] = {64u, s.heads_inside ? 1u : box_slots, s.heads_inside ? box_slots : 1u, 1u};
  const cuuint32_t step[4] = {1u, 1u, 1u, 1u};
  return encode(map, cache->dtype == QG_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                pool, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int DP, int MT, bool EXTRA>
cudaError_t launch_attn(const PagedView& c, const AttnArgs& a, const AttnMaps& maps, cudaStream_t stream) {
  using Shape = AttnShape<T, DP, MT, EXTRA>;
  const auto kernel = paged_attn_kernel<T, DP, MT, EXTRA>;
  static SmemAttr attr;
  const cudaError_t e = attr.set(reinterpret_cast<const void*>(kernel), Shape::kSmem);
  if (e != cudaSuccess) return e;
  const uint64_t blocks = static_cast<uint64_t>(c.batch) * c.n_kv * a.tiles *
                          ((std::min(a.max_len, c.capacity) + Shape::kBlock - 1u) / Shape::kBlock);
  const uint64_t fit = static_cast<uint64_t>(paged_sm_count()) * Shape::kCtasPerSm;
  const uint32_t grid = static_cast<uint32_t>(std::min<uint64_t>(std::min<uint64_t>(blocks, fit), kMaxCtas));
  if (blocks / grid >= (1ull << 29)) return cudaErrorInvalidValue;  // a CTA counts its units in 32 bits
  return launch_k(kernel, grid, kAttnThreads, Shape::kSmem, stream, c, a, maps);
}

template <typename T>
cudaError_t launch_attn(const AttnPlan& p, bool extra, const PagedView& c, const AttnArgs& a,
                        const AttnMaps& maps, cudaStream_t stream) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    if (extra) {
      if (p.dp == 64u && p.mt == 2u) return launch_attn<T, 64, 2, true>(c, a, maps, stream);
      if (p.dp == 64u) return launch_attn<T, 64, 1, true>(c, a, maps, stream);
      if (p.dp == 128u) return launch_attn<T, 128, 1, true>(c, a, maps, stream);
      return launch_attn<T, 256, 1, true>(c, a, maps, stream);
    }
  }
  if (p.dp == 64u && p.mt == 2u) return launch_attn<T, 64, 2, false>(c, a, maps, stream);
  if (p.dp == 64u) return launch_attn<T, 64, 1, false>(c, a, maps, stream);
  if (p.dp == 128u && p.mt == 2u) return launch_attn<T, 128, 2, false>(c, a, maps, stream);
  if (p.dp == 128u) return launch_attn<T, 128, 1, false>(c, a, maps, stream);
  return launch_attn<T, 256, 1, false>(c, a, maps, stream);
}

}  // namespace
}  // namespace qg

extern "C" cudaError_t qg_paged_attn_workspace_bytes(const qg_kv_pages* cache, uint32_t n_q_heads,
                                                     uint32_t max_len, int weights, size_t* bytes) {
  using namespace qg;
  PagedView c;
  AttnPlan p0, p1;
  if (bytes == nullptr || !paged_view(cache, &c)) return cudaErrorInvalidValue;
  // the type of the queries is not known here: the larger of both forms
  if (!plan_attn(c, n_q_heads, max_len, weights != 0, false, &p0) ||
      !plan_attn(c, n_q_heads, max_len, weights != 0, true, &p1)) {
    return cudaErrorInvalidValue;
  }
  *bytes = std::max(p0.bytes, p1.bytes);
  return cudaSuccess;
}

extern "C" cudaError_t qg_paged_attn(const qg_kv_pages* cache, const qg_attn* p, void* workspace,
                                     cudaStream_t stream) {
  using namespace qg;
  PagedView c;
  if (!paged_view(cache, &c) || p == nullptr || !dtype_ok(p->dtype)) return cudaErrorInvalidValue;
  const bool weights = p->weight_out != nullptr;
  const bool extra = cache->dtype == QG_BF16 && p->dtype == QG_F32;
  AttnPlan plan;
  if (!plan_attn(c, p->n_q_heads, p->max_len, weights, extra, &plan)) return cudaErrorInvalidValue;
  const uint64_t piece = 16u / dtype_bytes(p->dtype);
  if (p->q == nullptr || p->out == nullptr || p->lens == nullptr || workspace == nullptr ||
      p->q_stride % piece != 0u || p->out_stride % piece != 0u || !aligned16(p->q) || !aligned16(p->out) ||
      (reinterpret_cast<uintptr_t>(workspace) & 255u) != 0u ||
      (weights && p->weight_stride < p->max_len) || (!weights && p->weight_in != nullptr)) {
    return cudaErrorInvalidValue;
  }
  PoolStrides strides;
  if (!pool_strides(cache, &strides)) return cudaErrorInvalidValue;
  // a box is gcd(tile, page_size) slots
  const uint32_t log_box = std::min<uint32_t>(log_tile(plan.dp), __builtin_ctz(cache->page_size));
  const uint32_t box = 1u << log_box;
  AttnMaps maps;
  if (!encode_pool(&maps.k, cache->k, cache, strides, box) || !encode_pool(&maps.v, cache->v, cache, strides, box)) {
    return cudaErrorNotSupported;
  }
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  AttnArgs a{};
  a.log_boxes = log_tile(plan.dp) - log_box;
  a.heads_inside = strides.heads_inside;
  a.q = p->q;
  a.out = p->out;
  a.dtype = p->dtype;
  a.q_stride = p->q_stride;
  a.out_stride = p->out_stride;
  a.lens = p->lens;
  a.max_len = p->max_len;
  a.window = p->window;
  a.n_q = p->n_q_heads;
  a.group = p->n_q_heads / c.n_kv;
  a.tiles = plan.tiles;
  a.scale_log2 = p->scale * 1.44269504088896340736f;
  a.lse = p->lse;
  a.arrived = reinterpret_cast<uint32_t*>(ws);
  a.records = reinterpret_cast<float*>(ws + plan.records_at);
  a.scores = weights ? reinterpret_cast<float*>(ws + plan.scores_at) : nullptr;
  a.norm = weights ? reinterpret_cast<float*>(ws + plan.norm_at) : nullptr;
  a.score_stride = plan.score_stride;
  const cudaError_t e = cache->dtype == QG_F16 ? launch_attn<__half>(plan, extra, c, a, maps, stream)
                                               : launch_attn<__nv_bfloat16>(plan, extra, c, a, maps, stream);
  if (e != cudaSuccess || !weights) return e;
  constexpr uint32_t kSpan = kWeightThreads * kWeightSlots;
  const dim3 grid((std::min(p->max_len, c.capacity) + kSpan - 1u) / kSpan, c.n_kv, c.batch);
  return launch_k(attn_weight_kernel, grid, kWeightThreads, 0, stream, c, a, p->weight_in, p->weight_out,
                  p->weight_stride);
}

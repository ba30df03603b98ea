// qg_paged8_attn.cuh -- what the two attention kernels over the 8-bit paged cache share: a call's
// arguments, row tiles, the slots that a tile sees, and the list of tiles of a ragged call.
//
// A row is one query head of one new token.  The rows of a sequence and kv head that share its
// keys and values, token after token, are cut into tiles; a tile of one kv head is a segment of
// work over the blocks of slots that any of its rows sees: the first `sinks` slots, and those from
// `start` to `len`.
#pragma once

#include "qg_paged8.cuh"

namespace qg {

struct Attn8Args {
  const void* q;
  void* out;
  int dtype;
  uint64_t q_stride, out_stride;  // elements
  const int32_t *lens, *offsets;
  uint32_t tokens, window, sink;
  uint32_t n_q, tiles;            // query heads; row tiles of a sequence of a call of one row each
  FastDiv group;                  // query heads of a kv head
  float scale_log2;
  float* lse;
  uint32_t* arrived;              // counters, zero between calls
  float* records;                 // partial results
  // of a ragged call
  uint32_t* item_count;           // [0] tiles, [1] steps of the longest
  uint4* items;                   // [tile] {sequence, first token's row, its slot, first row's head | rows << 16}
  uint64_t* item_blocks;          // [tile + 1] blocks of all tiles before
  uint32_t* seq_tiles;            // [batch + 1] tiles of all sequences before
  uint32_t max_items;
  uint32_t log_boxes;             // log2 of the boxes of a copied tile
  bool heads_inside;              // a page's heads lie inside its slots ([place][head][dim])
};

// One segment: rows [0, rows) of the tile are query heads of kv head `kv`, the first one head `sub`
// of the row `token`, whose slot is p0.  Step j of the work is block j, or block j + gap from step
// `gap_at` on.
struct Segment8 {
  uint32_t item, line;  // of the call's segments: tile (sequence), kv head (kv head and tile)
  uint32_t b, kv, token, sub, rows;
  int32_t p0, p1;       // slots of the first and the last token
  uint32_t len, start, sinks;
  uint32_t j, j1, gap_at, gap;

  __device__ __forceinline__ void bounds(const Attn8Args& a, uint32_t log) {
    p1 = p0 + static_cast<int32_t>(div_by(sub + rows - 1u, a.group));
    len = static_cast<uint32_t>(max(p1 + 1, 0));
    start = a.window != 0u && p0 >= 0 && static_cast<uint32_t>(p0) >= a.window ? p0 + 1u - a.window : 0u;
    sinks = min(a.sink, start);
    const uint32_t end = len == 0u ? 1u : ((len - 1u) >> log) + 1u;  // an empty tile has one empty step
    const uint32_t first = start >> log, sink_blocks = (sinks + (1u << log) - 1u) >> log;
    gap = first > sink_blocks ? first - sink_blocks : 0u;
    gap_at = sink_blocks;
    j1 = end - gap;
  }
  __device__ __forceinline__ uint32_t block(uint32_t at) const { return at + (at >= gap_at ? gap : 0u); }
  // whether any row, and whether every row, sees slots [from, from + n)
  __device__ __forceinline__ bool some_see(uint32_t from, uint32_t n) const {
    return from < len && (from + n > start || from < sinks);
  }
  __device__ __forceinline__ bool all_see(const Attn8Args& a, uint32_t from, uint32_t n) const {
    return static_cast<int32_t>(from + n) <= p0 + 1 &&
           (a.window == 0u || static_cast<uint32_t>(p1) - from < a.window || from + n <= a.sink);
  }
};
// whether the token of slot p sees slot j
__device__ __forceinline__ bool sees(const Attn8Args& a, int32_t p, uint32_t j) {
  return static_cast<int32_t>(j) <= p && (a.window == 0u || static_cast<uint32_t>(p) - j < a.window || j < a.sink);
}

// Where unit r0 of a ragged call's line lies: the line is the blocks of all segments, `header` units before
// each segment's, `lines` segments a tile.  A whole warp takes part.
__device__ __forceinline__ void find_unit8(const Attn8Args& a, uint32_t n, uint32_t lines, uint32_t header, uint64_t r0,
                                           uint32_t& item, uint32_t& line, uint32_t& in_segment) {
  auto before = [&](uint32_t i) { return (a.item_blocks[i] + static_cast<uint64_t>(header) * i) * lines; };
  uint32_t lo = 0, hi = n;  // the tile lies in [lo, hi)
  while (hi - lo > 1u) {
    const uint32_t step = (hi - lo + 31u) / 32u, at = lo + (threadIdx.x & 31u) * step;
    const uint32_t ok = __ballot_sync(0xffffffffu, at < hi && before(at) <= r0);
    lo += (31u - __clz(ok)) * step;
    hi = min(hi, lo + step);
  }
  const uint64_t in = r0 - before(lo), units = (before(lo + 1u) - before(lo)) / lines;
  item = lo;
  line = static_cast<uint32_t>(in / units);
  in_segment = static_cast<uint32_t>(in % units);
}
// A tile of a ragged call and one of its kv heads.
__device__ __forceinline__ void take_item8(const Attn8Args& a, Segment8& s, bool fresh, uint32_t log) {
  if (fresh) {
    const uint4 it = a.items[s.item];
    s.b = it.x, s.token = it.y, s.p0 = static_cast<int32_t>(it.z);
    s.sub = it.w & 0xffffu, s.rows = it.w >> 16;
    s.bounds(a, log);
  }
  s.kv = s.line;
  s.j = 0u;
}

// The tiles of `rows` rows of a ragged call, how many blocks of 2^log slots each sees, and how many of
// 2^log_tile the longest, before the attention reads them.
cudaError_t launch_plan8(const Paged8View& c, const Attn8Args& a, uint32_t rows, uint32_t log, uint32_t log_tile,
                         cudaStream_t stream);

// ---- the kernel for many rows (qg_paged8_prompt.cu)
constexpr uint32_t kPromptRows = 256;
constexpr uint32_t kMaxPromptCtas = 148;
// bytes of its records
constexpr size_t prompt8_bytes(uint32_t dp) {
  return static_cast<size_t>(kMaxPromptCtas) * 2u * kPromptRows * (dp + 2u) * 4u;
}
// 16-bit queries and heads up to 128 wide, where a sequence has `kPromptFrom` rows or more for a kv head on average;
// us of this and of the other kernel, 16 sequences of 4000 slots (32/8 heads x 128): 16 rows 104 and 66, 32 rows 105
// and 94, 64 rows 106 and 149, 512 rows 203 and 919; of 600 slots 43 and 44, 45 and 51, 45 and 70, 78 and 205.
// The host knows the cache's sequences, not which of them have rows: the average is over all (over as many as
// rows where those are fewer).  So a lone prompt in a large cache can miss this kernel: 1000 tokens of 4000 slots, 64/8
// heads x 128, 175 us in a cache of up to 200 sequences, 746 in one of more.
constexpr uint32_t kPromptFrom = 40;
inline bool prompt8_fits(uint32_t dp, uint64_t tokens, uint32_t batch, uint32_t group) {
  return dp <= 128u && tokens * group >= static_cast<uint64_t>(kPromptFrom) * (tokens < batch ? tokens : batch);
}
cudaError_t launch_prompt8(const Paged8View& c, const Attn8Args& a, uint32_t dp, cudaStream_t stream);

// Largest number of tiles of `rows` rows: every sequence's last may be ragged.
inline uint64_t most_tiles(uint64_t tokens, uint32_t batch, uint32_t group, uint32_t rows) {
  return tokens * group / rows + (tokens < batch ? tokens : batch);
}

}  // namespace qg

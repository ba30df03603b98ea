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
  uint32_t* item_count;           // tiles
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

// The tiles of `rows` rows of a ragged call, and how many blocks of 2^log slots each sees, before
// the attention reads them.
cudaError_t launch_plan8(const Paged8View& c, const Attn8Args& a, uint32_t rows, uint32_t log, cudaStream_t stream);

// Largest number of tiles of `rows` rows: every sequence's last may be ragged.
inline uint64_t most_tiles(uint64_t tokens, uint32_t batch, uint32_t group, uint32_t rows) {
  return tokens * group / rows + (tokens < batch ? tokens : batch);
}

}  // namespace qg

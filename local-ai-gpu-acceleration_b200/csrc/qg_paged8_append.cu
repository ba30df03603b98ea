// qg_paged8_append.cu -- qg_qk_norm_rope_append8: per-head RMSNorm and rotation of new queries
// and keys, keys and values quantised into the blocks of an 8-bit paged cache, in one pass
// (declared in include/qgemv_b200.h).
//
// A block's codes depend on the largest of its new values and on the scale that it has, so the
// unit of work for keys and values is what a call writes to one (block, kv head): a CTA holds
// those rows in registers (in shared memory where they are more than one pass of its 8 to 64 rows),
// finds their maximum, and only then rounds.  Where the block was begun before and its scale
// grows, the CTA also scales the block's other codes down, so that they stand for what they stood
// for: scales are powers of two, so this moves exponents and rounds only what falls below e4m3's
// normal range.  Query rows need no neighbour: a warp takes a batch of one token's heads.  Both
// kinds of task are in one launch, the blocks first, because they wait the longest.  In a call with
// one row a sequence (decoding) nothing but that row is new in a block, so its keys and values go
// a batch of heads a warp too, without the CTA's barrier: 256 sequences of 64/8 heads x 128 bf16 are
// 640 CTAs and 10 us on the GPU, against 4608 and 25 us with a CTA for each block.
//
// Measured (B200, floor = bytes at 6.56 TB/s): 16384 tokens of 64/8 heads x 128 bf16, blocks of 64: 148 us
// (floor 98); a launch of the queries alone takes 115 us, one of the blocks alone 41, a chain of loads in CTAs
// of 3 to 4 us each.  32 tokens 2.9 us, 2047 of 32/8 x 80 17 us (queries 8, blocks 12).  Several heads a CTA, one
// after another, took 157 (2 heads) to 189 us (16).
//
// A row lies in LPR lanes as in qg_paged_append.cu: pairs never leave a lane, the sum of
// squares is log2(LPR) shuffles.
#include <algorithm>
#include <type_traits>

#include "qg_paged8.cuh"
#include "qg_rows.cuh"

namespace qg {
namespace {

constexpr uint32_t kWarps8 = 4;
constexpr uint32_t kThreads8 = kWarps8 * 32u;
template <typename T>
constexpr uint32_t kBatch8 = 4 / sizeof(T);  // rows that a lane has in flight: 64 bytes

struct Append8Args {
  const void *q, *k, *v;
  void* q_out;
  uint64_t q_stride, k_stride, v_stride, q_out_stride;  // elements, token to token
  const float *q_norm, *k_norm, *rope;
  const int32_t *positions, *lens, *offsets;
  float eps, inv_dim;
  uint32_t n_q, rot, rope_rows, tokens;
  uint32_t block_tasks;  // of one kv head, of a ragged call
  uint32_t q_parts, kv_parts;  // tasks of a token's queries; of its keys, and values, of a call with a row a sequence
};

// A begun block's other codes, when its scale grows by 1 / shrink: those of all rows but [at, at + n).
__device__ __forceinline__ void shrink_others(uint8_t* codes, uint64_t slot_bytes, uint32_t dim, uint32_t slots,
                                              uint32_t at, uint32_t n, float shrink, uint32_t tid, uint32_t threads) {
  const uint32_t pieces = dim / 16u;
#pragma unroll 4
  for (uint32_t i = tid; i < (slots - n) * pieces; i += threads) {
    uint32_t r = i / pieces;
    const uint32_t piece = i - r * pieces;
    if (r >= at) r += n;
    uint4* from = reinterpret_cast<uint4*>(codes + r * slot_bytes + piece * 16u);
    uint4 w = *from;
    auto less = [&](uint32_t u) {
      float x[4];
      codes_to_float(u, x);
      return float_to_codes(x[0] * shrink, x[1] * shrink, x[2] * shrink, x[3] * shrink);
    };
    w.x = less(w.x), w.y = less(w.y), w.z = less(w.z), w.w = less(w.w);
    *from = w;
  }
}

// What a CTA writes to one block: rows [token, token + n) of the call to slots from `slot` on.
struct Run {
  uint32_t b, token, slot, n;
};

// The run with index `want` among all sequences' of a ragged call (a sequence's runs are the blocks that
// its new tokens touch); n 0 where there are fewer.  All threads of the CTA take part.
__device__ __forceinline__ Run find_run(const Paged8View& c, const Append8Args& a, uint32_t want) {
  __shared__ uint32_t sums[kWarps8];
  __shared__ Run found;
  const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5;
  if (tid == 0u) found.n = 0u;
  uint32_t base = 0;
  for (uint32_t b0 = 0; b0 < c.c.batch; b0 += kThreads8) {
    const uint32_t b = b0 + tid;
    Rows8 r{0u, 0u, 0u};
    if (b < c.c.batch) r = rows_of(c.c, a.lens, a.offsets, a.tokens, b);
    const uint32_t slot0 = r.len - r.n;
    uint32_t count = 0;
    if (r.n != 0u && r.len != 0u) count = ((r.len - 1u) >> c.log_block) - (slot0 >> c.log_block) + 1u;
    uint32_t upto = count;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const uint32_t o = __shfl_up_sync(0xffffffffu, upto, off);
      if (lane >= static_cast<uint32_t>(off)) upto += o;
    }
    __syncthreads();
    if (lane == 31u) sums[warp] = upto;
    __syncthreads();
    uint32_t all = 0;
#pragma unroll
    for (uint32_t w = 0; w < kWarps8; ++w) {
      if (w < warp) upto += sums[w];
      all += sums[w];
    }
    const uint32_t from = base + upto - count;
    if (count != 0u && want >= from && want - from < count) {
      const uint32_t block = (slot0 >> c.log_block) + (want - from);
      const uint32_t first = max(slot0, block << c.log_block), end = min(r.len, (block + 1u) << c.log_block);
      found = Run{b, r.first + (first - slot0), first, end - first};
    }
    base += all;
    if (base > want) break;
  }
  __syncthreads();
  return found;
}

// The cosines and sines of a lane's 8 pairs.
struct Turn {
  F2 co[4], si[4];
  __device__ __forceinline__ void load(const float* angles, uint32_t half) {
    Piece<float> cos, sin;
    cos.load(angles);
    sin.load(angles + half);
    float cs[8], sn[8];
    cos.get(cs);
    sin.get(sn);
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      co[h] = f2(cs[2 * h], cs[2 * h + 1]);
      si[h] = f2(sn[2 * h], sn[2 * h + 1]);
    }
  }
};

// |x| as bits, 0 for infinities and NaN: ordered like the values.
__device__ __forceinline__ uint32_t finite_size(float x) {
  const uint32_t u = __float_as_uint(x) & 0x7fffffffu;
  return u < 0x7f800000u ? u : 0u;
}

// The least power of two (within the scales' range) whose 448-fold is `size` or more: 448 is
// 1.75 * 2^8.
__device__ __forceinline__ float least_scale(uint32_t size) {
  const int e = static_cast<int>(size >> 23) - 135 + ((size & 0x7fffffu) > 0x600000u ? 1 : 0);
  return __uint_as_float(static_cast<uint32_t>(127 + max(kLeastPower, min(kMostPower, e))) << 23);
}

__device__ __forceinline__ void put8(uint8_t* to, const float (&x)[8], float by) {
  *reinterpret_cast<uint2*>(to) = make_uint2(float_to_codes(x[0] * by, x[1] * by, x[2] * by, x[3] * by),
                                             float_to_codes(x[4] * by, x[5] * by, x[6] * by, x[7] * by));
}

// ONE: a row a sequence (no offsets).  Five CTAs an SM: 16384 tokens take 148 us, 173 with four, 169 with six.
template <typename T, int LPR, bool HALVES, bool ONE>
__global__ void __launch_bounds__(kThreads8, 5) append8_kernel(const Paged8View c, const Append8Args a) {
  constexpr uint32_t kSide = 32 / LPR;                 // rows side by side in a warp
  constexpr uint32_t kRows = kSide * kBatch8<T>;       // of a warp's pass
  extern __shared__ float4 kept[];                     // rows of passes after the first
  __shared__ uint32_t tops[kWarps8];
  const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, chunk = lane % LPR;
  const uint32_t block_ctas = ONE ? 0u : a.block_tasks * 2u * c.c.n_kv;
  bool is_q = blockIdx.x >= block_ctas, is_k = false;
  uint32_t head0 = 0, heads = 0, t = 0;
  if constexpr (ONE) {
    const uint32_t task = blockIdx.x * kWarps8 + warp, parts = a.q_parts + 2u * a.kv_parts;
    uint32_t part = task % parts;
    t = task / parts;
    is_q = part >= 2u * a.kv_parts;
    is_k = part < a.kv_parts;
    if (!is_k) part -= is_q ? 2u * a.kv_parts : a.kv_parts;
    head0 = part * kRows + lane / LPR;
    heads = is_q ? a.n_q : c.c.n_kv;
  } else if (is_q) {
    const uint32_t task = blockIdx.x - block_ctas, part = task % a.q_parts;
    t = task / a.q_parts * kWarps8 + warp;
    head0 = part * kRows + lane / LPR;
    heads = a.n_q;
  } else {
    const uint32_t which = blockIdx.x % (2u * c.c.n_kv);
    is_k = which < c.c.n_kv;
    head0 = is_k ? which : which - c.c.n_kv;
  }
  const bool turned = chunk * 16u < a.rot && (is_q || is_k);
  const uint32_t at0 = HALVES && turned ? chunk * 8u : chunk * 16u;
  const uint32_t at1 = HALVES && turned ? a.rot / 2u + chunk * 8u : chunk * 16u + 8u;
  const bool has0 = at0 < c.c.dim, has1 = at1 < c.c.dim;
  const bool some_stay = a.rot != c.c.dim;  // lanes whose pairs do not turn: 0 x infinity is kept out
  pdl_wait();
  pdl_trigger();

  const float* norm = is_q ? a.q_norm : is_k ? a.k_norm : nullptr;
  Pairs weight;
  {
    float wa[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f}, wb[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
    if (norm != nullptr) {
      Piece<float> w;
      if (has0) w.load(norm + at0), w.get(wa);
      if (has1) w.load(norm + at1), w.get(wb);
    }
    weight = pairs_of<HALVES>(wa, wb);
  }
  // a row's position; -1 for one that has none in the table
  auto place = [&](uint32_t token) {
    int32_t pos = a.positions[token];
    if (pos >= 0 && a.rot != 0u && static_cast<uint32_t>(pos) >= a.rope_rows) {
      atomicOr(&g_error_word, QG_ERR_POSITION);
      pos = -1;
    }
    return pos;
  };
  // 1 / sqrt(mean of the row's squares + eps); all lanes of the warp take part
  auto root = [&](const Pairs& p) {
    F2 s0 = p.u[0] * p.u[0], s1 = p.v[0] * p.v[0];
#pragma unroll
    for (int h = 1; h < 4; ++h) {
      s0 = fma(p.u[h], p.u[h], s0);
      s1 = fma(p.v[h], p.v[h], s1);
    }
    const float2 s = split(s0), z = split(s1);
    float ss = (s.x + s.y) + (z.x + z.y);
#pragma unroll
    for (int off = LPR / 2; off > 0; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off, LPR);
    return rsqrtf(__fadd_rn(__fmul_rn(ss, a.inv_dim), a.eps));
  };
  // Norm and rotation of a lane's share of a row, in place; all lanes of the warp take part.  A key that lies near
  // the border of two codes goes by its last bit, so keys take every product and sum rounded by itself, as the
  // formula is written, queries the cheaper fused ones.
  auto finish = [&](float (&xa)[8], float (&xb)[8], const Turn& turn, auto key) {
    constexpr bool kKey = decltype(key)::value;
    Pairs p = pairs_of<HALVES>(xa, xb);
    if (norm != nullptr) {
      const float inv = root(p);
      const F2 by = f2(inv, inv);
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        p.u[h] = kKey ? (p.u[h] * by) * weight.u[h] : p.u[h] * (by * weight.u[h]);
        p.v[h] = kKey ? (p.v[h] * by) * weight.v[h] : p.v[h] * (by * weight.v[h]);
      }
    }
    if (!some_stay || turned) {
      const F2 minus = f2(-1.f, -1.f);
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const F2 u = p.u[h], v = p.v[h], down = minus * (v * turn.si[h]);
        p.u[h] = kKey ? u * turn.co[h] + down : fma(u, turn.co[h], down);
        p.v[h] = kKey ? u * turn.si[h] + v * turn.co[h] : fma(v, turn.co[h], u * turn.si[h]);
      }
    }
    values_of<HALVES>(p, xa, xb);
  };

  if (is_q) {
    if (t >= a.tokens) return;
    if (!ONE && (static_cast<int64_t>(t) < a.offsets[0] || static_cast<int64_t>(t) >= a.offsets[c.c.batch])) {
      return;  // a row of no sequence
    }
    const T* src = static_cast<const T*>(a.q) + t * a.q_stride + head0 * c.c.dim;
    T* to = static_cast<T*>(a.q_out) + t * a.q_out_stride + head0 * c.c.dim;
    Piece<T> raw[kBatch8<T>][2];
#pragma unroll
    for (uint32_t i = 0; i < kBatch8<T>; ++i) {
      raw[i][0] = raw[i][1] = Piece<T>{};
      const bool live = head0 + i * kSide < heads;
      if (live && has0) raw[i][0].load(src + at0 + i * (kSide * c.c.dim));
      if (live && has1) raw[i][1].load(src + at1 + i * (kSide * c.c.dim));
    }
    const int32_t pos = place(t);
    Turn turn = {};
    if (turned && pos >= 0) turn.load(a.rope + static_cast<size_t>(pos) * a.rot + chunk * 8u, a.rot / 2u);
#pragma unroll
    for (uint32_t i = 0; i < kBatch8<T>; ++i) {
      float xa[8] = {}, xb[8] = {};
      if (pos >= 0) {  // the same in all lanes
        raw[i][0].get(xa);
        raw[i][1].get(xb);
        finish(xa, xb, turn, std::false_type());
      }
      const bool live = head0 + i * kSide < heads;
      if (live && has0) store8<T>(to + at0 + i * (kSide * c.c.dim), xa);
      if (live && has1) store8<T>(to + at1 + i * (kSide * c.c.dim), xb);
    }
    return;
  }

  if constexpr (ONE) {  // ---- a warp's heads of one token's keys or values
    if (t >= a.tokens) return;
    const Rows8 rows = rows_of(c.c, a.lens, nullptr, a.tokens, t);
    if (rows.len == 0u) return;
    const T* src = static_cast<const T*>(is_k ? a.k : a.v) + t * (is_k ? a.k_stride : a.v_stride) + head0 * c.c.dim;
    const uint32_t slot = rows.len - 1u, block_slots = 1u << c.log_block;
    const uint32_t in_block = slot & (block_slots - 1u), block0 = slot - in_block;
    const uint32_t on_page = div_by(block0, c.c.page), place0 = block0 - on_page * c.c.page.d;
    const uint32_t id = static_cast<uint32_t>(c.c.table[static_cast<size_t>(t) * c.c.table_stride + on_page]);
    Piece<T> raw[kBatch8<T>][2];
#pragma unroll
    for (uint32_t i = 0; i < kBatch8<T>; ++i) {
      raw[i][0] = raw[i][1] = Piece<T>{};
      const bool live = head0 + i * kSide < heads;
      if (live && has0) raw[i][0].load(src + at0 + i * (kSide * c.c.dim));
      if (live && has1) raw[i][1].load(src + at1 + i * (kSide * c.c.dim));
    }
    const int32_t pos = place(t);
    Turn turn = {};
    if (turned && pos >= 0) turn.load(a.rope + static_cast<size_t>(pos) * a.rot + chunk * 8u, a.rot / 2u);
    if (id >= c.c.num_pages) {
      if (lane == 0u) atomicOr(&g_error_word, QG_ERR_PAGE);
      return;
    }
    float* const scales = (is_k ? c.ks : c.vs) + id * c.scale_page + (place0 >> c.log_block);
    uint8_t* const codes = (is_k ? c.c.k : c.c.v) + id * c.c.page_bytes + place0 * c.c.slot_bytes;
    float old[kBatch8<T>];
#pragma unroll
    for (uint32_t i = 0; i < kBatch8<T>; ++i) {
      const uint32_t head = head0 + i * kSide;
      old[i] = in_block != 0u && head < heads ? scales[head * c.scale_head] : 0.f;
    }
#pragma unroll
    for (uint32_t i = 0; i < kBatch8<T>; ++i) {
      const uint32_t head = head0 + i * kSide;
      float xa[8] = {}, xb[8] = {};
      if (pos >= 0) {  // the same in all lanes
        raw[i][0].get(xa);
        raw[i][1].get(xb);
        if (is_k) finish(xa, xb, turn, std::true_type());
      }
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, max(finite_size(xa[e]), finite_size(xb[e])));
#pragma unroll
      for (int off = LPR / 2; off > 0; off >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, off, LPR));
      const float scale = fmaxf(least_scale(top), old[i]), by = 1.f / scale;
      __syncwarp();  // every lane has read the old scale
      if (head < heads) {
        if (chunk == 0u) scales[head * c.scale_head] = scale;
        uint8_t* to = codes + head * c.c.head_bytes + in_block * c.c.slot_bytes;
        if (has0) put8(to + at0, xa, by);
        if (has1) put8(to + at1, xb, by);
      }
      // blocks whose scale grew, one after another with all lanes
      uint32_t grown = __ballot_sync(0xffffffffu, chunk == 0u && head < heads && in_block != 0u && scale > old[i]);
      while (grown != 0u) {
        const int from = __ffs(static_cast<int>(grown)) - 1;
        grown &= grown - 1u;
        const float shrink = __shfl_sync(0xffffffffu, old[i] / scale, from);
        shrink_others(codes + __shfl_sync(0xffffffffu, head, from) * c.c.head_bytes, c.c.slot_bytes, c.c.dim,
                      block_slots, in_block, 1u, shrink, lane, 32u);
      }
    }
    return;
  }

  // ---- the rows of one block and kv head
  const Run run = find_run(c, a, blockIdx.x / (2u * c.c.n_kv));
  if (run.n == 0u) return;
  const uint32_t block_slots = 1u << c.log_block, block0 = run.slot & ~(block_slots - 1u);
  const int32_t* row = c.c.table + static_cast<size_t>(run.b) * c.c.table_stride;
  const uint32_t on_page = div_by(block0, c.c.page), place0 = block0 - on_page * c.c.page.d;
  const uint32_t id = static_cast<uint32_t>(row[on_page]);  // looked at once the rows are on their way
  float* scale_at = nullptr;
  float old = 0.f;
  const T* src = static_cast<const T*>(is_k ? a.k : a.v) + head0 * c.c.dim;
  const uint64_t stride = is_k ? a.k_stride : a.v_stride;
  constexpr uint32_t kPass = kRows * kWarps8;
  const uint32_t passes = (run.n + kPass - 1u) / kPass;
  float xa[kBatch8<T>][8], xb[kBatch8<T>][8];
  uint32_t top = 0;
  for (uint32_t p = passes; p-- > 0u;) {  // the first pass last: its rows stay in registers
    const uint32_t r0 = p * kPass + warp * kRows + lane / LPR;
    Piece<T> raw[kBatch8<T>][2];
    int32_t pos[kBatch8<T>];
#pragma unroll
    for (uint32_t i = 0; i < kBatch8<T>; ++i) {
      const uint32_t r = r0 + i * kSide;
      raw[i][0] = raw[i][1] = Piece<T>{};
      pos[i] = -1;
      if (r < run.n) {
        const T* from = src + (run.token + r) * stride;
        if (has0) raw[i][0].load(from + at0);
        if (has1) raw[i][1].load(from + at1);
        pos[i] = place(run.token + r);
      }
    }
    if (p + 1u == passes) {
      if (id >= c.c.num_pages) {  // the same for the whole CTA
        if (tid == 0u) atomicOr(&g_error_word, QG_ERR_PAGE);
        return;
      }
      scale_at = (is_k ? c.ks : c.vs) + id * c.scale_page + head0 * c.scale_head + (place0 >> c.log_block);
      if (run.slot != block0) old = *scale_at;
    }
#pragma unroll
    for (uint32_t i = 0; i < kBatch8<T>; ++i) {
      Turn turn = {};
      if (turned && pos[i] >= 0) turn.load(a.rope + static_cast<size_t>(pos[i]) * a.rot + chunk * 8u, a.rot / 2u);
      raw[i][0].get(xa[i]);
      raw[i][1].get(xb[i]);
      if (is_k) finish(xa[i], xb[i], turn, std::true_type());
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (pos[i] < 0) xa[i][e] = xb[i][e] = 0.f;
        top = max(top, max(finite_size(xa[i][e]), finite_size(xb[i][e])));
      }
      if (p != 0u) {
        float4* to = kept + ((p - 1u) * kBatch8<T> + i) * 4u * kThreads8 + tid;
        to[0] = make_float4(xa[i][0], xa[i][1], xa[i][2], xa[i][3]);
        to[kThreads8] = make_float4(xa[i][4], xa[i][5], xa[i][6], xa[i][7]);
        to[2u * kThreads8] = make_float4(xb[i][0], xb[i][1], xb[i][2], xb[i][3]);
        to[3u * kThreads8] = make_float4(xb[i][4], xb[i][5], xb[i][6], xb[i][7]);
      }
    }
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (lane == 0u) tops[warp] = top;
  __syncthreads();  // also: every thread has read the old scale
#pragma unroll
  for (uint32_t w = 0; w < kWarps8; ++w) top = max(top, tops[w]);
  const float scale = fmaxf(least_scale(top), old), by = 1.f / scale;
  if (tid == 0u) *scale_at = scale;
  uint8_t* const codes = (is_k ? c.c.k : c.c.v) + id * c.c.page_bytes + head0 * c.c.head_bytes + place0 * c.c.slot_bytes;
  if (scale > old && run.slot != block0) {
    shrink_others(codes, c.c.slot_bytes, c.c.dim, block_slots, run.slot - block0, run.n, old / scale, tid, kThreads8);
  }
  for (uint32_t p = 0; p < passes; ++p) {
#pragma unroll
    for (uint32_t i = 0; i < kBatch8<T>; ++i) {
      if (p != 0u) {
        const float4* from = kept + ((p - 1u) * kBatch8<T> + i) * 4u * kThreads8 + tid;
        const float4 f0 = from[0], f1 = from[kThreads8], f2_ = from[2u * kThreads8], f3 = from[3u * kThreads8];
        xa[i][0] = f0.x, xa[i][1] = f0.y, xa[i][2] = f0.z, xa[i][3] = f0.w;
        xa[i][4] = f1.x, xa[i][5] = f1.y, xa[i][6] = f1.z, xa[i][7] = f1.w;
        xb[i][0] = f2_.x, xb[i][1] = f2_.y, xb[i][2] = f2_.z, xb[i][3] = f2_.w;
        xb[i][4] = f3.x, xb[i][5] = f3.y, xb[i][6] = f3.z, xb[i][7] = f3.w;
      }
      const uint32_t r = p * kPass + warp * kRows + lane / LPR + i * kSide;
      if (r >= run.n) continue;
      uint8_t* to = codes + (run.slot - block0 + r) * c.c.slot_bytes;
      if (has0) put8(to + at0, xa[i], by);
      if (has1) put8(to + at1, xb[i], by);
    }
  }
}

template <typename T, int LPR, bool HALVES>
cudaError_t launch_append8(const Paged8View& c, const Append8Args& a, cudaStream_t stream) {
  constexpr uint32_t kRows = 32 / LPR * kBatch8<T>;
  Append8Args w = a;
  w.q_parts = (a.n_q + kRows - 1u) / kRows;
  w.kv_parts = (c.c.n_kv + kRows - 1u) / kRows;
  if (a.offsets == nullptr) {
    const uint64_t warps = static_cast<uint64_t>(a.tokens) * (w.q_parts + 2u * w.kv_parts);
    if (warps > 0x7fffffffull) return cudaErrorInvalidValue;
    return launch_k(append8_kernel<T, LPR, HALVES, true>, static_cast<uint32_t>((warps + kWarps8 - 1u) / kWarps8),
                    kThreads8, 0u, stream, c, w);
  }
  const uint32_t longest = std::min(1u << c.log_block, a.tokens);
  const uint32_t passes = (longest + kRows * kWarps8 - 1u) / (kRows * kWarps8);
  const uint32_t smem = (passes - 1u) * kBatch8<T> * 64u * kThreads8;
  static SmemAttr attr;
  constexpr uint32_t kMost = (128u / (kRows * kWarps8) - 1u) * kBatch8<T> * 64u * kThreads8;
  const auto kernel = append8_kernel<T, LPR, HALVES, false>;
  const cudaError_t e = attr.set(reinterpret_cast<const void*>(kernel), kMost);
  if (e != cudaSuccess) return e;
  const uint64_t ctas = static_cast<uint64_t>(a.block_tasks) * 2u * c.c.n_kv +
                        static_cast<uint64_t>((a.tokens + kWarps8 - 1u) / kWarps8) * w.q_parts;
  if (ctas > 0x7fffffffull) return cudaErrorInvalidValue;
  return launch_k(kernel, static_cast<uint32_t>(ctas), kThreads8, smem, stream, c, w);
}

template <typename T, int LPR>
cudaError_t launch_append8(const Paged8View& c, const Append8Args& a, bool halves, cudaStream_t stream) {
  return halves ? launch_append8<T, LPR, true>(c, a, stream) : launch_append8<T, LPR, false>(c, a, stream);
}

template <typename T>
cudaError_t launch_append8(const Paged8View& c, const Append8Args& a, bool halves, cudaStream_t stream) {
  if (c.c.dim <= 64u) return launch_append8<T, 4>(c, a, halves, stream);
  if (c.c.dim <= 128u) return launch_append8<T, 8>(c, a, halves, stream);
  return launch_append8<T, 16>(c, a, halves, stream);
}

}  // namespace
}  // namespace qg

extern "C" cudaError_t qg_qk_norm_rope_append8(const qg_kv_pages8* cache, const qg_append8* p, cudaStream_t stream) {
  using namespace qg;
  Paged8View c;
  if (!paged8_view(cache, &c) || p == nullptr || !dtype_ok(p->dtype)) return cudaErrorInvalidValue;
  if (p->tokens == 0u) return cudaSuccess;
  if (p->tokens > 0x7fffffffu || p->n_q_heads > 65535u || p->positions == nullptr || p->lens == nullptr ||
      p->k == nullptr || p->v == nullptr || (p->n_q_heads != 0u && (p->q == nullptr || p->q_out == nullptr))) {
    return cudaErrorInvalidValue;
  }
  if (p->offsets == nullptr && p->tokens > cache->batch) return cudaErrorInvalidValue;
  if (p->pairs != QG_PAIRS_ADJACENT && p->pairs != QG_PAIRS_HALVES) return cudaErrorInvalidValue;
  if (p->rot_dim % 16u != 0u || p->rot_dim > cache->head_dim ||
      (p->rot_dim != 0u && (p->rope == nullptr || !aligned16(p->rope) || p->rope_rows == 0u))) {
    return cudaErrorInvalidValue;
  }
  const uint64_t piece = 16u / dtype_bytes(p->dtype);
  if (p->q_stride % piece != 0u || p->k_stride % piece != 0u || p->v_stride % piece != 0u ||
      p->q_out_stride % piece != 0u || !aligned16(p->q) || !aligned16(p->k) || !aligned16(p->v) ||
      !aligned16(p->q_out) || !aligned16(p->q_norm) || !aligned16(p->k_norm)) {
    return cudaErrorInvalidValue;
  }
  Append8Args a{};
  a.q = p->q;
  a.k = p->k;
  a.v = p->v;
  a.q_out = p->q_out;
  a.q_stride = p->q_stride;
  a.k_stride = p->k_stride;
  a.v_stride = p->v_stride;
  a.q_out_stride = p->q_out_stride;
  a.q_norm = p->q_norm;
  a.k_norm = p->k_norm;
  a.rope = p->rope;
  a.positions = p->positions;
  a.lens = p->lens;
  a.offsets = p->offsets;
  a.eps = p->eps;
  a.inv_dim = 1.f / static_cast<float>(c.c.dim);
  a.n_q = p->n_q_heads;
  a.rot = p->rot_dim;
  a.rope_rows = p->rope_rows;
  a.tokens = p->tokens;
  // a sequence of n new tokens touches at most n / block + 2 blocks
  const uint64_t most = (static_cast<uint64_t>(p->tokens) >> c.log_block) + 2ull * std::min(p->tokens, cache->batch);
  a.block_tasks = static_cast<uint32_t>(std::min<uint64_t>(most, p->tokens));
  // find_run() stops behind its task's sequences: one more task, so that what does not fit is reported of all
  if (cache->batch > kThreads8) ++a.block_tasks;
  const bool halves = p->pairs == QG_PAIRS_HALVES;
  if (p->dtype == QG_F32) return launch_append8<float>(c, a, halves, stream);
  if (p->dtype == QG_F16) return launch_append8<__half>(c, a, halves, stream);
  return launch_append8<__nv_bfloat16>(c, a, halves, stream);
}

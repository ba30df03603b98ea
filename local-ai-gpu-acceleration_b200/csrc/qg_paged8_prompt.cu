// qg_paged8_prompt.cu -- attention of many new tokens a sequence over an 8-bit paged cache, on the
// tensor cores (a part of qg_paged_attn8; its entry point and the mathematics are in
// qg_paged8_attn.cu).
//
// A tile is 256 rows (query heads of a kv head, token after token) in two halves of 128, the lanes of
// tensor memory; a step is 128 slots.  For each half
//   S = Q C_k^T    both operands fp16 in shared memory, 128 x 128 fp32 in tensor memory
//   P = 2^(y - M)  one thread a row: it reads its row of S twice (maximum, then powers) and writes P
//                  as fp16 over S
//   O += P C_v     P from tensor memory, fp32 sums in tensor memory
// M is the largest y so far, but only moved (and O scaled) when it has grown by 2^8: powers carry 2^7, so
// they stay below fp16's largest value, and those down to 2^-21 of the largest keep 11 bits.
//
// Codes become fp16 once for 256 rows: four warps load a step's codes into registers a step ahead,
// convert them and write them as core matrices of 8 slots x 16 bytes, stored [16-byte chunk of dims][8 slots].
// This one layout is a K-major operand over dims (for K, slots are N) and an MN-major one over slots
// (for V, dims are N); no byte is transposed.
//
// Warps: 0-3 and 4-7 the rows of the halves, 8-11 codes, 12 issues the products.  The halves take turns
// on the tensor pipe: while one waits for its S, the other's powers are computed.
//
// Work.  Segments, blocks, equal ranges for one CTA an SM, records and joins as in
// qg_paged8_attn.cu.  Every wait is bounded; after one has run out (QG_ERR_WAIT_TIMEOUT) no wait
// waits, every role runs through its steps and the CTA ends.
#include <math_constants.h>

#include <algorithm>

#include "qg_mma.cuh"
#include "qg_paged8_attn.cuh"
#include "qg_umma.cuh"

namespace qg {
namespace {

constexpr uint32_t kHalf = 128;                  // rows of a half, and slots of a step
constexpr uint32_t kLogStep = 7;
constexpr uint32_t kRowWarps = 8, kCodeWarp0 = 8, kCodeWarps = 4, kIssueWarp = 12;
constexpr uint32_t kPromptThreads = (kIssueWarp + 1u) * 32u;
constexpr uint32_t kScaleRing = 4;
constexpr uint32_t kMaxPolls = 4000;             // of up to kPollNs each
constexpr float kCarry = 7.f, kSlack = 8.f;      // log2: the factor of powers, the growth of M that is let pass
constexpr float kLeastFactor = 1e-30f;           // of scores: zero would turn minus infinity into NaN
constexpr uint32_t kPromptHeader = 2;            // what a segment costs beside its blocks, in blocks
static_assert(2u * 256u * 4u <= QG_PAGED_ATTN_ZEROED && kMaxPromptCtas <= 256u, "a counter per CTA and half");
static_assert(kPromptRows == 2u * kHalf, "two halves");

template <int DP>
struct PromptShape {
  static constexpr uint32_t kChunks = DP / 8u;             // 16-byte chunks of a row in fp16
  static constexpr uint32_t kTileBytes = kHalf * DP * 2u;  // 128 rows or slots
  static constexpr uint32_t q_at = 0, k_at = 2u * kTileBytes, v_at = 4u * kTileBytes, end = 6u * kTileBytes;
  static constexpr uint32_t scales = end;                              // [ring][8] {key scale, log2 value scale, reciprocal}
  static constexpr uint32_t nan_bits = scales + kScaleRing * 8u * 16u;  // [2][128 slots][8 pieces] 16 columns each
  static constexpr uint32_t row_nan = nan_bits + 2u * kHalf * 16u;      // [256 rows] the columns that are NaN
  static constexpr uint32_t kSmem = row_nan + kPromptRows * 16u + 1024u;
  static constexpr uint32_t kRecord = kHalf * (DP + 2u);   // of a half: m[], l[], o[DP / 4][row] float4
};

// Descriptor of an operand stored as core matrices of 8 x 16 bytes, consecutive ones of a chunk 128 bytes
// apart, chunks 2048 bytes; no swizzle, version 1.
template <uint32_t LEADING, uint32_t STRIDE>
__device__ __forceinline__ uint64_t core_desc(uint32_t at) {
  return static_cast<uint64_t>((at >> 4) & 0x3FFFu) | (static_cast<uint64_t>(LEADING >> 4) << 16) |
         (static_cast<uint64_t>(STRIDE >> 4) << 32) | (1ull << 46);
}
constexpr uint32_t kChunkBytes = kHalf * 16u;
// fp16 operands, fp32 sums, M = 128
constexpr uint32_t score_idesc() { return (1u << 4) | ((kHalf >> 3) << 17) | ((kHalf >> 4) << 24); }
template <int DP>
constexpr uint32_t value_idesc() {  // B MN-major
  return (1u << 4) | (1u << 16) | ((DP >> 3) << 17) | ((kHalf >> 4) << 24);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

template <int DP>
__global__ void __launch_bounds__(kPromptThreads, 1) prompt8_kernel(const Paged8View cache, const Attn8Args a) {
  using Shape = PromptShape<DP>;
  const PagedView& c = cache.c;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t q_full[2], s_full[2], p_full[2], o_full[2], k_full[2], k_empty[2], v_full[2], v_empty[2],
      scale_full[kScaleRing], drained;
  __shared__ uint32_t tmem_slot, abort_flag, last_flag[2];
  __shared__ uint32_t nan_flag[2][kCodeWarps];
  const uint32_t tid = threadIdx.x, lane = tid & 31u;
  const uint32_t warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  uint8_t* const smem = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
  volatile uint32_t* const abort = &abort_flag;
  if (tid == 0u) {
    for (uint32_t i = 0; i < 2u; ++i) {
      mbar_init(&q_full[i], kHalf);
      mbar_init(&s_full[i], 1u);
      mbar_init(&p_full[i], kHalf);
      mbar_init(&o_full[i], 1u);
      mbar_init(&k_full[i], kCodeWarps);
      mbar_init(&k_empty[i], 1u);
      mbar_init(&v_full[i], kCodeWarps);
      mbar_init(&v_empty[i], 1u);
    }
    for (uint32_t i = 0; i < kScaleRing; ++i) mbar_init(&scale_full[i], 1u);
    mbar_init(&drained, 1u);
    abort_flag = 0u;
    fence_mbar_init();
  }
  if (warp == kIssueWarp) tmem_alloc_all(&tmem_slot);
  if (tid < kPromptRows) *reinterpret_cast<uint4*>(smem + Shape::row_nan + tid * 16u) = make_uint4(0u, 0u, 0u, 0u);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  pdl_wait();
  pdl_trigger();

  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (mbar_try_wait(bar, parity)) return;
    for (uint32_t i = 0; i < kMaxPolls; ++i) {
      if (*abort != 0u) return;
      if (mbar_try_wait_sleep(bar, parity)) return;
    }
    atomicOr(&g_error_word, QG_ERR_WAIT_TIMEOUT);
    *abort = 1u;
  };

  // ---- this CTA's range [r0, r1) of the line of units; every warp finds it
  const uint32_t n = *a.item_count, lines = c.n_kv;
  uint64_t total = 0, ctas = 0, r0 = 0, r1 = 0;
  uint32_t header = 0, left = 0;
  Segment8 use;
  auto skip_header = [&](uint32_t& units, uint32_t done) { units -= min(units, header - min(done, header)); };
  if (n != 0u) {
    const uint64_t blocks = a.item_blocks[n] * lines;
    if (blocks > gridDim.x) header = kPromptHeader;
    total = blocks + static_cast<uint64_t>(header) * n * lines;
    ctas = min(static_cast<uint64_t>(gridDim.x), total);
    if (blockIdx.x < ctas) {
      r0 = blockIdx.x * total / ctas;
      r1 = (blockIdx.x + 1u) * total / ctas;
      uint32_t in_segment;
      find_unit8(a, n, lines, header, r0, use.item, use.line, in_segment);
      take_item8(a, use, true, kLogStep);
      left = static_cast<uint32_t>(r1 - r0);
      skip_header(left, in_segment);
      use.j = in_segment - min(in_segment, header);
    }
  }
  // the segment after one that is done
  auto advance = [&](Segment8& s, uint32_t& units) {
    skip_header(units, 0u);
    if (units == 0u) return;
    const bool fresh = ++s.line == lines;
    if (fresh) s.line = 0u, ++s.item;
    take_item8(a, s, fresh, kLogStep);
  };

  uint32_t kt = 0;  // steps of the range

  if (warp < kRowWarps) {
    // ================= the rows of a half: a thread has one
    const uint32_t half = warp / 4u, row = tid % kHalf;      // of the half
    const uint32_t s_at = tmem + half * kHalf + ((warp & 3u) << 21), o_at = s_at + 2u * kHalf;
    uint4* const row_nan = reinterpret_cast<uint4*>(smem + Shape::row_nan) + half * kHalf + row;
    uint32_t parts = 0, steps = 0;                           // of this half
    for (; left != 0u; advance(use, left)) {
      const uint32_t from_j = use.j, to_j = min(use.j1, use.j + left);
      left -= to_j - from_j;
      if (use.rows <= half * kHalf) {  // this half has none
        kt += to_j - from_j;
        continue;
      }
      const uint32_t r = half * kHalf + row;                 // of the tile
      const bool has = r < use.rows;
      const uint32_t at = use.sub + (has ? r : 0u), down = div_by(at, a.group);
      const uint32_t token = use.token + down, head = use.kv * a.group.d + (at - down * a.group.d);
      const int32_t p = has ? use.p0 + static_cast<int32_t>(down) : use.p1;
      // ---- the query, scaled to a largest value in [1, 2); the scale's sign goes with it
      float mult = fabsf(a.scale_log2);
      {
        uint4 w[Shape::kChunks];
        float top = 0.f;
        const uint4* from = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) + token * a.q_stride +
                                                           static_cast<uint64_t>(head) * c.dim);
        auto two = [&](uint32_t u) { return a.dtype == QG_F16 ? unpack2(u, __half()) : unpack2(u, __nv_bfloat16()); };
#pragma unroll
        for (uint32_t i = 0; i < Shape::kChunks; ++i) {
          w[i] = make_uint4(0u, 0u, 0u, 0u);
          if (has && i * 8u < c.dim) w[i] = from[i];
        }
#pragma unroll
        for (uint32_t i = 0; i < Shape::kChunks; ++i) {
          const float2 x = two(w[i].x), y = two(w[i].y), z = two(w[i].z), u = two(w[i].w);
          top = max3(top, fabsf(x.x), fabsf(x.y));
          top = max3(top, fabsf(y.x), fabsf(y.y));
          top = max3(top, fabsf(z.x), fabsf(z.y));
          top = max3(top, fabsf(u.x), fabsf(u.y));
        }
        const int power = top == 0.f ? 0 : max(-126, min(126, static_cast<int>(__float_as_uint(top) >> 23) - 127));
        const float by = a.scale_log2 < 0.f ? -power_of_two(-power) : power_of_two(-power);
        mult *= power_of_two(power);
        uint8_t* const to = smem + Shape::q_at + half * Shape::kTileBytes + (row >> 3) * 128u + (row & 7u) * 16u;
#pragma unroll
        for (uint32_t i = 0; i < Shape::kChunks; ++i) {
          auto half2 = [&](uint32_t u) {
            const float2 x = two(u);
            return pack2(x.x * by, x.y * by, __half());
          };
          *reinterpret_cast<uint4*>(to + i * kChunkBytes) =
              make_uint4(half2(w[i].x), half2(w[i].y), half2(w[i].z), half2(w[i].w));
        }
        fence_proxy_async_smem();
        mbar_arrive(&q_full[half]);
      }
      float m = -CUDART_INF_F, l = 0.f;
      bool any_nan = false;  // columns of the row are NaN
      for (uint32_t j = from_j; j < to_j; ++j, ++kt, ++steps) {
        const uint32_t slot0 = use.block(j) << kLogStep, ring = kt % kScaleRing;
        const bool whole = use.all_see(a, slot0, kHalf);
        const float4* const scale = reinterpret_cast<const float4*>(smem + Shape::scales) + ring * 8u;
        // the row's slots of the step: up to hi, from lo on or before `first`
        const int32_t hi = p - static_cast<int32_t>(slot0);
        const int32_t lo = a.window == 0u || hi < 0 || a.window > static_cast<uint32_t>(hi)
                               ? INT32_MIN : hi - static_cast<int32_t>(a.window) + 1;
        const int32_t first = a.sink > slot0 ? static_cast<int32_t>(min(a.sink - slot0, kHalf)) : 0;
        wait(&s_full[half], steps & 1u);
        wait(&scale_full[ring], (kt / kScaleRing) & 1u);  // long done: S needed the step's codes
        tc_fence_after();
        // S comes 32 columns at a time, the next ones while these are worked on; columns that the row does
        // not see become minus infinity
        uint32_t s[2][32];
        auto mask = [&](uint32_t (&x)[32], int32_t at) {
          auto low = [](int32_t n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; };  // bits [0, n)
          const uint32_t bits = low(hi + 1 - at) & (low(first - at) | ~(lo <= at ? 0u : low(lo - at)));
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            if ((bits >> e & 1u) == 0u) x[e] = 0xff800000u;
          }
        };
        auto over = [&](auto work) {
          tmem_ld32(s_at, s[0]);
#pragma unroll 1
          for (int i = 0; i < 4; i += 2) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              tmem_wait_ld();
              if (k == 0 || i == 0) tmem_ld32(s_at + 32u * (i + k + 1), s[k ^ 1]);
              if (!whole) mask(s[k], 32 * (i + k));
              work(i + k, s[k]);
            }
          }
        };
        // ---- the largest y
        float top = -CUDART_INF_F;
        over([&](int i, const uint32_t (&raw)[32]) {
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            auto x = [&](int e) { return __uint_as_float(raw[16 * g + e]); };
            float u = max3(x(0), x(1), x(2)), v = max3(x(3), x(4), x(5));
            u = max3(u, x(6), x(7)), v = max3(v, x(8), x(9));
            u = max3(u, x(10), x(11)), v = max3(v, x(12), x(13));
            u = max3(u, x(14), x(15));
            const float4 sc = scale[2 * i + g];
            top = fmaxf(top, fmaf(fmaxf(u, v), fmaxf(mult * sc.x, kLeastFactor), sc.y));
          }
        });
        // ---- M moves at the first step, and when it has grown by more than the slack
        const float now = fmaxf(m, top);
        if (j == from_j) {
          m = now;
        } else if (__any_sync(0xffffffffu, now > m + kSlack)) {
          // the products before are done: they were issued before S was, and it is complete
          const float fade = exp2_fast(m - (now == -CUDART_INF_F ? 0.f : now));
          m = now;
          l *= fade;
#pragma unroll 1
          for (uint32_t i = 0; i < DP / 16u; ++i) {
            float v[16];
            uint32_t raw[16];
            tmem_ld16(o_at + 16u * i, v);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) raw[e] = __float_as_uint(v[e] * fade);
            tmem_st16(o_at + 16u * i, raw);
          }
        }
        // ---- powers, over S
        const float base = kCarry - (m == -CUDART_INF_F ? 0.f : m);
        over([&](int i, const uint32_t (&raw)[32]) {
          uint32_t out[16];
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const float4 sc = scale[2 * i + g];
            const float by = fmaxf(mult * sc.x, kLeastFactor), plus = sc.y + base;
            float sum[2] = {0.f, 0.f};
#pragma unroll
            for (int e = 0; e < 16; e += 2) {
              const float x = exp2_fast(fmaf(__uint_as_float(raw[16 * g + e]), by, plus));
              const float y = exp2_fast(fmaf(__uint_as_float(raw[16 * g + e + 1]), by, plus));
              sum[0] += x;
              sum[1] += y;
              out[8 * g + e / 2] = pack2(x, y, __half());
            }
            l = fmaf(sum[0] + sum[1], sc.z, l);
          }
          tmem_st16(s_at + 16u * i, out);
        });
        if (!whole) {  // a NaN value that some rows see and some do not was taken out of the codes
          wait(&v_full[kt & 1u], (kt >> 1) & 1u);
          for (uint32_t w = 0; w < kCodeWarps; ++w) {
            if (nan_flag[kt & 1u][w] == 0u) continue;
            for (uint32_t e = w * 32u; e < w * 32u + 32u; ++e) {
              const uint4 bits = reinterpret_cast<const uint4*>(smem + Shape::nan_bits)[(kt & 1u) * kHalf + e];
              if ((bits.x | bits.y | bits.z | bits.w) == 0u || !sees(a, p, slot0 + e)) continue;
              uint4 mine = *row_nan;
              mine.x |= bits.x, mine.y |= bits.y, mine.z |= bits.z, mine.w |= bits.w;
              *row_nan = mine;
              any_nan = true;
            }
          }
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&p_full[half]);
      }

      // ---- the end of the segment, or of the range inside it
      const bool mine = from_j == 0u && to_j == use.j1;
      float* const record = a.records + ((blockIdx.x * 2ull + (from_j == 0u ? 1u : 0u)) * 2u + half) * Shape::kRecord;
      auto put = [&](uint32_t at_col, const float* x, float top, float sum, float by) {  // 8 columns of the row
        if (!has || at_col >= c.dim) return;
        const uint64_t to = token * a.out_stride + static_cast<uint64_t>(head) * c.dim + at_col;
        auto two = [&](int e) {
          return a.dtype == QG_F16 ? pack2(x[e] * by, x[e + 1] * by, __half()) : pack2(x[e] * by, x[e + 1] * by, __nv_bfloat16());
        };
        *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + to) = make_uint4(two(0), two(2), two(4), two(6));
        if (at_col == 0u && a.lse != nullptr) {
          a.lse[static_cast<size_t>(token) * a.n_q + head] =
              sum == 0.f ? -CUDART_INF_F : (top + log2f(sum) - kCarry) * 0.69314718055994530942f;
        }
      };
      wait(&o_full[half], parts & 1u);
      ++parts;
      tc_fence_after();
      const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
      for (uint32_t i = 0; i < DP / 32u; ++i) {
        uint32_t raw[32];
        tmem_ld32(o_at + 32u * i, raw);
        tmem_wait_ld();
        float x[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) x[e] = __uint_as_float(raw[e]);
        if (any_nan) {
          const uint32_t bits = reinterpret_cast<const uint32_t*>(row_nan)[i];
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            if ((bits >> e & 1u) != 0u) x[e] = CUDART_NAN_F;
          }
        }
        if (mine) {
#pragma unroll
          for (int e = 0; e < 32; e += 8) put(32u * i + e, x + e, m, l, inv);
        } else {
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            reinterpret_cast<float4*>(record + 2u * kHalf)[(8u * i + e / 4) * kHalf + row] =
                make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
          }
        }
      }
      tc_fence_before();  // O is read; the next segment's first powers follow
      if (any_nan) *row_nan = make_uint4(0u, 0u, 0u, 0u);
      if (!mine) {
        record[row] = m;
        record[kHalf + row] = l;
        // the CTAs that share this segment own its first to its last block, in order
        const uint64_t seg0 = r1 - left - to_j, seg1 = seg0 + use.j1;
        const uint32_t c0 = static_cast<uint32_t>(((seg0 + 1u) * ctas - 1u) / total);
        const uint32_t count = static_cast<uint32_t>((seg1 * ctas - 1u) / total) - c0 + 1u;
        auto record_of = [&](uint32_t i) {
          return a.records + (((c0 + i) * 2ull + (i == 0u ? 1u : 0u)) * 2u + half) * Shape::kRecord;
        };
        auto half_sync = [&]() { asm volatile("bar.sync %0, 128;" ::"r"(1u + half) : "memory"); };
        half_sync();
        if (row == 0u) {
          __threadfence();  // this half's record, ordered before by the barrier, is out
          uint32_t* const counter = a.arrived + half * 256u + c0;
          const bool last = atomicAdd(counter, 1u) == count - 1u;
          if (last) *counter = 0u;
          last_flag[half] = last ? 1u : 0u;
          __threadfence();
        }
        half_sync();
        if (last_flag[half] != 0u) {  // the last CTA joins all records, in CTA order
          float most = -CUDART_INF_F, all = 0.f;
          for (uint32_t i = 0; i < count; ++i) most = fmaxf(most, __ldcg(record_of(i) + row));
          const float from = most == -CUDART_INF_F ? 0.f : most;
          for (uint32_t i = 0; i < count; ++i) {
            all = fmaf(__ldcg(record_of(i) + kHalf + row), exp2_fast(__ldcg(record_of(i) + row) - from), all);
          }
          const float by = all == 0.f ? 0.f : 1.f / all;
          for (uint32_t i0 = 0; i0 < DP / 16u; ++i0) {  // 16 columns at a time
            float x[16] = {};
            for (uint32_t i = 0; i < count; ++i) {
              const float f = exp2_fast(__ldcg(record_of(i) + row) - from);
              const float4* rec = reinterpret_cast<const float4*>(record_of(i) + 2u * kHalf) + (4u * i0) * kHalf + row;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float4 v = __ldcg(rec + e * kHalf);
                x[4 * e] = fmaf(v.x, f, x[4 * e]), x[4 * e + 1] = fmaf(v.y, f, x[4 * e + 1]);
                x[4 * e + 2] = fmaf(v.z, f, x[4 * e + 2]), x[4 * e + 3] = fmaf(v.w, f, x[4 * e + 3]);
              }
            }
            put(16u * i0, x, most, all, by);
            put(16u * i0 + 8u, x + 8, most, all, by);
          }
        }
        half_sync();  // the flag is free again
      }
    }
  } else if (warp < kIssueWarp) {
    // ================= codes to fp16: this thread has place r of the 8-slot groups 4 w to 4 w + 3 and every
    // fourth 16-code piece, so 8 lanes write 128 consecutive bytes and a group's lanes read 64 of a row
    constexpr uint32_t kMine = DP / 64u;                     // pieces of a row
    const uint32_t w = warp - kCodeWarp0, r = lane & 7u, pq = lane >> 3, thread = tid - kCodeWarp0 * 32u;
    Segment8 s = use;
    uint32_t rem = left;
    uint32_t id[4] = {}, scale_id = 0, flags = 0;            // flags: row i is seen by some, bit 4 + i: by all
    float ks = 0.f, vs = 1.f;
    uint64_t off[4] = {};
    uint4 kw[4][kMine], vw[4][kMine];
    auto slot_of = [&](uint32_t i) { return (s.block(s.j) << kLogStep) + (4u * w + i) * 8u + r; };
    auto look = [&]() {  // page ids of the step's rows
      const int32_t* list = c.table + static_cast<size_t>(s.b) * c.table_stride;
#pragma unroll
      for (uint32_t i = 0; i < 4u; ++i) {
        id[i] = 0xffffffffu;
        if (s.some_see(slot_of(i), 1u)) id[i] = static_cast<uint32_t>(list[div_by(slot_of(i), c.page)]);
      }
      if (thread < 8u) {
        const uint32_t slot = (s.block(s.j) << kLogStep) + thread * 16u;
        scale_id = 0xffffffffu;
        if (s.some_see(slot, 16u)) scale_id = static_cast<uint32_t>(list[div_by(slot, c.page)]);
      }
    };
    auto place = [&]() {  // where the rows lie, and the scales
      flags = 0u;
#pragma unroll
      for (uint32_t i = 0; i < 4u; ++i) {
        const uint32_t slot = slot_of(i), at = div_by(slot, c.page);
        if (!s.some_see(slot, 1u)) continue;
        if (s.all_see(a, slot, 1u)) flags |= 16u << i;
        if (id[i] >= c.num_pages) {
          atomicOr(&g_error_word, QG_ERR_PAGE);
          continue;
        }
        flags |= 1u << i;
        off[i] = id[i] * c.page_bytes + s.kv * c.head_bytes + (slot - at * c.page.d) * c.slot_bytes;
      }
      ks = 0.f;
      vs = 1.f;
      if (thread < 8u && scale_id < c.num_pages) {
        const uint32_t slot = (s.block(s.j) << kLogStep) + thread * 16u, at = div_by(slot, c.page);
        const uint64_t in = scale_id * cache.scale_page + s.kv * cache.scale_head + ((slot - at * c.page.d) >> cache.log_block);
        ks = cache.ks[in];
        vs = cache.vs[in];
      }
    };
    auto load = [&](const uint8_t* pool, uint4 (&to)[4][kMine]) {
#pragma unroll
      for (uint32_t i = 0; i < 4u; ++i) {
#pragma unroll
        for (uint32_t h = 0; h < kMine; ++h) {
          to[i][h] = make_uint4(0u, 0u, 0u, 0u);
          const uint32_t piece = pq + 4u * h;
          if ((flags >> i & 1u) != 0u && piece * 16u < c.dim) {
            to[i][h] = *reinterpret_cast<const uint4*>(pool + off[i] + piece * 16u);
          }
        }
      }
    };
    auto store = [&](uint32_t at, const uint4 (&from)[4][kMine]) {
#pragma unroll
      for (uint32_t i = 0; i < 4u; ++i) {
#pragma unroll
        for (uint32_t h = 0; h < kMine; ++h) {
          uint8_t* const to = smem + at + 2u * (pq + 4u * h) * kChunkBytes + (4u * w + i) * 128u + r * 16u;
          uint4 x, y;
          codes_to_half(from[i][h].x, x.x, x.y);
          codes_to_half(from[i][h].y, x.z, x.w);
          codes_to_half(from[i][h].z, y.x, y.y);
          codes_to_half(from[i][h].w, y.z, y.w);
          *reinterpret_cast<uint4*>(to) = x;
          *reinterpret_cast<uint4*>(to + kChunkBytes) = y;
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
    };
    bool next = rem != 0u;
    if (next) {
      look();
      place();
      load(c.k, kw);
      load(c.v, vw);
    }
    for (; next; ++kt) {
      const uint32_t buf = kt & 1u, ring = kt % kScaleRing, now_flags = flags;
      const float now_ks = ks, now_vs = fminf(fmaxf(vs, 0x1p-60f), 0x1p60f);
      ++s.j;
      --rem;
      if (s.j == s.j1) advance(s, rem);
      next = rem != 0u;
      if (next) look();
      if (kt >= 2u) wait(&k_empty[buf], ((kt >> 1) - 1u) & 1u);
      if (thread < 8u) {
        reinterpret_cast<float4*>(smem + Shape::scales)[ring * 8u + thread] = make_float4(now_ks, log2f(now_vs), 1.f / now_vs, 0.f);
      }
      store(Shape::k_at + buf * Shape::kTileBytes, kw);
      if (lane == 0u) mbar_arrive(&k_full[buf]);
      if (thread == 0u) mbar_arrive(&scale_full[ring]);
      if (next) {
        place();
        load(c.k, kw);
      }
      // NaN codes of rows that not all see: out of the codes, noted by column
      uint32_t odd = 0;
      if ((now_flags >> 4) != (now_flags & 15u)) {
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
#pragma unroll
          for (uint32_t h = 0; h < kMine; ++h) {
            if ((now_flags >> (4u + i) & 1u) != 0u) continue;
            auto nan = [](uint32_t u) { return ((u & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; };
            odd |= nan(vw[i][h].x) | nan(vw[i][h].y) | nan(vw[i][h].z) | nan(vw[i][h].w);
          }
        }
      }
      const bool flagged = __any_sync(0xffffffffu, odd != 0u);
      if (kt >= 2u) wait(&v_empty[buf], ((kt >> 1) - 1u) & 1u);
      if (flagged) {
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
#pragma unroll
          for (uint32_t h = 0; h < 2u; ++h) {  // both halves of a row's 128 columns
            uint32_t bits = 0;
            if (h < kMine && (now_flags >> (4u + i) & 1u) == 0u) {
              auto clean = [&](uint32_t& word, uint32_t e) {
                const uint32_t is = (((word & 0x7f7f7f7fu) + 0x01010101u) >> 7) & 0x01010101u;
                word &= ~(is * 0xffu);
                bits |= (is * 0x01020408u >> 24 & 15u) << (4u * e);
              };
              clean(vw[i][h % kMine].x, 0u), clean(vw[i][h % kMine].y, 1u);
              clean(vw[i][h % kMine].z, 2u), clean(vw[i][h % kMine].w, 3u);
            }
            reinterpret_cast<uint16_t*>(smem + Shape::nan_bits)[(buf * kHalf + (4u * w + i) * 8u + r) * 8u + pq + 4u * h] =
                static_cast<uint16_t>(bits);
          }
        }
      }
      if (lane == 0u) nan_flag[buf][w] = flagged ? 1u : 0u;
      store(Shape::v_at + buf * Shape::kTileBytes, vw);
      if (lane == 0u) mbar_arrive(&v_full[buf]);
      if (next) load(c.v, vw);
    }
  } else if (elect_one()) {
    // ================= the products, by one thread
    uint32_t parts[2] = {0u, 0u}, steps[2] = {0u, 0u};
    const uint32_t base = smem_addr(smem);
    auto scores = [&](uint32_t half, uint32_t buf) {
      if (*abort != 0u) return;
      const uint32_t q = base + Shape::q_at + half * Shape::kTileBytes, k = base + Shape::k_at + buf * Shape::kTileBytes;
#pragma unroll
      for (uint32_t i = 0; i < DP / 16u; ++i) {
        umma_ss(tmem + half * kHalf, core_desc<kChunkBytes, 128u>(q + i * 2u * kChunkBytes),
                core_desc<kChunkBytes, 128u>(k + i * 2u * kChunkBytes), score_idesc(), i != 0u ? 1u : 0u);
      }
    };
    auto values = [&](uint32_t half, uint32_t buf, bool more) {
      if (*abort != 0u) return;
      const uint32_t v = base + Shape::v_at + buf * Shape::kTileBytes;
#pragma unroll
      for (uint32_t i = 0; i < kHalf / 16u; ++i) {
        umma_ts(tmem + (2u + half) * kHalf, tmem + half * kHalf + 8u * i, core_desc<128u, kChunkBytes>(v + i * 256u),
                value_idesc<DP>(), more || i != 0u ? 1u : 0u);
      }
    };
    for (; left != 0u; advance(use, left)) {
      const uint32_t count = min(use.j1 - use.j, left), halves = use.rows > kHalf ? 2u : 1u;
      left -= count;
      for (uint32_t h = 0; h < halves; ++h) wait(&q_full[h], parts[h]++ & 1u);
      wait(&k_full[kt & 1u], (kt >> 1) & 1u);
      tc_fence_after();
      for (uint32_t h = 0; h < halves; ++h) {
        scores(h, kt & 1u);
        umma_commit(&s_full[h]);
      }
      umma_commit(&k_empty[kt & 1u]);
      for (uint32_t i = 0; i < count; ++i, ++kt) {
        const uint32_t buf = kt & 1u;
        const bool more = i + 1u < count;
        for (uint32_t h = 0; h < halves; ++h) {
          wait(&p_full[h], steps[h]++ & 1u);
          if (h == 0u) wait(&v_full[buf], (kt >> 1) & 1u);
          tc_fence_after();
          values(h, buf, i != 0u);
          if (h + 1u == halves) umma_commit(&v_empty[buf]);
          if (!more) {
            umma_commit(&o_full[h]);
            continue;
          }
          if (h == 0u) {
            wait(&k_full[buf ^ 1u], ((kt + 1u) >> 1) & 1u);
            tc_fence_after();
          }
          scores(h, buf ^ 1u);
          umma_commit(&s_full[h]);
          if (h + 1u == halves) umma_commit(&k_empty[buf ^ 1u]);
        }
      }
    }
    // what was issued ends before the CTA's memory goes, also after a wait that ran out
    umma_commit(&drained);
    for (uint32_t i = 0; i < kMaxPolls && !mbar_try_wait_sleep(&drained, 0u); ++i) {
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == kIssueWarp) {
    tc_fence_after();
    tmem_free_all(tmem);
  }
}

template <int DP>
cudaError_t launch_prompt8(const Paged8View& c, const Attn8Args& a, cudaStream_t stream) {
  using Shape = PromptShape<DP>;
  const auto kernel = prompt8_kernel<DP>;
  static SmemAttr attr;
  cudaError_t e = attr.set(reinterpret_cast<const void*>(kernel), Shape::kSmem);
  if (e != cudaSuccess) return e;
  const uint64_t blocks = most_tiles(a.tokens, c.c.batch, a.group.d, kPromptRows) * c.c.n_kv *
                          ((c.c.capacity + (1u << kLogStep) - 1u) >> kLogStep);
  const uint32_t fit = std::min<uint32_t>(static_cast<uint32_t>(paged_sm_count()), kMaxPromptCtas);
  const uint32_t grid = static_cast<uint32_t>(std::min<uint64_t>(blocks, fit));
  if (blocks / grid >= (1ull << 29)) return cudaErrorInvalidValue;  // a CTA counts its units in 32 bits
  e = launch_plan8(c, a, kPromptRows, kLogStep, stream);
  if (e != cudaSuccess) return e;
  return launch_k(kernel, grid, kPromptThreads, Shape::kSmem, stream, c, a);
}

}  // namespace

cudaError_t launch_prompt8(const Paged8View& c, const Attn8Args& a, uint32_t dp, cudaStream_t stream) {
  return dp == 64u ? launch_prompt8<64>(c, a, stream) : launch_prompt8<128>(c, a, stream);
}

}  // namespace qg

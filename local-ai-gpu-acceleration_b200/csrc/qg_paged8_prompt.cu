// qg_paged8_prompt.cu -- attention of many new tokens a sequence over an 8-bit paged cache, on the
// tensor cores (a part of qg_paged_attn8; its entry point and the mathematics are in
// qg_paged8_attn.cu).
//
// A tile is 256 rows (query heads of a kv head, token after token) in two halves of 128, the lanes of
// tensor memory; a step is 64 slots.  For each half
//   S = Q C_k^T    both operands fp16 in shared memory, 128 x 64 fp32 in tensor memory, two of them
//   P = 2^(y - M)  one thread a row: it takes its 64 scores into registers, finds the largest y and
//                  writes P as fp16 over S
//   O += P C_v     P from tensor memory, fp32 sums in tensor memory
// M is the largest y so far, but only moved (and O scaled) when it has grown by 2^8: powers carry 2^7, so
// they stay below fp16's largest value, and those down to 2^-21 of the largest keep 11 bits.  For the
// softmax's sum they are 2^64 times as large (why is in qg_paged8_attn.cu); that costs 3% of the time.  A branch for
// steps whose scales need it cost 9 to 13% in four forms.
//
// Codes become fp16 once for 256 rows: seven warps take turns at 16 slots, load their codes into
// registers a turn ahead, convert them and write them in panels of 64 dims, 128 swizzled bytes a slot.
// The one layout is a K-major operand over dims (for K, whose N are slots) and an MN-major one over
// slots (for V, whose N are dims), so no byte is transposed.
//
// Warps: 0 issues the products, 1-7 codes, 8-11 and 12-15 the rows of the halves.  With two S of a half
// the scores of the next step are there before the powers of this one are written, so the rows never
// wait for a product.  The four roles' loops have to stay small: unrolled further they left the
// instruction cache and took twice the time.
//
// Measured (B200): 4096 new tokens of 5600 slots, 64/8 heads x 128 bf16: 650 us, 733 TFLOP/s, 0.44 of what
// cuBLAS reaches; a step takes about 3100 cycles, its products 1024.  Leaving out any one of the powers, the
// products or the conversions saved under 8%: issuer, rows and codes each take about as long, by latency.
// 4 ragged prompts of 288 to 2500 tokens, 32/8 heads x 64, window 1000: 120 us.
//
// Work.  Segments, blocks, equal ranges for one CTA an SM, records and joins as in
// qg_paged8_attn.cu.  Every wait is bounded; after one has run out (QG_ERR_WAIT_TIMEOUT) no wait
// waits, every role runs through its steps and the CTA ends.
#include <math_constants.h>

#include <algorithm>

#include "qg_mma.cuh"
#include "qg_paged8_attn.cuh"
#include "qg_rows.cuh"
#include "qg_umma.cuh"

namespace qg {
namespace {

constexpr uint32_t kHalf = 128;                  // rows of a half
constexpr uint32_t kLogStep = 6, kStep = 1u << kLogStep;  // slots of a step
constexpr uint32_t kStages = 3;                  // steps of codes in fp16, for K and for V
constexpr uint32_t kGroups = kStep / 16u;        // 16-slot groups of a step, one scale each
constexpr uint32_t kIssueWarp = 0, kCodeWarp0 = 1, kCodeWarps = 7, kRowWarp0 = 8, kRowWarps = 8;
constexpr uint32_t kPromptThreads = (kRowWarp0 + kRowWarps) * 32u;  // four warps a scheduler: 128 registers a thread
constexpr uint32_t kScaleRing = 8;               // steps whose scales are kept: rows are up to 5 behind the K that is stored
constexpr uint32_t kMaxPolls = 4000;             // of up to kPollNs each
constexpr float kCarry = 7.f, kSlack = 8.f;      // log2: the factor of powers, the growth of M that is let pass
constexpr float kRaise = 64.f, kLower = 0x1p-64f;  // log2 of what the summed powers carry more, and what takes it off
constexpr float kLeastFactor = 1e-30f;           // of scores: zero would turn minus infinity into NaN
constexpr uint32_t kPromptHeader = 4;            // what a segment costs beside its blocks, in blocks
static_assert(2u * 256u * 4u <= QG_PAGED_ATTN_ZEROED && kMaxPromptCtas <= 256u, "a counter per CTA and half");
static_assert(kPromptRows == 2u * kHalf, "two halves");

template <int DP>
struct PromptShape {
  static constexpr uint32_t kChunks = DP / 8u;               // 16-byte chunks of a row in fp16
  static constexpr uint32_t kQBytes = kHalf * DP * 2u, kCodeBytes = kStep * DP * 2u;
  static constexpr uint32_t q_at = 0, k_at = 2u * kQBytes, v_at = k_at + kStages * kCodeBytes;
  static constexpr uint32_t scales = v_at + kStages * kCodeBytes;  // [ring][group] {key scale, log2 value scale, its reciprocal x kLower}
  static constexpr uint32_t nan_bits = scales + kScaleRing * kGroups * 16u;  // [stage][slot][8 pieces] 16 columns each
  static constexpr uint32_t row_nan = nan_bits + kStages * kStep * 16u;      // [256 rows] the columns that are NaN
  static constexpr uint32_t kSmem = row_nan + kPromptRows * 16u + 1024u;
  static constexpr uint32_t kRecord = kHalf * (DP + 2u);     // of a half: m[], l[], o[DP / 4][row] float4
};

// Descriptor of an operand in panels of rows of 64 values (128 bytes, swizzled in groups of 8 rows, 1024
// bytes): `panel` the bytes from panel to panel, used where columns are M or N; version 1, 128-byte swizzle.
__device__ __forceinline__ uint64_t panel_desc(uint32_t at, uint32_t panel) {
  return static_cast<uint64_t>((at >> 4) & 0x3FFFu) | (static_cast<uint64_t>(panel >> 4) << 16) |
         (static_cast<uint64_t>(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// the 16-byte piece of row r and values 8 c to 8 c + 7 of a panel
__device__ __forceinline__ uint32_t in_panel(uint32_t r, uint32_t c) { return r * 128u + ((c ^ (r & 7u)) << 4); }
constexpr uint32_t kQPanel = kHalf * 128u, kCodePanel = kStep * 128u;
// fp16 operands, fp32 sums, M = 128
constexpr uint32_t score_idesc() { return (1u << 4) | ((kStep >> 3) << 17) | ((kHalf >> 4) << 24); }
template <int DP>
constexpr uint32_t value_idesc() {  // B MN-major
  return (1u << 4) | (1u << 16) | ((DP >> 3) << 17) | ((kHalf >> 4) << 24);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// A wait that does not end at once, as a call: the roles' loops have to fit the instruction cache together.
__device__ __noinline__ void wait_long(uint64_t* bar, uint32_t parity, volatile uint32_t* abort) {
#pragma unroll 1
  for (uint32_t i = 0; i < kMaxPolls; ++i) {
    if (*abort != 0u) return;
    if (mbar_try_wait_sleep(bar, parity)) return;
  }
  atomicOr(&g_error_word, QG_ERR_WAIT_TIMEOUT);
  *abort = 1u;
}

template <int DP>
__global__ void __launch_bounds__(kPromptThreads, 1) prompt8_kernel(const Paged8View cache, const Attn8Args a) {
  using Shape = PromptShape<DP>;
  const PagedView& c = cache.c;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t q_full[2], s_full[2][2], p_full[2][2], pv_full[2][2], k_full[kStages], k_empty[kStages],
      v_full[kStages], v_empty[kStages], scale_full[kScaleRing], drained;
  __shared__ uint32_t tmem_slot, abort_flag, last_flag[2];
  __shared__ uint32_t nan_flag[kStages][kGroups];
  const uint32_t tid = threadIdx.x, lane = tid & 31u;
  const uint32_t warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  uint8_t* const smem = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
  volatile uint32_t* const abort = &abort_flag;
  if (tid == 0u) {
    for (uint32_t i = 0; i < 2u; ++i) {
      mbar_init(&q_full[i], kHalf / 32u);
      for (uint32_t k = 0; k < 2u; ++k) {
        mbar_init(&s_full[i][k], 1u);
        mbar_init(&p_full[i][k], kHalf / 32u);
        mbar_init(&pv_full[i][k], 1u);
      }
    }
    for (uint32_t i = 0; i < kStages; ++i) {
      mbar_init(&k_full[i], kGroups);
      mbar_init(&k_empty[i], 1u);
      mbar_init(&v_full[i], kGroups);
      mbar_init(&v_empty[i], 1u);
    }
    for (uint32_t i = 0; i < kScaleRing; ++i) mbar_init(&scale_full[i], kGroups);
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
    if (__builtin_expect(!mbar_try_wait(bar, parity), 0)) wait_long(bar, parity, abort);
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

  if (warp >= kRowWarp0) {
    // ================= the rows of a half: a thread has one
    const uint32_t half = (warp - kRowWarp0) / 4u, row = (warp & 3u) * 32u + lane;  // of the half: a lane of tensor memory
    const uint32_t s_at = tmem + half * kHalf + ((warp & 3u) << 21), o_at = s_at + 2u * kHalf;
    uint4* const row_nan = reinterpret_cast<uint4*>(smem + Shape::row_nan) + half * kHalf + row;
    uint32_t steps = 0;                                      // of this half
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
        const uint4* from = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) + token * a.q_stride +
                                                           static_cast<uint64_t>(head) * c.dim);
        auto two = [&](uint32_t u) { return a.dtype == QG_F16 ? unpack2(u, __half()) : unpack2(u, __nv_bfloat16()); };
        constexpr uint32_t kBatch = 4;  // pieces in flight
        auto each = [&](auto work) {
#pragma unroll 1
          for (uint32_t i = 0; i < Shape::kChunks; i += kBatch) {
            uint4 w[kBatch];
#pragma unroll
            for (uint32_t k = 0; k < kBatch; ++k) {
              w[k] = make_uint4(0u, 0u, 0u, 0u);
              if (has && (i + k) * 8u < c.dim) w[k] = from[i + k];
            }
#pragma unroll
            for (uint32_t k = 0; k < kBatch; ++k) work(i + k, w[k]);
          }
        };
        float top = 0.f;
        each([&](uint32_t, uint4 w) {
          const float2 x = two(w.x), y = two(w.y), z = two(w.z), u = two(w.w);
          top = max3(top, max3(fabsf(x.x), fabsf(x.y), fabsf(y.x)), fabsf(y.y));
          top = max3(top, max3(fabsf(z.x), fabsf(z.y), fabsf(u.x)), fabsf(u.y));
        });
        const int power = top == 0.f ? 0 : max(-126, min(126, static_cast<int>(__float_as_uint(top) >> 23) - 127));
        const float by = a.scale_log2 < 0.f ? -power_of_two(-power) : power_of_two(-power);
        mult *= power_of_two(power);
        uint8_t* const to = smem + Shape::q_at + half * Shape::kQBytes;
        each([&](uint32_t i, uint4 w) {
          auto half2 = [&](uint32_t u) {
            const float2 x = two(u);
            return pack2(x.x * by, x.y * by, __half());
          };
          *reinterpret_cast<uint4*>(to + (i >> 3) * kQPanel + in_panel(row, i & 7u)) = make_uint4(half2(w.x), half2(w.y), half2(w.z), half2(w.w));
        });
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0u) mbar_arrive(&q_full[half]);
      }
      float m = -CUDART_INF_F, l = 0.f;
      bool any_nan = false;  // columns of the row are NaN
      for (uint32_t j = from_j; j < to_j; ++j, ++kt, ++steps) {
        const uint32_t slot0 = use.block(j) << kLogStep, ring = kt % kScaleRing, s_now = s_at + (steps & 1u) * kStep;
        const bool whole = use.all_see(a, slot0, kStep);
        const float4* const scale = reinterpret_cast<const float4*>(smem + Shape::scales) + ring * kGroups;
        wait(&s_full[half][steps & 1u], (steps >> 1) & 1u);
        wait(&scale_full[ring], (kt / kScaleRing) & 1u);  // long done: S needed the step's codes
        tc_fence_after();
        uint32_t s[2][32];
        tmem_ld32(s_now, s[0]);
        tmem_ld32(s_now + 32u, s[1]);
        tmem_wait_ld();
        if (__builtin_expect(!whole, 0)) {  // columns that the row does not see become minus infinity
          // the row's slots of the step: up to hi, from lo on or before `first`
          const int32_t hi = p - static_cast<int32_t>(slot0);
          const int32_t lo = a.window == 0u || hi < 0 || a.window > static_cast<uint32_t>(hi)
                                 ? INT32_MIN : hi - static_cast<int32_t>(a.window) + 1;
          const int32_t first = a.sink > slot0 ? static_cast<int32_t>(min(a.sink - slot0, kStep)) : 0;
          auto low = [](int32_t n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; };  // bits [0, n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int32_t at = 32 * i;
            const uint32_t bits = low(hi + 1 - at) & (low(first - at) | ~(lo <= at ? 0u : low(lo - at)));
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              if ((bits >> e & 1u) == 0u) s[i][e] = 0xff800000u;
            }
          }
        }
        // ---- the largest y
        float top = -CUDART_INF_F;
#pragma unroll
        for (uint32_t g = 0; g < kGroups; ++g) {
          const float4 sc = scale[g];
          auto x = [&](int e) { return __uint_as_float(s[g / 2u][16 * (g & 1u) + e]); };
          float u = max3(x(0), x(1), x(2)), v = max3(x(3), x(4), x(5));
          u = max3(u, x(6), x(7)), v = max3(v, x(8), x(9));
          u = max3(u, x(10), x(11)), v = max3(v, x(12), x(13));
          u = max3(u, x(14), x(15));
          top = fmaxf(top, fmaf(fmaxf(u, v), fmaxf(mult * sc.x, kLeastFactor), sc.y));
        }
        // ---- M moves at the first step, and when it has grown by more than the slack
        const float now = fmaxf(m, top);
        if (j == from_j) {
          m = now;
        } else if (__builtin_expect(__any_sync(0xffffffffu, now > m + kSlack), 0)) {
          wait(&pv_full[half][(steps - 1u) & 1u], ((steps - 1u) >> 1) & 1u);  // the sums of the step before are in O
          tc_fence_after();
          const float root = exp2_fast(0.5f * (m - (now == -CUDART_INF_F ? 0.f : now))), fade = root * root;
          m = now;
          l = l * root * root;
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
        const float base = kCarry + kRaise - (m == -CUDART_INF_F ? 0.f : m);
#pragma unroll
        for (uint32_t i = 0; i < 2u; ++i) {
          uint32_t out[16];
#pragma unroll
          for (uint32_t h = 0; h < 2u; ++h) {
            const uint32_t g = 2u * i + h;
            const float4 sc = scale[g];
            const float by = fmaxf(mult * sc.x, kLeastFactor), plus = sc.y + base;
            const F2 by2 = f2(by, by), plus2 = f2(plus, plus);
            F2 sum = f2(0.f, 0.f);
#pragma unroll
            for (uint32_t e = 0; e < 16u; e += 2u) {
              const float2 y = split(fma(f2(__uint_as_float(s[i][16u * h + e]), __uint_as_float(s[i][16u * h + e + 1u])), by2, plus2));
              const F2 x = f2(exp2_fast(y.x), exp2_fast(y.y));
              sum = sum + x;
              const float2 power = split(x * f2(kLower, kLower));
              out[8u * h + e / 2u] = pack2(power.x, power.y, __half());
            }
            const float2 z = split(sum);
            l = fmaf(z.x + z.y, sc.z, l);
          }
          tmem_st16(s_now + 16u * i, out);
        }
        if (__builtin_expect(!whole, 0)) {  // a NaN value that some rows see and some do not was taken out of the codes
          const uint32_t stage = kt % kStages;
          wait(&v_full[stage], (kt / kStages) & 1u);
#pragma unroll 1
          for (uint32_t e = 0; e < kStep; ++e) {
            if (nan_flag[stage][e / 16u] == 0u) {
              e |= 15u;
              continue;
            }
            {
              const uint4 bits = reinterpret_cast<const uint4*>(smem + Shape::nan_bits)[stage * kStep + e];
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
        __syncwarp();
        if (lane == 0u) mbar_arrive(&p_full[half][steps & 1u]);
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
      wait(&pv_full[half][(steps - 1u) & 1u], ((steps - 1u) >> 1) & 1u);
      tc_fence_after();
      const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
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
            const float root = exp2_fast(0.5f * (__ldcg(record_of(i) + row) - from));
            all = fmaf(__ldcg(record_of(i) + kHalf + row) * root, root, all);
          }
          const float by = all == 0.f ? 0.f : 1.f / all;
#pragma unroll 1
          for (uint32_t i0 = 0; i0 < DP / 16u; ++i0) {  // 16 columns at a time
            float x[16] = {};
#pragma unroll 2
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
  } else if (warp >= kCodeWarp0) {
    // ================= codes to fp16, in turns: of a step's 16-slot group this thread has places r and 8 + r and
    // every fourth 16-code piece, so 8 lanes write 128 consecutive bytes and read 64 of a row
    constexpr uint32_t kMine = DP / 64u;                     // pieces of a row
    const uint32_t r = lane & 7u, pq = lane >> 3;
    Segment8 s = use;
    uint32_t rem = left;                                     // steps from s.j on
    uint32_t turn = warp - kCodeWarp0;                       // this warp's next, in groups from the step of s on
    uint32_t step = 0;                                       // of the range, where s is
    // Of a turn ahead: the group's page, first place on it, kv head, flags (row i is seen by some; bit 2 + i: by
    // all; bit 4: any), step and group.
    uint32_t id = 0, on = 0, kv = 0, seen = 0, at_step = 0, at_group = 0;
    bool ahead = false;                                      // there is a turn looked up
    auto look = [&]() {
#pragma unroll 1
      while (turn >= kGroups && rem != 0u) {
        turn -= kGroups;
        ++step;
        ++s.j;
        --rem;
        if (s.j == s.j1) advance(s, rem);
      }
      ahead = rem != 0u;
      if (!ahead) return;
      const uint32_t slot = (s.block(s.j) << kLogStep) + 16u * turn, at = div_by(slot, c.page);
      on = slot - at * c.page.d;
      kv = s.kv;
      at_step = step;
      at_group = turn;
      id = c.num_pages;
      if (s.all_see(a, slot, 16u)) {
        seen = 31u;
      } else {
        seen = s.some_see(slot, 16u) ? 16u : 0u;
#pragma unroll
        for (uint32_t i = 0; i < 2u; ++i) {
          if (s.some_see(slot + 8u * i + r, 1u)) seen |= 1u << i;
          if (s.all_see(a, slot + 8u * i + r, 1u)) seen |= 4u << i;
        }
      }
      if (seen > 15u) id = static_cast<uint32_t>(c.table[static_cast<size_t>(s.b) * c.table_stride + at]);
      turn += kCodeWarps;
    };
    uint32_t flags = 0, now_step = 0, now_group = 0;
    float ks = 0.f, vs = 1.f;
    uint64_t off = 0;
    uint4 kw[2][kMine], vw[2][kMine];
    auto place = [&]() {  // of the turn looked up last
      flags = seen & 15u;
      now_step = at_step;
      now_group = at_group;
      ks = 0.f;
      vs = 1.f;
      if (id >= c.num_pages) {
        flags = 0u;
        if (seen > 15u) atomicOr(&g_error_word, QG_ERR_PAGE);
        return;
      }
      off = id * c.page_bytes + kv * c.head_bytes + (on + r) * c.slot_bytes + pq * 16u;
      const uint64_t in = id * cache.scale_page + kv * cache.scale_head + (on >> cache.log_block);
      ks = cache.ks[in];
      vs = cache.vs[in];
    };
    auto load = [&](const uint8_t* pool, uint4 (&to)[2][kMine]) {
#pragma unroll
      for (uint32_t i = 0; i < 2u; ++i) {
#pragma unroll
        for (uint32_t h = 0; h < kMine; ++h) {
          to[i][h] = make_uint4(0u, 0u, 0u, 0u);
          if ((flags >> i & 1u) != 0u && (pq + 4u * h) * 16u < c.dim) {
            to[i][h] = *reinterpret_cast<const uint4*>(pool + off + i * 8u * c.slot_bytes + h * 64u);
          }
        }
      }
    };
    // piece pq + 4 h is chunks 2 pq and 2 pq + 1 of panel h
    const uint32_t chunk0 = in_panel(r, 2u * pq), chunk1 = in_panel(r, 2u * pq + 1u);
    auto store = [&](uint8_t* at, const uint4 (&from)[2][kMine]) {
#pragma unroll
      for (uint32_t i = 0; i < 2u; ++i) {
#pragma unroll
        for (uint32_t h = 0; h < kMine; ++h) {
          uint8_t* const to = at + h * kCodePanel + i * 1024u;
          uint4 x, y;
          codes_to_half(from[i][h].x, x.x, x.y);
          codes_to_half(from[i][h].y, x.z, x.w);
          codes_to_half(from[i][h].z, y.x, y.y);
          codes_to_half(from[i][h].w, y.z, y.w);
          *reinterpret_cast<uint4*>(to + chunk0) = x;
          *reinterpret_cast<uint4*>(to + chunk1) = y;
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
    };
    look();
    bool more = ahead;
    if (more) {
      place();
      load(c.k, kw);
      load(c.v, vw);
      look();
    }
    // A turn's codes are stored while the next one's are loaded and the page of the one after is looked up.
#pragma unroll 1
    while (more) {
      const uint32_t round = now_step / kStages, stage = now_step - round * kStages, ring = now_step % kScaleRing;
      const uint32_t group = now_group, now_flags = flags;
      uint8_t* const tile = smem + Shape::k_at + stage * Shape::kCodeBytes + group * 2048u;
      if (round != 0u) wait(&k_empty[stage], (round - 1u) & 1u);
      if (lane == 0u) {
        const float to = fminf(fmaxf(vs, 0x1p-60f), 0x1p60f);
        reinterpret_cast<float4*>(smem + Shape::scales)[ring * kGroups + group] = make_float4(ks, log2f(to), kLower / to, 0.f);
      }
      store(tile, kw);
      if (lane == 0u) {
        mbar_arrive(&k_full[stage]);
        mbar_arrive(&scale_full[ring]);
      }
      more = ahead;
      if (more) {
        place();
        load(c.k, kw);
        look();
      }
      // NaN codes of rows that not all see: out of the codes, noted by column
      bool flagged = false;
      if (__builtin_expect(now_flags != 15u, 0)) {
        uint32_t odd = 0;
#pragma unroll
        for (uint32_t i = 0; i < 2u; ++i) {
#pragma unroll
          for (uint32_t h = 0; h < kMine; ++h) {
            auto nan = [](uint32_t u) { return ((u & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; };
            if ((now_flags >> (2u + i) & 1u) == 0u) odd |= nan(vw[i][h].x) | nan(vw[i][h].y) | nan(vw[i][h].z) | nan(vw[i][h].w);
          }
        }
        flagged = odd != 0u;
      }
      flagged = __any_sync(0xffffffffu, flagged);
      if (round != 0u) wait(&v_empty[stage], (round - 1u) & 1u);
      if (__builtin_expect(flagged, 0)) {
#pragma unroll
        for (uint32_t i = 0; i < 2u; ++i) {
#pragma unroll
          for (uint32_t h = 0; h < 2u; ++h) {  // both halves of a row's 128 columns
            uint32_t bits = 0;
            if (h < kMine && (now_flags >> (2u + i) & 1u) == 0u) {
              auto clean = [&](uint32_t& word, uint32_t e) {
                const uint32_t is = (((word & 0x7f7f7f7fu) + 0x01010101u) >> 7) & 0x01010101u;
                word &= ~(is * 0xffu);
                bits |= (is * 0x01020408u >> 24 & 15u) << (4u * e);
              };
              uint4& w = vw[i][h % kMine];
              clean(w.x, 0u), clean(w.y, 1u), clean(w.z, 2u), clean(w.w, 3u);
            }
            reinterpret_cast<uint16_t*>(smem + Shape::nan_bits)[(stage * kStep + 16u * group + 8u * i + r) * 8u + pq + 4u * h] =
                static_cast<uint16_t>(bits);
          }
        }
      }
      if (lane == 0u) nan_flag[stage][group] = flagged ? 1u : 0u;
      store(tile + (Shape::v_at - Shape::k_at), vw);
      if (lane == 0u) mbar_arrive(&v_full[stage]);
      if (more) load(c.v, vw);
    }
  } else if (elect_one()) {
    // ================= the products, by one thread
    uint32_t parts[2] = {0u, 0u}, steps[2] = {0u, 0u};
    uint32_t k_stage = 0, k_round = 0, v_stage = 0, v_round = 0;
    const uint32_t base = smem_addr(smem);
    const uint64_t q0 = panel_desc(base + Shape::q_at, kQPanel), k0 = panel_desc(base + Shape::k_at, kCodePanel);
    const uint64_t v0 = panel_desc(base + Shape::v_at, kCodePanel);
    auto scores = [&](uint32_t half, uint32_t buffer) {  // of the K stage
      const uint64_t q = q0 + half * (Shape::kQBytes / 16u), k = k0 + k_stage * (Shape::kCodeBytes / 16u);
      const uint32_t s = tmem + half * kHalf + buffer * kStep;
#pragma unroll
      for (uint32_t i = 0; i < DP / 16u; ++i) {  // 32 bytes of the rows of panel i / 4
        umma_ss(s, q + (i / 4u * kQPanel + i % 4u * 32u) / 16u, k + (i / 4u * kCodePanel + i % 4u * 32u) / 16u, score_idesc(), i);
      }
    };
    auto values = [&](uint32_t half, uint32_t buffer, uint32_t more) {  // of the V stage
      const uint64_t v = v0 + v_stage * (Shape::kCodeBytes / 16u);
      const uint32_t p = tmem + half * kHalf + buffer * kStep, o = tmem + 2u * kHalf + half * kHalf;
#pragma unroll
      for (uint32_t i = 0; i < kStep / 16u; ++i) umma_ts(o, p + 8u * i, v + i * (2048u / 16u), value_idesc<DP>(), more | i);
    };
    for (; left != 0u; advance(use, left)) {
      const uint32_t count = min(use.j1 - use.j, left), halves = use.rows > kHalf ? 2u : 1u;
      left -= count;
#pragma unroll
      for (uint32_t h = 0; h < 2u; ++h) {
        if (h < halves) wait(&q_full[h], parts[h]++ & 1u);
      }
      // step i's scores two ahead of its sums: S(i) is free once the sums of step i - 2 have been issued
#pragma unroll 1
      for (uint32_t i = 0; i < count + 2u; ++i) {
        const bool sums = i >= 2u, more = i < count;
        if (sums) wait(&v_full[v_stage], v_round & 1u);
        if (more) wait(&k_full[k_stage], k_round & 1u);
#pragma unroll
        for (uint32_t h = 0; h < 2u; ++h) {
          if (h >= halves) break;
          const uint32_t buffer = steps[h] & 1u;
          if (sums) {
            wait(&p_full[h][buffer], ((steps[h] - 2u) >> 1) & 1u);
            tc_fence_after();
            values(h, buffer, i - 2u);
            umma_commit(&pv_full[h][buffer]);
          }
          if (more) {
            tc_fence_after();
            scores(h, buffer);
            umma_commit(&s_full[h][buffer]);
          }
          ++steps[h];
        }
        if (sums) {
          umma_commit(&v_empty[v_stage]);
          if (++v_stage == kStages) v_stage = 0u, ++v_round;
        }
        if (more) {
          umma_commit(&k_empty[k_stage]);
          if (++k_stage == kStages) k_stage = 0u, ++k_round;
        }
      }
#pragma unroll
      for (uint32_t h = 0; h < 2u; ++h) {
        if (h < halves) steps[h] -= 2u;
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
  e = launch_plan8(c, a, kPromptRows, kLogStep, kLogStep, stream);
  if (e != cudaSuccess) return e;
  return launch_k(kernel, grid, kPromptThreads, Shape::kSmem, stream, c, a);
}

}  // namespace

cudaError_t launch_prompt8(const Paged8View& c, const Attn8Args& a, uint32_t dp, cudaStream_t stream) {
  return dp == 64u ? launch_prompt8<64>(c, a, stream) : launch_prompt8<128>(c, a, stream);
}

}  // namespace qg

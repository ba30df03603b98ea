// qg_paged_append.cu -- qg_qk_norm_rope_append: per-head RMSNorm, rotation and paged-cache
// append of new queries, keys and values in one pass (declared in include/qgemv_b200.h).
//
// One row is one head of one token.  A row is held by LPR lanes with two pieces of 8 values
// each: of the rotated part lane c has pairs 8 c to 8 c + 7 whole, as values 16 c to 16 c + 15
// where pairs are neighbours and as 8 c .. + 7 of either half where they lie half a width
// apart, so the rotation never leaves a lane and takes the same eight cosines and sines for
// every head of the token; the norm's weights are multiplied into them once.  The sum of
// squares is log2(LPR) shuffles.  Arithmetic is on pairs of fp32 (f32x2).
//
// Bound by memory: a value is read once and written once for ~7 flops.  A warp's task is one
// batch of query, key or value rows of one token; it asks for all of it before it looks up
// where the token goes, so 2 KB are in flight behind one latency and no warp waits for another.
// 16384 tokens of 64/8 heads x 128 bf16: 132 us, 5.1 TB/s of the bytes that have to move, 80%
// of a plain copy's rate; issue and latency share the rest (24 warps an SM).
#include "qg_paged.cuh"

namespace qg {
namespace {

constexpr uint32_t kAppendWarps = 4;
// Rows that a lane has in flight: 64 bytes.  (128 bytes a lane take 126 registers; 16 warps an
// SM then measured 144 us where 24 warps with half as much each measure 131 us.)
template <typename T>
constexpr uint32_t kBatch = 4 / sizeof(T);

struct AppendArgs {
  const void *q, *k, *v;
  void* q_out;
  uint64_t q_stride, k_stride, v_stride, q_out_stride;  // elements, token to token
  const float *q_norm, *k_norm, *rope;
  const int32_t *positions, *slots, *seqs;
  float eps, inv_dim;
  uint32_t n_q, rot, rope_rows, tokens;
  uint32_t q_parts, kv_parts;                           // tasks of a token's queries, keys (values)
};

// Two fp32 values in a register pair, worked on by one instruction.
struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 split(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// Eight consecutive values as loaded, and stored.
template <typename T>
struct Piece {
  uint4 w;
  __device__ __forceinline__ void load(const void* p) { w = *static_cast<const uint4*>(p); }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    const float2 a = unpack2(w.x, T()), b = unpack2(w.y, T()), c = unpack2(w.z, T()), d = unpack2(w.w, T());
    x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y, x[4] = c.x, x[5] = c.y, x[6] = d.x, x[7] = d.y;
  }
};
template <>
struct Piece<float> {
  float4 a, b;
  __device__ __forceinline__ void load(const void* p) {
    a = static_cast<const float4*>(p)[0];
    b = static_cast<const float4*>(p)[1];
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  }
};
template <typename T>
__device__ __forceinline__ void store8(void* p, const float (&x)[8]) {
  *static_cast<uint4*>(p) = make_uint4(pack2(x[0], x[1], T()), pack2(x[2], x[3], T()), pack2(x[4], x[5], T()),
                                       pack2(x[6], x[7], T()));
}
template <>
__device__ __forceinline__ void store8<float>(void* p, const float (&x)[8]) {
  static_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  static_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}

// A lane's two pieces as 8 pairs (u, v) to be turned; u[h] and v[h] hold pairs 2 h, 2 h + 1.
struct Pairs {
  F2 u[4], v[4];
};
template <bool HALVES>
__device__ __forceinline__ Pairs pairs_of(const float (&a)[8], const float (&b)[8]) {
  if constexpr (HALVES) {
    return {{f2(a[0], a[1]), f2(a[2], a[3]), f2(a[4], a[5]), f2(a[6], a[7])},
            {f2(b[0], b[1]), f2(b[2], b[3]), f2(b[4], b[5]), f2(b[6], b[7])}};
  }
  return {{f2(a[0], a[2]), f2(a[4], a[6]), f2(b[0], b[2]), f2(b[4], b[6])},
          {f2(a[1], a[3]), f2(a[5], a[7]), f2(b[1], b[3]), f2(b[5], b[7])}};
}
template <bool HALVES>
__device__ __forceinline__ void values_of(const Pairs& p, float (&a)[8], float (&b)[8]) {
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    const float2 u = split(p.u[h]), v = split(p.v[h]);
    if constexpr (HALVES) {
      a[2 * h] = u.x, a[2 * h + 1] = u.y, b[2 * h] = v.x, b[2 * h + 1] = v.y;
    } else {
      float(&x)[8] = h < 2 ? a : b;
      const int e = 4 * (h & 1);
      x[e] = u.x, x[e + 1] = v.x, x[e + 2] = u.y, x[e + 3] = v.y;
    }
  }
}

// T: type of q, k, v, q_out; C: type of the cache; HALVES: pairs half a width apart.
template <typename T, typename C, int LPR, bool HALVES>
__global__ void __launch_bounds__(kAppendWarps * 32, 6) append_kernel(const PagedView c, const AppendArgs a) {
  constexpr uint32_t kSide = 32 / LPR;               // rows side by side
  constexpr uint32_t kRows = kSide * kBatch<T>;      // rows of a task
  const uint32_t lane = threadIdx.x % 32u, chunk = lane % LPR;
  const uint32_t t = blockIdx.x * kAppendWarps + threadIdx.x / 32u;
  if (t >= a.tokens) return;
  // the task's rows: heads [first, heads) of the queries, the keys or the values, kRows at most
  uint32_t part = blockIdx.y;
  const bool is_q = part < a.q_parts, is_k = !is_q && part < a.q_parts + a.kv_parts;
  if (!is_q) part -= is_k ? a.q_parts : a.q_parts + a.kv_parts;
  const uint32_t heads = is_q ? a.n_q : c.n_kv, first = part * kRows, head0 = first + lane / LPR;
  const bool turned = chunk * 16u < a.rot && (is_q || is_k);
  // the lane's pieces
  const uint32_t at0 = HALVES && turned ? chunk * 8u : chunk * 16u;
  const uint32_t at1 = HALVES && turned ? a.rot / 2u + chunk * 8u : chunk * 16u + 8u;
  const bool has0 = at0 < c.dim, has1 = at1 < c.dim;
  pdl_wait();
  pdl_trigger();
  const bool full = c.dim == LPR * 16u && first + kRows <= heads;  // every lane holds rows
  const T* src = static_cast<const T*>(is_q ? a.q : is_k ? a.k : a.v) +
                 t * (is_q ? a.q_stride : is_k ? a.k_stride : a.v_stride) + head0 * c.dim;
  const uint32_t src_step = kSide * c.dim;
  Piece<T> raw[kBatch<T>][2];
  if (full) {
#pragma unroll
    for (uint32_t i = 0; i < kBatch<T>; ++i) {
      raw[i][0].load(src + at0 + i * src_step);
      raw[i][1].load(src + at1 + i * src_step);
    }
  } else {
#pragma unroll
    for (uint32_t i = 0; i < kBatch<T>; ++i) {
      raw[i][0] = raw[i][1] = Piece<T>{};
      if (has0 && head0 + i * kSide < heads) raw[i][0].load(src + at0 + i * src_step);
      if (has1 && head0 + i * kSide < heads) raw[i][1].load(src + at1 + i * src_step);
    }
  }
  int32_t pos = a.positions[t];
  const int32_t given_slot = a.slots != nullptr ? a.slots[t] : pos;
  const uint32_t seq = a.seqs != nullptr ? static_cast<uint32_t>(a.seqs[t]) : t;
  const float* norm = is_q ? a.q_norm : is_k ? a.k_norm : nullptr;
  float wa[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f}, wb[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
  if (norm != nullptr) {
    Piece<float> w;
    if (has0) w.load(norm + at0), w.get(wa);
    if (has1) w.load(norm + at1), w.get(wb);
  }
  if (pos >= 0 && a.rot != 0u && static_cast<uint32_t>(pos) >= a.rope_rows) {
    if (lane == 0u) atomicOr(&g_error_word, QG_ERR_POSITION);
    pos = -1;
  }
  // where the task's rows go: the first, and the bytes from one step to the next
  uint8_t* to = nullptr;
  uint64_t to_step = kSide * c.head_bytes;
  if (is_q) {
    to = reinterpret_cast<uint8_t*>(static_cast<T*>(a.q_out) + t * a.q_out_stride + head0 * c.dim);
    to_step = kSide * c.dim * sizeof(T);
  } else if (pos >= 0 && given_slot >= 0) {
    if (static_cast<uint32_t>(given_slot) < c.capacity && seq < c.batch) {
      const uint64_t at = paged_row(c, c.table + static_cast<size_t>(seq) * c.table_stride,
                                    static_cast<uint32_t>(given_slot), head0);
      if (at != kNoRow) to = (is_k ? c.k : c.v) + at;
    } else if (lane == 0u) {
      atomicOr(&g_error_word, QG_ERR_PAGE);
    }
  }
  if (to == nullptr) return;  // nothing to append

  if (pos < 0 || !(is_q || is_k)) {  // a padding row's queries are zero; values are rounded alone
#pragma unroll
    for (uint32_t i = 0; i < kBatch<T>; ++i) {
      if (first + i * kSide >= heads) break;
      const bool live = head0 + i * kSide < heads;
      float xa[8] = {}, xb[8] = {};
      if (pos >= 0) {
        raw[i][0].get(xa);
        raw[i][1].get(xb);
      }
      uint8_t* row = to + i * to_step;
      if (live && has0) is_q ? store8<T>(row + at0 * sizeof(T), xa) : store8<C>(row + at0 * 2u, xa);
      if (live && has1) is_q ? store8<T>(row + at1 * sizeof(T), xb) : store8<C>(row + at1 * 2u, xb);
    }
    return;
  }

  // u <- u uu + v uv, v <- v vv + u vu: the rotation with the weights in it
  Pairs w = pairs_of<HALVES>(wa, wb);
  F2 uu[4], uv[4], vu[4], vv[4];
#pragma unroll
  for (int h = 0; h < 4; ++h) {
    uu[h] = w.u[h];
    vv[h] = w.v[h];
    uv[h] = vu[h] = f2(0.f, 0.f);
  }
  if (turned) {
    const float* angles = a.rope + static_cast<size_t>(pos) * a.rot + chunk * 8u;
    Piece<float> cos, sin;
    cos.load(angles);
    sin.load(angles + a.rot / 2u);
    float cs[8], sn[8];
    cos.get(cs);
    sin.get(sn);
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const F2 co = f2(cs[2 * h], cs[2 * h + 1]), si = f2(sn[2 * h], sn[2 * h + 1]);
      uv[h] = w.v[h] * f2(-sn[2 * h], -sn[2 * h + 1]);
      vu[h] = w.u[h] * si;
      uu[h] = w.u[h] * co;
      vv[h] = w.v[h] * co;
    }
  }
  const bool some_stay = a.rot != c.dim;  // lanes whose pairs do not turn: 0 x infinity is kept out
  auto head = [&](uint32_t i, float (&xa)[8], float (&xb)[8]) {
    raw[i][0].get(xa);
    raw[i][1].get(xb);
    Pairs p = pairs_of<HALVES>(xa, xb);
    float inv = 1.f;
    if (norm != nullptr) {
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
      inv = rsqrtf(ss * a.inv_dim + a.eps);
    }
    const F2 by = f2(inv, inv);
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const F2 u = by * p.u[h], v = by * p.v[h];
      if (some_stay && !turned) {
        p.u[h] = u * uu[h];
        p.v[h] = v * vv[h];
      } else {
        p.u[h] = fma(u, uu[h], v * uv[h]);
        p.v[h] = fma(v, vv[h], u * vu[h]);
      }
    }
    values_of<HALVES>(p, xa, xb);
  };
#pragma unroll
  for (uint32_t i = 0; i < kBatch<T>; ++i) {
    if (first + i * kSide >= heads) break;
    float xa[8], xb[8];
    head(i, xa, xb);
    const bool live = full || head0 + i * kSide < heads;
    uint8_t* row = to + i * to_step;
    if (is_q) {
      if (live && has0) store8<T>(row + at0 * sizeof(T), xa);
      if (live && has1) store8<T>(row + at1 * sizeof(T), xb);
    } else {
      if (live && has0) store8<C>(row + at0 * 2u, xa);
      if (live && has1) store8<C>(row + at1 * 2u, xb);
    }
  }
}

template <typename T, typename C, int LPR>
cudaError_t launch_append(const PagedView& c, const AppendArgs& a, bool halves,
                          cudaStream_t stream) {
  constexpr uint32_t kRows = 32 / LPR * kBatch<T>;
  AppendArgs w = a;
  w.q_parts = (a.n_q + kRows - 1u) / kRows;
  w.kv_parts = (c.n_kv + kRows - 1u) / kRows;
  const dim3 grid((a.tokens + kAppendWarps - 1u) / kAppendWarps, w.q_parts + 2u * w.kv_parts);
  if (halves) return launch_k(append_kernel<T, C, LPR, true>, grid, kAppendWarps * 32, 0, stream, c, w);
  return launch_k(append_kernel<T, C, LPR, false>, grid, kAppendWarps * 32, 0, stream, c, w);
}

template <typename T, typename C>
cudaError_t launch_append(const PagedView& c, const AppendArgs& a, bool halves,
                          cudaStream_t stream) {
  if (c.dim <= 64u) return launch_append<T, C, 4>(c, a, halves, stream);
  if (c.dim <= 128u) return launch_append<T, C, 8>(c, a, halves, stream);
  return launch_append<T, C, 16>(c, a, halves, stream);
}

template <typename C>
cudaError_t launch_append(int dtype, const PagedView& c, const AppendArgs& a, bool halves, cudaStream_t stream) {
  if (dtype == QG_F32) return launch_append<float, C>(c, a, halves, stream);
  if (dtype == QG_F16) return launch_append<__half, C>(c, a, halves, stream);
  return launch_append<__nv_bfloat16, C>(c, a, halves, stream);
}

}  // namespace
}  // namespace qg

extern "C" cudaError_t qg_qk_norm_rope_append(const qg_kv_pages* cache, const qg_append* p,
                                              cudaStream_t stream) {
  using namespace qg;
  PagedView c;
  if (!paged_view(cache, &c) || p == nullptr || !dtype_ok(p->dtype)) return cudaErrorInvalidValue;
  if (p->tokens == 0u) return cudaSuccess;
  if (p->tokens > 0x7fffffffu || static_cast<uint64_t>(p->n_q_heads) + 2u * c.n_kv > 65535u || p->positions == nullptr || p->k == nullptr ||
      p->v == nullptr || (p->n_q_heads != 0u && (p->q == nullptr || p->q_out == nullptr))) {
    return cudaErrorInvalidValue;
  }
  if (p->seqs == nullptr && p->tokens > cache->batch) return cudaErrorInvalidValue;
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
  AppendArgs a{};
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
  a.slots = p->slots;
  a.seqs = p->seqs;
  a.eps = p->eps;
  a.inv_dim = 1.f / static_cast<float>(c.dim);
  a.n_q = p->n_q_heads;
  a.rot = p->rot_dim;
  a.rope_rows = p->rope_rows;
  a.tokens = p->tokens;
  const bool halves = p->pairs == QG_PAIRS_HALVES;
  return cache->dtype == QG_F16 ? launch_append<__half>(p->dtype, c, a, halves, stream)
                                : launch_append<__nv_bfloat16>(p->dtype, c, a, halves, stream);
}

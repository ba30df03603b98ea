// qg_paged_append.cu -- qg_qk_norm_rope_append: per-head RMSNorm, rotation and paged-cache
// append of new queries, keys and values in one pass (declared in include/qgemv_b200.h).
//
// One row is one head of one token.  A row is held by LPR lanes, 8 consecutive values each
// (16 bytes of a 16-bit type, two 16-byte loads of fp32), so the sum of squares is log2(LPR)
// shuffles; the rotation of adjacent pairs stays inside a lane and that of half-width pairs
// takes one shuffle a value (the partner lies rot_dim / 16 lanes away, in the same place).
//
// Bound by memory: a value is read once and written once for ~7 flops.
#include "qg_paged.cuh"

namespace qg {
namespace {

constexpr uint32_t kAppendThreads = 256;

struct AppendArgs {
  const void *q, *k, *v;
  void* q_out;
  uint64_t q_stride, k_stride, v_stride, q_out_stride;  // elements, token to token
  const float *q_norm, *k_norm, *rope;
  const int32_t *positions, *slots, *seqs;
  float eps;
  uint32_t n_q, rows, rot, rope_rows;
  bool halves;
};

// T: type of q, k, v, q_out; C: type of the cache.
template <typename T, typename C, int LPR>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const PagedView c, const AppendArgs a) {
  constexpr uint32_t kRows = kAppendThreads / LPR;  // rows in flight
  const uint32_t t = blockIdx.x, chunk = threadIdx.x % LPR;
  const uint32_t lane_mask = 0xffffffffu;
  const uint32_t i0 = chunk * 8u;
  const bool active = i0 < c.dim;
  pdl_wait();
  pdl_trigger();
  int32_t pos = a.positions[t];
  if (pos >= 0 && a.rot != 0u && static_cast<uint32_t>(pos) >= a.rope_rows) {
    if (threadIdx.x == 0u) atomicOr(&g_error_word, QG_ERR_POSITION);
    pos = -1;
  }
  // the sequence's page list and slot, or nothing to append
  const int32_t* pages = nullptr;
  uint32_t slot = 0;
  if (pos >= 0) {
    const int32_t s = a.slots != nullptr ? a.slots[t] : pos;
    if (s >= 0) {
      const uint32_t seq = a.seqs != nullptr ? static_cast<uint32_t>(a.seqs[t]) : t;
      if (static_cast<uint32_t>(s) < c.capacity && seq < c.batch) {
        slot = static_cast<uint32_t>(s);
        pages = c.table + static_cast<size_t>(seq) * c.table_stride;
      } else if (threadIdx.x == 0u) {
        atomicOr(&g_error_word, QG_ERR_PAGE);
      }
    }
  }
  // x[e] <- x[e] cs[e] + partner[e] sn[e]: the second of a pair adds, the first subtracts
  const bool turns = pos >= 0 && i0 < a.rot;
  const uint32_t half = a.rot / 2u;
  float cs[8], sn[8];
  if (turns) {
    const float* row = a.rope + static_cast<size_t>(pos) * a.rot;
    if (a.halves) {
      const uint32_t at = i0 < half ? i0 : i0 - half;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        cs[e] = row[at + e];
        sn[e] = i0 < half ? -row[half + at + e] : row[half + at + e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        cs[e] = row[i0 / 2u + e / 2];
        sn[e] = (e & 1) ? row[half + i0 / 2u + e / 2] : -row[half + i0 / 2u + e / 2];
      }
    }
  }
  const uint32_t first = threadIdx.x / LPR;
  for (uint32_t r0 = 0; r0 < a.rows; r0 += kRows) {
    const uint32_t r = r0 + first;
    const bool is_q = r < a.n_q, is_k = !is_q && r < a.n_q + c.n_kv;
    const uint32_t head = is_q ? r : is_k ? r - a.n_q : r - a.n_q - c.n_kv;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (active && r < a.rows && pos >= 0) {
      const T* src = is_q ? static_cast<const T*>(a.q) + t * a.q_stride
                     : is_k ? static_cast<const T*>(a.k) + t * a.k_stride
                            : static_cast<const T*>(a.v) + t * a.v_stride;
      Raw8<T> raw;
      raw.load(src + head * c.dim + i0);
      raw.get(x);
    }
    const float* w = is_q ? a.q_norm : is_k ? a.k_norm : nullptr;
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(x[e], x[e], ss);
#pragma unroll
    for (int off = LPR / 2; off > 0; off >>= 1) ss += __shfl_xor_sync(lane_mask, ss, off, LPR);
    if (w != nullptr && active && pos >= 0) {  // a padding row stays zero for any eps
      const float inv = rsqrtf(ss / static_cast<float>(c.dim) + a.eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] *= inv * w[i0 + e];
    }
    float partner[8];
    if (a.halves) {
      const int from = static_cast<int>(i0 < half ? chunk + half / 8u : chunk - half / 8u);
#pragma unroll
      for (int e = 0; e < 8; ++e) partner[e] = __shfl_sync(lane_mask, x[e], from, LPR);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) partner[e] = x[e ^ 1];
    }
    if (turns && (is_q || is_k)) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = fmaf(x[e], cs[e], partner[e] * sn[e]);
    }
    if (!active || r >= a.rows) continue;
    if (is_q) {
      store8(static_cast<T*>(a.q_out) + t * a.q_out_stride + head * c.dim + i0, x);
    } else if (pages != nullptr) {
      const uint64_t at = paged_row(c, pages, slot, head);
      if (at != kNoRow) store8(reinterpret_cast<C*>((is_k ? c.k : c.v) + at) + i0, x);
    }
  }
}

template <typename T, typename C>
cudaError_t launch_append(const PagedView& c, const AppendArgs& a, uint32_t tokens, cudaStream_t stream) {
  const dim3 grid(tokens);
  if (c.dim <= 64u) return launch_k(append_kernel<T, C, 8>, grid, kAppendThreads, 0, stream, c, a);
  if (c.dim <= 128u) return launch_k(append_kernel<T, C, 16>, grid, kAppendThreads, 0, stream, c, a);
  return launch_k(append_kernel<T, C, 32>, grid, kAppendThreads, 0, stream, c, a);
}

template <typename C>
cudaError_t launch_append(int dtype, const PagedView& c, const AppendArgs& a, uint32_t tokens,
                          cudaStream_t stream) {
  if (dtype == QG_F32) return launch_append<float, C>(c, a, tokens, stream);
  if (dtype == QG_F16) return launch_append<__half, C>(c, a, tokens, stream);
  return launch_append<__nv_bfloat16, C>(c, a, tokens, stream);
}

}  // namespace
}  // namespace qg

extern "C" cudaError_t qg_qk_norm_rope_append(const qg_kv_pages* cache, const qg_append* p,
                                              cudaStream_t stream) {
  using namespace qg;
  PagedView c;
  if (!paged_view(cache, &c) || p == nullptr || !dtype_ok(p->dtype)) return cudaErrorInvalidValue;
  if (p->tokens == 0u) return cudaSuccess;
  if (p->tokens > 0x7fffffffu || p->n_q_heads > 65535u || p->positions == nullptr || p->k == nullptr ||
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
  a.n_q = p->n_q_heads;
  a.rows = p->n_q_heads + 2u * c.n_kv;
  a.rot = p->rot_dim;
  a.rope_rows = p->rope_rows;
  a.halves = p->pairs == QG_PAIRS_HALVES;
  return cache->dtype == QG_F16 ? launch_append<__half>(p->dtype, c, a, p->tokens, stream)
                                : launch_append<__nv_bfloat16>(p->dtype, c, a, p->tokens, stream);
}

// qg_paged8.cuh -- what the operators of the 8-bit paged cache share: the checked view of pools,
// scales and table, the rows of a call, and e4m3 codes.
#pragma once

#include <cuda_fp8.h>

#include "qg_paged.cuh"

namespace qg {

struct Paged8View {
  PagedView c;                      // pools in bytes
  float *ks, *vs;
  uint64_t scale_page, scale_head;  // elements
  uint32_t log_block;               // log2 of the slots of a block
};

constexpr int kLeastPower = -60, kMostPower = 60;   // of a block's scale

// Four codes as two fp16 pairs (exact).
__device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\t"
      "mov.b32 {l, h}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, l;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, h;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}
__device__ __forceinline__ void codes_to_float(uint32_t w, float (&x)[4]) {
  uint32_t lo, hi;
  codes_to_half(w, lo, hi);
  const float2 a = unpack2(lo, __half()), b = unpack2(hi, __half());
  x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
}
// Four values as codes, to nearest even, saturating; NaN is 0x7f.
__device__ __forceinline__ uint32_t float_to_codes(float a, float b, float c, float d) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}

// Rows [first, first + n) of a call that are sequence b's, and its slots; n 0 for a sequence that
// is padding, has no rows or does not fit (QG_ERR_PAGE).
struct Rows8 {
  uint32_t first, n, len;
};
__device__ __forceinline__ Rows8 rows_of(const PagedView& c, const int32_t* lens, const int32_t* offsets,
                                         uint32_t tokens, uint32_t b) {
  Rows8 r{b, 1u, 0u};
  const int32_t len = lens[b];
  if (offsets != nullptr) {
    const int32_t o0 = offsets[b], o1 = offsets[b + 1];
    if (o0 < 0 || o1 < o0 || static_cast<uint32_t>(o1) > tokens) {
      atomicOr(&g_error_word, QG_ERR_PAGE);
      return Rows8{0u, 0u, 0u};
    }
    r.first = static_cast<uint32_t>(o0);
    r.n = static_cast<uint32_t>(o1 - o0);
  }
  if (len > 0) {
    r.len = static_cast<uint32_t>(len);
    if (r.len > c.capacity || r.n > r.len) {
      atomicOr(&g_error_word, QG_ERR_PAGE);
      r.len = 0u;
    }
  }
  return r;
}

// Host side: checks the cache description and fills the view; false for one that is refused.
inline bool paged8_view(const qg_kv_pages8* c, Paged8View* out) {
  if (c == nullptr || c->k == nullptr || c->v == nullptr || c->k_scale == nullptr || c->v_scale == nullptr ||
      c->table == nullptr) {
    return false;
  }
  if (c->num_pages == 0u || c->num_pages > 0x7fffffffu || c->page_size == 0u || c->n_kv_heads == 0u ||
      c->n_kv_heads > 32767u || c->batch == 0u || c->batch > 65535u || c->table_pages == 0u ||
      c->table_stride < c->table_pages) {
    return false;
  }
  if (c->head_dim == 0u || c->head_dim % 16u != 0u || c->head_dim > kMaxPagedDim) return false;
  if (c->block < 16u || c->block > 128u || (c->block & (c->block - 1u)) != 0u || c->page_size % c->block != 0u) {
    return false;
  }
  if (c->page_stride % 16u != 0u || c->head_stride % 16u != 0u || c->slot_stride % 16u != 0u) return false;
  if (!aligned16(c->k) || !aligned16(c->v) || (reinterpret_cast<uintptr_t>(c->k_scale) & 3u) != 0u ||
      (reinterpret_cast<uintptr_t>(c->v_scale) & 3u) != 0u) {
    return false;
  }
  const uint64_t slots = static_cast<uint64_t>(c->table_pages) * c->page_size;
  if (slots > 0x7fffff00ull) return false;  // a tile past the end still counts in 31 bits
  out->c.k = static_cast<uint8_t*>(c->k);
  out->c.v = static_cast<uint8_t*>(c->v);
  out->c.table = c->table;
  out->c.page_bytes = c->page_stride;
  out->c.head_bytes = c->head_stride;
  out->c.slot_bytes = c->slot_stride;
  out->c.page = fast_div(c->page_size);
  out->c.num_pages = c->num_pages;
  out->c.n_kv = c->n_kv_heads;
  out->c.dim = c->head_dim;
  out->c.batch = c->batch;
  out->c.table_stride = c->table_stride;
  out->c.capacity = static_cast<uint32_t>(slots);
  out->ks = c->k_scale;
  out->vs = c->v_scale;
  out->scale_page = c->scale_page_stride;
  out->scale_head = c->scale_head_stride;
  out->log_block = static_cast<uint32_t>(__builtin_ctz(c->block));
  return true;
}

}  // namespace qg

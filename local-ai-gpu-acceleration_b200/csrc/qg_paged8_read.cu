// qg_paged8_read.cu -- qg_kv_read8: rows of an 8-bit paged cache as the values that they stand
// for (declared in include/qgemv_b200.h).
//
// out = T(code * scale), one multiplication a value: bound by memory, 1 byte read and 2 or 4
// written a value.  A thread takes 16 codes, a 16-byte piece, of a key row and of the value row
// beside it, for kTake pieces a CTA's width apart, so that their loads are in flight together and a
// warp writes whole lines.  Where a row comes from is looked up once a piece; the sequence of a
// CTA's first row is found by all its threads at once, its later rows go on from there.
// Measured (B200): 8 x 9000..30001 rows of 8 x 128 to fp16 155 us, 85% of a plain copy's rate; 700 rows 5.1 us.
#include <algorithm>

#include "qg_paged8.cuh"

namespace qg {
namespace {

constexpr uint32_t kReadThreads = 256;
constexpr uint32_t kTake = 2;  // pieces of a thread

struct Read8Args {
  const int32_t *starts, *offsets;
  void *k, *v;
  uint64_t k_stride, v_stride;
  uint32_t tokens;
  FastDiv row_pieces, head_pieces;  // 16-code pieces of a row (all heads), of a head
};

template <typename T>
__device__ __forceinline__ void put16(T* to, uint4 w, float scale) {
  const uint32_t words[4] = {w.x, w.y, w.z, w.w};
  uint32_t out[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float x[4];
    codes_to_float(words[i], x);
    if constexpr (sizeof(T) == 4) {
      reinterpret_cast<float4*>(to)[i] = make_float4(x[0] * scale, x[1] * scale, x[2] * scale, x[3] * scale);
    } else {
      out[2 * i] = pack2(x[0] * scale, x[1] * scale, T());
      out[2 * i + 1] = pack2(x[2] * scale, x[3] * scale, T());
    }
  }
  if constexpr (sizeof(T) == 2) {
    reinterpret_cast<uint4*>(to)[0] = make_uint4(out[0], out[1], out[2], out[3]);
    reinterpret_cast<uint4*>(to)[1] = make_uint4(out[4], out[5], out[6], out[7]);
  }
}

template <typename T>
__global__ void __launch_bounds__(kReadThreads) read8_kernel(const Paged8View c, const Read8Args a) {
  pdl_wait();
  pdl_trigger();
  const uint64_t piece0 = static_cast<uint64_t>(blockIdx.x) * (kReadThreads * kTake);
  const uint32_t row0 = static_cast<uint32_t>(piece0 / a.row_pieces.d);
  const uint32_t in0 = static_cast<uint32_t>(piece0 - static_cast<uint64_t>(row0) * a.row_pieces.d);
  // sequences that end at or before the CTA's first row
  uint32_t before = 0;
  for (uint32_t b0 = 0; b0 < c.c.batch; b0 += kReadThreads) {
    const uint32_t b = b0 + threadIdx.x;
    const int n = __syncthreads_count(b < c.c.batch && a.offsets[b + 1u] <= static_cast<int64_t>(row0));
    before += static_cast<uint32_t>(n);
    if (n < static_cast<int>(kReadThreads)) break;
  }
  if (blockIdx.x == 0u && threadIdx.x == 0u && a.offsets[c.c.batch] > static_cast<int64_t>(a.tokens)) {
    atomicOr(&g_error_word, QG_ERR_PAGE);
  }
  uint32_t b = before;
  uint4 kw[kTake], vw[kTake];
  float ks[kTake], vs[kTake];
  uint32_t row[kTake], in[kTake];
#pragma unroll
  for (uint32_t i = 0; i < kTake; ++i) {
    const uint32_t p = in0 + threadIdx.x + i * kReadThreads;  // from the CTA's first row on
    const uint32_t down = div_by(p, a.row_pieces);
    row[i] = row0 + down;
    in[i] = p - down * a.row_pieces.d;
    kw[i] = vw[i] = make_uint4(0u, 0u, 0u, 0u);
    ks[i] = vs[i] = 0.f;
    while (b < c.c.batch && a.offsets[b + 1u] <= static_cast<int64_t>(row[i])) ++b;
    const int32_t first = b < c.c.batch ? a.offsets[b] : 0x7fffffff;
    if (row[i] >= a.tokens || first > static_cast<int64_t>(row[i])) {
      row[i] = 0xffffffffu;  // a row of no sequence
      continue;
    }
    const int64_t slot = static_cast<int64_t>(a.starts[b]) + row[i] - first;
    if (first < 0 || slot < 0 || slot >= c.c.capacity) {
      atomicOr(&g_error_word, QG_ERR_PAGE);
      continue;
    }
    const uint32_t s = static_cast<uint32_t>(slot), head = div_by(in[i], a.head_pieces);
    const int32_t* list = c.c.table + static_cast<size_t>(b) * c.c.table_stride;
    const uint64_t at = paged_row(c.c, list, s, head);
    if (at == kNoRow) continue;
    const uint64_t code = at + (in[i] - head * a.head_pieces.d) * 16u;
    kw[i] = *reinterpret_cast<const uint4*>(c.c.k + code);
    vw[i] = *reinterpret_cast<const uint4*>(c.c.v + code);
    const uint32_t page = div_by(s, c.c.page);
    const uint64_t scale = static_cast<uint32_t>(list[page]) * c.scale_page + head * c.scale_head +
                           ((s - page * c.c.page.d) >> c.log_block);
    ks[i] = c.ks[scale];
    vs[i] = c.vs[scale];
  }
#pragma unroll
  for (uint32_t i = 0; i < kTake; ++i) {
    if (row[i] == 0xffffffffu) continue;
    put16(static_cast<T*>(a.k) + row[i] * a.k_stride + in[i] * 16u, kw[i], ks[i]);
    put16(static_cast<T*>(a.v) + row[i] * a.v_stride + in[i] * 16u, vw[i], vs[i]);
  }
}

}  // namespace
}  // namespace qg

extern "C" cudaError_t qg_kv_read8(const qg_kv_pages8* cache, const qg_read8* p, cudaStream_t stream) {
  using namespace qg;
  Paged8View c;
  if (!paged8_view(cache, &c) || p == nullptr || !dtype_ok(p->dtype)) return cudaErrorInvalidValue;
  if (p->tokens == 0u) return cudaSuccess;
  const uint64_t piece = 16u / dtype_bytes(p->dtype);
  if (p->tokens > 0x7fffffffu || p->starts == nullptr || p->offsets == nullptr || p->k_out == nullptr ||
      p->v_out == nullptr || p->k_stride % piece != 0u || p->v_stride % piece != 0u || !aligned16(p->k_out) ||
      !aligned16(p->v_out)) {
    return cudaErrorInvalidValue;
  }
  Read8Args a{};
  a.starts = p->starts;
  a.offsets = p->offsets;
  a.k = p->k_out;
  a.v = p->v_out;
  a.k_stride = p->k_stride;
  a.v_stride = p->v_stride;
  a.tokens = p->tokens;
  a.head_pieces = fast_div(c.c.dim / 16u);
  a.row_pieces = fast_div(c.c.n_kv * (c.c.dim / 16u));
  const uint64_t pieces = static_cast<uint64_t>(p->tokens) * a.row_pieces.d;
  const uint64_t ctas = (pieces + kReadThreads * kTake - 1u) / (kReadThreads * kTake);
  if (ctas > 0x7fffffffull) return cudaErrorInvalidValue;
  const uint32_t grid = static_cast<uint32_t>(ctas);
  if (p->dtype == QG_F32) return launch_k(read8_kernel<float>, grid, kReadThreads, 0, stream, c, a);
  if (p->dtype == QG_F16) return launch_k(read8_kernel<__half>, grid, kReadThreads, 0, stream, c, a);
  return launch_k(read8_kernel<__nv_bfloat16>, grid, kReadThreads, 0, stream, c, a);
}

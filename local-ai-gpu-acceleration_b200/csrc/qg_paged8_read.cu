// qg_paged8_read.cu -- qg_kv_read8: rows of an 8-bit paged cache as the values that they stand
// for (declared in include/qgemv_b200.h).
//
// out = T(code * scale), one multiplication a value: bound by memory, 1 byte read and 2 or 4
// written a value.  A thread takes 16 codes, a 16-byte piece, of a key row and of the value row
// beside it, and writes 32 bytes at a time, a whole sector, where the outputs' rows begin on 32 bytes.  Where
// a row comes from is looked up once a piece; the sequence of a CTA's first row is found by all its
// threads at once, its later rows go on from there.
// Measured (B200; a plain copy's rate is 100%): 8 x 9000..30001 rows of 8 x 128 to fp16 141 us, 94%, and 8 x 20000 to
// fp32 258 us, 97%; in stores of 16 bytes 147 and 367.  With 256 threads and two pieces each 158 us for the former.
#include <algorithm>

#include "qg_paged8.cuh"

namespace qg {
namespace {

constexpr uint32_t kReadThreads = 128;

struct Read8Args {
  const int32_t *starts, *offsets;
  void *k, *v;
  uint64_t k_stride, v_stride;
  uint32_t tokens;
  FastDiv row_pieces, head_pieces;  // 16-code pieces of a row (all heads), of a head
};

// 32 bytes at once
__device__ __forceinline__ void put32(void* to, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

// WIDE: rows begin on 32 bytes
template <typename T, bool WIDE>
__device__ __forceinline__ void put16(T* to, uint4 w, float scale) {
  const uint32_t words[4] = {w.x, w.y, w.z, w.w};
  uint32_t out[8];
  if constexpr (WIDE && sizeof(T) == 4) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float x[4];
        codes_to_float(words[2 * h + i], x);
#pragma unroll
        for (int e = 0; e < 4; ++e) out[4 * i + e] = __float_as_uint(x[e] * scale);
      }
      put32(to + 8 * h, out);
    }
    return;
  }
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
  if constexpr (WIDE) {
    put32(to, out);
  } else if constexpr (sizeof(T) == 2) {
    reinterpret_cast<uint4*>(to)[0] = make_uint4(out[0], out[1], out[2], out[3]);
    reinterpret_cast<uint4*>(to)[1] = make_uint4(out[4], out[5], out[6], out[7]);
  }
}

template <typename T, bool WIDE>
__global__ void __launch_bounds__(kReadThreads) read8_kernel(const Paged8View c, const Read8Args a) {
  pdl_wait();
  pdl_trigger();
  const uint64_t piece0 = static_cast<uint64_t>(blockIdx.x) * kReadThreads;
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
  // offsets that do not ascend or lie outside the call; the look-ups below stay inside whatever they are
  for (uint64_t b = piece0 + threadIdx.x; b < c.c.batch; b += static_cast<uint64_t>(gridDim.x) * kReadThreads) {
    const int32_t o0 = a.offsets[b], o1 = a.offsets[b + 1u];
    if (o0 < 0 || o1 < o0 || static_cast<uint32_t>(o1) > a.tokens) atomicOr(&g_error_word, QG_ERR_PAGE);
  }
  const uint32_t p = in0 + threadIdx.x, down = div_by(p, a.row_pieces);  // from the CTA's first row on
  const uint32_t row = row0 + down, in = p - down * a.row_pieces.d;
  uint32_t b = before;
  while (b < c.c.batch && a.offsets[b + 1u] <= static_cast<int64_t>(row)) ++b;
  const int32_t first = b < c.c.batch ? a.offsets[b] : 0x7fffffff;
  if (row >= a.tokens || first > static_cast<int64_t>(row)) return;  // a row of no sequence
  const int64_t slot = static_cast<int64_t>(a.starts[b]) + row - first;
  uint4 kw = make_uint4(0u, 0u, 0u, 0u), vw = kw;
  float ks = 0.f, vs = 0.f;
  if (first < 0 || slot < 0 || slot >= c.c.capacity) {
    atomicOr(&g_error_word, QG_ERR_PAGE);
  } else {
    const uint32_t s = static_cast<uint32_t>(slot), head = div_by(in, a.head_pieces);
    const int32_t* list = c.c.table + static_cast<size_t>(b) * c.c.table_stride;
    const uint64_t at = paged_row(c.c, list, s, head);
    if (at != kNoRow) {
      const uint64_t code = at + (in - head * a.head_pieces.d) * 16u;
      kw = *reinterpret_cast<const uint4*>(c.c.k + code);
      vw = *reinterpret_cast<const uint4*>(c.c.v + code);
      const uint32_t page = div_by(s, c.c.page);
      const uint64_t scale = static_cast<uint32_t>(list[page]) * c.scale_page + head * c.scale_head +
                             ((s - page * c.c.page.d) >> c.log_block);
      ks = c.ks[scale];
      vs = c.vs[scale];
    }
  }
  put16<T, WIDE>(static_cast<T*>(a.k) + row * a.k_stride + in * 16u, kw, ks);
  put16<T, WIDE>(static_cast<T*>(a.v) + row * a.v_stride + in * 16u, vw, vs);
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
  const uint64_t ctas = (pieces + kReadThreads - 1u) / kReadThreads;
  if (ctas > 0x7fffffffull) return cudaErrorInvalidValue;
  const uint32_t grid = static_cast<uint32_t>(ctas);
  const uint64_t bytes = dtype_bytes(p->dtype);
  const bool wide = ((reinterpret_cast<uintptr_t>(p->k_out) | reinterpret_cast<uintptr_t>(p->v_out) | p->k_stride * bytes |
                      p->v_stride * bytes) & 31u) == 0u;
  auto launch = [&](auto t) {
    using T = decltype(t);
    return wide ? launch_k(read8_kernel<T, true>, grid, kReadThreads, 0, stream, c, a)
                : launch_k(read8_kernel<T, false>, grid, kReadThreads, 0, stream, c, a);
  };
  if (p->dtype == QG_F32) return launch(0.f);
  if (p->dtype == QG_F16) return launch(__half());
  return launch(__nv_bfloat16());
}

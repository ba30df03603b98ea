// qg_paged.cuh -- what the paged key-value cache operators share: the checked view of the
// pools and page table that their kernels take, 16-bit / 32-bit element access in 16-byte
// pieces, and the host-side argument checks.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

#include "qg_common.cuh"
#include "qg_host.h"

namespace qg {

constexpr uint32_t kMaxPagedDim = 256;

// n / d for n < 2^31, d >= 1, by a multiplication (Granlund and Montgomery, Division by Invariant
// Integers using Multiplication, 1994): q = (umulhi(n, mul) + n) >> shift.
struct FastDiv {
  uint32_t d, mul, shift;
};
inline FastDiv fast_div(uint32_t d) {
  FastDiv f{d, 0u, 0u};
  while ((1ull << f.shift) < d) ++f.shift;
  f.mul = static_cast<uint32_t>(((1ull << 32) * ((1ull << f.shift) - d)) / d + 1u);
  return f;
}
__device__ __forceinline__ uint32_t div_by(uint32_t n, const FastDiv& f) {
  return (__umulhi(n, f.mul) + n) >> f.shift;
}

// The cache as the kernels see it.
struct PagedView {
  uint8_t *k, *v;
  const int32_t* table;
  uint64_t page_bytes, head_bytes, slot_bytes;  // strides of the pools
  FastDiv page;                                 // slots per page
  uint32_t num_pages, n_kv, dim, batch, table_stride;
  uint32_t capacity;                            // slots that a table row names (< 2^31)
};

constexpr uint64_t kNoRow = ~0ull;

// Byte offset of (slot, head) of the sequence whose page list is `row`, in either pool;
// kNoRow and QG_ERR_PAGE when the page id is not one of the pool's.  slot < capacity.
__device__ __forceinline__ uint64_t paged_row(const PagedView& c, const int32_t* row, uint32_t slot,
                                              uint32_t head) {
  const uint32_t at = div_by(slot, c.page);
  const uint32_t id = static_cast<uint32_t>(row[at]);
  if (id >= c.num_pages) {
    atomicOr(&g_error_word, QG_ERR_PAGE);
    return kNoRow;
  }
  return id * c.page_bytes + head * c.head_bytes + (slot - at * c.page.d) * c.slot_bytes;
}

// lens[b] as a count: negative is 0, past `most` is `most` and QG_ERR_PAGE.
__device__ __forceinline__ uint32_t paged_len(int32_t len, uint32_t most) {
  if (len <= 0) return 0u;
  if (static_cast<uint32_t>(len) > most) {
    atomicOr(&g_error_word, QG_ERR_PAGE);
    return most;
  }
  return static_cast<uint32_t>(len);
}

// Pairs of 16-bit values as fp32 and back.
__device__ __forceinline__ float2 unpack2(uint32_t w, __half) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ float2 unpack2(uint32_t w, __nv_bfloat16) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w));
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Host side.
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0u; }
inline uint32_t dtype_bytes(int dtype) { return dtype == QG_F32 ? 4u : 2u; }
inline bool dtype_ok(int dtype) { return dtype == QG_F32 || dtype == QG_F16 || dtype == QG_BF16; }

constexpr int kMaxDevices = 64;  // whose attributes are remembered

// Raises a kernel's dynamic shared memory limit, once a device.  (No locks or containers:
// nothing at a C entry point may throw, and setting it twice does no harm.)
struct SmemAttr {
  std::atomic<bool> done[kMaxDevices] = {};
  cudaError_t set(const void* kernel, uint32_t bytes) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const bool known = dev >= 0 && dev < kMaxDevices;
    if (known && done[dev].load(std::memory_order_acquire)) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes));
    if (e == cudaSuccess && known) done[dev].store(true, std::memory_order_release);
    return e;
  }
};

// SMs of the current device, asked for once a device.
inline int paged_sm_count() {
  static std::atomic<int> count[kMaxDevices] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return device_sm_count();
  int n = count[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    n = device_sm_count();
    count[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

// Checks the cache description and fills the kernels' view; false for one that the
// operators refuse.
inline bool paged_view(const qg_kv_pages* c, PagedView* out) {
  if (c == nullptr || c->k == nullptr || c->v == nullptr || c->table == nullptr) return false;
  if (c->dtype != QG_F16 && c->dtype != QG_BF16) return false;
  if (c->num_pages == 0u || c->num_pages > 0x7fffffffu || c->page_size == 0u || c->n_kv_heads == 0u ||
      c->n_kv_heads > 65535u || c->batch == 0u || c->batch > 65535u || c->table_pages == 0u ||
      c->table_stride < c->table_pages) {
    return false;
  }
  if (c->head_dim == 0u || c->head_dim % 8u != 0u || c->head_dim > kMaxPagedDim) return false;
  if (c->page_stride % 8u != 0u || c->head_stride % 8u != 0u || c->slot_stride % 8u != 0u) return false;
  if (!aligned16(c->k) || !aligned16(c->v)) return false;
  const uint64_t slots = static_cast<uint64_t>(c->table_pages) * c->page_size;
  if (slots > 0x7fffffffull) return false;
  out->k = static_cast<uint8_t*>(c->k);
  out->v = static_cast<uint8_t*>(c->v);
  out->table = c->table;
  out->page_bytes = c->page_stride * 2u;
  out->head_bytes = c->head_stride * 2u;
  out->slot_bytes = c->slot_stride * 2u;
  out->page = fast_div(c->page_size);
  out->num_pages = c->num_pages;
  out->n_kv = c->n_kv_heads;
  out->dim = c->head_dim;
  out->batch = c->batch;
  out->table_stride = c->table_stride;
  out->capacity = static_cast<uint32_t>(slots);
  return true;
}

}  // namespace qg

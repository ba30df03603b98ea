// qg_rows.cuh -- rows of heads as the append kernels hold them: pieces of 8 values of any type,
// pairs of fp32 worked on by one instruction, and the pairs that a rotation turns.
#pragma once

#include "qg_paged.cuh"

namespace qg {

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
__device__ __forceinline__ F2 operator+(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
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

}  // namespace qg

// What the attention kernels with few rows a unit share: the matrix instruction,
// and the merge of partial results.
#pragma once

#include "common.cuh"

namespace ffai {

namespace {

template <int F16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  if constexpr (F16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A merge of partial softmax results of one row, 8 head dims a thread.
struct Merged {
  float m, l, o[8];
  __device__ __forceinline__ void add(const float2 ml, const float4 a, const float4 b) {
    if (ml.y == 0.f) return;  // nothing in it (NaN: scores that were none)
    const float M = fmaxf(m, ml.x);
    const float f0 = m == -INFINITY ? 0.f : ex2_approx(m - M), f1 = ex2_approx(ml.x - M);
    m = M;
    l = l * f0 + ml.y * f1;
    const float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = o[e] * f0 + x[e] * f1;
  }
};

// Which halves of a pair are infinite or NaN.
template <int F16>
__device__ __forceinline__ uint32_t odd_halves(uint32_t x) {
  constexpr uint32_t kExp = F16 ? 0x7c00u : 0x7f80u;
  return ((x & kExp) == kExp ? 0xffffu : 0u) | ((x >> 16 & kExp) == kExp ? 0xffff0000u : 0u);
}

}  // namespace

}  // namespace ffai

// Whole weights of logits, as sampling and verification share them:
//   d = fl(fl(x - xmax) * fl(1 / T)), w = floor(2^36 e^d), e^d in f32.
#pragma once

#include <type_traits>

#include "common.cuh"

namespace ffai {

namespace {

// NaN counts as -inf (never chosen), -0 as 0 (they tie).
__device__ __forceinline__ float clean(float x) { return x != x ? -INFINITY : x + 0.0f; }
// x - xmax, with 0 for the maximum itself (also when it is infinite).
__device__ __forceinline__ float delta(float x, float xmax) {
  return x == xmax ? 0.0f : __fadd_rn(x, -xmax);
}
// floor(2^36 e) for e in [0, 1], as two 18-bit halves: adding 2^23 and
// rounding towards zero leaves the whole part in the low mantissa bits.
struct Halves {
  uint32_t hi, lo;
};
__device__ __forceinline__ Halves halves(float e) {
  const float x = __fmul_rn(e, 262144.0f);
  const float t = __fadd_rz(x, 8388608.0f);
  const float r = __fmul_rn(__fadd_rn(x, -__fadd_rn(t, -8388608.0f)), 262144.0f);
  return {__float_as_uint(t) & 0x7fffffu, __float_as_uint(__fadd_rz(r, 8388608.0f)) & 0x7fffffu};
}
__device__ __forceinline__ unsigned long long weight(float d) {
  if (!(d >= -25.0f)) return 0;
  const Halves h = halves(expf(d));
  return (static_cast<unsigned long long>(h.hi) << 18) + h.lo;
}

// The logits of a 16-byte piece.
template <typename T>
__device__ __forceinline__ void unpack(const uint4& w, float (&x)[16 / sizeof(T)]) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int e = 0; e < 16 / static_cast<int>(sizeof(T)); ++e) {
    if constexpr (sizeof(T) == 4)
      x[e] = __uint_as_float(u[e]);
    else
      x[e] = e & 1 ? hi_half(u[e / 2], std::is_same<T, __half>::value)
                   : lo_half(u[e / 2], std::is_same<T, __half>::value);
  }
}

}  // namespace

}  // namespace ffai

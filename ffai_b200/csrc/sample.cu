// Sampling of one token per row of logits from a given uniform number, with
// temperature, top-k, top-p and min-p.
//
// A row's tokens are ordered by (logit descending, index ascending).  With
//   d_i = fl(fl(x_i - xmax) * fl(1 / T))          two f32 roundings
//   w_i = floor(2^36 e^(d_i))                     e^d in f32, then whole
// every sum is a sum of whole numbers, hence the same in any order, and the
// sampled token depends on the inputs alone.  In that order, with C the
// running sum of w:
//   M_k = C after the first k tokens              (all of them without top-k)
//   M_p = least C >= top_p * M_k
//   M_m = sum of w with d >= ln(min_p)            (a prefix too: d falls)
//   M   = min(M_p, M_m);  token = the first with C > floor(u * M).
// Prefix masses alone are compared, so no cut needs its token count.
//
// One CTA per row.  A prefix position is found by descending the bits of an
// order-preserving 32-bit key (11 + 11 + 10): a histogram of the elements
// that share the bits found so far, a scan of its bins from the largest key
// down, and the bin where the running count or mass reaches the goal.
#include "common.cuh"
#include "kernels.h"

namespace ffai {

namespace {

constexpr int kSmThreads = 1024;
constexpr int kSmWarps = kSmThreads / 32;
constexpr int kSmBins = 2048;
constexpr float kSmScale = 68719476736.0f;  // 2^36

// Logits as f32; NaN counts as -inf (never chosen), -0 as 0 (they tie).
template <typename T>
__device__ __forceinline__ float load_logit(const T* row, int i) {
  const float x = to_f32<T>(row[i]);
  return x != x ? -INFINITY : x + 0.0f;
}

// Larger logit, larger key.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

struct RowScale {
  float xmax, inv;
};
// x - xmax, with 0 for the maximum itself (also when it is infinite).
__device__ __forceinline__ float delta(float x, float xmax) {
  return x == xmax ? 0.0f : __fadd_rn(x, -xmax);
}
__device__ __forceinline__ float exponent(float x, const RowScale& r) {
  return x == -INFINITY ? -INFINITY : __fmul_rn(delta(x, r.xmax), r.inv);
}
__device__ __forceinline__ unsigned long long weight(float d) {
  return static_cast<unsigned long long>(__fmul_rn(expf(d), kSmScale));
}

template <typename V, typename Op>
__device__ __forceinline__ V block_reduce(V v, V* s_red, Op op) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (lane == 0) s_red[warp] = v;
  __syncthreads();
  v = s_red[0];
  for (int w = 1; w < kSmWarps; ++w) v = op(v, s_red[w]);
  __syncthreads();
  return v;
}

struct SampleShared {
  uint32_t cnt[kSmBins], lo[kSmBins], hi[kSmBins];
  unsigned long long red64[kSmWarps];
  float redf[kSmWarps];
  double redd[kSmWarps];
  uint32_t warp_cnt[kSmWarps];
  unsigned long long warp_mass[kSmWarps];
  int bin;
  uint32_t bin_cnt;            // elements before the bin found
  unsigned long long bin_mass; // mass before it
  int token;
};

struct Found {
  uint32_t key;               // the element's key
  uint32_t rank;              // 1-based rank among the equal keys, by index
  unsigned long long before;  // mass of the elements with larger keys
};

// The element where the running count (BY_COUNT) or mass first reaches
// `goal` >= 1; the totals reach it (the caller's concern).
template <typename T, bool BY_COUNT>
__device__ Found find_prefix(const T* row, int V, const RowScale& rs, unsigned long long goal,
                             SampleShared& s) {
  uint32_t prefix = 0, cnt0 = 0;
  unsigned long long mass0 = 0;
  constexpr int kShift[3] = {21, 10, 0}, kBits[3] = {11, 11, 10};
  for (int level = 0; level < 3; ++level) {
    const int shift = kShift[level], bits = kBits[level];
    for (int i = threadIdx.x; i < kSmBins; i += kSmThreads) s.cnt[i] = s.lo[i] = s.hi[i] = 0;
    __syncthreads();
    const uint32_t mask = (1u << bits) - 1;
    for (int i = threadIdx.x; i < V; i += kSmThreads) {
      const float x = load_logit(row, i);
      const uint32_t key = key_of(x);
      if (level > 0 && (key >> (shift + bits)) != prefix) continue;
      const uint32_t b = (key >> shift) & mask;
      const unsigned long long w = weight(exponent(x, rs));
      atomicAdd(&s.cnt[b], 1u);
      // a 64-bit sum as two 32-bit halves: each wrap of the low half is
      // seen by exactly one adder, which carries it
      const uint32_t wl = static_cast<uint32_t>(w);
      const uint32_t old = atomicAdd(&s.lo[b], wl);
      const uint32_t up = static_cast<uint32_t>(w >> 32) + (old + wl < old ? 1u : 0u);
      if (up) atomicAdd(&s.hi[b], up);
    }
    __syncthreads();
    // Running sums from the largest key down: thread t takes bins
    // kSmBins - 1 - 2t and the one below.
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int hi_bin = kSmBins - 1 - 2 * threadIdx.x;
    uint32_t c[2];
    unsigned long long m[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      c[e] = s.cnt[hi_bin - e];
      m[e] = (static_cast<unsigned long long>(s.hi[hi_bin - e]) << 32) + s.lo[hi_bin - e];
    }
    uint32_t ci = c[0] + c[1];
    unsigned long long mi = m[0] + m[1];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t cu = __shfl_up_sync(0xffffffffu, ci, o);
      const unsigned long long mu = __shfl_up_sync(0xffffffffu, mi, o);
      if (lane >= o) {
        ci += cu;
        mi += mu;
      }
    }
    if (lane == 31) {
      s.warp_cnt[warp] = ci;
      s.warp_mass[warp] = mi;
    }
    __syncthreads();
    uint32_t cb = cnt0 + ci - c[0] - c[1];
    unsigned long long mb = mass0 + mi - m[0] - m[1];
    for (int w = 0; w < warp; ++w) {
      cb += s.warp_cnt[w];
      mb += s.warp_mass[w];
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const bool before = BY_COUNT ? cb < goal : mb < goal;
      const bool reached = BY_COUNT ? cb + c[e] >= goal : mb + m[e] >= goal;
      if (before && reached) {  // one bin only
        s.bin = hi_bin - e;
        s.bin_cnt = cb;
        s.bin_mass = mb;
      }
      cb += c[e];
      mb += m[e];
    }
    __syncthreads();
    prefix = (prefix << bits) | static_cast<uint32_t>(s.bin);
    cnt0 = s.bin_cnt;
    mass0 = s.bin_mass;
    __syncthreads();
  }
  Found f{prefix, 0, mass0};
  if constexpr (BY_COUNT) {
    f.rank = static_cast<uint32_t>(goal - cnt0);
  } else {
    const unsigned long long w = weight(exponent(logit_of(prefix), rs));
    f.rank = static_cast<uint32_t>((goal - mass0 + w - 1) / w);
  }
  return f;
}

// Index of the `rank`-th (1-based) element with this key, by index.
template <typename T>
__device__ int find_index(const T* row, int V, uint32_t key, uint32_t rank, SampleShared& s) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int per = ((V + kSmWarps - 1) / kSmWarps + 31) / 32 * 32;
  const int i0 = min(V, warp * per), i1 = min(V, i0 + per);
  uint32_t n = 0;
  for (int i = i0 + lane; i < i1; i += 32) n += key_of(load_logit(row, i)) == key;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  if (lane == 0) s.warp_cnt[warp] = n;
  __syncthreads();
  uint32_t before = 0;
  for (int w = 0; w < warp; ++w) before += s.warp_cnt[w];
  if (before < rank && before + n >= rank) {  // one warp
    for (int i = i0; i < i1; i += 32) {
      const bool hit = i + lane < i1 && key_of(load_logit(row, i + lane)) == key;
      const uint32_t m = __ballot_sync(0xffffffffu, hit);
      const uint32_t here = __popc(m);
      if (before + here >= rank) {
        if (hit && before + __popc(m & ((1u << lane) - 1)) + 1 == rank) s.token = i + lane;
        break;
      }
      before += here;
    }
  }
  __syncthreads();
  return s.token;
}

template <typename T>
__global__ void __launch_bounds__(kSmThreads) sample_kernel(SampleParams p) {
  __shared__ SampleShared s;
  const int b = blockIdx.x, V = p.vocab;
  const T* row = static_cast<const T*>(p.logits) + b * p.ld;
  const auto add64 = [](unsigned long long a, unsigned long long c) { return a + c; };
  const auto addd = [](double a, double c) { return a + c; };
  const auto maxf = [](float a, float c) { return fmaxf(a, c); };

  float mx = -INFINITY;
  for (int i = threadIdx.x; i < V; i += kSmThreads) mx = fmaxf(mx, load_logit(row, i));
  RowScale rs{block_reduce(mx, s.redf, maxf), 1.0f};
  if (rs.xmax == -INFINITY) {  // nothing to choose from
    if (threadIdx.x == 0) {
      p.tokens[b] = -1;
      if (p.logprobs) p.logprobs[b] = -INFINITY;
    }
    return;
  }
  const float T0 = p.temperature ? p.temperature[b] : 1.0f;
  rs.inv = __fdiv_rn(1.0f, T0);
  uint32_t key = key_of(rs.xmax), rank = 1;  // greedy: the first maximum
  if (T0 > 0.0f && rs.inv < INFINITY) {
    const int k = p.top_k ? p.top_k[b] : 0;
    const float tp = p.top_p ? p.top_p[b] : 1.0f;
    const float mp = p.min_p ? p.min_p[b] : 0.0f;
    const float dmin = mp > 0.0f ? fminf(static_cast<float>(log(static_cast<double>(mp))), 0.0f)
                                 : -INFINITY;
    unsigned long long all = 0, above = 0;
    for (int i = threadIdx.x; i < V; i += kSmThreads) {
      const float d = exponent(load_logit(row, i), rs);
      const unsigned long long w = weight(d);
      all += w;
      if (d >= dmin) above += w;
    }
    unsigned long long mass = block_reduce(all, s.red64, add64);
    above = block_reduce(above, s.red64, add64);
    if (k > 0 && k < V) {
      const Found f = find_prefix<T, true>(row, V, rs, static_cast<unsigned long long>(k), s);
      mass = f.before + f.rank * weight(exponent(logit_of(f.key), rs));
    }
    if (tp < 1.0f) {
      const double want = ceil(static_cast<double>(fmaxf(tp, 0.0f)) * static_cast<double>(mass));
      const unsigned long long goal =
          max(1ull, min(mass, static_cast<unsigned long long>(want)));
      const Found f = find_prefix<T, false>(row, V, rs, goal, s);
      mass = f.before + f.rank * weight(exponent(logit_of(f.key), rs));
    }
    mass = min(mass, above);
    const double t = floor(static_cast<double>(p.u[b]) * static_cast<double>(mass));
    const unsigned long long target =
        t > 0.0 ? min(mass - 1, static_cast<unsigned long long>(t)) : 0ull;
    const Found f = find_prefix<T, false>(row, V, rs, target + 1, s);
    key = f.key;
    rank = f.rank;
  }
  const int token = find_index(row, V, key, rank, s);
  if (threadIdx.x == 0) p.tokens[b] = token;
  if (p.logprobs) {
    // f64 sum of the f32 exponentials: a peaked row adds tens of thousands of
    // tiny terms to 1, which f32 partial sums would lose
    double z = 0.0;
    for (int i = threadIdx.x; i < V; i += kSmThreads)
      z += static_cast<double>(expf(delta(load_logit(row, i), rs.xmax)));
    z = block_reduce(z, s.redd, addd);
    if (threadIdx.x == 0) {
      const float x = logit_of(key);
      const double dx = x == rs.xmax ? 0.0 : static_cast<double>(x) - rs.xmax;
      p.logprobs[b] = static_cast<float>(dx - log(z));
    }
  }
}

}  // namespace

cudaError_t launch_sample(const SampleParams& p, cudaStream_t s) {
  switch (p.dtype) {
    case 0: sample_kernel<float><<<p.batch, kSmThreads, 0, s>>>(p); break;
    case 1: sample_kernel<__nv_bfloat16><<<p.batch, kSmThreads, 0, s>>>(p); break;
    case 2: sample_kernel<__half><<<p.batch, kSmThreads, 0, s>>>(p); break;
    default: return cudaErrorInvalidValue;
  }
  return cudaGetLastError();
}

}  // namespace ffai

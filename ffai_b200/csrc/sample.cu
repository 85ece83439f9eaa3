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
// Three launches, each over (row, stretch of tokens) with thousands of threads
// per row, the first reading the logits from memory, the others from L2 as far as
// it holds them (300 rows of 128000 f32 it does not: each pass reads memory):
//  1. sample_max_kernel: the row's first maximum, by an atomic maximum of
//     (order-preserving key, ~index);
//  2. sample_bins_kernel: weights, and a histogram of their sums (and counts, for
//     top-k) over bins 1/64 wide in d, which order the tokens coarsely.  The last
//     CTA of a row to finish scans the bins and works out which of them can hold
//     the three prefix positions asked for (top-k, top-p, the token): a position
//     known to lie in one bin bounds the next one's goal to an interval, almost
//     always within a bin or two;
//  3. sample_pick_kernel: lists the tokens of those bins; the last CTA of a row
//     finds each position in its list (finer bins, then one warp ranks the few
//     tokens left).
// A set with more tokens than a list holds (flat or coarsely rounded rows) is
// split by the logits' own bits, by that CTA alone, until a part fits.
// Weights are summed as two 18-bit halves in 32-bit words, which a stretch of
// less than 2^14 tokens cannot overflow, so plain shared-memory reductions
// suffice: a 64-bit shared-memory add is a compare-and-swap loop.
//
// Measured (device, us): 25 at 5 rows of 51865 f32 logits, 44 at 64 rows bf16 with
// every setting, 160 at 300 rows of 128000 f32 (28 + 75 + 60; one read of the
// logits takes 24).  A few rows are bound by the chain of dependent passes, many
// by the instructions of the second pass (about 35 a token).  The alternative,
// a cluster of CTAs per row that keeps the logits in shared memory, took 25, 40
// and 269: it reads them once, but its exchanges and single-CTA phases leave
// only two stretches per SM in flight.  Rows whose cut falls among many equal or
// close logits pay for long lists, or for splitting by one CTA: 64 rows of 51865
// with top-p 36 us ordinary, 45 at bf16 logits about -10, 74 (f32) and 82 (bf16)
// at temperature 4, 150 all equal; 300 of 128000 f32 170, 302 and 776.
#include <stddef.h>

#include <type_traits>

#include "common.cuh"
#include "kernels.h"

namespace ffai {

namespace {

constexpr int kSmThreads = 512;
constexpr int kSmWarps = kSmThreads / 32;
constexpr int kSmPer = 4;        // bins per scanning thread
constexpr int kSmQueue = 1024;   // tokens of a stretch that may be in a set
constexpr int kSmPair = 256;     // tokens of a short list
constexpr int kSmSub = 512;      // finer bins of a list: 2^-15 wide in d
static_assert(kSmSub == kSmThreads && 2 * kSmPair == kSmThreads && kSmBins % kSmPer == 0 && kSmBins / kSmPer <= kSmThreads, "scan");
// The high half of the weight 2^36 is 2^18.
static_assert((static_cast<unsigned long long>(kSmChunk) << 18) < (1ull << 32), "halves");

// NaN counts as -inf (never chosen), -0 as 0 (they tie).
__device__ __forceinline__ float clean(float x) { return x != x ? -INFINITY : x + 0.0f; }
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
// NaN for a NaN or masked logit; NaN and -inf both weigh nothing.
__device__ __forceinline__ float exponent(float x, const RowScale& r) {
  return __fmul_rn(delta(x, r.xmax), r.inv);
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
// The bin of an exponent in [-25, 0]: floor(-64 d), at most 1600.
__device__ __forceinline__ int bin_of(float d) {
  return min(static_cast<int>(__float_as_uint(__fmaf_rz(d, -64.0f, 8388608.0f)) & 0x7fffffu),
             kSmBins - 1);
}
// Its finer bin within a set that starts at `first` of them.
__device__ __forceinline__ int fine_of(float d) {
  return static_cast<int>(__float_as_uint(__fmaf_rz(d, -64.0f * kSmSub, 8388608.0f)) & 0x7fffffu);
}

struct SampleShared {
  union {
    struct {
      uint32_t lo[kSmBins], hi[kSmBins];  // sums of the weights' halves
    };
    unsigned long long mass[kSmBins];     // then: mass before each bin
  };
  uint32_t cnt[kSmBins];  // tokens of weight; then: those before each bin
  union {
    unsigned long long list[kSmList];
    float2 queue[kSmQueue];  // (logit, index) of tokens that may be in a set
  };
  unsigned long long pair[3][kSmPair], pair_w[3][kSmPair];  // short lists and weights
  uint2 sub[kSmSub];      // a list's finer bins
  uint32_t sub_cnt[kSmSub];
  unsigned long long red[kSmWarps];
  unsigned long long red2[kSmWarps];
  unsigned long long few[32];  // a fine bin's tokens
  uint32_t n_few, n_list;
  unsigned long long total;  // mass and tokens of all bins
  uint32_t total_cnt;
  int bin, token, last;
  unsigned long long found;
  uint32_t found_key, found_rank;
};

static_assert(offsetof(SampleShared, cnt) == kSmBins * 8, "add_weight");
__shared__ SampleShared sm_shared;
#define SM_SHARED sm_shared

template <typename V, typename Op>
__device__ __forceinline__ V block_reduce(V v, V* s_red, Op op) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (lane == 0) s_red[warp] = v;
  __syncthreads();
  v = s_red[lane % kSmWarps];
#pragma unroll
  for (int o = kSmWarps / 2; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  return v;
}

// Exclusive prefix sums over the CTA of a 64-bit and a 32-bit number.
struct Sums {
  unsigned long long a;
  uint32_t c;
};
__device__ __forceinline__ Sums warp_inclusive(Sums v) {
  const int lane = threadIdx.x % 32;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long x = __shfl_up_sync(0xffffffffu, v.a, o);
    const uint32_t y = __shfl_up_sync(0xffffffffu, v.c, o);
    if (lane >= o) {
      v.a += x;
      v.c += y;
    }
  }
  return v;
}
__device__ __noinline__ Sums block_exclusive(Sums v, Sums* total) {
  SampleShared& s = SM_SHARED;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const Sums in = warp_inclusive(v);
  if (lane == 31) {
    s.red[warp] = in.a;
    s.red2[warp] = in.c;
  }
  __syncthreads();
  Sums w{0, 0};
  if (lane < kSmWarps) {
    w.a = s.red[lane];
    w.c = static_cast<uint32_t>(s.red2[lane]);
  }
  w = warp_inclusive(w);
  total->a = __shfl_sync(0xffffffffu, w.a, 31);
  total->c = __shfl_sync(0xffffffffu, w.c, 31);
  const unsigned long long ba = __shfl_sync(0xffffffffu, w.a, (warp + 31) & 31);
  const uint32_t bc = __shfl_sync(0xffffffffu, w.c, (warp + 31) & 31);
  __syncthreads();
  return {(warp ? ba : 0) + in.a - v.a, (warp ? bc : 0) + in.c - v.c};
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
// f(x, i) for tokens [0, n) of a stretch in global memory, in no order: 16-byte
// loads where the stretch allows, kUnroll of them in flight a thread.
template <typename T, typename F>
__device__ __forceinline__ void each(const T* src, int n, F f) {
  constexpr int kVec = 16 / sizeof(T), kUnroll = 4;
  const int skew = static_cast<int>(reinterpret_cast<uintptr_t>(src) % 16 / sizeof(T));
  const int head = min(n, (kVec - skew) % kVec), vecs = (n - head) / kVec;
  const int t = threadIdx.x;
  const uint4* mid = reinterpret_cast<const uint4*>(src + head);
#pragma unroll 1
  for (int v0 = t; v0 < vecs; v0 += kUnroll * kSmThreads) {
    uint4 w[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k)
      if (v0 + k * kSmThreads < vecs) w[k] = __ldg(mid + v0 + k * kSmThreads);
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      if (v0 + k * kSmThreads >= vecs) break;
      float x[kVec];
      unpack<T>(w[k], x);
#pragma unroll
      for (int e = 0; e < kVec; ++e) f(x[e], head + (v0 + k * kSmThreads) * kVec + e);
    }
  }
  // the tokens before and behind the pieces: fewer than 2 kVec, one a thread
  const int rest = n - vecs * kVec;
  if (t < rest) {
    const int i = t < head ? t : vecs * kVec + t;
    f(to_f32<T>(src[i]), i);
  }
}
// take(x, i) for the few tokens near(x) holds for: the test sets a bit a token,
// without a branch, and the bits of four pieces are gone through afterwards.
template <typename T, typename N, typename F>
__device__ __forceinline__ void each_near(const T* src, int n, N near, F take) {
  constexpr int kVec = 16 / sizeof(T), kUnroll = 4;  // at most 32 tokens
  const int skew = static_cast<int>(reinterpret_cast<uintptr_t>(src) % 16 / sizeof(T));
  const int head = min(n, (kVec - skew) % kVec), vecs = (n - head) / kVec;
  const int t = threadIdx.x;
  const uint4* mid = reinterpret_cast<const uint4*>(src + head);
#pragma unroll 1
  for (int v0 = t; v0 < vecs; v0 += kUnroll * kSmThreads) {
    uint4 w[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      w[k] = make_uint4(0, 0, 0, 0);
      if (v0 + k * kSmThreads < vecs) w[k] = __ldg(mid + v0 + k * kSmThreads);
    }
    uint32_t bits = 0;
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      float x[kVec];
      unpack<T>(w[k], x);
      uint32_t part = 0;
#pragma unroll
      for (int e = 0; e < kVec; ++e) part |= near(x[e]) ? 1u << (k * kVec + e) : 0u;
      if (v0 + k * kSmThreads < vecs) bits |= part;
    }
    while (bits) {
      const int j = __ffs(bits) - 1;
      bits &= bits - 1;
      const int i = head + (v0 + j / kVec * kSmThreads) * kVec + j % kVec;
      take(to_f32<T>(src[i]), i);  // read again: a register cannot be indexed
    }
  }
  const int rest = n - vecs * kVec;
  if (t < rest) {
    const int i = t < head ? t : vecs * kVec + t;
    const float x = to_f32<T>(src[i]);
    if (near(x)) take(x, i);
  }
}

// The row's bins into mass and tokens before each; the bins are cleared.
__device__ __noinline__ void finish_bins(unsigned long long* bins, uint32_t* bins_cnt, bool counts) {
  SampleShared& s = SM_SHARED;
  unsigned long long m[kSmPer] = {0, 0, 0, 0};
  uint32_t c[kSmPer] = {0, 0, 0, 0};
  const int b0 = threadIdx.x * kSmPer;
  __syncthreads();
  if (b0 < kSmBins) {
    // written by other CTAs' atomics: read and clear at L2
    ulonglong2* g = reinterpret_cast<ulonglong2*>(bins + b0);
    const ulonglong2 x = __ldcg(g), y = __ldcg(g + 1);
    m[0] = x.x, m[1] = x.y, m[2] = y.x, m[3] = y.y;
    __stcg(g, make_ulonglong2(0, 0));
    __stcg(g + 1, make_ulonglong2(0, 0));
    if (counts) {
      const uint4 n = __ldcg(reinterpret_cast<const uint4*>(bins_cnt + b0));
      c[0] = n.x, c[1] = n.y, c[2] = n.z, c[3] = n.w;
      __stcg(reinterpret_cast<uint4*>(bins_cnt + b0), make_uint4(0, 0, 0, 0));
    }
  }
  __syncthreads();
  Sums v{0, 0}, total;
#pragma unroll
  for (int e = 0; e < kSmPer; ++e) {
    v.a += m[e];
    v.c += c[e];
  }
  v = block_exclusive(v, &total);
  if (b0 < kSmBins) {
#pragma unroll
    for (int e = 0; e < kSmPer; ++e) {
      s.mass[b0 + e] = v.a;
      s.cnt[b0 + e] = v.c;
      v.a += m[e];
      v.c += c[e];
    }
  }
  if (threadIdx.x == 0) {
    s.total = total.a;
    s.total_cnt = total.c;
  }
  __syncthreads();
}

// The bin where the running count or mass reaches `goal` (1 .. the total): the
// last one with less before it.  One warp: every lane probes the last bin of
// each 32nd of what is left.
__device__ __forceinline__ int find_bin(bool by_count, unsigned long long goal) {
  SampleShared& s = SM_SHARED;
  const int lane = threadIdx.x % 32;
  int lo = 0;
#pragma unroll 1
  for (int step = 1024; step > 0; step /= 32) {
    const int b = lo + lane * step;  // rising: the lanes below the goal come first
    const bool below = b < kSmBins && (by_count ? s.cnt[b] : s.mass[b]) < goal;
    lo += max(__popc(__ballot_sync(0xffffffffu, below)) - 1, 0) * step;
  }
  return lo;
}
__device__ __forceinline__ unsigned long long mass_before(int b) {
  return b < kSmBins ? SM_SHARED.mass[b] : SM_SHARED.total;
}

__device__ __forceinline__ void clear_bins() {
  SampleShared& s = SM_SHARED;
  for (int i = threadIdx.x; i < kSmBins; i += kSmThreads) {
    s.lo[i] = s.hi[i] = s.cnt[i] = 0;
  }
  __syncthreads();
}

// The goals that follow from the mass kept so far: top-p's, and the token's.
__device__ __forceinline__ unsigned long long goal_p(unsigned long long mass, float top_p) {
  const double want = ceil(static_cast<double>(fmaxf(top_p, 0.0f)) * static_cast<double>(mass));
  return max(1ull, min(mass, static_cast<unsigned long long>(want)));
}
__device__ __forceinline__ unsigned long long goal_t(unsigned long long mass, float u) {
  const double t = floor(static_cast<double>(u) * static_cast<double>(mass));
  return (t > 0.0 ? min(mass - 1, static_cast<unsigned long long>(t)) : 0ull) + 1;
}

// Adds the weight of an exponent to its bin (and 1 to the bin's count), without
// a branch: the bin's address comes straight from the bits of floor(-64 d) +
// 2^23, and tokens that weigh nothing (d below -25, NaN, masked) add nothing
// and, wherever they would fall, touch no bin.  (A weight above zero means d >
// -24.96: a bin below 1598.)
template <bool COUNT>
__device__ __forceinline__ Halves add_weight(float d, uint32_t lo_bins) {
  d = fmaxf(d, -26.0f);
  const Halves h = halves(expf(d));
  const uint32_t at = (__float_as_uint(__fmaf_rz(d, -64.0f, 8388608.0f)) << 2) + lo_bins -
                      (0x4b000000u << 2);
  if constexpr (COUNT)
    asm volatile(
        "{\n\t.reg .pred p, q, r;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "setp.ne.u32 q, %2, 0;\n\t"
        "or.pred r, p, q;\n\t"
        "@p red.shared.add.u32 [%0], %1;\n\t"
        "@q red.shared.add.u32 [%0 + %3], %2;\n\t"
        "@r red.shared.add.u32 [%0 + %4], 1;\n\t}" ::"r"(at),
        "r"(h.lo), "r"(h.hi), "n"(kSmBins * 4), "n"(kSmBins * 8)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "setp.ne.u32 q, %2, 0;\n\t"
        "@p red.shared.add.u32 [%0], %1;\n\t"
        "@q red.shared.add.u32 [%0 + %3], %2;\n\t}" ::"r"(at),
        "r"(h.lo), "r"(h.hi), "n"(kSmBins * 4)
        : "memory");
  return h;
}

// A set of tokens: exponent bins b0 .. b1, or a range of keys.
struct Pick {
  int b0, b1;  // b0 -1: keys klo .. khi
  uint32_t klo, khi;
  float xlo, xhi;  // every token of the set lies between them
  // The bins' logits, widened by more than the roundings of the exponent.
  __device__ __forceinline__ void bin_range(int first, int last, float xmax, float T0) {
    b0 = first;
    b1 = last;
    const float far = (last + 1) / 64.0f * T0;
    const float slack = 4e-6f * (fabsf(xmax) + far) + 1e-30f;
    xlo = xmax - far - slack;
    xhi = xmax - first / 64.0f * T0 + slack;
    if (!(far < 1e30f && slack < 1e30f)) {
      xlo = -INFINITY;
      xhi = INFINITY;
    }
  }
  __device__ __forceinline__ void nothing() {  // no logit lies in its range
    b0 = b1 = 0;
    xlo = INFINITY;
    xhi = -INFINITY;
  }
  __device__ __forceinline__ void key_range(uint32_t lo, uint32_t hi) {
    b0 = -1;
    klo = lo;
    khi = hi;
    xlo = logit_of(lo);
    xhi = logit_of(hi);
  }
  __device__ __forceinline__ bool has(float x, const RowScale& rs, uint32_t& key) const {
    if (!(x >= xlo && x <= xhi)) return false;
    key = key_of(x + 0.0f);
    if (b0 < 0) return key >= klo && key <= khi;
    const float d = exponent(x, rs);
    if (!(d >= -25.0f)) return false;
    const int b = bin_of(d);
    return b >= b0 && b <= b1;
  }
};

struct Found {
  unsigned long long mass;  // prefix mass up to and with the token
  int token;                // its index, or -1: the rank-th token with `key`
  uint32_t key, rank;
};

// The token of the list (n tokens, all of a set) where the running count or
// mass reaches `goal`, counted from the set's start: in s.found (the mass up to
// and with it), s.token, s.found_key.  The list is binned again, finer (2^-15
// 2^coarse in the exponent, from fine bin fine0 on), and the few tokens of the
// fine bin that holds the goal are ranked by one warp; should they be many, the
// list is sorted.
__device__ __noinline__ void find_listed(bool by_count, uint32_t n, unsigned long long goal,
                                         int fine0, int coarse, float xmax, float inv) {
  SampleShared& s = SM_SHARED;
  const RowScale rs{xmax, inv};
  const int lane = threadIdx.x % 32;
  s.sub[threadIdx.x] = make_uint2(0, 0);
  s.sub_cnt[threadIdx.x] = 0;
  if (threadIdx.x == 0) {
    // (The goal lies within the list.  Should a racing write to the logits make
    // that untrue, every index below stays in range.)
    s.n_few = 0;
    s.bin = 0;
    s.token = 0;
    s.found = 0;
    s.found_key = s.found_rank = 0;
  }
  __syncthreads();
  int fine[2] = {-1, -1};
#pragma unroll
  for (int e = 0; e < kSmList / kSmThreads; ++e) {
    const uint32_t i = threadIdx.x + e * kSmThreads;
    if (i >= n) continue;
    const float d = exponent(logit_of(~static_cast<uint32_t>(s.list[i] >> 32)), rs);
    const Halves h = halves(expf(d));
    fine[e] = min(max(fine_of(d) - fine0, 0) >> coarse, kSmSub - 1);
    atomicAdd(&s.sub[fine[e]].x, h.lo);
    if (h.hi) atomicAdd(&s.sub[fine[e]].y, h.hi);
    atomicAdd(&s.sub_cnt[fine[e]], 1u);
  }
  __syncthreads();
  const uint2 h = s.sub[threadIdx.x];
  const Sums v{(static_cast<unsigned long long>(h.y) << 18) + h.x, s.sub_cnt[threadIdx.x]};
  Sums total;
  const Sums at = block_exclusive(v, &total);
  if (by_count ? at.c < goal && goal <= at.c + v.c : at.a < goal && goal <= at.a + v.a) {
    s.bin = threadIdx.x;  // one bin only
    s.found = at.a;
    s.found_rank = at.c;
  }
  __syncthreads();
  const int bin = s.bin;
  const unsigned long long mass0 = s.found;
  const uint32_t cnt0 = s.found_rank, few = s.sub_cnt[bin];
  if (few <= 32) {
#pragma unroll
    for (int e = 0; e < kSmList / kSmThreads; ++e)
      if (fine[e] == bin) s.few[atomicAdd(&s.n_few, 1u) % 32] = s.list[threadIdx.x + e * kSmThreads];
    __syncthreads();
    if (threadIdx.x < 32) {
      const bool real = lane < static_cast<int>(few);
      const unsigned long long mine = real ? s.few[lane] : ~0ull;
      unsigned long long w = 0;
      if (real) w = weight(exponent(logit_of(~static_cast<uint32_t>(mine >> 32)), rs));
      unsigned long long mass = mass0;  // up to and with this token
      uint32_t cnt = cnt0;
#pragma unroll 1
      for (uint32_t j = 0; j < few; ++j) {
        const unsigned long long other = __shfl_sync(0xffffffffu, mine, j);
        const unsigned long long ow = __shfl_sync(0xffffffffu, w, j);
        if (other <= mine) {
          mass += ow;
          ++cnt;
        }
      }
      if (real && (by_count ? cnt == goal : mass - w < goal && goal <= mass)) {
        s.found = mass;
        s.token = static_cast<int>(mine & 0xffffffffu);
        s.found_key = ~static_cast<uint32_t>(mine >> 32);
      }
    }
    __syncthreads();
    return;
  }
  // ---- sort the list (bitonic, ascending: the largest logit, lowest index first)
  uint32_t size = 2;
  while (size < n) size <<= 1;
  for (uint32_t i = n + threadIdx.x; i < size; i += kSmThreads) s.list[i] = ~0ull;
  __syncthreads();
#pragma unroll 1
  for (uint32_t k = 2; k <= size; k <<= 1)
#pragma unroll 1
    for (uint32_t j = k >> 1; j > 0; j >>= 1) {
      for (uint32_t i = threadIdx.x; i < size / 2; i += kSmThreads) {
        const uint32_t lo = ((i & ~(j - 1)) << 1) | (i & (j - 1)), hi = lo | j;
        const unsigned long long a = s.list[lo], b = s.list[hi];
        if ((a > b) == ((lo & k) == 0)) {
          s.list[lo] = b;
          s.list[hi] = a;
        }
      }
      __syncthreads();
    }
  // ---- running mass over it, two tokens a thread
  const uint32_t i = 2 * threadIdx.x;
  unsigned long long w[2];
#pragma unroll
  for (int e = 0; e < 2; ++e)
    w[e] = i + e < n ? weight(exponent(logit_of(~static_cast<uint32_t>(s.list[i + e] >> 32)), rs)) : 0;
  unsigned long long a = block_exclusive({w[0] + w[1], 0}, &total).a;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const bool hit = by_count ? i + e + 1 == goal : a < goal && goal <= a + w[e];
    a += w[e];
    if (hit && i + e < n) {
      s.found = a;
      s.token = static_cast<int>(s.list[i + e] & 0xffffffffu);
      s.found_key = ~static_cast<uint32_t>(s.list[i + e] >> 32);
    }
  }
  __syncthreads();
}

// The same in a list of at most kSmPair tokens (in s.pair, with weights in
// s.pair_w): eight threads a token add up what comes before it.
__device__ __noinline__ void find_paired(bool by_count, int set, uint32_t n, unsigned long long goal) {
  SampleShared& s = SM_SHARED;
  __syncthreads();  // the last result is read
  const uint32_t part = threadIdx.x % 8;
  for (uint32_t base = 0; base < n; base += kSmThreads / 8) {
    const uint32_t i = base + threadIdx.x / 8;
    const unsigned long long mine = i < n ? s.pair[set][i] : 0;
    unsigned long long mass = 0;  // up to and with this token
    uint32_t cnt = 0;
    for (uint32_t j = part; j < n; j += 8)
      if (s.pair[set][j] <= mine) {
        mass += s.pair_w[set][j];
        ++cnt;
      }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
      mass += __shfl_xor_sync(0xffffffffu, mass, o);
      cnt += __shfl_xor_sync(0xffffffffu, cnt, o);
    }
    if (part == 0 && i < n &&
        (by_count ? cnt == goal : mass - s.pair_w[set][i] < goal && goal <= mass)) {  // one token
      s.found = mass;
      s.token = static_cast<int>(mine & 0xffffffffu);
      s.found_key = ~static_cast<uint32_t>(mine >> 32);
    }
  }
  __syncthreads();
}

// The slow way to the token where the running count or mass of the row first
// reaches `goal`, for a set that its list did not hold, by this CTA alone: bins
// first .. last of the exponent hold the goal, and before / before_cnt come
// before them.
template <typename T>
__device__ __noinline__ Found find_by_splitting(const T* row, int vocab, RowScale rs, float T0,
                                                bool by_count, unsigned long long goal, int first,
                                                int last, unsigned long long before,
                                                uint32_t before_cnt) {
  SampleShared& s = SM_SHARED;
  Pick pick;
  pick.bin_range(first, last, rs.xmax, T0);
  {
    uint32_t kmin = 0xffffffffu, kmax = 0;
    each(row, vocab, [&](float x, int) {
      uint32_t key;
      if (!pick.has(x, rs, key)) return;
      kmin = min(kmin, key);
      kmax = max(kmax, key);
    });
    uint32_t* red = reinterpret_cast<uint32_t*>(s.red);
    kmin = block_reduce(kmin, red, [](uint32_t a, uint32_t b) { return min(a, b); });
    kmax = block_reduce(kmax, red, [](uint32_t a, uint32_t b) { return max(a, b); });
    pick.key_range(kmin, kmax);
  }
  for (int level = 0;; ++level) {
    // equal logits: the rank follows from the goal.  (32 key bits, 10 a level:
    // the fourth split leaves one key.)
    if (pick.klo >= pick.khi || level == 5) {
      const unsigned long long w = max(1ull, weight(exponent(logit_of(pick.klo), rs)));
      const uint32_t rank = by_count ? static_cast<uint32_t>(goal - before_cnt)
                                     : static_cast<uint32_t>((goal - before + w - 1) / w);
      return {before + rank * w, -1, pick.klo, rank};
    }
    const uint32_t range = pick.khi - pick.klo;
    const int shift = max(0, 32 - __clz(range) - 10);  // at most 1024 bins
    // The row is histogrammed by stretches whose halves cannot overflow, into
    // 64-bit sums, two bins a thread.
    if (threadIdx.x == 0) {
      s.bin = 0;
      s.found = 0;
      s.found_rank = 0;
    }
    unsigned long long mass[2] = {0, 0};
    uint32_t cnt[2] = {0, 0};
    for (int i0 = 0; i0 < vocab; i0 += kSmChunk) {
      __syncthreads();
      clear_bins();
      each(row + i0, min(vocab - i0, kSmChunk), [&](float x, int) {
        uint32_t key;
        if (!pick.has(x, rs, key)) return;
        const uint32_t b = (pick.khi - key) >> shift;
        const unsigned long long w = weight(exponent(logit_of(key), rs));
        atomicAdd(&s.lo[b], static_cast<uint32_t>(w) & 0x3ffffu);
        atomicAdd(&s.hi[b], static_cast<uint32_t>(w >> 18));
        atomicAdd(&s.cnt[b], 1u);
      });
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        mass[e] += (static_cast<unsigned long long>(s.hi[2 * threadIdx.x + e]) << 18) +
                   s.lo[2 * threadIdx.x + e];
        cnt[e] += s.cnt[2 * threadIdx.x + e];
      }
    }
    Sums total;
    Sums at = block_exclusive({mass[0] + mass[1], cnt[0] + cnt[1]}, &total);
    const unsigned long long want = goal - (by_count ? before_cnt : before);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const Sums end{at.a + mass[e], at.c + cnt[e]};
      if (by_count ? at.c < want && want <= end.c : at.a < want && want <= end.a) {
        s.bin = 2 * threadIdx.x + e;  // one bin only
        s.found = at.a;
        s.found_rank = at.c;
      }
      at = end;
    }
    if (threadIdx.x == 0) s.n_list = 0;
    __syncthreads();
    const uint32_t top = pick.khi - (static_cast<uint32_t>(s.bin) << shift);
    const uint32_t low = shift == 0 ? top : top - min(top - pick.klo, (1u << shift) - 1);
    before += s.found;
    before_cnt += s.found_rank;
    pick.key_range(low, top);
    each(row, vocab, [&](float x, int i) {
      uint32_t key;
      if (!pick.has(x, rs, key)) return;
      const uint32_t n = atomicAdd(&s.n_list, 1u);
      if (n < kSmList)
        s.list[n] = (static_cast<unsigned long long>(~key) << 32) | static_cast<uint32_t>(i);
    });
    __syncthreads();
    const uint32_t n = s.n_list;
    if (n <= kSmList) {
      find_listed(by_count, n, goal - (by_count ? before_cnt : before),
                  fine_of(exponent(logit_of(top), rs)), 0, rs.xmax, rs.inv);
      return {before + s.found, s.token, s.found_key, 0};
    }
    __syncthreads();
  }
}

// Index of the `rank`-th (1-based) token of the row with this key.
template <typename T>
__device__ __noinline__ int find_ranked(const T* row, int vocab, uint32_t key, uint32_t rank) {
  SampleShared& s = SM_SHARED;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int per = ((vocab + kSmWarps - 1) / kSmWarps + 31) / 32 * 32;
  const int i0 = min(vocab, warp * per), i1 = min(vocab, i0 + per);
  uint32_t n = 0;
  for (int i = i0 + lane; i < i1; i += 32) n += key_of(clean(to_f32<T>(row[i]))) == key;
  n = __reduce_add_sync(0xffffffffu, n);
  __syncthreads();
  if (lane == 0) s.red[warp] = n;
  __syncthreads();
  uint32_t before = 0;
  for (int w = 0; w < warp; ++w) before += static_cast<uint32_t>(s.red[w]);
  if (threadIdx.x == 0) s.token = 0;
  __syncthreads();
  if (before < rank && before + n >= rank) {  // one warp
    for (int i = i0; i < i1; i += 32) {
      const bool hit = i + lane < i1 && key_of(clean(to_f32<T>(row[i + lane]))) == key;
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

// ---------------------------------------------------------------- the launches

// The row's settings.
struct Setting {
  float T0, inv, top_p, min_p, u;
  int top_k;
  bool greedy;
};
__device__ __forceinline__ Setting setting(const SampleParams& p, int b) {
  Setting c;
  c.T0 = p.temperature ? __ldg(p.temperature + b) : 1.0f;
  c.top_k = p.top_k ? __ldg(p.top_k + b) : 0;
  c.top_p = p.top_p ? __ldg(p.top_p + b) : 1.0f;
  c.min_p = p.min_p ? __ldg(p.min_p + b) : 0.0f;
  c.u = __ldg(p.u + b);
  c.inv = __fdiv_rn(1.0f, c.T0);
  c.greedy = !(c.T0 > 0.0f && c.inv < INFINITY);
  return c;
}
// The stretch of a CTA.
template <typename T>
struct Stretch {
  const T* row;
  int b, i0, n, parts, part;
  SampleRow* ws;
  __device__ __forceinline__ Stretch(const SampleParams& p, int chunk) {
    parts = (p.vocab + chunk - 1) / chunk;
    b = blockIdx.x / parts;
    part = blockIdx.x - b * parts;
    i0 = part * chunk;
    n = min(p.vocab - i0, chunk);
    row = static_cast<const T*>(p.logits) + b * p.ld;
    ws = p.rows + b;
  }
};
__device__ __forceinline__ float best_logit(unsigned long long best) {
  return logit_of(static_cast<uint32_t>(best >> 32));
}
// True for the last CTA of the row to come here; everything the others wrote
// before is then visible.  The ticket is left at zero.
__device__ __forceinline__ bool last_of_row(uint32_t* ticket, int parts) {
  SampleShared& s = SM_SHARED;
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    const bool last = atomicAdd(ticket, 1u) == static_cast<uint32_t>(parts) - 1;
    if (last) *ticket = 0;
    __threadfence();
    s.last = last;
  }
  __syncthreads();
  return s.last != 0;
}

template <typename T>
__global__ void __launch_bounds__(kSmThreads) sample_max_kernel(SampleParams p) {
  griddep_launch_dependents();
  griddep_wait();  // the logits, and the previous call's use of the workspace
  const Stretch<T> st(p, p.long_chunk);
  // The largest logit and where a thread met it first: of the 16-byte pieces
  // only the piece is noted (a comparison a piece, not a token), the token in
  // it looked up at the end.  fmaxf passes over NaN; -0 ties with 0.
  constexpr int kVec = 16 / sizeof(T), kUnroll = 4;
  const T* src = st.row + st.i0;
  const int skew = static_cast<int>(reinterpret_cast<uintptr_t>(src) % 16 / sizeof(T));
  const int head = min(st.n, (kVec - skew) % kVec), vecs = (st.n - head) / kVec;
  const uint4* mid = reinterpret_cast<const uint4*>(src + head);
  const int t = threadIdx.x, tail = head + vecs * kVec + t;
  float mx = -INFINITY;
  int piece = -1;
  for (int v0 = t; v0 < vecs; v0 += kUnroll * kSmThreads) {
    uint4 w[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k)
      if (v0 + k * kSmThreads < vecs) w[k] = __ldg(mid + v0 + k * kSmThreads);
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      if (v0 + k * kSmThreads >= vecs) break;
      float x[kVec];
      unpack<T>(w[k], x);
      float m = x[0];
#pragma unroll
      for (int e = 1; e < kVec; ++e) m = fmaxf(m, x[e]);
      if (m > mx) {
        mx = m;
        piece = v0 + k * kSmThreads;
      }
    }
  }
  float ends = -INFINITY;  // the tokens before and behind the pieces
  if (t < head) ends = fmaxf(ends, to_f32<T>(src[t]));
  if (tail < st.n) ends = fmaxf(ends, to_f32<T>(src[tail]));
  const float top = block_reduce(fmaxf(mx, ends), reinterpret_cast<float*>(SM_SHARED.red),
                                 [](float a, float b) { return fmaxf(a, b); });
  int at = INT32_MAX;
  if (t < head && to_f32<T>(src[t]) == top) at = t;
  if (at == INT32_MAX && piece >= 0 && mx == top) {
    float x[kVec];
    unpack<T>(__ldg(mid + piece), x);
#pragma unroll
    for (int e = kVec - 1; e >= 0; --e)
      if (x[e] == top) at = head + piece * kVec + e;
  }
  if (at == INT32_MAX && tail < st.n && to_f32<T>(src[tail]) == top) at = tail;
  at = block_reduce(at, reinterpret_cast<int*>(SM_SHARED.red), [](int a, int b) { return min(a, b); });
  if (at == INT32_MAX) at = 0;  // nothing above -inf here
  const unsigned long long best =
      (static_cast<unsigned long long>(key_of(top + 0.0f)) << 32) | ~static_cast<uint32_t>(st.i0 + at);
  if (threadIdx.x == 0) atomicMax(&st.ws->best, best);
}

template <typename T>
__global__ void __launch_bounds__(kSmThreads, 3) sample_bins_kernel(SampleParams p) {
  SampleShared& s = SM_SHARED;
  griddep_launch_dependents();
  const Stretch<T> st(p, p.chunk);
  clear_bins();
  griddep_wait();
  const Setting c = setting(p, st.b);
  const RowScale rs{best_logit(__ldcg(&st.ws->best)), c.inv};
  const bool empty = rs.xmax == -INFINITY;
  if (empty || (c.greedy && !p.logprobs)) return;  // every CTA of the row alike
  const bool sampled = !c.greedy, counts = sampled && c.top_k > 0 && c.top_k < p.vocab;
  const float dmin = c.min_p > 0.0f
                         ? fminf(static_cast<float>(log(static_cast<double>(c.min_p))), 0.0f)
                         : -INFINITY;
  const bool floor_p = sampled && c.min_p > 0.0f;
  unsigned long long above = 0;  // weight above the min-p cut
  const uint32_t lo_bins = smem_u32(s.lo);
  if (sampled && !counts && !floor_p && rs.xmax < INFINITY) {
    // the plain case, with nothing decided per token but the weight itself
    each(st.row + st.i0, st.n, [&](float x, int) {
      add_weight<false>(__fmul_rn(__fadd_rn(x, -rs.xmax), rs.inv), lo_bins);
    });
  } else if (sampled) {
    const float from = floor_p ? dmin : INFINITY;
    each(st.row + st.i0, st.n, [&](float x, int) {
      const float d = exponent(x, rs);
      const Halves h = add_weight<true>(d, lo_bins);
      if (d >= from) above += (static_cast<unsigned long long>(h.hi) << 18) + h.lo;
    });
  }
  if (p.logprobs) {
    // sum of e^(x - max): f64 over f32 sums of a piece, because a peaked row
    // adds tens of thousands of tiny terms to 1 (a logit 200 below weighs 0, as
    // do NaN; an infinite maximum is 0 from itself)
    double z = 0.0;
    float part = 0.0f;
    int n = 0;
    each(st.row + st.i0, st.n, [&](float x, int) {
      part += expf(fmaxf(delta(x, rs.xmax), -200.0f));
      if (++n % 4 == 0) {
        z += static_cast<double>(part);
        part = 0.0f;
      }
    });
    z = block_reduce(z + static_cast<double>(part), reinterpret_cast<double*>(s.red),
                     [](double a, double b) { return a + b; });
    if (threadIdx.x == 0) st.ws->z[st.part] = z;
  }
  if (floor_p) {
    above = block_reduce(above, s.red, [](unsigned long long a, unsigned long long b) { return a + b; });
    if (threadIdx.x == 0) atomicAdd(&st.ws->above, above);
  }
  if (sampled) {  // the row's bins: whole numbers, in any order
    __syncthreads();
    for (int b = threadIdx.x; b < kSmBins; b += kSmThreads) {
      unsigned long long m = (static_cast<unsigned long long>(s.hi[b]) << 18) + s.lo[b];
      if (m) atomicAdd(&st.ws->bins[b], m);
      if (counts && s.cnt[b]) atomicAdd(&st.ws->cnt[b], s.cnt[b]);
    }
  }
  if (!last_of_row(&st.ws->ticket, st.parts)) return;

  // ---- the whole row is in: where each position can lie
  if (p.logprobs && threadIdx.x >= kSmThreads - 32) {  // in one order, whatever CTA does it
    double sum = 0.0;
    for (int r = threadIdx.x % 32; r < st.parts; r += 32) sum += __ldcg(&st.ws->z[r]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (threadIdx.x % 32 == 0) st.ws->log_z = log(sum);
  }
  if (!sampled) return;
  if (floor_p) above = __ldcg(&st.ws->above);
  finish_bins(st.ws->bins, st.ws->cnt, counts);
  if (threadIdx.x >= 32) return;
  // One warp, all lanes alike (they search together); lane k writes set k.
  const int lane = threadIdx.x;
  const bool cut_k = counts && static_cast<uint32_t>(c.top_k) < s.total_cnt, cut_p = c.top_p < 1.0f;
  int b0 = -1, b1 = -1;  // this lane's set; -1: not asked for
  unsigned long long lo = s.total, hi = lo;  // the mass kept so far lies between
  if (cut_k) {
    const int b = find_bin(true, c.top_k);
    if (lane == 0) b0 = b1 = b;
    lo = max(1ull, mass_before(b));
    hi = mass_before(b + 1);
  }
  if (cut_p) {
    const int first = find_bin(false, goal_p(lo, c.top_p));
    const int last = hi == lo ? first : find_bin(false, goal_p(hi, c.top_p));
    if (lane == 1) b0 = first, b1 = last;
    lo = max(1ull, mass_before(first));
    hi = mass_before(last + 1);
  }
  if (floor_p) {
    lo = min(lo, above);
    hi = min(hi, above);
  }
  {
    const int first = find_bin(false, goal_t(lo, c.u));
    const int last = hi == lo ? first : find_bin(false, goal_t(hi, c.u));
    if (lane == 2) b0 = first, b1 = last;
  }
  if (lane < 3) {
    Pick pick;
    pick.nothing();
    if (b0 >= 0) pick.bin_range(b0, b1, rs.xmax, c.T0);
    SampleSet& q = st.ws->set[lane];
    q.b0 = b0;
    q.b1 = b1;
    q.xlo = pick.xlo;
    q.xhi = pick.xhi;
    q.before = b0 >= 0 ? mass_before(b0) : 0;
    q.before_cnt = b0 >= 0 && counts ? s.cnt[b0] : 0;
  }
  if (lane == 0) {
    st.ws->total = s.total;
    st.ws->floor = floor_p ? above : ~0ull;
    st.ws->above = 0;
  }
}

template <typename T>
__global__ void __launch_bounds__(kSmThreads, 2) sample_pick_kernel(SampleParams p) {
  SampleShared& s = SM_SHARED;
  griddep_launch_dependents();
  const Stretch<T> st(p, p.long_chunk);
  griddep_wait();
  const Setting c = setting(p, st.b);
  const unsigned long long best = __ldcg(&st.ws->best);
  const RowScale rs{best_logit(best), c.inv};
  const bool empty = rs.xmax == -INFINITY;
  uint32_t key = static_cast<uint32_t>(best >> 32);
  int token = empty ? -1 : static_cast<int>(~static_cast<uint32_t>(best));
  const bool sampled = !empty && !c.greedy;
  const SampleSet* set = st.ws->set;
  if (sampled) {  // ---- this stretch's tokens of the sets
    Pick pick[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const int b0 = __ldcg(&set[k].b0), b1 = __ldcg(&set[k].b1);
      pick[k].b0 = b0;
      pick[k].b1 = b1;
      pick[k].xlo = __ldcg(&set[k].xlo);
      pick[k].xhi = __ldcg(&set[k].xhi);
    }
    const auto take = [&](float x, int i) {
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        uint32_t kx;
        if (!pick[k].has(x, rs, kx)) continue;
        const uint32_t at = atomicAdd(&st.ws->n[k], 1u);
        if (at < kSmList)
          st.ws->list[k][at] =
              (static_cast<unsigned long long>(~kx) << 32) | static_cast<uint32_t>(st.i0 + i);
      }
    };
    // In the pass only the ranges of x are tested; what passes is queued (one
    // token in a hundred, but one warp instruction in four would branch).
    if (threadIdx.x == 0) s.n_list = 0;
    __syncthreads();
    const auto queue = [&](float x, int i) {
      const uint32_t at = atomicAdd(&s.n_list, 1u);
      if (at < kSmQueue)
        s.queue[at] = make_float2(x, __int_as_float(i));
      else
        take(x, i);
    };
    const float a0 = pick[0].xlo, a1 = pick[0].xhi, b0 = pick[1].xlo, b1 = pick[1].xhi,
                c0 = pick[2].xlo, c1 = pick[2].xhi;
    if (a0 > a1)  // without top-k, two ranges to test
      each_near(st.row + st.i0, st.n,
                [&](float x) { return (x >= b0 && x <= b1) || (x >= c0 && x <= c1); }, queue);
    else
      each_near(st.row + st.i0, st.n,
                [&](float x) {
                  return (x >= a0 && x <= a1) || (x >= b0 && x <= b1) || (x >= c0 && x <= c1);
                },
                queue);
    __syncthreads();
    for (uint32_t q = threadIdx.x; q < min(s.n_list, static_cast<uint32_t>(kSmQueue)); q += kSmThreads)
      take(s.queue[q].x, __float_as_int(s.queue[q].y));
  }
  if (!last_of_row(&st.ws->ticket, st.parts)) return;
  if (sampled) {  // ---- each position in its list
    // Short lists are loaded together, with their tokens' weights.
    uint32_t len[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) len[k] = __ldcg(&st.ws->n[k]);
    {
      const int k = threadIdx.x / kSmPair, i = threadIdx.x % kSmPair;
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // sets 0 and 1, then 2
        const int set_of = k + 2 * h;
        if (set_of >= 3 || len[set_of] > kSmPair) continue;
        if (i < static_cast<int>(len[set_of])) {
          const unsigned long long e = __ldcg(&st.ws->list[set_of][i]);
          s.pair[set_of][i] = e;
          s.pair_w[set_of][i] = weight(exponent(logit_of(~static_cast<uint32_t>(e >> 32)), rs));
        }
      }
    }
    if (threadIdx.x == 0) {
      s.token = 0;
      s.found = 0;
      s.found_key = key;
    }
    __syncthreads();
    const auto find = [&](int k, bool by_count, unsigned long long goal) -> Found {
      const int b0 = __ldcg(&set[k].b0), b1 = __ldcg(&set[k].b1);
      const unsigned long long before = __ldcg(&set[k].before);
      const uint32_t before_cnt = __ldcg(&set[k].before_cnt);
      const uint32_t n = len[k];
      const unsigned long long want = goal - (by_count ? before_cnt : before);
      if (n <= kSmPair) {
        find_paired(by_count, k, n, want);
        return {before + s.found, s.token, s.found_key, 0};
      }
      if (n > kSmList)
        return find_by_splitting(st.row, p.vocab, rs, c.T0, by_count, goal, b0, b1, before,
                                 before_cnt);
      __syncthreads();
      for (uint32_t i = threadIdx.x; i < n; i += kSmThreads) s.list[i] = __ldcg(&st.ws->list[k][i]);
      find_listed(by_count, n, want, b0 * kSmSub, b1 > b0 ? 32 - __clz(b1 - b0) : 0, rs.xmax, rs.inv);
      return {before + s.found, s.token, s.found_key, 0};
    };
    unsigned long long mass = __ldcg(&st.ws->total);
    if (__ldcg(&set[0].b0) >= 0) mass = find(0, true, c.top_k).mass;
    if (__ldcg(&set[1].b0) >= 0) mass = find(1, false, goal_p(mass, c.top_p)).mass;
    mass = min(mass, __ldcg(&st.ws->floor));
    const Found f = find(2, false, goal_t(mass, c.u));
    key = f.key;
    token = f.token >= 0 ? f.token : find_ranked(st.row, p.vocab, f.key, f.rank);
    __syncthreads();
    if (threadIdx.x < 3) st.ws->n[threadIdx.x] = 0;
  }
  if (threadIdx.x == 0) {
    st.ws->best = 0;  // for the next call; every CTA of the row has read it
    p.tokens[st.b] = token;
    if (p.logprobs) {
      const float v = logit_of(key);
      const double dx = v == rs.xmax ? 0.0 : static_cast<double>(v) - rs.xmax;
      p.logprobs[st.b] = empty ? -INFINITY : static_cast<float>(dx - __ldcg(&st.ws->log_z));
    }
  }
}

template <typename K>
cudaError_t launch_k(K kernel, const SampleParams& p, int grid, cudaStream_t s) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(kSmThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <typename T>
cudaError_t launch_t(const SampleParams& p, cudaStream_t s) {
  const int grid = p.batch * ((p.vocab + p.chunk - 1) / p.chunk);
  const int long_grid = p.batch * ((p.vocab + p.long_chunk - 1) / p.long_chunk);
  cudaError_t e = launch_k(sample_max_kernel<T>, p, long_grid, s);
  if (e == cudaSuccess) e = launch_k(sample_bins_kernel<T>, p, grid, s);
  if (e == cudaSuccess) e = launch_k(sample_pick_kernel<T>, p, long_grid, s);
  return e;
}

}  // namespace

// Tokens per CTA: one wave of two CTAs per SM where the batch allows, within
// kSmMinChunk and `most` (a CTA's fixed work, some hundreds of instructions a
// warp, is worth about 2000 tokens of a plain pass).
int sample_chunk(int batch, int vocab, int sms, int most) {
  const int parts = 2 * sms / batch > 1 ? 2 * sms / batch : 1;
  const int want = ((vocab + parts - 1) / parts + 7) / 8 * 8;
  return want < kSmMinChunk ? kSmMinChunk : want > most ? most : want;
}

cudaError_t launch_sample(const SampleParams& p, cudaStream_t s) {
  switch (p.dtype) {
    case 0: return launch_t<float>(p, s);
    case 1: return launch_t<__nv_bfloat16>(p, s);
    case 2: return launch_t<__half>(p, s);
  }
  return cudaErrorInvalidValue;
}

}  // namespace ffai

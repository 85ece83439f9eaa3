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
// A row is spread over a cluster of C CTAs (1 to 16), each keeping its stretch
// of the logits in shared memory, so they are read from global memory once:
//  1. load, the row's maximum (exchanged through distributed shared memory);
//  2. weights, and a histogram of their sums (and counts, for top-k) over bins
//     1/64 wide in d, which order the tokens coarsely: the CTAs add up a slice
//     of the bins each, and all of them read all slices and scan them;
//  3. each prefix position asked for (top-k, top-p, the token) lies in one bin,
//     whose tokens every CTA lists and sorts by (logit, index).
// A bin with more tokens than the list holds (flat or coarsely rounded rows)
// is split by the logits' own bits until one is small or holds equal logits.
// Weights are summed as two 18-bit halves in 32-bit words, which a stretch of
// at most 2^14 tokens does not overflow (but for one case, noted below), so plain
// shared-memory reductions suffice: a 64-bit shared-memory add is a
// compare-and-swap loop.
#include <atomic>

#include "common.cuh"
#include "kernels.h"

namespace ffai {

namespace {

constexpr int kSmThreads = 512;
constexpr int kSmWarps = kSmThreads / 32;
constexpr int kSmBins = 1600;    // d in (-25, 0]; e^-25 2^36 < 1: nothing beyond
constexpr int kSmPer = 4;        // bins per scanning thread
constexpr int kSmLocal = 512;    // listed tokens per CTA
constexpr int kSmList = 1024;    // per row
constexpr int kSmMaxCluster = 16;
constexpr int kSmChunk = 16384;  // tokens per CTA
static_assert(kSmChunk * kSmMaxCluster >= kSmMaxVocab, "stretches");
static_assert(kSmBins % kSmPer == 0 && kSmBins / kSmPer <= kSmThreads, "scan");
// A stretch's low halves sum to at most 2^14 (2^18 - 1), its high ones to 2^14
// 2^18: 2^32 exactly, when a whole stretch of 2^14 tokens is at the maximum.
// The add that then wraps to 0 is noted in SampleShared::wrapped.
static_assert((static_cast<unsigned long long>(kSmChunk) << 18) <= (1ull << 32), "halves");

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

// What the CTAs of a cluster tell one another, one entry per CTA.
struct Slot {
  float xmax;
  int first;                  // lowest index of the maximum
  double z;                   // sum of e^(x - max)
  unsigned long long above;   // weight above the min-p cut
  uint32_t count[2];          // listed tokens, by search parity
  uint32_t kmin, kmax;        // keys of a bin to be split
  uint32_t ties;              // tokens with one key
};

struct SampleShared {
  uint32_t lo[kSmBins], hi[kSmBins];  // then: mass before each bin (64 bits)
  uint32_t cnt[kSmBins];              // then: tokens before each bin
  uint32_t wrapped;                   // hi[0] passed 2^32
  unsigned long long local[2][kSmLocal];
  unsigned long long list[kSmList];
  unsigned long long red[kSmWarps];
  unsigned long long red2[kSmWarps];
  Slot mine;                  // read by the other CTAs
  unsigned long long total;   // mass and tokens of all bins
  uint32_t total_cnt;
  int bin;
  unsigned long long before;
  uint32_t before_cnt, bin_cnt;
  uint32_t n;                 // local list's length
  int token;
  unsigned long long found;
  uint32_t found_key, found_rank;
};
constexpr size_t kSmSlice = (kSmBins + 1) / 2 * 12;  // a CTA's slice of the bins (C >= 2)

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
__device__ __forceinline__ void block_exclusive(unsigned long long& a, uint32_t& c,
                                                unsigned long long& ta, uint32_t& tc,
                                                SampleShared& s) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  unsigned long long ai = a;
  uint32_t ci = c;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long x = __shfl_up_sync(0xffffffffu, ai, o);
    const uint32_t y = __shfl_up_sync(0xffffffffu, ci, o);
    if (lane >= o) {
      ai += x;
      ci += y;
    }
  }
  if (lane == 31) {
    s.red[warp] = ai;
    s.red2[warp] = ci;
  }
  __syncthreads();
  unsigned long long ba = 0;
  uint32_t bc = 0;
  ta = 0;
  tc = 0;
#pragma unroll
  for (int w = 0; w < kSmWarps; ++w) {
    if (w == warp) {
      ba = ta;
      bc = tc;
    }
    ta += s.red[w];
    tc += static_cast<uint32_t>(s.red2[w]);
  }
  __syncthreads();
  a = ba + ai - a;
  c = bc + ci - c;
}

__device__ __forceinline__ void cluster_sync_all() {
  __syncwarp();
  cluster_arrive();
  cluster_wait();
}
template <typename V>
__device__ __forceinline__ V ld_cluster(const V* local, int rank) {
  V v;
  const uint32_t a = mapa_shared(smem_u32(local), rank);
  if constexpr (sizeof(V) == 8) {
    unsigned long long x;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(x) : "r"(a) : "memory");
    v = *reinterpret_cast<V*>(&x);
  } else {
    uint32_t x;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(x) : "r"(a) : "memory");
    v = *reinterpret_cast<V*>(&x);
  }
  return v;
}

template <typename T>
struct Row {
  const T* x;   // this CTA's stretch, in shared memory
  int n, i0;    // its tokens, and the index of the first
  int C, rank;  // CTAs of the row, and this one
  RowScale rs;
};

// The local histograms of all CTAs into mass and tokens before each bin.
__device__ __forceinline__ void finish_bins(SampleShared& s, uint8_t* slice, int C, int rank) {
  unsigned long long m[kSmPer];
  uint32_t c[kSmPer];
  const int b0 = threadIdx.x * kSmPer;
  if (C == 1) {
    __syncthreads();
    if (b0 < kSmBins) {
#pragma unroll
      for (int e = 0; e < kSmPer; ++e) {
        m[e] = (static_cast<unsigned long long>(s.hi[b0 + e]) << 18) + s.lo[b0 + e];
        c[e] = s.cnt[b0 + e];
      }
      if (b0 == 0) m[0] += static_cast<unsigned long long>(s.wrapped) << 50;
    }
    __syncthreads();
  } else {
    const int per = (kSmBins + C - 1) / C;
    unsigned long long* sm = reinterpret_cast<unsigned long long*>(slice);
    uint32_t* sc = reinterpret_cast<uint32_t*>(slice + (kSmBins + 1) / 2 * 8);
    cluster_sync_all();
    for (int i = threadIdx.x; i < per; i += kSmThreads) {
      const int b = rank * per + i;
      unsigned long long mass = 0;
      uint32_t cnt = 0;
      if (b < kSmBins) {
#pragma unroll 4
        for (int r = 0; r < C; ++r) {
          mass += (static_cast<unsigned long long>(ld_cluster(&s.hi[b], r)) << 18) +
                  ld_cluster(&s.lo[b], r);
          cnt += ld_cluster(&s.cnt[b], r);
          if (b == 0) mass += static_cast<unsigned long long>(ld_cluster(&s.wrapped, r)) << 50;
        }
      }
      sm[i] = mass;
      sc[i] = cnt;
    }
    cluster_sync_all();
    if (b0 < kSmBins) {
#pragma unroll
      for (int e = 0; e < kSmPer; ++e) {
        const int r = (b0 + e) / per, i = b0 + e - r * per;
        m[e] = ld_cluster(sm + i, r);
        c[e] = ld_cluster(sc + i, r);
      }
    }
  }
  unsigned long long a = 0, ta;
  uint32_t k = 0, tk;
  if (b0 < kSmBins) {
#pragma unroll
    for (int e = 0; e < kSmPer; ++e) {
      a += m[e];
      k += c[e];
    }
  }
  block_exclusive(a, k, ta, tk, s);
  if (b0 < kSmBins) {
    // bin b's mass at word b of the joined lo / hi arrays
    unsigned long long* mass = reinterpret_cast<unsigned long long*>(s.lo);
#pragma unroll
    for (int e = 0; e < kSmPer; ++e) {
      mass[b0 + e] = a;
      s.cnt[b0 + e] = k;
      a += m[e];
      k += c[e];
    }
  }
  if (threadIdx.x == 0) {
    s.total = ta;
    s.total_cnt = tk;
  }
  __syncthreads();
}

// The bin where the running count or mass reaches `goal` (1 .. the total).
template <bool BY_COUNT>
__device__ __forceinline__ void find_bin(unsigned long long goal, SampleShared& s) {
  const unsigned long long* mass = reinterpret_cast<const unsigned long long*>(s.lo);
  for (int b = threadIdx.x; b < kSmBins; b += kSmThreads) {
    const bool end = b + 1 == kSmBins;
    const unsigned long long m1 = end ? s.total : mass[b + 1];
    const uint32_t c1 = end ? s.total_cnt : s.cnt[b + 1];
    const unsigned long long v0 = BY_COUNT ? s.cnt[b] : mass[b], v1 = BY_COUNT ? c1 : m1;
    if (v0 < goal && goal <= v1) {  // one bin only
      s.bin = b;
      s.before = mass[b];
      s.before_cnt = s.cnt[b];
      s.bin_cnt = c1 - s.cnt[b];
    }
  }
  __syncthreads();
}

__device__ __forceinline__ void clear_bins(SampleShared& s) {
  for (int i = threadIdx.x; i < kSmBins; i += kSmThreads) s.lo[i] = s.hi[i] = s.cnt[i] = 0;
  if (threadIdx.x == 0) s.wrapped = 0;
  __syncthreads();
}

// Histogram over the exponents.
template <typename T>
__device__ __forceinline__ void exponent_bins(const Row<T>& row, bool counts, SampleShared& s) {
  clear_bins(s);
  for (int i = threadIdx.x; i < row.n; i += kSmThreads) {
    const float d = exponent(to_f32<T>(row.x[i]), row.rs);
    if (!(d >= -25.0f)) continue;
    const Halves h = halves(expf(d));
    const int b = bin_of(d);
    atomicAdd(&s.lo[b], h.lo);
    if (h.hi < (1u << 18)) {
      if (h.hi) atomicAdd(&s.hi[b], h.hi);
    } else if (atomicAdd(&s.hi[b], 1u << 18) == 0u - (1u << 18)) {
      s.wrapped = 1;
    }
    if (counts) atomicAdd(&s.cnt[b], 1u);
  }
}

// A set of tokens: one exponent bin, or a range of keys.
struct Pick {
  int bin;  // -1: keys klo .. khi
  uint32_t klo, khi;
  template <typename T>
  __device__ __forceinline__ bool has(const Row<T>& row, int i, uint32_t& key) const {
    const float x = to_f32<T>(row.x[i]);
    if (bin >= 0) {
      const float d = exponent(x, row.rs);
      if (!(d >= -25.0f) || bin_of(d) != bin) return false;
      key = key_of(x + 0.0f);
      return true;
    }
    key = key_of(clean(x));
    return key >= klo && key <= khi;
  }
};

struct Found {
  unsigned long long mass;  // prefix mass up to and with the token
  int token;                // its index, or -1: the rank-th token with `key`
  uint32_t key, rank;
};

// The token where the running count or mass of the whole row first reaches
// `goal`.  `nth` counts the searches of the row; the exponent bins are valid
// on entry if `*bins`, which a split clears.
template <typename T, bool BY_COUNT>
__device__ Found find_prefix(const Row<T>& row, unsigned long long goal, int& nth, bool& bins,
                             bool counts, SampleShared& s, uint8_t* slice) {
  if (!bins) {
    exponent_bins(row, counts, s);
    finish_bins(s, slice, row.C, row.rank);
    bins = true;
  }
  find_bin<BY_COUNT>(goal, s);
  Pick pick{s.bin, 0, 0};
  while (true) {
    const unsigned long long before = s.before;
    const uint32_t before_cnt = s.before_cnt;
    // ---- list the set's tokens
    const int par = nth++ & 1;
    __syncthreads();
    if (threadIdx.x == 0) s.n = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < row.n; i += kSmThreads) {
      uint32_t key;
      if (!pick.has(row, i, key)) continue;
      const uint32_t at = atomicAdd(&s.n, 1u);
      if (at < kSmLocal)
        s.local[par][at] = (static_cast<unsigned long long>(~key) << 32) |
                           static_cast<uint32_t>(row.i0 + i);
    }
    __syncthreads();
    if (threadIdx.x == 0) s.mine.count[par] = s.n;
    cluster_sync_all();
    uint32_t total = 0;
    bool fits = true;
    for (int r = 0; r < row.C; ++r) {
      const uint32_t n = ld_cluster(&s.mine.count[par], r);
      fits = fits && n <= kSmLocal;
      if (fits && total + n <= kSmList)
        for (uint32_t i = threadIdx.x; i < n; i += kSmThreads)
          s.list[total + i] = ld_cluster(&s.local[par][i], r);
      total += n;
    }
    if (fits && total <= kSmList) {
      // ---- sort it (bitonic, ascending: the largest logit, lowest index first)
      uint32_t size = 2;
      while (size < total) size <<= 1;
      for (uint32_t i = total + threadIdx.x; i < size; i += kSmThreads) s.list[i] = ~0ull;
      __syncthreads();
      for (uint32_t k = 2; k <= size; k <<= 1)
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
      unsigned long long w[2], a, ta;
      uint32_t c = 0, tc;
#pragma unroll
      for (int e = 0; e < 2; ++e)
        w[e] = i + e < total
                   ? weight(exponent(logit_of(~static_cast<uint32_t>(s.list[i + e] >> 32)), row.rs))
                   : 0;
      a = w[0] + w[1];
      block_exclusive(a, c, ta, tc, s);
      a += before;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const bool hit = BY_COUNT ? before_cnt + i + e + 1 == goal
                                  : a < goal && goal <= a + w[e];
        a += w[e];
        if (hit && i + e < total) {
          s.found = a;
          s.token = static_cast<int>(s.list[i + e] & 0xffffffffu);
          s.found_key = ~static_cast<uint32_t>(s.list[i + e] >> 32);
        }
      }
      __syncthreads();
      return {s.found, s.token, s.found_key, 0};
    }
    // ---- too many: split the set by its keys
    if (pick.bin >= 0) {
      uint32_t kmin = 0xffffffffu, kmax = 0;
      for (int i = threadIdx.x; i < row.n; i += kSmThreads) {
        uint32_t key;
        if (!pick.has(row, i, key)) continue;
        kmin = min(kmin, key);
        kmax = max(kmax, key);
      }
      uint32_t* red = reinterpret_cast<uint32_t*>(s.red);
      kmin = block_reduce(kmin, red, [](uint32_t a, uint32_t b) { return min(a, b); });
      kmax = block_reduce(kmax, red, [](uint32_t a, uint32_t b) { return max(a, b); });
      if (threadIdx.x == 0) {
        s.mine.kmin = kmin;
        s.mine.kmax = kmax;
      }
      cluster_sync_all();
      for (int r = 0; r < row.C; ++r) {
        kmin = min(kmin, ld_cluster(&s.mine.kmin, r));
        kmax = max(kmax, ld_cluster(&s.mine.kmax, r));
      }
      pick = {-1, kmin, kmax};
    }
    if (pick.klo == pick.khi) {  // equal logits: the rank follows from the goal
      const unsigned long long w = weight(exponent(logit_of(pick.klo), row.rs));
      const uint32_t rank = BY_COUNT ? static_cast<uint32_t>(goal - before_cnt)
                                     : static_cast<uint32_t>((goal - before + w - 1) / w);
      return {before + rank * w, -1, pick.klo, rank};
    }
    bins = false;
    const uint32_t range = pick.khi - pick.klo;
    const int shift = max(0, 32 - __clz(range) - 10);  // at most 1024 bins
    clear_bins(s);
    for (int i = threadIdx.x; i < row.n; i += kSmThreads) {
      uint32_t key;
      if (!pick.has(row, i, key)) continue;
      const uint32_t b = (pick.khi - key) >> shift;
      const unsigned long long w = weight(exponent(logit_of(key), row.rs));
      atomicAdd(&s.lo[b], static_cast<uint32_t>(w) & 0x3ffffu);
      atomicAdd(&s.hi[b], static_cast<uint32_t>(w >> 18));
      atomicAdd(&s.cnt[b], 1u);
    }
    finish_bins(s, slice, row.C, row.rank);
    // the goal counts from the row's start, the bins from the set's
    find_bin<BY_COUNT>(goal - (BY_COUNT ? before_cnt : before), s);
    const uint32_t top = pick.khi - (static_cast<uint32_t>(s.bin) << shift);
    const uint32_t low = shift == 0 ? top : top - min(top - pick.klo, (1u << shift) - 1);
    __syncthreads();
    if (threadIdx.x == 0) {
      s.before += before;
      s.before_cnt += before_cnt;
    }
    __syncthreads();
    pick = {-1, low, top};
  }
}

// Writes the index of the `rank`-th (1-based) token of the row with this key.
template <typename T>
__device__ void write_ranked(const Row<T>& row, uint32_t key, uint32_t rank, int* out,
                             SampleShared& s) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int per = ((row.n + kSmWarps - 1) / kSmWarps + 31) / 32 * 32;
  const int i0 = min(row.n, warp * per), i1 = min(row.n, i0 + per);
  uint32_t n = 0;
  for (int i = i0 + lane; i < i1; i += 32) n += key_of(clean(to_f32<T>(row.x[i]))) == key;
  n = __reduce_add_sync(0xffffffffu, n);
  if (lane == 0) s.red[warp] = n;
  __syncthreads();
  uint32_t before = 0, mine = 0;
  for (int w = 0; w < kSmWarps; ++w) {
    if (w == warp) before = mine;
    mine += static_cast<uint32_t>(s.red[w]);
  }
  if (threadIdx.x == 0) s.mine.ties = mine;
  cluster_sync_all();
  for (int r = 0; r < row.rank; ++r) before += ld_cluster(&s.mine.ties, r);
  if (before < rank && before + n >= rank) {  // one warp of the row
    for (int i = i0; i < i1; i += 32) {
      const bool hit = i + lane < i1 && key_of(clean(to_f32<T>(row.x[i + lane]))) == key;
      const uint32_t m = __ballot_sync(0xffffffffu, hit);
      const uint32_t here = __popc(m);
      if (before + here >= rank) {
        if (hit && before + __popc(m & ((1u << lane) - 1)) + 1 == rank) *out = row.i0 + i + lane;
        break;
      }
      before += here;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kSmThreads) sample_kernel(SampleParams p, int C) {
  extern __shared__ __align__(16) uint8_t sm_smem[];
  SampleShared& s = *reinterpret_cast<SampleShared*>(sm_smem);
  uint8_t* slice = sm_smem + (sizeof(SampleShared) + 15) / 16 * 16;
  T* data = reinterpret_cast<T*>(slice + (C > 1 ? (kSmSlice + 15) / 16 * 16 : 0));
  const int b = blockIdx.x / C, rank = blockIdx.x - b * C;
  const int per = (p.vocab + C - 1) / C;
  Row<T> row;
  row.C = C;
  row.rank = rank;
  row.i0 = min(p.vocab, rank * per);
  row.n = min(p.vocab, row.i0 + per) - row.i0;
  const T* src = static_cast<const T*>(p.logits) + b * p.ld + row.i0;

  // ---- 1. the stretch into shared memory, at the source's offset within 16
  // bytes so that the middle goes by 16-byte copies
  constexpr int kVec = 16 / sizeof(T);
  const int skew = static_cast<int>(reinterpret_cast<uintptr_t>(src) % 16 / sizeof(T));
  T* x = data + skew;
  row.x = x;
  const int head = min(row.n, (kVec - skew) % kVec), vecs = (row.n - head) / kVec;
  for (int i = threadIdx.x; i < vecs; i += kSmThreads)
    cp_async16(x + head + i * kVec, src + head + i * kVec, true);
  if (threadIdx.x < head) x[threadIdx.x] = src[threadIdx.x];
  const int tail = head + vecs * kVec + threadIdx.x;
  if (tail < row.n) x[tail] = src[tail];
  const float T0 = p.temperature ? p.temperature[b] : 1.0f;
  const int k = p.top_k ? p.top_k[b] : 0;
  const float tp = p.top_p ? p.top_p[b] : 1.0f;
  const float mp = p.min_p ? p.min_p[b] : 0.0f;
  row.rs.inv = __fdiv_rn(1.0f, T0);
  const bool greedy = !(T0 > 0.0f && row.rs.inv < INFINITY);
  cp_async_wait_all();
  __syncthreads();
  float mx = -INFINITY;
  for (int i = threadIdx.x; i < row.n; i += kSmThreads) mx = fmaxf(mx, to_f32<T>(x[i]));
  mx = block_reduce(mx, reinterpret_cast<float*>(s.red), [](float a, float c) { return fmaxf(a, c); });
  if (threadIdx.x == 0) s.mine.xmax = mx;
  cluster_sync_all();
  for (int r = 0; r < C; ++r) mx = fmaxf(mx, ld_cluster(&s.mine.xmax, r));
  row.rs.xmax = mx + 0.0f;

  if (mx == -INFINITY) {  // nothing to choose from
    if (rank == 0 && threadIdx.x == 0) {
      p.tokens[b] = -1;
      if (p.logprobs) p.logprobs[b] = -INFINITY;
    }
    cluster_sync_all();  // shared memory is read by the other CTAs until here
    return;
  }

  // ---- sums that need no order: e^(x - max) for the log-probability (f64 over
  // f32 terms: a peaked row adds tens of thousands of tiny terms to 1), the
  // weight above the min-p cut, and the first maximum of a greedy row
  const float dmin = mp > 0.0f ? fminf(static_cast<float>(log(static_cast<double>(mp))), 0.0f)
                               : -INFINITY;
  double z = 0.0;
  if (p.logprobs) {
    for (int i = threadIdx.x; i < row.n; i += kSmThreads) {
      const float e = expf(delta(to_f32<T>(x[i]), mx));
      z += e == e ? static_cast<double>(e) : 0.0;
    }
    z = block_reduce(z, reinterpret_cast<double*>(s.red), [](double a, double c) { return a + c; });
  }
  unsigned long long above = 0;
  if (!greedy && mp > 0.0f) {
    for (int i = threadIdx.x; i < row.n; i += kSmThreads) {
      const float d = exponent(to_f32<T>(x[i]), row.rs);
      if (d >= dmin) above += weight(d);
    }
    above = block_reduce(above, s.red, [](unsigned long long a, unsigned long long c) { return a + c; });
  }
  int first = INT32_MAX;
  if (greedy) {
    for (int i = threadIdx.x; i < row.n; i += kSmThreads)
      if (to_f32<T>(x[i]) == mx) first = min(first, row.i0 + i);
    first = block_reduce(first, reinterpret_cast<int*>(s.red), [](int a, int c) { return min(a, c); });
  }
  if (threadIdx.x == 0) {
    s.mine.z = z;
    s.mine.above = above;
    s.mine.first = first;
  }
  uint32_t key = key_of(row.rs.xmax), tie_rank = 0;
  int token = -1;
  if (!greedy) {
    // ---- 2. and 3.
    const bool counts = k > 0 && k < p.vocab;
    int nth = 0;
    bool bins = false;
    exponent_bins(row, counts, s);
    finish_bins(s, slice, C, rank);
    bins = true;
    if (C == 1) __syncthreads();
    unsigned long long mass = s.total;
    if (counts && static_cast<unsigned long long>(k) < s.total_cnt)
      mass = find_prefix<T, true>(row, static_cast<unsigned long long>(k), nth, bins, counts, s, slice).mass;
    if (tp < 1.0f) {
      const double want = ceil(static_cast<double>(fmaxf(tp, 0.0f)) * static_cast<double>(mass));
      const unsigned long long goal = max(1ull, min(mass, static_cast<unsigned long long>(want)));
      mass = find_prefix<T, false>(row, goal, nth, bins, counts, s, slice).mass;
    }
    if (mp > 0.0f) {  // (the slots were written before the bins' barriers)
      above = 0;
      for (int r = 0; r < C; ++r) above += ld_cluster(&s.mine.above, r);
      mass = min(mass, above);
    }
    const double t = floor(static_cast<double>(p.u[b]) * static_cast<double>(mass));
    const unsigned long long target =
        t > 0.0 ? min(mass - 1, static_cast<unsigned long long>(t)) : 0ull;
    const Found f = find_prefix<T, false>(row, target + 1, nth, bins, counts, s, slice);
    key = f.key;
    token = f.token;
    tie_rank = f.rank;
    if (token < 0) write_ranked(row, key, tie_rank, p.tokens + b, s);
  } else {
    cluster_sync_all();
    for (int r = 0; r < C; ++r) first = min(first, ld_cluster(&s.mine.first, r));
    token = first;
  }
  if (rank == 0 && threadIdx.x == 0) {
    if (token >= 0) p.tokens[b] = token;
    if (p.logprobs) {
      z = 0.0;
      for (int r = 0; r < C; ++r) z += ld_cluster(&s.mine.z, r);
      const float v = logit_of(key);
      p.logprobs[b] = static_cast<float>((v == mx ? 0.0 : static_cast<double>(v) - mx) - log(z));
    }
  }
  cluster_sync_all();  // shared memory is read by the other CTAs until here
}

template <typename T>
cudaError_t launch_t(const SampleParams& p, int C, cudaStream_t s) {
  const size_t smem = (sizeof(SampleShared) + 15) / 16 * 16 +
                      (C > 1 ? (kSmSlice + 15) / 16 * 16 : 0) +
                      static_cast<size_t>((p.vocab + C - 1) / C) * sizeof(T) + 32;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  static std::atomic<bool> configured[64];
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
    configured[dev].store(true, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(p.batch) * C);
  cfg.blockDim = dim3(kSmThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = C;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, sample_kernel<T>, p, C);
}

}  // namespace

// CTAs per row: enough that a stretch fits (kSmChunk tokens), and up to 8 while
// the batch leaves SMs idle.
int sample_cluster(int batch, int vocab, int sms) {
  int C = 1;
  while ((vocab + C - 1) / C > kSmChunk) C *= 2;
  while (C < 8 && batch * 2ll * C <= sms && vocab > 1024 * C) C *= 2;
  return C;
}

cudaError_t launch_sample(const SampleParams& p, int C, cudaStream_t s) {
  switch (p.dtype) {
    case 0: return launch_t<float>(p, C, s);
    case 1: return launch_t<__nv_bfloat16>(p, C, s);
    case 2: return launch_t<__half>(p, C, s);
  }
  return cudaErrorInvalidValue;
}

}  // namespace ffai

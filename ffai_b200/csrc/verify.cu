// Verification of drafted tokens against the target's distribution, from given
// uniform numbers.
//
// Request b has the rows cu[b] .. cu[b + 1] - 1: its last token and its drafts.
// Row i's target distribution p is the softmax of its logits over the
// temperature T; the token of row i + 1 was drafted from q, likewise of the draft
// model's logits of row i, or given (q is 1 there).  The draft x of row i stands if
//   u_i q(x) < p(x),
// and with the first that does not the request takes a token from the
// distribution max(0, p - q) / sum of it, or, if all stand, from the last row's p:
// what is emitted is distributed as if the target alone had been sampled.
//
// In whole weights w = floor(2^36 e^d) (weights.cuh) of sum W, v and V for the
// draft's, all sums are exact and the tokens depend on the inputs alone:
//   x stands if  fl(fl(u v_x) W) < fl(w_x V)                        (f64 products)
//   r_i = max(0, w_i - floor(fl(v_i fl(W / V)))),  R their sum
//   the token is the first i with r_0 + .. + r_i > floor(fl(u' R)),
// with w in r's place if R is 0.  T = 0 puts all weight on the first maximum, an
// infinite T the same on every finite logit.
//
// Two launches.  In the first a cluster of CTAs takes a row at a time, of target
// and draft: the maximum, then the sum of the weights, the logits coming from L1 or
// L2 the second time.  Rows are taken by their place in the request, all first ones
// first, and a row behind one that is known to have failed is left out: it
// cannot matter.  (Which ones are left out depends on timing, the results do not.)
// In the second launch a cluster per request walks the row of its token again.
//
// Bound by waiting: for the exchange behind each of a row's two passes, for loads that
// start anew behind it (about 20 instructions a logit for the exact weight's two halves use
// 14 to 35 % of the first launch's issue slots, up to 45 % of the second's), and for few
// rows by the chain of all these: 96 requests of four drafts with the draft model's
// logits, 128000 f32: 141 us, the launches 97 and 56 apart (198 MB at least, 30 us); 64 of
// seven looked-up drafts, 51865 bf16: 43 us; five with a draft model's, f32: 26 us.
#include <algorithm>

#include "common.cuh"
#include "kernels.h"
#include "weights.cuh"

namespace ffai {

namespace {

constexpr int kVfThreads = 512;
constexpr int kVfWarps = kVfThreads / 32;
constexpr int kVfCluster = 8;  // CTAs per row, at most
constexpr int kVfParts = kVfWarps * kVfCluster;  // warps per row
constexpr int kVfNone = 1 << 25;  // more than a request has rows

__device__ __forceinline__ void st_cluster_u64(uint32_t caddr, unsigned long long v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(caddr), "l"(v) : "memory");
}
// v, the same in all lanes, to *at of every CTA of the cluster, there after the
// next row_sync.
__device__ __forceinline__ void tell_all(unsigned long long* at, unsigned long long v, int ctas) {
  const int lane = threadIdx.x % 32;
  if (ctas == 1) {
    if (lane == 0) *at = v;
  } else if (lane < ctas) {
    st_cluster_u64(mapa_shared(smem_u32(at), lane), v);
  }
}
__device__ __forceinline__ void row_sync(int ctas) {
  if (ctas > 1) {
    cluster_arrive();
    cluster_wait();
  } else {
    __syncthreads();
  }
}
// Over a warp: the maximum (no NaN; -0 is below 0), and the sum (of less than 2^59).
__device__ __forceinline__ float warp_max(float x) {
  const int b = __float_as_int(x);
  const int m = __reduce_max_sync(0xffffffffu, b < 0 ? b ^ 0x7fffffff : b);
  return __int_as_float(m < 0 ? m ^ 0x7fffffff : m);
}
__device__ __forceinline__ unsigned long long warp_sum(unsigned long long x) {
  constexpr uint32_t kMask = (1u << 20) - 1;
  const uint32_t a = __reduce_add_sync(0xffffffffu, static_cast<uint32_t>(x) & kMask);
  const uint32_t b = __reduce_add_sync(0xffffffffu, static_cast<uint32_t>(x >> 20) & kMask);
  const uint32_t c = __reduce_add_sync(0xffffffffu, static_cast<uint32_t>(x >> 40));
  return a + (static_cast<unsigned long long>(b) << 20) + (static_cast<unsigned long long>(c) << 40);
}

struct Request {
  int r0, n;  // first row, rows
};
// Rows of request b; those that cannot be told are none.
__device__ __forceinline__ Request request(const VerifyParams& p, int b, bool& bad) {
  const int r0 = __ldg(p.cu_rows + b), r1 = __ldg(p.cu_rows + b + 1);
  if (r0 < 0 || r1 < r0 || r1 > p.rows) {
    bad = true;
    return {0, 0};
  }
  return {r0, r1 - r0};
}

__device__ __forceinline__ float inverse(const float* temperature, int b) {
  const float t = temperature ? __ldg(temperature + b) : 1.0f;
  const float inv = t > 0.0f ? __fdiv_rn(1.0f, t) : INFINITY;
  return isinf(inv) ? -1.0f : inv;  // (0 is an infinite T's)
}
// The first maximum has all weight.
__device__ __forceinline__ bool greedy(float inv) { return inv < 0.0f; }

// A weight's halves with the magic numbers' bits in them: fma and add towards zero
// leave the whole part in the low mantissa bits.  e < 1 / 2^36 gives none.
struct Half2 {
  uint32_t hi, lo;
};
__device__ __forceinline__ Half2 raw_halves(float e) {
  const float t = __fmaf_rz(e, 262144.0f, 8388608.0f);
  const float r = __fmaf_rn(e, 262144.0f, -__fadd_rn(t, -8388608.0f));
  return {__float_as_uint(t), __float_as_uint(__fmaf_rz(r, 262144.0f, 8388608.0f))};
}
constexpr uint32_t kMagic = 0x4b000000u;
// The weight itself, in 64 bits of floating point: the whole number's bits in the
// mantissa of 2^52, less 2^52.
__device__ __forceinline__ double whole_weight(float e) {
  const Half2 h = raw_halves(e);
  const unsigned long long w = static_cast<unsigned long long>(h.hi - kMagic) * 262144ull + (h.lo - kMagic);
  return __dadd_rn(__longlong_as_double(static_cast<long long>(w | 0x4330000000000000ull)), -4503599627370496.0);
}

// The same of two powers at once.
__device__ __forceinline__ uint64_t f2_fma_rz(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rz.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ void add_halves(float e0, float e1, uint32_t& hi, uint32_t& lo) {
  const uint64_t e = f2_pack(e0, e1), scale = f2_pack(262144.0f, 262144.0f);
  const uint64_t magic = f2_pack(8388608.0f, 8388608.0f);
  const uint64_t t = f2_fma_rz(e, scale, magic);
  const uint64_t r = f2_fma(e, scale, f2_sub(magic, t));
  const uint64_t l = f2_fma_rz(r, scale, magic);
  hi += static_cast<uint32_t>(t) + static_cast<uint32_t>(t >> 32);
  lo += static_cast<uint32_t>(l) + static_cast<uint32_t>(l >> 32);
}

// The distribution of a row: what its weights are relative to.
struct Dist {
  float xmax, inv;
  int first;  // index of the first maximum, if greedy(inv)
  // ordinary: weights are e^d; else all weight lies on some maxima, or there is none
  __device__ __forceinline__ bool ordinary() const { return !greedy(inv) && !isinf(xmax); }
  // e^d; what is not a number gives none
  __device__ __forceinline__ float power(float x) const {
    return expf(fmaxf(__fmul_rn(__fadd_rn(x, -xmax), inv), -100.0f));
  }
  __device__ __forceinline__ unsigned long long at(float x, int i) const {
    if (xmax == -INFINITY) return 0;
    if (greedy(inv)) return i == first ? 1ull << 36 : 0;
    return weight(__fmul_rn(delta(clean(x), xmax), inv));
  }
};

// The 16-byte pieces that hold a row, from the one its first logit lies in.
template <typename T>
struct RowPieces {
  static constexpr int kVec = 16 / sizeof(T);
  const T* row;
  int skew, vocab, pieces;
  __device__ __forceinline__ RowPieces(const void* base, long long ld, int r, int v)
      : row(static_cast<const T*>(base) + r * ld), vocab(v) {
    skew = static_cast<int>(reinterpret_cast<uintptr_t>(row) % 16 / sizeof(T));
    pieces = (skew + v + kVec - 1) / kVec;
  }
  __device__ __forceinline__ int index(int piece) const { return piece * kVec - skew; }
  __device__ __forceinline__ bool whole(int i) const {
    return index(i) >= 0 && index(i) + kVec <= vocab;
  }
  __device__ __forceinline__ uint4 load(int i) const {
    return __ldg(reinterpret_cast<const uint4*>(row + index(i)));
  }
  // Element e of piece i, -inf outside the row.
  __device__ __forceinline__ float element(int i, int e) const {
    const int at = index(i) + e;
    return at >= 0 && at < vocab ? to_f32<T>(row[at]) : -INFINITY;
  }
  // f(x, i) for the logits (index i) of pieces [i0, i1) that no vector load may
  // take, one a thread: at the row's ends.  The others are lo .. hi - 1.
  template <typename F>
  __device__ __forceinline__ void edges(int i0, int i1, int& lo, int& hi, F f) const {
    lo = i0 < i1 && !whole(i0) ? i0 + 1 : i0;
    hi = i1 > lo && !whole(i1 - 1) ? i1 - 1 : i1;
    const int t = threadIdx.x, edge = t < kVec ? i0 : i1 - 1;
    if (t < 2 * kVec && (t < kVec ? lo > i0 : hi < i1)) {
      const int i = index(edge) + t % kVec;
      if (i >= 0 && i < vocab) f(to_f32<T>(row[i]), i);
    }
  }
};

// The passes over a CTA's part [lo, hi) of a row's pieces, functions of their own
// so that the loops have all registers (inlined they kept theirs in local memory).
template <typename T>
__device__ __noinline__ float max_pass(const uint4* pieces, int lo, int hi) {
  constexpr int kVec = 16 / sizeof(T), kUnroll = 4;
  float m = -INFINITY;  // NaN counts as -inf: fmaxf passes it over
#pragma unroll 1
  for (int i = lo + static_cast<int>(threadIdx.x); i < hi; i += kUnroll * kVfThreads) {
    uint4 w[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) w[k] = __ldg(pieces + min(i + k * kVfThreads, hi - 1));  // (some twice)
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      float x[kVec];
      unpack<T>(w[k], x);
#pragma unroll
      for (int e = 0; e < kVec; e += 2) m = max3f(m, x[e], x[e + 1]);
    }
  }
  return m;
}

// Sum of the weights, and of e^(x - top).
struct PassSums {
  unsigned long long mass;
  float z;
};
template <typename T, bool LOGS>
__device__ __noinline__ PassSums sum_pass(const uint4* pieces, int lo, int hi, float top, float inv) {
  constexpr int kVec = 16 / sizeof(T);
  const uint64_t top2 = f2_pack(-top, -top), inv2 = f2_pack(inv, inv);
  uint32_t hs = 0, ls = 0, n = 0;
  float z = 0.0f;
  int i = lo + static_cast<int>(threadIdx.x);
  uint4 next = i < hi ? __ldg(pieces + i) : make_uint4(0, 0, 0, 0);
#pragma unroll 1
  for (; i < hi; i += kVfThreads) {
    const uint4 w = next;
    next = __ldg(pieces + min(i + kVfThreads, hi - 1));
    float x[kVec];
    unpack<T>(w, x);
    n += kVec;
#pragma unroll
    for (int e = 0; e < kVec; e += 2) {
      const uint64_t below = f2_add(f2_pack(x[e], x[e + 1]), top2);
      float a, b;
      f2_unpack(f2_mul(below, inv2), a, b);
      // (what is not a number, and all below, weighs nothing)
      a = expf(fmaxf(a, -100.0f)), b = expf(fmaxf(b, -100.0f));
      add_halves(a, b, hs, ls);
      if constexpr (LOGS) {
        if (inv != 1.0f) {
          f2_unpack(below, a, b);
          a = expf(fmaxf(a, -100.0f)), b = expf(fmaxf(b, -100.0f));
        }
        z += a + b;
      }
    }
  }
  return {(static_cast<unsigned long long>(hs - n * kMagic) << 18) + (ls - n * kMagic), z};
}

// A row to take: what the warps that walk logits need to know.
struct Job {
  long long pair;  // place in the request * batch + request
  int row, flags;  // flags 1: a token was drafted there, 2: with a draft model's logits
  float inv[2];
};
// Pair n in order, if it has a row that matters: the request has so many, and none
// before it is known to have failed.
__device__ __forceinline__ Job job_of(const VerifyParams& p, long long n, long long end, bool fails) {
  Job job{n, -1, 0, {0.0f, 0.0f}};
  if (n >= end) return job;
  int k, b;
  bool bad = false;
  if (end <= INT32_MAX) {
    k = static_cast<int>(static_cast<uint32_t>(n) / static_cast<uint32_t>(p.batch));
    b = static_cast<int>(n) - k * p.batch;
  } else {
    k = static_cast<int>(n / p.batch);
    b = static_cast<int>(n - static_cast<long long>(k) * p.batch);
  }
  const Request req = request(p, b, bad);
  if (k < req.n && (!fails || k <= kVfNone - __ldcg(p.fails + b))) {
    job.row = req.r0 + k;
    job.flags = k + 1 < req.n ? (p.draft ? 3 : 1) : 0;
    job.inv[0] = inverse(p.temperature, b);
    job.inv[1] = job.flags & 2 ? inverse(p.draft_temperature, b) : 0.0f;
  }
  return job;
}
// The row a cluster takes next, off the queue of pairs (the first `clusters` went
// out without it).  One warp, which may keep a few: where few pairs have a row it
// takes 32 at a time.  Row -1: no more.
struct Queue {
  long long base;
  unsigned left;  // lanes of the pairs base .. that are still to be looked at
};
__device__ __forceinline__ Job next_job(const VerifyParams& p, Queue& q, int clusters, int places) {
  const int lane = threadIdx.x % 32;
  const long long end = static_cast<long long>(places) * p.batch;
  const int take = end > 8LL * p.rows ? 32 : 1;
  while (end > clusters) {
    if (!q.left) {
      unsigned long long n = 0;
      if (lane == 0) n = atomicAdd(p.queue, static_cast<unsigned long long>(take));
      q.base = static_cast<long long>(__shfl_sync(0xffffffffu, n, 0)) + clusters;
      if (q.base >= end) return {end, -1, 0, {0.0f, 0.0f}};
      q.left = take == 32 ? ~0u : 1u;
    }
    Job job = job_of(p, q.left >> lane & 1u ? q.base + lane : end, end, true);
    q.left &= __ballot_sync(0xffffffffu, job.row >= 0);
    if (!q.left) continue;
    const int l = __ffs(q.left) - 1;
    q.left &= q.left - 1;
    job.pair = __shfl_sync(0xffffffffu, job.pair, l);
    job.row = __shfl_sync(0xffffffffu, job.row, l);
    job.flags = __shfl_sync(0xffffffffu, job.flags, l);
    job.inv[0] = __shfl_sync(0xffffffffu, job.inv[0], l);
    job.inv[1] = __shfl_sync(0xffffffffu, job.inv[1], l);
    return job;
  }
  return {end, -1, 0, {0.0f, 0.0f}};
}

// What the warps of a row's CTAs tell one another, of target and draft.
struct RowParts {
  unsigned long long top[2][kVfParts], val[2][kVfParts], z[kVfParts];
  unsigned long long job[3];  // the next: pair, row and flags, inverse temperatures
  int places;
};
__device__ __forceinline__ Job read_job(const RowParts& s) {
  Job j;
  j.pair = static_cast<long long>(s.job[0]);
  j.row = static_cast<int>(s.job[1] & 0xffffffffu);
  j.flags = static_cast<int>(s.job[1] >> 32);
  j.inv[0] = __uint_as_float(static_cast<uint32_t>(s.job[2]));
  j.inv[1] = __uint_as_float(static_cast<uint32_t>(s.job[2] >> 32));
  return j;
}
__device__ __forceinline__ void tell_job(RowParts& s, const Job& j, int ctas) {
  tell_all(&s.job[0], static_cast<unsigned long long>(j.pair), ctas);
  tell_all(&s.job[1], static_cast<uint32_t>(j.row) | static_cast<unsigned long long>(static_cast<uint32_t>(j.flags)) << 32, ctas);
  tell_all(&s.job[2], __float_as_uint(j.inv[0]) | static_cast<unsigned long long>(__float_as_uint(j.inv[1])) << 32, ctas);
}
// The maximum of all warps of a row.
__device__ __forceinline__ float all_max(const unsigned long long* part, int parts) {
  float m = -INFINITY;
  for (int i = threadIdx.x % 32; i < parts; i += 32) m = fmaxf(m, __uint_as_float(static_cast<uint32_t>(part[i])));
  return warp_max(m);
}

// What is known of a row once its parts are: a warp, in the order of its steps.
template <typename T>
__device__ __noinline__ void finish_row(const VerifyParams& p, const RowParts& s, const Job& job, int parts,
                                        const float* top, int token, const float* at, float u) {
  const int lane = threadIdx.x % 32, both = job.flags & 2 ? 2 : 1;
  unsigned long long w[2] = {0, 1}, mass[2] = {0, 1};
#pragma unroll 1
  for (int which = 0; which < both; ++which) {
    const float inv = job.inv[which], t = top[which];
    unsigned long long v = greedy(inv) ? ~0ull : 0;
    for (int i = lane; i < parts; i += 32) v = greedy(inv) ? min(v, s.val[which][i]) : v + s.val[which][i];
    v = greedy(inv) ? __reduce_min_sync(0xffffffffu, static_cast<uint32_t>(v)) : warp_sum(v);
    double z = 0.0;
    if (!which && p.logprobs) {
      for (int i = lane; i < parts; i += 32) z += __longlong_as_double(s.z[i]);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
    }
    VerifyRow r;
    r.xmax = t;
    r.first = greedy(inv) ? static_cast<int>(v) : 0;
    r.mass = t == -INFINITY ? 0 : greedy(inv) ? 1ull << 36 : isinf(t) ? v << 36 : v;
    r.log_z = !which && p.logprobs ? static_cast<float>(log(z)) : 0.0f;
    w[which] = token >= 0 ? Dist{t, inv, r.first}.at(at[which], token) : 0;
    mass[which] = r.mass;
    if (lane == 0) p.stats[which * p.rows + job.row] = r;
  }
  if ((job.flags & 1) && lane == 0) {
    const double left = __dmul_rn(__dmul_rn(static_cast<double>(u), __ull2double_rn(w[1])), __ull2double_rn(mass[0]));
    if (!(left < __dmul_rn(__ull2double_rn(w[0]), __ull2double_rn(mass[1])))) {
      const int place = static_cast<int>(job.pair / p.batch);
      atomicMax(p.fails + static_cast<int>(job.pair - static_cast<long long>(place) * p.batch), kVfNone - place);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kVfThreads + 32, 2) verify_rows_kernel(const __grid_constant__ VerifyParams p) {
  __shared__ RowParts s;
  griddep_launch_dependents();
  const int shift = p.row_shift, ctas = 1 << shift, cluster = blockIdx.x >> shift, rank = blockIdx.x & (ctas - 1);
  const int clusters = gridDim.x >> shift, warp = threadIdx.x / 32;
  const int parts = kVfWarps << shift, part = rank * kVfWarps + warp;
  const bool steers = warp == kVfWarps;  // the last warp: it walks no logits
  if (ctas > 1) cluster_arrive_relaxed();  // waited for below: every CTA of the cluster runs
  // ---- nothing is emitted yet; the most rows a request has
  if (threadIdx.x == 0) s.places = 0;
  const int threads = kVfThreads + 32;
  for (int i = blockIdx.x * threads + threadIdx.x; i < p.rows; i += gridDim.x * threads) {
    p.tokens_out[i] = -1;
    if (p.logprobs) p.logprobs[i] = 0.0f;
  }
  int most = 0;
  bool bad = false;
#pragma unroll 4
  for (int b = threadIdx.x; b < p.batch; b += threads) most = max(most, request(p, b, bad).n);
  __syncthreads();
  if (warp * 32 < p.batch) {
    most = __reduce_max_sync(0xffffffffu, most);
    if (threadIdx.x % 32 == 0 && most > 0) atomicMax(&s.places, most);
  }
  if (ctas > 1) cluster_wait();
  __syncthreads();
  const int places = s.places;
  // (the first one without a look at what failed: all CTAs of the cluster agree on
  // it, also that there is none)
  const long long end = static_cast<long long>(places) * p.batch;
  if (steers) tell_job(s, job_of(p, cluster, end, false), 1);
  __syncthreads();
  Job job = read_job(s);
  Queue queue{0, 0};
  if (job.row < 0 && job.pair < end) {
    if (ctas > 1) row_sync(ctas);  // (each has read its own)
    if (steers && rank == 0) tell_job(s, next_job(p, queue, clusters, places), ctas);
    row_sync(ctas);
    job = read_job(s);
  }

  while (job.row >= 0) {
    const int both = job.flags & 2 ? 2 : 1;
    float at[2] = {-INFINITY, -INFINITY}, u = 0.0f;
    int token = -1;
    if (steers && rank == 0 && (job.flags & 1)) {  // the logits of the token drafted there
      token = __ldg(p.tokens + job.row + 1);
      u = __ldg(p.u + job.row);
      if (token >= 0 && token < p.vocab) {
        at[0] = to_f32<T>(static_cast<const T*>(p.logits)[job.row * p.ld + token]);
        if (both == 2) at[1] = to_f32<T>(static_cast<const T*>(p.draft)[job.row * p.draft_ld + token]);
      } else {
        token = -1;
      }
    }
    // Maximum and sum of target and draft: a single CTA finishes one after the
    // other, so that fewer rows are to stay in L2; a cluster exchanges both at once.
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll 1
    for (int step = 0; step < 4; ++step) {
      const int which = ctas > 1 ? step & 1 : step >> 1, phase = ctas > 1 ? step >> 1 : step & 1;
      if (which < both && !steers) {
        const RowPieces<T> src(which ? p.draft : p.logits, which ? p.draft_ld : p.ld, job.row, p.vocab);
        const int per = (src.pieces + ctas - 1) >> shift;
        const int i0 = min(src.pieces, rank * per), i1 = min(src.pieces, i0 + per);
        const uint4* pieces = reinterpret_cast<const uint4*>(src.row - src.skew);
        int lo, hi;
        if (phase == 0) {
          float m = -INFINITY;
          src.edges(i0, i1, lo, hi, [&](float x, int) { m = fmaxf(m, x); });
          m = warp_max(fmaxf(m, max_pass<T>(pieces, lo, hi))) + 0.0f;
          tell_all(&s.top[which][part], __float_as_uint(m), ctas);
        } else {
          const Dist d{which ? top[1] : top[0], which ? job.inv[1] : job.inv[0], 0};
          const bool logs = !which && p.logprobs;
          float z = 0.0f;
          unsigned long long v = 0;
          if (d.ordinary()) {
            src.edges(i0, i1, lo, hi, [&](float x, int) {
              v = weight(__fmul_rn(__fadd_rn(x, -d.xmax), d.inv));
              if (logs) z = expf(fmaxf(__fadd_rn(x, -d.xmax), -100.0f));
            });
            const PassSums r = logs ? sum_pass<T, true>(pieces, lo, hi, d.xmax, d.inv)
                                    : sum_pass<T, false>(pieces, lo, hi, d.xmax, d.inv);
            v = warp_sum(v + r.mass);
            z += r.z;
          } else {
            // the first maximum, or the number of infinite logits
            uint32_t first = ~0u, n = 0;
#pragma unroll 1
            for (int i = max(0, src.index(i0)) + static_cast<int>(threadIdx.x); i < min(p.vocab, src.index(i1)); i += kVfThreads) {
              const float x = to_f32<T>(src.row[i]);
              if (x == d.xmax) {
                first = min(first, static_cast<uint32_t>(i));
                ++n;
              }
              if (logs) z += x == x ? expf(delta(x, d.xmax)) : 0.0f;
            }
            v = greedy(d.inv) ? __reduce_min_sync(0xffffffffu, first) : __reduce_add_sync(0xffffffffu, n);
          }
          tell_all(&s.val[which][part], v, ctas);
          if (logs) {
            double zd = z;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) zd += __shfl_xor_sync(0xffffffffu, zd, o);
            tell_all(&s.z[part], __double_as_longlong(zd), ctas);
          }
        }
      }
      if (step == 3 && steers && rank == 0)  // (one answer for all CTAs of the cluster: they might not see the same)
        tell_job(s, next_job(p, queue, clusters, places), ctas);
      if (which == 1 || ctas == 1) {
        if (which < both || ctas > 1 || step == 3) row_sync(ctas);
        if (phase == 0) {
          if (which == 0 || ctas > 1) top[0] = all_max(s.top[0], parts);
          if (which == 1 && both == 2) top[1] = all_max(s.top[1], parts);
        }
      }
    }
    // (while the others begin the next row: they wait for this warp before they tell more)
    if (steers && rank == 0) finish_row<T>(p, s, job, parts, top, token, at, u);
    job = read_job(s);
  }
}

// The weights of a row's token: the target's, or what it has beyond the draft's.
template <typename T>
__global__ void __launch_bounds__(kVfThreads, 2) verify_pick_kernel(const __grid_constant__ VerifyParams p) {
  constexpr int kVec = 16 / sizeof(T);
  __shared__ unsigned long long s_part[2][kVfParts];
  const int ctas = p.pick_ctas, b = blockIdx.x / ctas, rank = blockIdx.x - b * ctas;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int parts = ctas * kVfWarps, part = rank * kVfWarps + warp;
  bool bad = false;
  const Request req = request(p, b, bad);
  const float inv = inverse(p.temperature, b), draft_inv = inverse(p.draft_temperature, b);
  if (ctas > 1) cluster_arrive_relaxed();  // waited for below: every CTA of the request runs
  griddep_wait();
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.queue = 0;  // for the next call
  if (req.n == 0) {
    if (rank == 0 && threadIdx.x == 0) {
      p.accepted[b] = 0;
      p.next[b] = -1;
      if (bad && p.err) atomicOr(p.err, kErrBadArgs);
    }
    if (ctas > 1) cluster_wait();
    return;
  }
  // ---- the first draft that does not stand; the last row has none
  const int failed = __ldcg(p.fails + b);
  const int fail = failed ? kVfNone - failed : req.n - 1;
  const int row = req.r0 + fail;
  const VerifyRow t = p.stats[row];
  const Dist target{t.xmax, inv, t.first};
  const int drafted = failed ? __ldg(p.tokens + row + 1) : -1;
  Dist draft{-INFINITY, 0.0f, 0};
  double rho = 0.0;
  if (failed && p.draft) {
    const VerifyRow d = p.stats[p.rows + row];
    draft = Dist{d.xmax, draft_inv, d.first};
    rho = d.mass ? __ddiv_rn(__ull2double_rn(t.mass), __ull2double_rn(d.mass)) : 0.0;
  }

  // ---- its weights once more: a warp takes a run of pieces
  const RowPieces<T> src(p.logits, p.ld, row, p.vocab);
  const RowPieces<T> other(failed && p.draft ? p.draft : p.logits, failed && p.draft ? p.draft_ld : p.ld, row, p.vocab);
  const int per = (src.pieces + parts - 1) / parts;
  const int i0 = min(src.pieces, part * per), i1 = min(src.pieces, i0 + per);
  const bool ordinary = target.ordinary() && (!(failed && p.draft) || draft.ordinary());
  bool rest = failed;  // what the draft leaves
  struct Raw {
    uint4 x, y;
  };
  const bool alike = other.skew == src.skew;
  const auto fetch = [&](int i) {
    Raw r{};
    if (i < i1 && src.whole(i)) {
      r.x = src.load(i);
      if (rest && p.draft && alike) r.y = other.load(i);
    }
    return r;
  };
  // the sum of piece i's weights, which are w: whole numbers below 2^52 in 64 bits
  // of floating point, whose sums stay exact over a warp's pieces
  const auto piece = [&](int i, const Raw& raw, double (&w)[kVec]) {
    float x[kVec], y[kVec];
    const int at = src.index(i);
    const bool inside = src.whole(i), beside = rest && p.draft;
    if (inside) {
      unpack<T>(raw.x, x);
    } else {
#pragma unroll
      for (int e = 0; e < kVec; ++e) x[e] = src.element(i, e);
    }
    if (beside) {
      if (inside && alike) {
        unpack<T>(raw.y, y);
      } else {
#pragma unroll
        for (int e = 0; e < kVec; ++e)
          y[e] = at + e >= 0 && at + e < p.vocab ? to_f32<T>(other.row[at + e]) : -INFINITY;
      }
    }
    double sum = 0.0;
    if (ordinary) {
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        double r = whole_weight(target.power(x[e]));
        if (beside) {
          // w - floor(v rho): adding 2^52 towards zero leaves the whole part (of
          // what is larger than that, something larger than w)
          const double less = __dmul_rn(whole_weight(draft.power(y[e])), rho);
          r = __dadd_rn(r, -__dadd_rn(__dadd_rz(less, 4503599627370496.0), -4503599627370496.0));
          r = __double2hiint(r) < 0 ? 0.0 : r;
        } else if (rest) {
          r = at + e == drafted ? 0.0 : r;
        }
        w[e] = r;
        sum += r;
      }
    } else {
#pragma unroll 1
      for (int e = 0; e < kVec; ++e) {
        float xe = -INFINITY, ye = -INFINITY;
#pragma unroll
        for (int k = 0; k < kVec; ++k)
          if (k == e) {
            xe = x[k];
            if (beside) ye = y[k];
          }
        double r = at + e >= 0 && at + e < p.vocab ? __ull2double_rn(target.at(xe, at + e)) : 0.0;
        if (beside && r > 0.0) {
          const double v = __ull2double_rn(draft.at(ye, at + e));
          r = fmax(0.0, r - floor(__dmul_rn(v, rho)));
        } else if (rest && !p.draft && at + e == drafted) {
          r = 0.0;
        }
#pragma unroll
        for (int k = 0; k < kVec; ++k)
          if (k == e) w[k] = r;
        sum += r;
      }
    }
    return sum;
  };
  unsigned long long total = 0, before = 0, mine = 0;
  unsigned long long run = 0;  // lane n: the sum of the warp's n-th kRun * 32 pieces
  constexpr int kRun = 2;
  // (the launcher gives more than 2048 pieces a warp to no row)
#pragma unroll 1
  for (int round = 0; round < 2; ++round) {
    mine = 0;
    int n = 0;
#pragma unroll 1
    for (int i = i0; i < i1; i += 32 * kRun, ++n) {
      double sum = 0.0;
      Raw raw[kRun];
#pragma unroll
      for (int k = 0; k < kRun; ++k) raw[k] = fetch(i + 32 * k + lane);
#pragma unroll
      for (int k = 0; k < kRun; ++k) {
        double w[kVec];
        if (i + 32 * k + lane < i1) sum += piece(i + 32 * k + lane, raw[k], w);
      }
      const unsigned long long all = warp_sum(static_cast<unsigned long long>(__double2ll_rn(sum)));
      if (lane == n) run = all;
      mine += all;
    }
    if (ctas > 1 && round == 0) cluster_wait();
    tell_all(&s_part[round][part], mine, ctas);
    row_sync(ctas);
    total = before = 0;
    for (int i = lane; i < parts; i += 32) {
      const unsigned long long x = s_part[round][i];
      total += x;
      if (i < part) before += x;
    }
    total = warp_sum(total);
    before = warp_sum(before);
    if (total > 0 || !rest) break;
    rest = false;  // the draft's distribution was the target's, as far as weights tell
  }
  if (rank == 0) {  // (every CTA has read p.fails by now)
    if (threadIdx.x == 0) {
      p.accepted[b] = fail;
      p.fails[b] = 0;  // for the next call
      if (total == 0) p.next[b] = -1;
    }
    for (int i = threadIdx.x; i < fail; i += kVfThreads) {
      const int r = req.r0 + i, x = __ldg(p.tokens + r + 1);
      p.tokens_out[r] = x;
      if (p.logprobs)
        p.logprobs[r] = delta(clean(to_f32<T>(static_cast<const T*>(p.logits)[r * p.ld + x])), p.stats[r].xmax) - p.stats[r].log_z;
    }
  }
  if (total == 0) return;
  // ---- the token: warp, 32 pieces, piece, place
  const long long wanted = __double2ll_rd(__dmul_rn(static_cast<double>(__ldg(p.u_last + b)), __ull2double_rn(total)));
  const unsigned long long goal = min(wanted < 0 ? 0 : static_cast<unsigned long long>(wanted), total - 1);
  if (goal < before || goal >= before + mine) return;
  int at_run = 0;
  for (; at_run < 31; ++at_run) {
    const unsigned long long x = __shfl_sync(0xffffffffu, run, at_run);
    if (goal < before + x) break;
    before += x;
  }
#pragma unroll 1
  for (int i = i0 + at_run * 32 * kRun; i < i1; i += 32) {
    double w[kVec];
    const unsigned long long sum = i + lane < i1 ? static_cast<unsigned long long>(__double2ll_rn(piece(i + lane, fetch(i + lane), w))) : 0;
    unsigned long long upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + upto > goal);
    if (hit) {
      if (lane == __ffs(hit) - 1) {
        unsigned long long c = before + upto - sum;
        int token = -1;
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          c += static_cast<unsigned long long>(__double2ll_rn(w[e]));
          if (token < 0 && c > goal) token = src.index(i + lane) + e;
        }
        p.next[b] = p.tokens_out[row] = token;
        if (p.logprobs)
          p.logprobs[row] = delta(clean(to_f32<T>(src.row[token])), t.xmax) - t.log_z;
      }
      return;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
}

template <typename K>
cudaError_t launch_clusters(K kernel, const VerifyParams& p, long long jobs, int ctas, int threads,
                            bool dependent, cudaStream_t s) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(jobs * ctas));
  cfg.blockDim = dim3(threads);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dependent ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <typename T>
cudaError_t launch_t(VerifyParams p, int sms, cudaStream_t s) {
  constexpr int kVec = 16 / sizeof(T);
  const int pieces = (p.vocab + kVec - 1) / kVec;
  const int slots = 2 * sms;
  if (p.rows > 0) {
    // As many CTAs a row as fill the GPU, or as leave the rows that are walked at the
    // same time in L2 for their second pass: 260 rows of 51865 bf16 (31 MB at one CTA
    // each) take 47 us with one CTA, 51 with two, 65 with eight, 241 rows of 128000 f32
    // with the draft's 258, 245, 166 and, with eight (19 MB), 147.
    int ctas = 1;
    while (ctas < kVfCluster && pieces >= 2 * ctas * kVfThreads &&
           (2LL * p.rows * ctas <= slots || 16LL * pieces * slots / ctas > (32 << 20)))
      ctas *= 2;
    p.row_shift = 0;
    while (1 << p.row_shift < ctas) ++p.row_shift;
    const long long clusters = slots / ctas;  // (a place and request each, in turn: not all have a row)
    cudaError_t e = launch_clusters(verify_rows_kernel<T>, p, clusters, ctas, kVfThreads + 32, false, s);
    if (e != cudaSuccess) return e;
  }
  int ctas = 1;
  while (ctas < kVfCluster && pieces >= 2 * ctas * kVfThreads &&
         (2LL * p.batch * ctas <= slots || pieces >= 8 * ctas * kVfThreads))
    ctas *= 2;
  p.pick_ctas = ctas;
  return launch_clusters(verify_pick_kernel<T>, p, p.batch, ctas, kVfThreads, p.rows > 0, s);
}

}  // namespace

cudaError_t launch_verify(const VerifyParams& p, int sms, cudaStream_t s) {
  switch (p.dtype) {
    case 0: return launch_t<float>(p, sms, s);
    case 1: return launch_t<__nv_bfloat16>(p, sms, s);
    case 2: return launch_t<__half>(p, sms, s);
  }
  return cudaErrorInvalidValue;
}

}  // namespace ffai

// Attention of a chunk of new tokens over a paged KV cache, sequences with few
// query rows: single tokens, a handful of drafted ones.
//
// Sequence b brings n_b = cu_q[b + 1] - cu_q[b] tokens, the newest of the
// len_b = seq_lens[b] keys in its pages.  Query row (token i, head h) sees the
// keys j < len_b - (n_b - 1 - i), all len_b of them without the causal mask; query
// head h reads KV head h / G, G = heads / kv_heads:
//   s_j = scale q.k_j,  o = sum_j e^(s_j - m) v_j / l,  l = sum_j e^(s_j - m).
// A row that sees no key gives zeros and an lse of -inf.
//
// A unit is 16 R of a (sequence, KV head)'s n_b G rows; a team of W R warps (R = 1
// or 4) passes over its keys: R warps with 16 rows each (the matrix instruction's)
// share a ring of 32-key steps, W such groups take the steps in turn.  The steps of
// all units lie on one line (chunk.cuh), and team c takes the steps [c S, (c + 1) S):
// a long cache is read by many teams, whatever the batch, and no length passes
// through the host.  A unit that lies in one stretch is finished there; else each
// team leaves a partial result (running maximum, sum, unnormalised output), and
// the last of the unit's teams to come (a ticket) merges all of them, in their
// order on the line, so equal inputs give equal bits.  A team has at most two such
// partials, of its first and its last unit.
//
// Keys and values come by TMA, half a page a step, swizzled so that ldmatrix reads
// them without bank conflicts: as they are for the scores, transposed for the second
// product.  Only steps that some row does not see in full are masked.
//
// f32 queries with an f32 output: q and the weights are sums of two f16 or three bf16
// numbers, the products' terms smallest first, so that what is left of a rounding is
// 2^-22 or 2^-24 (of a weight in f16 2^-40 of the largest, where that is more): at 28 / 4
// heads and 6000 bf16 keys the error is 3.6e-7, that of a plain form in f32 1.1e-6 (two
// terms of the weights: 1.9e-6 and a tenth less time).
//
// Bound by HBM where the caches are long (192 units of one token behind up to 30000
// keys, f16: 831 MB in 136 us = 6.1 TB/s); by the latency of a team's first pages, its
// merge and uneven ends, and by a second pass over the keys of a pair with more than
// 16 rows, where they are short (64 requests of up to 8 tokens, 32 / 8 heads, up to 2000
// keys: 151 MB in 51 us = 3.0 TB/s; a short batch 10.5 us); by the products with several
// terms (36 sequences, 28 / 4 heads, f32: 466 us, tensor pipe 45 %, where the long chunks
// meet the shorter caches; 640 on average).
#include <atomic>

#include "chunk.cuh"

namespace ffai {

namespace {

constexpr int kCrWarps = 4;
constexpr int kCrThreads = kCrWarps * 32;
constexpr int kCrKeys = 32;  // keys per step of a group (half a page)
constexpr int kCrStage = 2 * kCrKeys * 128;  // bytes: keys, then values
constexpr int kCrStages = 8;                 // of a CTA, 2 R a ring
constexpr int kCrPitch = 68;  // floats per row of a state: m, l, -, -, o[64]
constexpr size_t kCrSmem = kCrStages * kCrStage;

struct CrBars {
  uint64_t full[kCrStages], empty[kCrStages];
  int abort_flag;
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}

// A warp's 16 rows: lane (g, t) = (lane / 4, lane % 4) holds rows g and g + 8;
// o[j][2 v + x] is row g + 8 v, head dim 8 j + 2 t + x.
struct RowState {
  float m[2], l[2];
  float o[8][4];
};
// The rows as A operands, in TERMS numbers of the cache's type that sum to them, and
// what their scores are to be multiplied by (scale log2 e).
template <int TERMS>
struct RowQ {
  uint32_t a[TERMS][4][4];
  float scale_log2[2];
};

// Rows row0 .. end - 1 of the sequence and KV head (16 at most).  Two f16 terms hold 22
// bits of a number only while the second is no subnormal, and nothing above 65504: a row
// is multiplied by the power of two that brings its largest element to 2^14 .. 2^15, so
// that what is left of an element is 2^-22 of it, or 2^-39 of the largest.
template <int TERMS>
__device__ __forceinline__ void load_rows(RowQ<TERMS>& q, RowState& st, const ChunkParams& p,
                                          const ChunkSeq& s, int kvh, int row0, int end) {
  const int lane = threadIdx.x % 32, g = lane >> 2, t = lane & 3;
  const int G = p.heads / p.kv_heads, f16 = p.kv_dtype == 2;
#pragma unroll
  for (int v = 0; v < 2; ++v) {
    const int row = row0 + g + 8 * v, i = row / G;
    const size_t off = static_cast<size_t>(s.t0 + i) * p.q_st + static_cast<size_t>(kvh * G + row - i * G) * p.q_sh;
    const auto pair = [&](int k, int x) {  // two head dims of an f32 row
      return row < end ? __ldg(reinterpret_cast<const float2*>(static_cast<const float*>(p.q) + off + 16 * k + 8 * x + 2 * t))
                       : make_float2(0.f, 0.f);
    };
    float up = 1.f, down = 1.f;
    if constexpr (TERMS == 2) {
      float most = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const float2 y = pair(k, x);
          most = max3f(most, fabsf(y.x), fabsf(y.y));
        }
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
      most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
      if (most > 0.f && most < INFINITY) {
        // (2^126 at most: both powers are normal numbers)
        const int e = min(14 - (static_cast<int>(__float_as_uint(most) >> 23) - 127), 126);
        up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
        down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
      }
    }
    q.scale_log2[v] = p.scale_log2 * down;
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        uint32_t w[TERMS] = {};
        if (p.q_dtype == 0) {  // f32 queries are rounded to the cache's type, and what that leaves again
          float2 y = pair(k, x);
          y.x *= up, y.y *= up;
#pragma unroll
          for (int n = 0; n < TERMS; ++n) {
            w[n] = f16 ? pack_f16x2(y.x, y.y) : pack_bf16x2(y.x, y.y);
            y.x -= lo_half(w[n], f16);
            y.y -= hi_half(w[n], f16);
          }
        } else if (row < end) {
          w[0] = __ldg(reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(p.q) + off + 16 * k + 8 * x + 2 * t));
        }
#pragma unroll
        for (int n = 0; n < TERMS; ++n) q.a[n][k][2 * x + v] = w[n];
      }
    st.m[v] = -INFINITY;
    st.l[v] = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) st.o[j][2 * v] = st.o[j][2 * v + 1] = 0.f;
  }
}

// Value rows lo .. hi - 1 of a step are seen by some rows and not by others, whose
// weight 0 a value that is not finite would turn into a NaN.  If there is one, it is
// added to the rows that see it, and true returned: the product of all then takes 0
// in its place.
template <int F16>
__device__ __forceinline__ bool guard_values(RowState& st, const uint8_t* v, const int (&see)[2], int lo, int hi) {
  const int lane = threadIdx.x % 32, t = lane & 3;
  bool any = false;
  for (int i = lo * 8 + lane; i < hi * 8; i += 32) {
    const uint4 x = *reinterpret_cast<const uint4*>(v + i * 16);
    any = any || (odd_halves<F16>(x.x) | odd_halves<F16>(x.y) | odd_halves<F16>(x.z) | odd_halves<F16>(x.w));
  }
  if (!__any_sync(0xffffffffu, any)) return false;
#pragma unroll 1
  for (int key = lo; key < hi; ++key)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t x = *reinterpret_cast<const uint32_t*>(v + key * 128 + ((j ^ (key & 7)) << 4) + 4 * t);
      const uint32_t odd = odd_halves<F16>(x);
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        if (key >= see[r]) continue;
        if (odd & 0xffffu) st.o[j][2 * r] += lo_half(x, F16);
        if (odd >> 16) st.o[j][2 * r + 1] += hi_half(x, F16);
      }
    }
  return true;
}

// One step: 32 keys and values at buf, row v of this lane sees the first see[v].
// tail: not all rows see all, but all the first lo, and the cache ends at key hi
// (behind which lies whatever was there).  With several terms the weights
// enter the second product in as many, and that product starts from zero, since
// the matrix instruction's sums are cut, not rounded.
template <int F16, int TERMS>
__device__ __forceinline__ void step32(RowState& st, const RowQ<TERMS>& q, const uint8_t* buf,
                                       const int (&see)[2], bool tail, int lo, int hi) {
  const int lane = threadIdx.x % 32, t = lane & 3;
  const uint32_t base = smem_u32(buf);
  // matrix m of a load: 8 rows of 16 bytes, lane 8 m + r gives row r's address
  const int row = lane & 7, mat = lane >> 3;
  float s[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {  // keys 8 i ..
    uint32_t k[2][4];            // head dims 32 h + 8 m ..
#pragma unroll
    for (int h = 0; h < 2; ++h)
      ldsm4(k[h], base + (8 * i + row) * 128 + (((4 * h + mat) ^ row) << 4));
#pragma unroll
    for (int e = 0; e < 4; ++e) s[i][e] = 0.f;
#pragma unroll
    for (int n = TERMS - 1; n >= 0; --n)  // the smallest first
#pragma unroll
      for (int x = 0; x < 4; ++x) mma16816<F16>(s[i], q.a[n][x], k[x / 2][2 * (x & 1)], k[x / 2][2 * (x & 1) + 1]);
  }
  if (tail) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        // a key the row does not see weighs nothing, whatever it holds
        if (8 * i + 2 * t + x >= see[0]) s[i][x] = -INFINITY;
        if (8 * i + 2 * t + x >= see[1]) s[i][2 + x] = -INFINITY;
      }
  }
  float mx[2];
#pragma unroll
  for (int r = 0; r < 2; ++r)
    mx[r] = max3f(fmaxf(s[0][2 * r], s[0][2 * r + 1]), max3f(s[1][2 * r], s[1][2 * r + 1], s[2][2 * r]),
                  max3f(s[2][2 * r + 1], s[3][2 * r], s[3][2 * r + 1]));
  // The maximum moves at once, so that the largest weight is 1, which has no rounding; in
  // f16 it is 2^15, so that none above 2^-29 of it is a subnormal number.
  constexpr float kLift = F16 ? 15.f : 0.f;
  if (__any_sync(0xffffffffu, fmaf(mx[0], q.scale_log2[0], -kLift) > st.m[0] ||
                                  fmaf(mx[1], q.scale_log2[1], -kLift) > st.m[1])) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
      const float m_new = fmaf(mx[r], q.scale_log2[r], -kLift);
      if (m_new > st.m[r]) {
        const float corr = ex2_approx(st.m[r] - m_new);
        st.m[r] = m_new;
        st.l[r] *= corr;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          st.o[j][2 * r] *= corr;
          st.o[j][2 * r + 1] *= corr;
        }
      }
    }
  }
  uint32_t p[2][4], rest[TERMS][2][4];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const float neg = st.m[r] == -INFINITY ? 0.f : -st.m[r];
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float p0 = ex2_approx(fmaf(s[i][2 * r], q.scale_log2[r], neg));
      const float p1 = ex2_approx(fmaf(s[i][2 * r + 1], q.scale_log2[r], neg));
      sum += p0 + p1;
      // the weights enter the second product in the cache's 16-bit type (off by
      // 2^-8 or 2^-11 of them at most, in f16 by 2^-40 of the largest where that is
      // more); their sum stays unrounded f32
      const uint32_t w = F16 ? pack_f16x2(p0, p1) : pack_bf16x2(p0, p1);
      p[i >> 1][(i & 1) * 2 + r] = w;
      if constexpr (TERMS > 1) {
        float r0 = p0 - lo_half(w, F16), r1 = p1 - hi_half(w, F16);
#pragma unroll
        for (int n = 1; n < TERMS; ++n) {
          const uint32_t x = F16 ? pack_f16x2(r0, r1) : pack_bf16x2(r0, r1);
          rest[n][i >> 1][(i & 1) * 2 + r] = x;
          r0 -= lo_half(x, F16), r1 -= hi_half(x, F16);
        }
      }
    }
    st.l[r] += sum;
  }
  bool fix = false;
  if (tail && lo < hi) fix = guard_values<F16>(st, buf + kCrKeys * 128, see, lo, hi);
  float part[8][4];
  if constexpr (TERMS > 1) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) part[j][e] = 0.f;
  }
  float(&o)[8][4] = TERMS > 1 ? part : st.o;
#pragma unroll
  for (int h = 0; h < 2; ++h)      // keys 16 h ..
#pragma unroll
    for (int c = 0; c < 4; ++c) {  // head dims 16 c ..
      uint32_t v[4];               // (keys, dims) + (0, 0), (8, 0), (0, 8), (8, 8)
      ldsm4_t(v, base + kCrKeys * 128 + (16 * h + 8 * (mat & 1) + row) * 128 + (((2 * c + (mat >> 1)) ^ row) << 4));
      if (tail) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = 16 * h + 8 * (e & 1) + 2 * t;
          v[e] &= (key < hi ? 0xffffu : 0u) | (key + 1 < hi ? 0xffff0000u : 0u);
          if (fix)
            v[e] &= ~(odd_halves<F16>(v[e]) & ((key >= lo ? 0xffffu : 0u) | (key + 1 >= lo ? 0xffff0000u : 0u)));
        }
      }
#pragma unroll
      for (int n = TERMS - 1; n > 0; --n) {
        mma16816<F16>(o[2 * c], rest[n][h], v[0], v[1]);
        mma16816<F16>(o[2 * c + 1], rest[n][h], v[2], v[3]);
      }
      mma16816<F16>(o[2 * c], p[h], v[0], v[1]);
      mma16816<F16>(o[2 * c + 1], p[h], v[2], v[3]);
    }
  if constexpr (TERMS > 1) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) st.o[j][e] += part[j][e];
  }
}

// The warps of a team meet.
template <int WARPS>
__device__ __forceinline__ void team_sync(int slot) {
  if constexpr (WARPS == 1)
    __syncwarp();
  else
    named_bar_sync(1 + slot, WARPS * 32);
}

// A warp's state of its rows into shared memory, kCrPitch floats a row; and a row of
// one, 8 head dims, into a merge.
__device__ __forceinline__ void put_state(const RowState& st, float* rows) {
  const int lane = threadIdx.x % 32, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    float l = st.l[r];
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    float* w = rows + (g + 8 * r) * kCrPitch;
    if (t == 0) *reinterpret_cast<float2*>(w) = make_float2(st.m[r], l);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      *reinterpret_cast<float2*>(w + 4 + 8 * j + 2 * t) = make_float2(st.o[j][2 * r], st.o[j][2 * r + 1]);
  }
}
__device__ __forceinline__ void add_state(Merged& acc, const float* x, int part) {
  acc.add(*reinterpret_cast<const float2*>(x), *reinterpret_cast<const float4*>(x + 4 + 8 * part),
          *reinterpret_cast<const float4*>(x + 8 + 8 * part));
}

template <int F16, int TERMS, int W, int R>
__global__ void __launch_bounds__(kCrThreads, TERMS > 1 ? 2 : 3)
    chunk_rows_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                      const __grid_constant__ ChunkParams p) {
  constexpr int kWarps = W * R, kTeams = kCrWarps / kWarps, kKeys = W * kCrKeys, kRows = R * kChRows;
  constexpr int kThreads = kWarps * 32, kDepth = 2 * R;
  // steps on their way: all of the ring's, or short of it what lets the first warp
  // of a group run ahead of the others
  constexpr int kAhead = R > 1 ? kDepth - 2 : kDepth;
  extern __shared__ __align__(1024) uint8_t cr_smem[];
  __shared__ CrBars bars;
  __shared__ Stretch s_start[kTeams];
  __shared__ int2 s_warp[kCrWarps];
  __shared__ int s_last[kTeams];
  if (smem_u32(cr_smem) % 1024 != 0) {  // the whole grid alike
    if (threadIdx.x == 0 && p.err) atomicOr(p.err, kErrBadArgs);
    return;
  }
  const int slot = threadIdx.x / kThreads, jt = threadIdx.x % kThreads;
  // this warp's share of the keys (a group with a ring), and of the rows
  const int split = jt / 32 / R, group = jt / 32 % R, lane = threadIdx.x % 32;
  const int stage0 = (slot * W + split) * kDepth;  // of the group's ring
  const int G = p.heads / p.kv_heads;
  uint64_t* full = bars.full + stage0;
  uint64_t* empty = bars.empty + stage0;
  uint8_t* ring = cr_smem + stage0 * kCrStage;
  // the states of a team's warps while they are joined, in the place of its rings
  float* states = reinterpret_cast<float*>(cr_smem + slot * W * kDepth * kCrStage);
  static_assert(kWarps * 16 * kCrPitch * sizeof(float) <= W * kDepth * kCrStage, "a team's rings");
  if (threadIdx.x == 0) {
    for (int i = 0; i < kCrStages; ++i) {
      mbar_init(&bars.full[i], 1);
      mbar_init(&bars.empty[i], R);
    }
    bars.abort_flag = 0;
    fence_mbar_init();
    prefetch_tensormap(&tmK);
    prefetch_tensormap(&tmV);
  }
  find_stretch<kRows, kKeys, kCrThreads, kTeams>(p, s_start, s_warp);
  Stretch w = s_start[slot];
  const int team = static_cast<int>(blockIdx.x) * kTeams + slot;
  bool bad = false;
  ChunkSeq s{};
  if (w.left > 0) s = chunk_seq(p, w.b, bad);
  uint32_t before = 0;  // steps of the group's ring before this unit
  bool ok = true;       // no wait ran out; else nothing more is sent for or computed
  while (w.left > 0) {
    // ---- the unit's rows, and the team's n of its steps
    const int row0 = w.m * kRows, rows = min(kRows, s.n * G - row0), end = row0 + rows;
    const int steps = unit_steps<kRows, kKeys>(p, s, G, w.m), n = min(w.left, steps - w.step);
    const int mine = row0 + group * kChRows;  // this warp's rows: mine .. end - 1, 16 at most
    const int k0 = w.step * kKeys + split * kCrKeys;  // the group's first key
    const int len = min(chunk_limit(p, s, (end - 1) / G), (w.step + n) * kKeys) - k0;
    const int count = len > 0 ? (len + kKeys - 1) / kKeys : 0;  // the group's steps
    const int* table = p.block_table + static_cast<size_t>(w.b) * p.max_pages;
    RowQ<TERMS> q;
    RowState st;
    load_rows(q, st, p, s, w.h, mine, end);
    int see[2], common = chunk_limit(p, s, min(mine, end - 1) / G) - k0, live = s.len - k0;
#pragma unroll
    for (int v = 0; v < 2; ++v)
      see[v] = chunk_limit(p, s, min(mine + (lane >> 2) + 8 * v, end - 1) / G) - k0;
    // The group's first warp sends for the copies: of kAhead steps before the first
    // one is taken, and behind each of one more, whose stage is that step's or an
    // older one's.
    int ids = 0, issued = 0;  // lanes hold the pages of 32 steps
#pragma unroll 1
    for (int i = -kAhead; i < count; ++i) {
      if (i >= 0 && ok) {
        const uint32_t it = before + i;
        const int at = it % kDepth;
        ok = __all_sync(0xffffffffu, mbar_wait(&full[at], (it / kDepth) & 1, &bars.abort_flag, p.err,
                                               kErrTimeoutConsumer));
        if (common >= kCrKeys)
          step32<F16, TERMS>(st, q, ring + at * kCrStage, see, false, kCrKeys, kCrKeys);
        else
          step32<F16, TERMS>(st, q, ring + at * kCrStage, see, true, max(common, 0), min(live, kCrKeys));
        see[0] -= kKeys, see[1] -= kKeys, common -= kKeys, live -= kKeys;
        __syncwarp();
        if (R > 1) mbar_arrive_w(&empty[at]);
      }
      if (group == 0 && issued < count && ok) {
        if (issued % 32 == 0) {
          ids = issued + lane < count ? __ldg(table + (k0 + (issued + lane) * kKeys) / kPageKeys) : 0;
          if (ids < 0 || ids >= p.num_pages) {  // reported; page 0 is read in its place
            if (p.err) atomicOr(p.err, kErrBadArgs);
            ids = 0;
          }
        }
        const uint32_t it = before + issued;
        const int at = it % kDepth, page = __shfl_sync(0xffffffffu, ids, issued % 32);
        if (R > 1 && it >= kDepth) {
          ok = __all_sync(0xffffffffu, mbar_wait(&empty[at], ((it / kDepth) - 1) & 1, &bars.abort_flag,
                                                 p.err, kErrTimeoutProducer));
          if (!ok) continue;
        }
        const int half = (k0 + issued * kKeys) % kPageKeys;
        __syncwarp();
        mbar_arrive_expect_tx_w(&full[at], kCrStage);
        tma_load_3d_w(ring + at * kCrStage, &tmK, &full[at], 0, half, page * p.kv_heads + w.h);
        tma_load_3d_w(ring + at * kCrStage + kCrStage / 2, &tmV, &full[at], 0, half, page * p.kv_heads + w.h);
        ++issued;
      }
    }
    if (issued > 0 && !ok) {  // every copy lands before its place is used again
      int none = 0;
      for (uint32_t st0 = 0, it = before + issued; st0 < kDepth && st0 < it; ++st0)
        mbar_wait(&full[st0], ((it - 1 - st0) / kDepth) & 1, &none, p.err, kErrTimeoutDrain);
    }
    before += count;
    team_sync<kWarps>(slot);  // the rings are done with: the warps' states take their place
    put_state(st, states + (split * R + group) * 16 * kCrPitch);
    team_sync<kWarps>(slot);
    // ---- the states joined: 8 threads a row, 8 head dims each
    const int c0 = w.unit0 / w.share;
    const UnitParts u{c0, min((w.unit0 + steps - 1) / w.share, static_cast<int>(gridDim.x) * kTeams - 1),
                      kRows, 0, row0, rows, s.t0, w.h};
    const bool whole = n == steps;
#pragma unroll 1
    for (int row = jt / 8; row < rows; row += kThreads / 8) {
      const int part = jt % 8;
      Merged acc{-INFINITY, 0.f, {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}};
#pragma unroll 1
      for (int x = 0; x < W; ++x) add_state(acc, states + ((x * R + row / 16) * 16 + row % 16) * kCrPitch, part);
      if (whole) {
        store_unit_row(p, u, acc, row, part);
      } else {
        const size_t at = part_row(u, team, row);
        float4* o = reinterpret_cast<float4*>(p.part_o + at * 64 + 8 * part);
        __stcg(o, make_float4(acc.o[0], acc.o[1], acc.o[2], acc.o[3]));
        __stcg(o + 1, make_float4(acc.o[4], acc.o[5], acc.o[6], acc.o[7]));
        if (part == 0) __stcg(reinterpret_cast<float2*>(p.part_ml + 2 * at), make_float2(acc.m, acc.l));
      }
    }
    if (!whole) {
      // ---- a part of the unit: the last of its teams merges all, in their order
      __threadfence();
      team_sync<kWarps>(slot);
      if (jt == 0) {
        const unsigned others = static_cast<unsigned>(u.c1 - u.c0);
        s_last[slot] = atomicInc(p.tickets + u.c0, others) == others;
        __threadfence();
      }
      team_sync<kWarps>(slot);
      if (s_last[slot]) merge_rows<kThreads>(p, u, jt);
    }
    // the states are read, and by ordinary loads: the rings may be filled again
    fence_proxy_async_smem();
    team_sync<kWarps>(slot);
    // ---- on to the next unit
    w.left -= n;
    if (w.left > 0) {
      w.step = 0;
      w.unit0 += steps;
      if (++w.m == chunk_units<kRows>(s, G)) {
        w.m = 0;
        if (++w.h == p.kv_heads) {
          w.h = 0;
          s.n = 0;
          while (s.n == 0 && ++w.b < p.batch) s = chunk_seq(p, w.b, bad);
          if (s.n == 0) break;
        }
      }
    }
  }
}

template <int F16, int TERMS>
cudaError_t launch_w(const CUtensorMap& tmK, const CUtensorMap& tmV, const ChunkParams& p, int grid,
                     int w, int r, cudaStream_t s) {
  // (64 rows share their keys where the products are many; else two tiles of 16 that
  // read the keys twice take less: 64 x 32 tokens, 32 / 8 heads, 2000 keys 107 and 116 us)
  const int which = TERMS > 1 && r == 4 ? 0 : w == 1 ? 1 : w == 2 ? 2 : 3;
  auto kern = which == 0   ? chunk_rows_kernel<F16, TERMS, 1, (TERMS > 1 ? 4 : 1)>
              : which == 1 ? chunk_rows_kernel<F16, TERMS, 1, 1>
              : which == 2 ? chunk_rows_kernel<F16, TERMS, 2, 1>
                           : chunk_rows_kernel<F16, TERMS, 4, 1>;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  static std::atomic<bool> configured[4][64];
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[which][dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kCrSmem));
    if (e != cudaSuccess) return e;
    configured[which][dev].store(true, std::memory_order_release);
  }
  kern<<<grid, kCrThreads, kCrSmem, s>>>(tmK, tmV, p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t launch_chunk_rows(const CUtensorMap& tmK, const CUtensorMap& tmV, const ChunkParams& p,
                              int grid, int w, int r, cudaStream_t s) {
  // f16: two terms hold 22 of 24 bits, bf16: three hold all
  if (p.kv_dtype == 2)
    return p.precise ? launch_w<1, 2>(tmK, tmV, p, grid, w, r, s) : launch_w<1, 1>(tmK, tmV, p, grid, w, r, s);
  return p.precise ? launch_w<0, 3>(tmK, tmV, p, grid, w, r, s) : launch_w<0, 1>(tmK, tmV, p, grid, w, r, s);
}

}  // namespace ffai

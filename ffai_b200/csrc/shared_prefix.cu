// Attention of a batch whose sequences share long prefixes, over a paged KV
// cache: group g of consecutive sequences shares prefix_lens[g] keys; sequence
// b adds seq_lens[b] keys of its own.  Query row (b, i, h), i < q_len, sees
// the whole prefix of its group and its own keys j < seq_lens[b] - (q_len - 1
// - i), i.e. up to its own position; query head h reads KV head h / G, G =
// heads / kv_heads:
//   s_j = scale q.k_j,  o = sum_j e^(s_j - m) v_j / l,  l = sum_j e^(s_j - m).
// A row that sees no key gives zeros and an lse of -inf.
//
// The R = q_len * G rows of one (sequence, KV head) are served together, in
// tiles of 16 (the matrix instruction's rows).  A tile is a job for W = 1, 2 or
// 4 warps of a CTA's four: as few as still fill the GPU, because a job's fixed
// costs (first loads, merge) are paid by all its warps.  Each takes every W-th
// step of 32 keys with a softmax state of its own, and the warps merge at the
// end.  A warp copies its steps' key and value rows two steps
// ahead into shared memory of its own (no barrier), and takes its operands
// from there in 16-byte pieces: the products' inner order is free, so it is
// chosen such that a lane's operands are whole pieces of the rows.
//
// The prefixes' share comes from one of three places, by size (the rule, with
// both sides' times, stands in ffai_attn_shared_prefix):
//  * this kernel walks them too, each sequence for itself (short prefixes: the
//    repeated reads hit L2 and a second launch costs more);
//  * prefix_rows_kernel, the same walk over a group's rows, when a group has few
//    rows: its partial results are merged here;
//  * prefix_tc_kernel (prefix_tc.cu), on tcgen05, otherwise.  Its partial results
//    are merged here too; but where the sequences' own keys are a sizeable share,
//    it leaves some SMs free, and own_rows_kernel attends those keys there
//    meanwhile (jobs from a queue, so that it spreads over all SMs once the prefix
//    is done), and merge_rows_kernel joins both.
//
// Bounds.  Of the first and second: the reads (own keys and prefix once) from
// HBM, and below some 10 MB the chain of dependent loads: lengths, page ids,
// keys, values, merge.  Of the third: the exponentials and the moves between
// tensor memory and registers.  Device time, bf16 or f16 caches, on one B200:
//   5 sequences, 12 heads, 224 + up to 224 keys            6.9 us (2.4 MB)
//   12 groups of 5, 20 heads, up to 1500 + up to 448 keys 35 us   (145 MB, 4.1 TB/s)
//   64 sequences, 32 / 8 heads, 8200 + up to 1000 keys    32 us   (82 MB)
//   96 in 3 groups, 4 queries, 32768 + up to 700 keys      163 us (89 GFLOP, 0.55 PFLOP/s)
#include <algorithm>

#include "shared_prefix.cuh"

namespace ffai {

namespace {

constexpr int kSpWarps = 4;
constexpr int kSpThreads = kSpWarps * 32;
constexpr int kSpKeys = 32;  // keys per warp step (divides a page)

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

// Softmax state of a warp's 16 rows: lane (g, t) = (lane / 4, lane % 4) holds
// rows g and g + 8; o[j][2 v + w] is row g + 8 v, head dim 16 t + 8 w + j.
struct RowState {
  float m[2], l[2];
  float o[8][4];
};

// The 16 query rows as A operands: k-step s (16 of the 64 head dims) holds
// dims 32 (s / 2) + 8 t + 4 (s % 2) + {0, 1} and + {2, 3}, so that the lane's
// part of a key row is the two 16-byte pieces at dims 8 t and 32 + 8 t.
struct RowQ {
  uint32_t a[4][4];
};

// A warp's copies: kSpDepth steps of 32 key rows, then 32 value rows.
constexpr int kSpDepth = 2;
constexpr int kSpStep = 2 * kSpKeys * 128;  // bytes
constexpr int kSpRing = kSpDepth * kSpStep;

// Piece c (16 bytes) of row `key` sits where the eight lanes that read together
// meet eight different banks: key rows are read by row pairs, four pieces each;
// value rows by the rows 0, 2, 4, 6 (or 1, 3, 5, 7), two pieces each.
__device__ __forceinline__ int k_piece(int key, int c) {
  return key * 128 + ((c ^ ((key & 1) << 2)) << 4);
}
__device__ __forceinline__ int v_piece(int key, int c) {
  return kSpKeys * 128 + key * 128 + ((c ^ (((key >> 1) & 3) << 1)) << 4);
}

// Start copying one step (32 keys of one page at kp / vp, `live` of them to be
// read, zeros behind them) into buf.
__device__ __forceinline__ void fetch32(uint8_t* buf, const uint16_t* kp, const uint16_t* vp, int live) {
  const int lane = threadIdx.x % 32, c = lane & 7;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int key = 4 * i + (lane >> 3);
    const bool have = key < live;
    const int off = have ? key * 64 + c * 8 : 0;
    cp_async16(buf + k_piece(key, c), kp + off, have);
    cp_async16(buf + v_piece(key, c), vp + off, have);
  }
}

// Value rows lo .. hi of a step are seen by some rows and not by others, whose
// weight 0 a value that is not finite would turn into a NaN.  If there is one,
// it is added to the rows that see it, and is 0 for the product of all.
template <int F16>
__device__ __forceinline__ void guard_values(RowState& st, const uint32_t (&p)[2][4], uint8_t* buf,
                                             const int (&see)[2], int lo, int hi) {
  constexpr uint32_t kExp = F16 ? 0x7c00u : 0x7f80u;
  const int lane = threadIdx.x % 32, t = lane & 3;
  const auto bad = [](uint32_t x) {  // which halves are infinite or NaN
    return ((x & kExp) == kExp ? 0xffffu : 0u) | ((x >> 16 & kExp) == kExp ? 0xffff0000u : 0u);
  };
  bool any = false;
  for (int i = lo * 8 + lane; i < hi * 8; i += 32) {
    const uint4 v = *reinterpret_cast<const uint4*>(buf + v_piece(i >> 3, i & 7));
    any = any || (bad(v.x) | bad(v.y) | bad(v.z) | bad(v.w));
  }
  if (!__any_sync(0xffffffffu, any)) return;
#pragma unroll 1
  for (int key = lo; key < hi; ++key) {
    const int n = key >> 3;  // the weights' n-tile, and the lane that holds them
    uint32_t w[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      w[r] = n == 0 ? p[0][r] : n == 1 ? p[0][2 + r] : n == 2 ? p[1][r] : p[1][2 + r];
      w[r] = __shfl_sync(0xffffffffu, w[r], (lane & ~3) | ((key & 7) >> 1)) >> 16 * (key & 1);
    }
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const uint4 v = *reinterpret_cast<const uint4*>(buf + v_piece(key, 2 * t + x));
      const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (!(bad(u[j / 2]) >> 16 * (j & 1) & 1u)) continue;
        const float f = j & 1 ? hi_half(u[j / 2], F16) : lo_half(u[j / 2], F16);
#pragma unroll
        for (int r = 0; r < 2; ++r)
          if (key < see[r]) st.o[j][2 * r + x] = fmaf(lo_half(w[r], F16), f, st.o[j][2 * r + x]);
      }
    }
  }
  __syncwarp();
  for (int i = lo * 8 + lane; i < hi * 8; i += 32) {
    uint4* at = reinterpret_cast<uint4*>(buf + v_piece(i >> 3, i & 7));
    const uint4 v = *at;
    *at = make_uint4(v.x & ~bad(v.x), v.y & ~bad(v.y), v.z & ~bad(v.z), v.w & ~bad(v.w));
  }
  __syncwarp();
}

// One step from buf; row v of this lane sees the first `see[v]` of its keys.  TAIL:
// not all rows alike, but all the first lo, and none those from hi on.
template <int F16, bool TAIL>
__device__ __forceinline__ void step32(RowState& st, const RowQ& q, uint8_t* buf,
                                       const int (&see)[2], int lo, int hi, float scale_log2) {
  const int lane = threadIdx.x % 32, g = lane >> 2, t = lane & 3;
  uint4 k[4][2];  // n-tile i: key 8 i + g
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    k[i][0] = *reinterpret_cast<const uint4*>(buf + k_piece(8 * i + g, t));
    k[i][1] = *reinterpret_cast<const uint4*>(buf + k_piece(8 * i + g, 4 + t));
  }
  float s[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int e = 0; e < 4; ++e) s[i][e] = 0.f;
    mma16816<F16>(s[i], q.a[0], k[i][0].x, k[i][0].y);
    mma16816<F16>(s[i], q.a[1], k[i][0].z, k[i][0].w);
    mma16816<F16>(s[i], q.a[2], k[i][1].x, k[i][1].y);
    mma16816<F16>(s[i], q.a[3], k[i][1].z, k[i][1].w);
  }
  uint32_t p[2][4];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        // a key the row does not see weighs nothing, whatever it holds
        const float x = 8 * i + 2 * t + e < see[r] ? s[i][2 * r + e] * scale_log2 : -INFINITY;
        s[i][2 * r + e] = x;
        mx = fmaxf(mx, x);
      }
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    const float m_new = fmaxf(st.m[r], mx);
    const float base = m_new == -INFINITY ? 0.f : m_new;
    const float corr = ex2_approx(st.m[r] - base);
    st.m[r] = m_new;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float p0 = ex2_approx(s[i][2 * r] - base), p1 = ex2_approx(s[i][2 * r + 1] - base);
      sum += p0 + p1;
      // the weights enter the second product in the cache's 16-bit type (at
      // most 1, relative error 2^-9 or 2^-12); their sum stays unrounded f32
      p[i >> 1][(i & 1) * 2 + r] = F16 ? pack_f16x2(p0, p1) : pack_bf16x2(p0, p1);
    }
    st.l[r] = fmaf(st.l[r], corr, sum);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      st.o[j][2 * r] *= corr;
      st.o[j][2 * r + 1] *= corr;
    }
  }
  if constexpr (TAIL)
    if (lo < hi) guard_values<F16>(st, p, buf, see, lo, hi);
  uint4 v[2][4];  // 16-key half h: keys 16 h + 2 t + {0, 1, 8, 9}, dims 8 g ..
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      v[h][e] = *reinterpret_cast<const uint4*>(
          buf + v_piece(16 * h + 2 * t + (e & 1) + 8 * (e >> 1), g));
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t e0[4] = {v[h][0].x, v[h][0].y, v[h][0].z, v[h][0].w};
    const uint32_t e1[4] = {v[h][1].x, v[h][1].y, v[h][1].z, v[h][1].w};
    const uint32_t e2[4] = {v[h][2].x, v[h][2].y, v[h][2].z, v[h][2].w};
    const uint32_t e3[4] = {v[h][3].x, v[h][3].y, v[h][3].z, v[h][3].w};
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      mma16816<F16>(st.o[2 * c], p[h], __byte_perm(e0[c], e1[c], 0x5410),
                    __byte_perm(e2[c], e3[c], 0x5410));
      mma16816<F16>(st.o[2 * c + 1], p[h], __byte_perm(e0[c], e1[c], 0x7632),
                    __byte_perm(e2[c], e3[c], 0x7632));
    }
  }
}

__device__ __forceinline__ uint32_t q_pair(const SharedParams& p, const void* row, int dim) {
  if (p.q_dtype == 0) {  // f32 queries are rounded to the cache's type
    const float2 x = __ldg(reinterpret_cast<const float2*>(static_cast<const float*>(row) + dim));
    return p.kv_dtype == 2 ? pack_f16x2(x.x, x.y) : pack_bf16x2(x.x, x.y);
  }
  return __ldg(reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(row) + dim));
}

__device__ __forceinline__ const void* q_row(const SharedParams& p, int b, int tok, int h) {
  const size_t off = static_cast<size_t>(b) * p.q_sb + static_cast<size_t>(tok) * p.q_st +
                     static_cast<size_t>(h) * p.q_sh;
  return static_cast<const uint8_t*>(p.q) + off * (p.q_dtype == 0 ? 4 : 2);
}

// The group whose sequences hold b, or -1 (a whole warp): starts[] rises, so
// it is the last group that starts at or before b, if b is before its end.  If
// it does not rise within the batch, no sequence has a group.
__device__ __forceinline__ int group_of(const SharedParams& p, int b) {
  const int lane = threadIdx.x % 32;
  int n = 0;  // groups that start at or before b
  bool bad = false;
  for (int base = 0; base < p.groups; base += 32) {
    const int g = base + lane;
    if (g < p.groups) bad = bad || !group_ok(p, g, false);
    const bool in = g < p.groups && __ldg(p.group_starts + g) <= b;
    n += __popc(__ballot_sync(0xffffffffu, in));
  }
  if (__any_sync(0xffffffffu, bad)) return -1;
  return n > 0 && b < __ldg(p.group_starts + n) ? n - 1 : -1;
}

// The same for a lane by itself.
__device__ __forceinline__ int group_of_lane(const SharedParams& p, int b) {
  int lo = 0, hi = p.groups;  // groups below lo start at or before b, those from hi on behind it
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(p.group_starts + mid) <= b)
      lo = mid + 1;
    else
      hi = mid;
  }
  return lo > 0 && __ldg(p.group_starts + lo - 1) <= b && b < __ldg(p.group_starts + lo) ? lo - 1 : -1;
}

// Page ids of a warp's next 32 steps, one per lane: warp w of the job's W takes
// the steps w, w + W, ... of 32 keys, and `first` counts the warp's own.
template <int W>
__device__ __forceinline__ int step_page(const int* table, int pages, int warp, int first) {
  const int page = (warp + W * (first + static_cast<int>(threadIdx.x % 32))) / 2;
  return page < pages ? __ldg(table + page) : -1;
}

// Walk `len` keys of a list of pages (TAIL: the first `common` of which all rows
// see; else all rows see all).  `ids` holds the first 32 steps' page ids, loaded ahead (the table does not depend on the lengths).  `ring`: this
// warp's kSpRing bytes, not in use.
template <int F16, int W, bool TAIL>
__device__ __forceinline__ void walk(RowState& st, const RowQ& q, const SharedParams& p, int kvh,
                                     const int* table, int pages, int ids, int len, int common,
                                     const int (&see)[2], int warp, uint8_t* ring) {
  const uint16_t* kpool = static_cast<const uint16_t*>(p.k_pool);
  const uint16_t* vpool = static_cast<const uint16_t*>(p.v_pool);
  constexpr int kStride = W * kSpKeys;
  const int steps = (len - warp * kSpKeys + kStride - 1) / kStride;
  int first = 0;  // ids are those of steps first .. first + 31
  const auto fetch = [&](int i) {
    if (i < steps) {
      if (i - first == 32) {
        first = i;
        ids = step_page<W>(table, pages, warp, first);
      }
      const int k0 = i * kStride + warp * kSpKeys;
      const int page = __shfl_sync(0xffffffffu, ids, i - first);
      const bool ok = page >= 0 && page < p.num_pages;
      if (!ok && p.err && threadIdx.x % 32 == 0) atomicOr(p.err, kErrBadArgs);  // not read
      const size_t off = ((static_cast<size_t>(ok ? page : 0) * p.kv_heads + kvh) * kPageKeys +
                          k0 % kPageKeys) * 64;
      fetch32(ring + i % kSpDepth * kSpStep, kpool + off, vpool + off, ok ? len - k0 : 0);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kSpDepth; ++i) fetch(i);
#pragma unroll 1
  for (int i = 0; i < steps; ++i) {
    cp_async_wait<kSpDepth - 1>();
    __syncwarp();
    const int k0 = i * kStride + warp * kSpKeys;
    const int rel[2] = {see[0] - k0, see[1] - k0};
    step32<F16, TAIL>(st, q, ring + i % kSpDepth * kSpStep, rel, max(common - k0, 0),
                min(len - k0, kSpKeys), p.scale_log2);
    __syncwarp();
    fetch(i + kSpDepth);
  }
}

// The 16 query rows of a tile as operands: row r is token tok[r] (of a lane's
// two rows; -1: none) of sequence b[r], head h[r].
__device__ __forceinline__ void load_rows(RowQ& q, RowState& st, const SharedParams& p,
                                          const int (&b)[2], const int (&tok)[2], const int (&h)[2]) {
  const int t = threadIdx.x & 3;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const void* src = tok[r] >= 0 ? q_row(p, b[r], tok[r], h[r]) : nullptr;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int dim = 32 * (s / 2) + 8 * t + 4 * (s % 2);
      q.a[s][r] = src ? q_pair(p, src, dim) : 0u;
      q.a[s][2 + r] = src ? q_pair(p, src, dim + 2) : 0u;
    }
    st.m[r] = -INFINITY;
    st.l[r] = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) st.o[j][2 * r] = st.o[j][2 * r + 1] = 0.f;
  }
}

constexpr int kSpStage = 8;  // partials a thread stages at a time

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

// Shared memory of a job: its warps' rings while they walk; then their states,
// the staged partials, and the threads' merges.
constexpr int kSpPitch = 68;  // floats per state row: m, l, -, -, o[64]
template <int THREADS>
struct alignas(16) Staging {
  float o[kSpStage][THREADS][8];
  float ml[kSpStage][THREADS][2];
};
template <int W>
struct RowsMerge {
  float state[W][16][kSpPitch];
  Staging<W * 32> stage;
  float merged[W * 32][10];
};
static_assert(sizeof(RowsMerge<1>) <= kSpRing && sizeof(RowsMerge<4>) <= 4 * kSpRing, "a job's rings");
constexpr size_t kSpSmem = kSpWarps * kSpRing;
static_assert(kSpSmem <= 75 * 1024, "three CTAs per SM");

// The warps of a job meet.
template <int W>
__device__ __forceinline__ void job_sync(int slot) {
  if constexpr (W == 1)
    __syncwarp();
  else
    named_bar_sync(1 + slot, W * 32);
}

// The warps' states of the tile into shared memory.
template <int W>
__device__ __forceinline__ void put_state(const RowState& st, RowsMerge<W>& m, int warp) {
  const int lane = threadIdx.x % 32, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    float l = st.l[r];
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    float* w = m.state[warp][g + 8 * r];
    if (t == 0) *reinterpret_cast<float2*>(w) = make_float2(st.m[r], l);
    float4* o = reinterpret_cast<float4*>(w + 4 + 16 * t);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      o[e] = make_float4(st.o[4 * e][2 * r], st.o[4 * e + 1][2 * r], st.o[4 * e + 2][2 * r],
                         st.o[4 * e + 3][2 * r]);
      o[2 + e] = make_float4(st.o[4 * e][2 * r + 1], st.o[4 * e + 1][2 * r + 1],
                             st.o[4 * e + 2][2 * r + 1], st.o[4 * e + 3][2 * r + 1]);
    }
  }
}
template <int W>
__device__ __forceinline__ void add_state(Merged& acc, const RowsMerge<W>& m, int w, int row, int part) {
  const float* x = m.state[w][row];
  acc.add(*reinterpret_cast<const float2*>(x), *reinterpret_cast<const float4*>(x + 4 + 8 * part),
          *reinterpret_cast<const float4*>(x + 8 + 8 * part));
}

// Copy `n` partials of a row (rows at, at + step, ..  of part_o) into this
// thread's places of the staging buffer, a few at a time so that their latencies
// overlap, and fold them into acc.  A thread reads its own pieces: no barrier.
template <int THREADS>
__device__ __forceinline__ void fold_run(Merged& acc, Staging<THREADS>& sm, const SharedParams& p,
                                         size_t at, size_t step, int n, int part, int jt) {
  for (int base = 0; base < n; base += kSpStage) {
    const int m = min(n - base, kSpStage);
#pragma unroll 1
    for (int i = 0; i < m; ++i, at += step) {
      cp_async16(sm.o[i][jt], p.part_o + at * 64 + 8 * part, true);
      cp_async16(sm.o[i][jt] + 4, p.part_o + at * 64 + 8 * part + 4, true);
      cp_async8(sm.ml[i][jt], p.part_ml + 2 * at);
    }
    cp_async_wait_all();
#pragma unroll 1
    for (int i = 0; i < m; ++i)
      acc.add(*reinterpret_cast<const float2*>(sm.ml[i][jt]),
              *reinterpret_cast<const float4*>(sm.o[i][jt]),
              *reinterpret_cast<const float4*>(sm.o[i][jt] + 4));
  }
}

// The n partials from `slot` on, if the workspace holds them.  It always does
// (its size is a bound on the plan's slots), unless the lengths or starts were
// written between the prefix kernel's look at them and this one.
__device__ __forceinline__ int in_slots(const SharedParams& p, int slot, int n) {
  if (slot >= 0 && n <= p.part_slots - slot) return n;
  if (p.err) atomicOr(p.err, kErrNoSlot);
  return 0;
}

// The prefix kernel's partials of row `row` of sequence b's R rows of a KV head,
// folded into `acc` in the order of the line: copy k of `copies` takes every
// copies-th.
template <int THREADS>
__device__ __forceinline__ void fold_partials(Merged& acc, Staging<THREADS>& sm, const SharedParams& p,
                                              int group, int b, int kvh, int row, int R, int copy,
                                              int copies, int part, int jt) {
  const GroupDims d = group_dims(p, group);
  const int rg = (b - d.b0) * R + row;
  // the plan was written by the preceding kernel, which may have run beside this one
  const int plan = __ldcg(p.part_plan);
  if (plan == kBadPlan) return;
  if (p.splits > 0) {  // prefix_rows_kernel's: one per split that has pages
    const int pages = (d.plen + kPageKeys - 1) / kPageKeys;
    if (pages == 0) return;
    const int tiles = (d.rows + 15) / 16, per = (pages + p.splits - 1) / p.splits;
    const int slot = (__ldcg(p.part_plan + 1 + group) + kvh * tiles + rg / 16) * p.splits;
    const int n = in_slots(p, slot, (pages + per - 1) / per);
    fold_run(acc, sm, p, static_cast<size_t>(slot + copy) * 16 + rg % 16,
             static_cast<size_t>(copies) * 16, (n - copy + copies - 1) / copies, part, jt);
    return;
  }
  // prefix_tc_kernel's: segments of the line, each one per CTA that has a share of it
  const int share = abs(plan), lin0 = __ldcg(p.part_plan + 1 + 2 * group),
            seg0 = __ldcg(p.part_plan + 2 + 2 * group);
  if (d.nb == 0 || in_slots(p, 0, share > 0 ? 1 : INT_MAX) == 0) return;
  const int cl = chunk_blocks(d, share), chunks = (d.nb + cl - 1) / cl;
  const int head0 = lin0 + kvh * line_steps(d, share, plan < 0), m = rg / kPxRows;
  int skip = copy;  // partials to pass over before this copy's next
#pragma unroll 1
  for (int q = 0; q < chunks; ++q) {
    const int len = min(cl, d.nb - q * cl);
    const int l0 = head0 + head_steps(d, q * cl) + m * len;
    const int seg = seg0 + (kvh * chunks + q) * d.mu + m;
    const int c0 = l0 / share, c1 = (l0 + unit_steps(d, m, len) - 1) / share;
    const int n = in_slots(p, c0 + seg, c1 - c0 + 1);
    fold_run(acc, sm, p, static_cast<size_t>(c0 + seg + skip) * kPxRows + rg % kPxRows,
             static_cast<size_t>(copies) * kPxRows, (n - skip + copies - 1) / copies, part, jt);
    // the next chunk's go on being dealt where this one's stopped (copies: a power of two)
    skip = (skip - n) & (copies - 1);
  }
}

// Store one row's result, 8 head dims a thread.
__device__ __forceinline__ void store_row(const SharedParams& p, Merged& acc, int b, int rr, int kvh,
                                          int G, int part) {
  const int ti = rr / G, h = kvh * G + rr % G;
  const size_t at = static_cast<size_t>(b) * p.o_sb + static_cast<size_t>(ti) * p.o_st +
                    static_cast<size_t>(h) * p.o_sh + 8 * part;
  const float inv = acc.l == 0.f ? 0.f : 1.f / acc.l;  // 0: the row saw no key
#pragma unroll
  for (int e = 0; e < 8; ++e) acc.o[e] *= inv;
  if (p.out_dtype == 0) {
    float4* o = reinterpret_cast<float4*>(static_cast<float*>(p.out) + at);
    o[0] = make_float4(acc.o[0], acc.o[1], acc.o[2], acc.o[3]);
    o[1] = make_float4(acc.o[4], acc.o[5], acc.o[6], acc.o[7]);
  } else {
    uint4 x;
    if (p.out_dtype == 1)
      x = make_uint4(pack_bf16x2(acc.o[0], acc.o[1]), pack_bf16x2(acc.o[2], acc.o[3]),
                     pack_bf16x2(acc.o[4], acc.o[5]), pack_bf16x2(acc.o[6], acc.o[7]));
    else
      x = make_uint4(pack_f16x2(acc.o[0], acc.o[1]), pack_f16x2(acc.o[2], acc.o[3]),
                     pack_f16x2(acc.o[4], acc.o[5]), pack_f16x2(acc.o[6], acc.o[7]));
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.out) + at) = x;
  }
  if (p.lse && part == 0)
    p.lse[static_cast<size_t>(b) * p.lse_sb + static_cast<size_t>(ti) * p.lse_st +
          static_cast<size_t>(h) * p.lse_sh] =
        acc.l == 0.f ? -INFINITY : (acc.m + log2f(acc.l)) * 0.69314718055994530942f;
}

template <int F16, int W, bool TAIL>
__global__ void __launch_bounds__(kSpThreads, 3) shared_rows_kernel(SharedParams p, int jobs) {
  extern __shared__ __align__(128) uint8_t sp_smem[];
  const int warp = threadIdx.x / 32 % W, slot = threadIdx.x / 32 / W, jt = threadIdx.x % (W * 32);
  const int lane = threadIdx.x % 32, g = lane >> 2;
  const int G = p.heads / p.kv_heads, R = p.q_len * G;
  const int tiles = (R + 15) / 16;
  const int id = static_cast<int>(blockIdx.x) * (kSpWarps / W) + slot, job = id / tiles;
  if (id >= jobs) return;
  uint8_t* ring = sp_smem + threadIdx.x / 32 * kSpRing;
  RowsMerge<W>& sm = *reinterpret_cast<RowsMerge<W>*>(sp_smem + slot * W * kSpRing);
  const int tile = id - job * tiles;
  const int b = job / p.kv_heads, kvh = job - b * p.kv_heads;

  const int* table = p.block_table + static_cast<size_t>(b) * p.max_pages;
  const int ids = step_page<W>(table, p.max_pages, warp, 0);
  int len = __ldg(p.seq_lens + b);
  RowQ q;
  RowState st;
  int tok[2], head[2];
  const int seq[2] = {b, b};
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = tile * 16 + g + 8 * r;
    tok[r] = row < R ? row / G : -1;
    head[r] = kvh * G + row % G;
  }
  load_rows(q, st, p, seq, tok, head);
  if (len < 0 || len > p.max_pages * kPageKeys) {
    if (p.err && jt == 0) atomicOr(p.err, kErrBadArgs);
    len = min(max(len, 0), p.max_pages * kPageKeys);
  }
  const int see[2] = {tok[0] < 0 ? 0 : max(0, len - (p.q_len - 1 - tok[0])),
                      tok[1] < 0 ? 0 : max(0, len - (p.q_len - 1 - tok[1]))};
  // the tile's first token sees the fewest
  const int common = max(0, len - (p.q_len - 1 - tile * 16 / G));
  walk<F16, W, TAIL>(st, q, p, kvh, table, p.max_pages, ids, len, common, see, warp, ring);
  const int group = group_of(p, b);
  if (!p.part_o && blockIdx.x == 0 && threadIdx.x < 32)  // a prefix kernel's business otherwise
    for (int gi = lane; gi < p.groups; gi += 32) group_ok(p, gi, true);
  if (!p.part_o && group >= 0) {  // the prefix too
    const int plen = min(max(__ldg(p.prefix_lens + group), 0), p.prefix_pages * kPageKeys);
    const int all[2] = {plen, plen};
    table = p.prefix_table + static_cast<size_t>(group) * p.prefix_pages;
    walk<F16, W, false>(st, q, p, kvh, table, p.prefix_pages,
                 step_page<W>(table, p.prefix_pages, warp, 0), plen, plen, all, warp, ring);
  }

  cp_async_wait_all();
  job_sync<W>(slot);  // the rings are done with
  put_state(st, sm, warp);
  job_sync<W>(slot);
  if (p.part_o) griddep_wait();  // the prefix kernel's partials
  // Merge: 8 threads a row, 8 head dims each.  With fewer rows than the job has
  // thread octets, copies of a row share its parts (four of them, or all there
  // are when the prefix is in many); with more, the octets pass over the rows.
  constexpr int kOctets = W * 4;
  const int rows = min(16, R - tile * 16), part = jt % 8, octet = jt / 8;
  const int rows2 = rows <= 1 ? 1 : 1 << (32 - __clz(rows - 1));  // a power of two
  const int copies = max(1, min(kOctets / rows2, p.splits > 16 ? 16 : 4));
  const int copy = octet / rows2;  // 0 where the rows outnumber the octets
#pragma unroll 1
  for (int row = octet % rows2; row < rows2; row += kOctets) {
    const int rr = tile * 16 + row;
    Merged acc{-INFINITY, 0.f, {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}};
    if (row < rows && copy < copies) {
#pragma unroll 1
      for (int w = copy; w < W; w += copies) add_state(acc, sm, w, row, part);
      if (p.part_o && group >= 0)
        fold_partials(acc, sm.stage, p, group, b, kvh, rr, R, copy, copies, part, jt);
    }
    if (copies > 1) {  // one pass: the whole job is here
      // pairwise, in a fixed order
      float* mine = sm.merged[jt];
#pragma unroll 1
      for (int half = copies; half > 0; half >>= 1) {
        if (half < copies && copy < half) {
          const float* x = sm.merged[jt + half * rows2 * 8];
          acc.add(make_float2(x[0], x[1]), make_float4(x[2], x[3], x[4], x[5]),
                  make_float4(x[6], x[7], x[8], x[9]));
        }
        if (half == 1) break;
        if (copy < half) {
          mine[0] = acc.m;
          mine[1] = acc.l;
#pragma unroll
          for (int e = 0; e < 8; ++e) mine[2 + e] = acc.o[e];
        }
        job_sync<W>(slot);
      }
      if (copy > 0) return;
    }
    if (row >= rows) continue;
    store_row(p, acc, b, rr, kvh, G, part);
  }
}

// The sequences' own keys beside the prefix kernel: teams of W warps take jobs
// (a tile of 16 rows of a sequence and KV head) from the queue and leave one
// partial per row in own_o / own_ml.
template <int F16, int W, bool TAIL>
__global__ void __launch_bounds__(kSpThreads, 3) own_rows_kernel(SharedParams p, int jobs) {
  extern __shared__ __align__(128) uint8_t sp_smem[];
  __shared__ int s_job[kSpWarps];
  const int warp = threadIdx.x / 32 % W, slot = threadIdx.x / 32 / W, jt = threadIdx.x % (W * 32);
  const int lane = threadIdx.x % 32, g = lane >> 2;
  const int G = p.heads / p.kv_heads, R = p.q_len * G;
  const int tiles = (R + 15) / 16;
  uint8_t* ring = sp_smem + threadIdx.x / 32 * kSpRing;
  RowsMerge<W>& sm = *reinterpret_cast<RowsMerge<W>*>(sp_smem + slot * W * kSpRing);
  griddep_launch_dependents();
  while (true) {
    if (jt == 0) s_job[slot] = static_cast<int>(atomicAdd(p.queue, 1u));
    job_sync<W>(slot);
    const int id = s_job[slot];
    if (id >= jobs) break;
    const int job = id / tiles, tile = id - job * tiles;
    const int b = job / p.kv_heads, kvh = job - b * p.kv_heads;
    const int* table = p.block_table + static_cast<size_t>(b) * p.max_pages;
    const int ids = step_page<W>(table, p.max_pages, warp, 0);
    int len = __ldg(p.seq_lens + b);
    RowQ q;
    RowState st;
    int tok[2], head[2];
    const int seq[2] = {b, b};
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = tile * 16 + g + 8 * r;
      tok[r] = row < R ? row / G : -1;
      head[r] = kvh * G + row % G;
    }
    load_rows(q, st, p, seq, tok, head);
    if (len < 0 || len > p.max_pages * kPageKeys) {
      if (p.err && jt == 0) atomicOr(p.err, kErrBadArgs);
      len = min(max(len, 0), p.max_pages * kPageKeys);
    }
    const int see[2] = {tok[0] < 0 ? 0 : max(0, len - (p.q_len - 1 - tok[0])),
                        tok[1] < 0 ? 0 : max(0, len - (p.q_len - 1 - tok[1]))};
    const int common = max(0, len - (p.q_len - 1 - tile * 16 / G));
    walk<F16, W, TAIL>(st, q, p, kvh, table, p.max_pages, ids, len, common, see, warp, ring);
    cp_async_wait_all();
    job_sync<W>(slot);
    put_state(st, sm, warp);
    job_sync<W>(slot);
    const int rows = min(16, R - tile * 16), part = jt % 8;
#pragma unroll 1
    for (int row = jt / 8; row < rows; row += W * 4) {
      Merged acc{-INFINITY, 0.f, {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}};
#pragma unroll 1
      for (int w = 0; w < W; ++w) add_state(acc, sm, w, row, part);
      const size_t pr = static_cast<size_t>(job) * R + tile * 16 + row;
      float4* o = reinterpret_cast<float4*>(p.own_o + pr * 64 + 8 * part);
      o[0] = make_float4(acc.o[0], acc.o[1], acc.o[2], acc.o[3]);
      o[1] = make_float4(acc.o[4], acc.o[5], acc.o[6], acc.o[7]);
      if (part == 0) *reinterpret_cast<float2*>(p.own_ml + 2 * pr) = make_float2(acc.m, acc.l);
    }
    job_sync<W>(slot);  // the states are read: the rings may be filled again
  }
  // This grid ends after the prefix kernel, so that one dependency of the merge
  // covers both.
  griddep_wait();
}

// A row's own partial and its group's, joined: COPIES octets of threads a row,
// sharing the parts.
template <int COPIES>
__global__ void __launch_bounds__(kSpThreads) merge_rows_kernel(SharedParams p, int rows) {
  __shared__ Staging<kSpThreads> sm;
  const int R = p.q_len * (p.heads / p.kv_heads);
  const int id = blockIdx.x * (kSpThreads / 8 / COPIES) + threadIdx.x / 8 / COPIES;
  const int copy = threadIdx.x / 8 % COPIES, part = threadIdx.x % 8;
  griddep_wait();
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.queue = 0;  // for the next call
  const bool real = id < rows;
  const int job = real ? id / R : 0, rr = id - job * R, b = job / p.kv_heads, kvh = job - b * p.kv_heads;
  const int group = group_of_lane(p, b);
  Merged acc{-INFINITY, 0.f, {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}};
  if (real && copy == 0) {
    const float4* o = reinterpret_cast<const float4*>(p.own_o + static_cast<size_t>(id) * 64 + 8 * part);
    acc.add(__ldcg(reinterpret_cast<const float2*>(p.own_ml) + id), __ldcg(o), __ldcg(o + 1));
  }
  if (real && group >= 0) {
    fold_partials(acc, sm, p, group, b, kvh, rr, R, copy, COPIES, part, threadIdx.x);
  }
  __syncwarp();
#pragma unroll
  for (int o = 8; o < 8 * COPIES; o <<= 1) {
    const float2 ml = make_float2(__shfl_xor_sync(0xffffffffu, acc.m, o),
                                  __shfl_xor_sync(0xffffffffu, acc.l, o));
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = __shfl_xor_sync(0xffffffffu, acc.o[e], o);
    acc.add(ml, make_float4(x[0], x[1], x[2], x[3]), make_float4(x[4], x[5], x[6], x[7]));
  }
  if (real && copy == 0) store_row(p, acc, b, rr, kvh, p.heads / p.kv_heads, part);
}

// The prefixes of groups with few rows: CTA (unit, split) takes split `split` of
// p.splits of the pages for unit `unit`, 16 rows of a (group, KV head), and
// leaves one partial per row in slot unit * splits + split.
template <int F16>
__global__ void __launch_bounds__(kSpThreads, 3) prefix_rows_kernel(SharedParams p) {
  extern __shared__ __align__(128) uint8_t sp_smem[];
  RowsMerge<kSpWarps>& sm = *reinterpret_cast<RowsMerge<kSpWarps>*>(sp_smem);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane >> 2;
  griddep_launch_dependents();
  const int G = p.heads / p.kv_heads, R = p.q_len * G;
  const int unit = blockIdx.x / p.splits, split = blockIdx.x - unit * p.splits;
  // ---- the unit's group: every warp scans the groups' unit counts
  int group = -1, unit0 = 0, before = 0;
  bool bad = false;
#pragma unroll 1
  for (int base = 0; base < p.groups; base += 32) {
    const int gi = base + lane;
    int n = 0;
    if (gi < p.groups) {
      n = p.kv_heads * ((group_dims(p, gi).rows + 15) / 16);
      bad = bad || !group_ok(p, gi, blockIdx.x == 0 && warp == 0);
    }
    int upto = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const int from = before + upto - n;
    if (blockIdx.x == 0 && warp == 0 && gi < p.groups) p.part_plan[1 + gi] = from;
    const unsigned hit = __ballot_sync(0xffffffffu, from <= unit && unit < from + n);
    if (hit) {
      group = base + __ffs(hit) - 1;
      unit0 = __shfl_sync(0xffffffffu, from, __ffs(hit) - 1);
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  bad = __any_sync(0xffffffffu, bad);
  if (blockIdx.x == 0 && threadIdx.x == 0) p.part_plan[0] = bad ? kBadPlan : 0;
  if (bad || group < 0 || static_cast<int>(blockIdx.x) >= p.part_slots) return;
  const GroupDims d = group_dims(p, group);
  const int tiles = (d.rows + 15) / 16, kvh = (unit - unit0) / tiles;
  const int row0 = (unit - unit0 - kvh * tiles) * 16;
  const int pages = (d.plen + kPageKeys - 1) / kPageKeys, per = (pages + p.splits - 1) / p.splits;
  const int len = min(d.plen - split * per * kPageKeys, per * kPageKeys);
  if (len <= 0) return;
  const int* table = p.prefix_table + static_cast<size_t>(group) * p.prefix_pages + split * per;
  const int mine = min(per, pages - split * per);
  const int ids = step_page<kSpWarps>(table, mine, warp, 0);
  RowQ q;
  RowState st;
  int seq[2], tok[2], head[2], see[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = row0 + g + 8 * r, rb = row / R, rr = row - rb * R;
    seq[r] = d.b0 + rb;
    tok[r] = row < d.rows ? rr / G : -1;
    head[r] = kvh * G + rr % G;
    see[r] = row < d.rows ? len : 0;
  }
  load_rows(q, st, p, seq, tok, head);
  walk<F16, kSpWarps, false>(st, q, p, kvh, table, mine, ids, len, len, see, warp, sp_smem + warp * kSpRing);
  cp_async_wait_all();
  __syncthreads();
  put_state(st, sm, warp);
  __syncthreads();
  const int part = threadIdx.x % 8, row = threadIdx.x / 8;
  if (row0 + row >= d.rows) return;
  Merged acc{-INFINITY, 0.f, {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}};
#pragma unroll 1
  for (int w = 0; w < kSpWarps; ++w) add_state(acc, sm, w, row, part);
  const size_t pr = static_cast<size_t>(blockIdx.x) * 16 + row;
  float4* o = reinterpret_cast<float4*>(p.part_o + pr * 64 + 8 * part);
  o[0] = make_float4(acc.o[0], acc.o[1], acc.o[2], acc.o[3]);
  o[1] = make_float4(acc.o[4], acc.o[5], acc.o[6], acc.o[7]);
  if (part == 0) *reinterpret_cast<float2*>(p.part_ml + 2 * pr) = make_float2(acc.m, acc.l);
}

template <typename K, typename... A>
cudaError_t launch_rows(K kernel, long long ctas, size_t smem, bool dependent, cudaStream_t s,
                        A... args) {
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(smem));
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(kSpThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dependent ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// TAIL: several queries a sequence, which see different numbers of its keys (without
// it a walk is 2 to 4 % shorter).
template <int F16, bool TAIL>
cudaError_t launch_rows_f(const SharedParams& p, int sms, cudaStream_t s) {
  const int R = p.q_len * (p.heads / p.kv_heads);
  const int jobs = p.batch * p.kv_heads * ((R + 15) / 16);
  const int room = 3 * kSpWarps * sms;  // warps in flight
  const bool dep = p.part_o != nullptr;
  const auto ctas = [&](int w) { return (static_cast<long long>(jobs) * w + kSpWarps - 1) / kSpWarps; };
  if (jobs <= room / 4)
    return launch_rows(shared_rows_kernel<F16, 4, TAIL>, ctas(4), kSpSmem, dep, s, p, jobs);
  if (jobs <= room / 2)
    return launch_rows(shared_rows_kernel<F16, 2, TAIL>, ctas(2), kSpSmem, dep, s, p, jobs);
  return launch_rows(shared_rows_kernel<F16, 1, TAIL>, ctas(1), kSpSmem, dep, s, p, jobs);
}

template <int F16, bool TAIL>
cudaError_t launch_own_f(const SharedParams& p, int sms, cudaStream_t s) {
  const int R = p.q_len * (p.heads / p.kv_heads);
  const int jobs = p.batch * p.kv_heads * ((R + 15) / 16);
  // Teams of four warps where there are keys for them: 64 sequences of up to 1000
  // keys 31.3 us against 32.2 with two, 100 of two queries and up to 300 keys 57
  // against 54.
  const int w = p.max_pages >= 8 ? 4 : 2;
  const long long ctas = std::min<long long>(
      3LL * sms, (static_cast<long long>(jobs) * w + kSpWarps - 1) / kSpWarps);
  cudaError_t e = w == 4 ? launch_rows(own_rows_kernel<F16, 4, TAIL>, ctas, kSpSmem, true, s, p, jobs)
                         : launch_rows(own_rows_kernel<F16, 2, TAIL>, ctas, kSpSmem, true, s, p, jobs);
  if (e != cudaSuccess) return e;
  const int rows = p.batch * p.kv_heads * R;
  // as many octets a row as leave the merge in one wave
  const long long room = 1024LL * sms / 8;
  if (rows * 4LL <= room) return launch_rows(merge_rows_kernel<4>, (rows + 3LL) / 4, 0, true, s, p, rows);
  if (rows * 2LL <= room) return launch_rows(merge_rows_kernel<2>, (rows + 7LL) / 8, 0, true, s, p, rows);
  return launch_rows(merge_rows_kernel<1>, (rows + 15LL) / 16, 0, true, s, p, rows);
}

// f<element is f16, several queries a sequence>
#define FFAI_ROWS(f, ...)                                                               \
  (p.kv_dtype == 2 ? (p.q_len > 1 ? f<1, true>(__VA_ARGS__) : f<1, false>(__VA_ARGS__)) \
                   : (p.q_len > 1 ? f<0, true>(__VA_ARGS__) : f<0, false>(__VA_ARGS__)))

}  // namespace

// Behind a prefix kernel the rows kernel is a programmatic dependent: sequences'
// own keys are attended while the last of the prefix finishes.
cudaError_t launch_shared_rows(const SharedParams& p, int sms, cudaStream_t s) {
  return FFAI_ROWS(launch_rows_f, p, sms, s);
}

cudaError_t launch_own_and_merge(const SharedParams& p, int sms, cudaStream_t s) {
  return FFAI_ROWS(launch_own_f, p, sms, s);
}

cudaError_t launch_prefix_rows(const SharedParams& p, int units, cudaStream_t s) {
  return launch_rows(p.kv_dtype == 2 ? prefix_rows_kernel<1> : prefix_rows_kernel<0>,
                     static_cast<long long>(units) * p.splits, kSpSmem, false, s, p);
}

}  // namespace ffai

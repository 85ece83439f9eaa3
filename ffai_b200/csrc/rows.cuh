// Attention of 16 query rows by one warp over keys in pages, on mma.sync: what the
// kernels with few rows a unit share.  P: the kernel's parameters (q and its
// strides, pools, kv_heads, num_pages, types, scale_log2, err).
#pragma once

#include "common.cuh"
#include "kernels.h"

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
// not all rows alike, but all the first lo, and none those from hi on.  TERMS: of
// the queries, whose sum they are; with more than one the weights enter the second
// product in two terms as well, and that product starts from zero, since the
// matrix instruction's sums are cut, not rounded.
template <int F16, bool TAIL, int TERMS>
__device__ __forceinline__ void step32(RowState& st, const RowQ (&q)[TERMS], uint8_t* buf,
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
#pragma unroll
    for (int n = TERMS - 1; n >= 0; --n) {  // the smallest first
      mma16816<F16>(s[i], q[n].a[0], k[i][0].x, k[i][0].y);
      mma16816<F16>(s[i], q[n].a[1], k[i][0].z, k[i][0].w);
      mma16816<F16>(s[i], q[n].a[2], k[i][1].x, k[i][1].y);
      mma16816<F16>(s[i], q[n].a[3], k[i][1].z, k[i][1].w);
    }
  }
  uint32_t p[2][4], rest[2][4];
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
      const uint32_t w = F16 ? pack_f16x2(p0, p1) : pack_bf16x2(p0, p1);
      p[i >> 1][(i & 1) * 2 + r] = w;
      if constexpr (TERMS > 1) {
        const float r0 = p0 - lo_half(w, F16), r1 = p1 - hi_half(w, F16);
        rest[i >> 1][(i & 1) * 2 + r] = F16 ? pack_f16x2(r0, r1) : pack_bf16x2(r0, r1);
      }
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
  float part[8][4];
  if constexpr (TERMS > 1) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) part[j][e] = 0.f;
  }
  float(&o)[8][4] = TERMS > 1 ? part : st.o;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t e0[4] = {v[h][0].x, v[h][0].y, v[h][0].z, v[h][0].w};
    const uint32_t e1[4] = {v[h][1].x, v[h][1].y, v[h][1].z, v[h][1].w};
    const uint32_t e2[4] = {v[h][2].x, v[h][2].y, v[h][2].z, v[h][2].w};
    const uint32_t e3[4] = {v[h][3].x, v[h][3].y, v[h][3].z, v[h][3].w};
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if constexpr (TERMS > 1) {
        mma16816<F16>(o[2 * c], rest[h], __byte_perm(e0[c], e1[c], 0x5410),
                      __byte_perm(e2[c], e3[c], 0x5410));
        mma16816<F16>(o[2 * c + 1], rest[h], __byte_perm(e0[c], e1[c], 0x7632),
                      __byte_perm(e2[c], e3[c], 0x7632));
      }
      mma16816<F16>(o[2 * c], p[h], __byte_perm(e0[c], e1[c], 0x5410),
                    __byte_perm(e2[c], e3[c], 0x5410));
      mma16816<F16>(o[2 * c + 1], p[h], __byte_perm(e0[c], e1[c], 0x7632),
                    __byte_perm(e2[c], e3[c], 0x7632));
    }
  }
  if constexpr (TERMS > 1) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) st.o[j][e] += part[j][e];
  }
}

template <typename P, int TERMS>
__device__ __forceinline__ void q_pair(const P& p, const void* row, int dim, uint32_t (&w)[TERMS]) {
  if (p.q_dtype == 0) {  // f32 queries are rounded to the cache's type, and what that leaves again
    float2 x = __ldg(reinterpret_cast<const float2*>(static_cast<const float*>(row) + dim));
    const int f16 = p.kv_dtype == 2;
#pragma unroll
    for (int n = 0; n < TERMS; ++n) {
      w[n] = f16 ? pack_f16x2(x.x, x.y) : pack_bf16x2(x.x, x.y);
      if (n + 1 < TERMS) {
        x.x -= lo_half(w[n], f16);
        x.y -= hi_half(w[n], f16);
      }
    }
  } else {
    w[0] = __ldg(reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(row) + dim));
#pragma unroll
    for (int n = 1; n < TERMS; ++n) w[n] = 0u;
  }
}

template <typename P>
__device__ __forceinline__ const void* q_row(const P& p, int b, int tok, int h) {
  const size_t off = static_cast<size_t>(b) * p.q_sb + static_cast<size_t>(tok) * p.q_st +
                     static_cast<size_t>(h) * p.q_sh;
  return static_cast<const uint8_t*>(p.q) + off * (p.q_dtype == 0 ? 4 : 2);
}

// Page ids of a warp's next 32 steps, one per lane: warp w of the job's W takes
// the steps w, w + W, ... of 32 keys, and `first` counts the warp's own.
template <int W>
__device__ __forceinline__ int step_page(const int* table, int pages, int warp, int first) {
  const int page = (warp + W * (first + static_cast<int>(threadIdx.x % 32))) / 2;
  return page < pages ? __ldg(table + page) : -1;
}

// Walk `len` keys of a list of pages (TAIL: the first `common` of which all rows
// see; else all rows see all).  `ids` holds the first 32 steps' page ids, loaded
// ahead (the table does not depend on the lengths).  `ring`: this warp's kSpRing
// bytes, not in use.
template <int F16, int W, bool TAIL, int TERMS, typename P>
__device__ __forceinline__ void walk(RowState& st, const RowQ (&q)[TERMS], const P& p, int kvh,
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
    step32<F16, TAIL, TERMS>(st, q, ring + i % kSpDepth * kSpStep, rel, max(common - k0, 0),
                min(len - k0, kSpKeys), p.scale_log2);
    __syncwarp();
    fetch(i + kSpDepth);
  }
}

// The 16 query rows of a tile as operands: row r is token tok[r] (of a lane's
// two rows; -1: none) of sequence seq[r], head h[r].
template <int TERMS, typename P>
__device__ __forceinline__ void load_rows(RowQ (&q)[TERMS], RowState& st, const P& p,
                                          const int (&seq)[2], const int (&tok)[2], const int (&h)[2]) {
  const int t = threadIdx.x & 3;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const void* src = tok[r] >= 0 ? q_row(p, seq[r], tok[r], h[r]) : nullptr;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int dim = 32 * (s / 2) + 8 * t + 4 * (s % 2);
      uint32_t a[TERMS] = {}, b[TERMS] = {};
      if (src) {
        q_pair(p, src, dim, a);
        q_pair(p, src, dim + 2, b);
      }
#pragma unroll
      for (int n = 0; n < TERMS; ++n) {
        q[n].a[s][r] = a[n];
        q[n].a[s][2 + r] = b[n];
      }
    }
    st.m[r] = -INFINITY;
    st.l[r] = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) st.o[j][2 * r] = st.o[j][2 * r + 1] = 0.f;
  }
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

constexpr int kSpStage = 8;  // partials a thread stages at a time

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

}  // namespace

}  // namespace ffai

// What the kernels of ffai_attn_chunk_paged agree on.
#pragma once

#include <limits.h>

#include "common.cuh"
#include "kernels.h"
#include "rows.cuh"

namespace ffai {

namespace {

constexpr int kChKeys = 128;  // keys per block of the tensor kernel (two pages)

// A sequence's new tokens, and the keys it holds with them.
struct ChunkSeq {
  int t0, n, len;
};
__device__ __forceinline__ ChunkSeq chunk_seq(const ChunkParams& p, int b, bool& bad) {
  const int t0 = __ldg(p.cu_q + b), t1 = __ldg(p.cu_q + b + 1);
  ChunkSeq s{t0, t1 - t0, __ldg(p.seq_lens + b)};
  if (t0 < 0 || t1 < t0 || t1 > p.tokens) {  // no rows that can be told
    bad = true;
    s.t0 = s.n = 0;
  }
  if (s.len < 0 || s.len > p.max_pages * kPageKeys) {
    bad = true;
    s.len = min(max(s.len, 0), p.max_pages * kPageKeys);
  }
  return s;
}

// Rows of a sequence and KV head are ordered by (token, head within the group);
// a unit is RU of them.
template <int RU>
__device__ __forceinline__ int chunk_units(const ChunkSeq& s, int G) {
  return (s.n * G + RU - 1) / RU;
}
// Keys that the unit's last row sees (not below 0).
__device__ __forceinline__ int chunk_limit(const ChunkParams& p, const ChunkSeq& s, int tok) {
  return p.causal ? max(0, s.len - (s.n - 1 - tok)) : s.len;
}
// Blocks of keys up to there; one at least, so that every row has a place where
// it is written.
template <int KEYS>
__device__ __forceinline__ int chunk_blocks(int limit) {
  return max(1, (limit + KEYS - 1) / KEYS);
}
// Steps of a unit on the line: a block of KEYS keys each, or two where a unit of two
// tiles of 128 rows has only one.
template <int RU, int KEYS>
__device__ __forceinline__ int unit_steps(const ChunkParams& p, const ChunkSeq& s, int G, int m) {
  const int rows = min((m + 1) * RU, s.n * G), blocks = chunk_blocks<KEYS>(chunk_limit(p, s, (rows - 1) / G));
  return RU == kPxRows && rows - m * RU <= RU / 2 ? (blocks + 1) >> 1 : blocks;
}
// Steps of a (sequence, KV head), and with each unit's rounded up to whole shares.
struct HeadSteps {
  int n, padded;
};
template <int RU, int KEYS>
__device__ __forceinline__ HeadSteps head_steps(const ChunkParams& p, const ChunkSeq& s, int G) {
  const int units = chunk_units<RU>(s, G);
  HeadSteps h{0, 0};
#pragma unroll 1
  for (int m = 0; m < units; ++m) {
    const int n = unit_steps<RU, KEYS>(p, s, G, m);
    h.n += n;
    h.padded += (n + p.min_share - 1) / p.min_share * p.min_share;
  }
  return h;
}

// A team's stretch of the line (a CTA is one team, or a few): where it starts, and
// how long it is.
struct Stretch {
  int b, h, m, step;  // sequence, KV head, unit, step within the unit
  int left;           // steps
  int share;          // of a team
  int unit0;          // the unit's first step on the line
};

// Where cu_q falls, sequences may name the same tokens many times, and the line
// would be longer than the host allowed for: there is nothing to do then.
__device__ __noinline__ bool repeats_rows(const ChunkParams& p) {
  long long rows = 0;
  bool bad = false;
#pragma unroll 1
  for (int b = 0; b < p.batch; ++b) rows += chunk_seq(p, b, bad).n;
  return rows > p.tokens;
}

// All threads of a CTA: every CTA scans the sequences.  The line is dealt out
// evenly, min_share steps a team at least.  Where so little is to be done that
// every unit can begin with a team of its own at that share, it does: most units
// then lie within one and need no merge.  s_warp: two words per warp.
template <int RU, int KEYS, int THREADS, int TEAMS>
__device__ __forceinline__ void find_stretch(const ChunkParams& p, Stretch* out, int2* s_warp) {
  const int G = p.heads / p.kv_heads;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int per = (p.batch + THREADS - 1) / THREADS;
  const int b0 = min(p.batch, static_cast<int>(threadIdx.x) * per), b1 = min(p.batch, b0 + per);
  bool bad = false, falls = false;
  HeadSteps sum{0, 0};
#pragma unroll 4
  for (int b = b0; b < b1; ++b) {
    falls |= __ldg(p.cu_q + b) > __ldg(p.cu_q + b + 1);
    const HeadSteps h = head_steps<RU, KEYS>(p, chunk_seq(p, b, bad), G);
    sum.n += p.kv_heads * h.n;
    sum.padded += p.kv_heads * h.padded;
  }
  if (bad && blockIdx.x == 0 && p.err) atomicOr(p.err, kErrBadArgs);
  HeadSteps at = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, at.n, o), y = __shfl_up_sync(0xffffffffu, at.padded, o);
    if (lane >= o) {
      at.n += x;
      at.padded += y;
    }
  }
  if (lane == 31) s_warp[warp] = make_int2(at.n, at.padded);
  if (threadIdx.x < TEAMS) out[threadIdx.x].left = 0;
  if (__syncthreads_or(falls) && repeats_rows(p)) return;  // (reported as bad above; all CTAs alike)
  HeadSteps total{0, 0};
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    const int2 x = s_warp[w];
    if (w < warp) {
      at.n += x.x;
      at.padded += x.y;
    }
    total.n += x.x;
    total.padded += x.y;
  }
  const int teams = static_cast<int>(gridDim.x) * TEAMS;
  const bool own = total.padded <= teams * p.min_share;  // a team of its own for every unit
  const int all = own ? total.padded : total.n;
  const int share = own ? p.min_share : max(p.min_share, (total.n + teams - 1) / teams);
  const int mine = own ? sum.padded : sum.n, from = (own ? at.padded : at.n) - mine;
#pragma unroll 1
  for (int t = 0; t < TEAMS; ++t) {
    const int first = (static_cast<int>(blockIdx.x) * TEAMS + t) * share;
    if (!(from <= first && first < from + mine)) continue;  // one thread goes on
    int at0 = from, b = b0, per_head = 0;
    ChunkSeq s{};
    for (; b < b1; ++b) {
      s = chunk_seq(p, b, bad);
      const HeadSteps h = head_steps<RU, KEYS>(p, s, G);
      per_head = own ? h.padded : h.n;
      if (first < at0 + p.kv_heads * per_head) break;
      at0 += p.kv_heads * per_head;
    }
    if (b == b1) continue;  // (never, unless the lengths are written meanwhile)
    Stretch w{};
    w.b = b;
    w.h = (first - at0) / per_head;
    at0 += w.h * per_head;
    const int units = chunk_units<RU>(s, G);
    int n = 0;
    for (;; ++w.m) {
      n = unit_steps<RU, KEYS>(p, s, G, w.m);
      const int line = own ? (n + share - 1) / share * share : n;
      if (w.m == units - 1 || first < at0 + line) break;
      at0 += line;
    }
    w.unit0 = at0;
    w.step = first - at0;
    w.left = own ? min(share, n - w.step) : min(all, first + share) - first;
    w.share = share;
    out[t] = w;
  }
  __syncthreads();
}

// One row's result, 8 head dims a thread.
__device__ __forceinline__ void store_row(const ChunkParams& p, Merged& acc, int tok, int h, int part) {
  const size_t at = (static_cast<size_t>(tok) * p.heads + h) * 64 + 8 * part;
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
    p.lse[static_cast<size_t>(h) * p.tokens + tok] =
        acc.l == 0.f ? -INFINITY : (acc.m + log2f(acc.l)) * 0.69314718055994530942f;
}

// Where a unit's partial results lie, and its rows: slots of slot_rows rows, from row
// `side` of them on; rows row0 .. row0 + rows - 1 of the sequence whose first token is
// t0 and of a KV head.
struct UnitParts {
  int c0, c1;  // its teams
  int slot_rows, side;
  int row0, rows, t0, kvh;
};
// Row `row` in team c's: two slots a team, the second for the unit that begins in its stretch.
__device__ __forceinline__ size_t part_row(const UnitParts& u, int c, int row) {
  return static_cast<size_t>(2 * c + (c == u.c0 ? 1 : 0)) * u.slot_rows + u.side + row;
}
__device__ __forceinline__ void store_unit_row(const ChunkParams& p, const UnitParts& u, Merged& acc, int row, int part) {
  const int G = p.heads / p.kv_heads, i = (u.row0 + row) / G;
  store_row(p, acc, u.t0 + i, u.kvh * G + u.row0 + row - i * G, part);
}

// All partial results of a unit's rows, teams c0 .. c1 in that order, by THREADS
// threads: 8 a row, 8 head dims each, and where the rows are few up to four such
// octets a row, which share its parts.
template <int THREADS>
__device__ __noinline__ void merge_rows(const ChunkParams& p, const UnitParts u, int thread) {
  constexpr int kOctets = THREADS / 8, kAhead = 4;
  const int part = thread % 8, octet = thread / 8;
  const int shift = 4 * u.rows <= kOctets ? 2 : 2 * u.rows <= kOctets ? 1 : 0;
  const int copy = octet & ((1 << shift) - 1);
#pragma unroll 1
  for (int r0 = 0; r0 < u.rows; r0 += kOctets >> shift) {
    const int row = r0 + (octet >> shift);
    Merged acc{-INFINITY, 0.f, {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}};
#pragma unroll 1
    for (int c = u.c0 + copy; c <= u.c1; c += kAhead << shift) {
      float2 ml[kAhead];
      float4 a[kAhead], b[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int from = c + (k << shift);
        ml[k] = make_float2(-INFINITY, 0.f);
        if (from <= u.c1 && row < u.rows) {
          const size_t i = part_row(u, from, row);
          const float4* o = reinterpret_cast<const float4*>(p.part_o + i * 64 + 8 * part);
          ml[k] = __ldcg(reinterpret_cast<const float2*>(p.part_ml + 2 * i));
          a[k] = __ldcg(o);
          b[k] = __ldcg(o + 1);
        }
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) acc.add(ml[k], a[k], b[k]);
    }
#pragma unroll 1
    for (int o = 8; o < 8 << shift; o <<= 1) {
      const float2 ml = make_float2(__shfl_xor_sync(0xffffffffu, acc.m, o), __shfl_xor_sync(0xffffffffu, acc.l, o));
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = __shfl_xor_sync(0xffffffffu, acc.o[e], o);
      acc.add(ml, make_float4(x[0], x[1], x[2], x[3]), make_float4(x[4], x[5], x[6], x[7]));
    }
    if (row < u.rows && copy == 0) store_unit_row(p, u, acc, row, part);
  }
}

}  // namespace

}  // namespace ffai

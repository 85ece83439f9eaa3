// What the kernels of ffai_attn_chunk_paged agree on.
#pragma once

#include <limits.h>

#include "common.cuh"
#include "kernels.h"
#include "rows.cuh"

namespace ffai {

namespace {

constexpr int kChKeys = 128;  // keys per block (two pages)

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
__device__ __forceinline__ int chunk_blocks(int limit) {
  return max(1, (limit + kChKeys - 1) / kChKeys);
}

// Steps of a unit on the line: a block of keys each, or two where a unit of two
// tiles of 128 rows has only one.
template <int RU>
__device__ __forceinline__ int unit_steps(const ChunkParams& p, const ChunkSeq& s, int G, int m) {
  const int rows = min((m + 1) * RU, s.n * G), blocks = chunk_blocks(chunk_limit(p, s, (rows - 1) / G));
  return RU == kPxRows && rows - m * RU <= RU / 2 ? (blocks + 1) >> 1 : blocks;
}
template <int RU>
__device__ __forceinline__ int head_steps(const ChunkParams& p, const ChunkSeq& s, int G) {
  const int units = chunk_units<RU>(s, G);
  if (units == 0) return 0;
  int n = 0;
  for (int m = 0; m < units; ++m) n += unit_steps<RU>(p, s, G, m);
  return n;
}

// A CTA's stretch of the line: where it starts, and how long it is.
struct Stretch {
  int b, h, m, step;  // sequence, KV head, unit, step within the unit
  int left;           // steps
  int share;          // of a CTA
  int unit0;          // the unit's first step on the line
};

// All threads of a CTA: every CTA scans the sequences.  s_warp: a word per warp.
template <int RU, int THREADS>
__device__ __forceinline__ void find_stretch(const ChunkParams& p, Stretch* out, int* s_warp) {
  const int G = p.heads / p.kv_heads;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  const int per = (p.batch + THREADS - 1) / THREADS;
  const int b0 = min(p.batch, static_cast<int>(threadIdx.x) * per), b1 = min(p.batch, b0 + per);
  bool bad = false;
  int sum = 0;
#pragma unroll 4
  for (int b = b0; b < b1; ++b) sum += p.kv_heads * head_steps<RU>(p, chunk_seq(p, b, bad), G);
  if (bad && blockIdx.x == 0 && p.err) atomicOr(p.err, kErrBadArgs);
  int at = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, at, o);
    if (lane >= o) at += x;
  }
  if (lane == 31) s_warp[warp] = at;
  __syncthreads();
  int total = 0, base = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) base += s_warp[w];
    total += s_warp[w];
  }
  at += base - sum;
  const int grid = static_cast<int>(gridDim.x);
  const int share = max(p.min_share, (total + grid - 1) / grid);
  const int first = static_cast<int>(blockIdx.x) * share;
  const int left = min(total, first + share) - first;
  if (threadIdx.x == 0) out->left = 0;
  __syncthreads();
  if (left > 0 && at <= first && first < at + sum) {  // one thread
    int b = b0;
    ChunkSeq s{};
    int per_head = 0;
    for (; b < b1; ++b) {
      s = chunk_seq(p, b, bad);
      per_head = head_steps<RU>(p, s, G);
      if (first < at + p.kv_heads * per_head) break;
      at += p.kv_heads * per_head;
    }
    Stretch w{};
    if (b < b1) {  // (always, unless the lengths are written meanwhile)
      w.b = b;
      w.h = (first - at) / per_head;
      at += w.h * per_head;
      const int units = chunk_units<RU>(s, G);
      for (; w.m < units - 1; ++w.m) {
        const int n = unit_steps<RU>(p, s, G, w.m);
        if (first < at + n) break;
        at += n;
      }
      w.unit0 = at;
      w.step = first - at;
      w.left = left;
      w.share = share;
    }
    *out = w;
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

}  // namespace

}  // namespace ffai

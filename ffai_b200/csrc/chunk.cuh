// What the kernels of ffai_attn_chunk_paged agree on.
#pragma once

#include <limits.h>

#include "common.cuh"
#include "kernels.h"

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

}  // namespace

}  // namespace ffai

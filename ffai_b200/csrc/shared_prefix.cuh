// What the two kernels of ffai_attn_shared_prefix agree on.
#pragma once

#include <limits.h>

#include "common.cuh"
#include "kernels.h"

namespace ffai {

// A group's query rows per KV head, in units of 256 (two tiles of 128), and
// the prefix's blocks of 128 keys.  Rows are ordered by (sequence, token, head
// within the KV head's group).
struct GroupDims {
  int b0;    // first sequence
  int rows;  // sequences * q_len * G
  int mu;    // units
  int single;  // 1: the last unit has one tile
  int plen;  // prefix keys
  int nb;    // key blocks; 0 without rows or keys
};
__device__ __forceinline__ GroupDims group_dims(const SharedParams& p, int g) {
  GroupDims d;
  d.b0 = min(max(__ldg(p.group_starts + g), 0), p.batch);
  const int b1 = min(max(__ldg(p.group_starts + g + 1), d.b0), p.batch);
  d.rows = (b1 - d.b0) * p.q_len * (p.heads / p.kv_heads);
  d.mu = (d.rows + kPxRows - 1) / kPxRows;
  d.single = d.rows - (d.mu - 1) * kPxRows <= 128 ? 1 : 0;
  d.plen = min(max(__ldg(p.prefix_lens + g), 0), p.prefix_pages * kPageKeys);
  d.nb = d.rows > 0 ? (d.plen + kPxKeys - 1) / kPxKeys : 0;
  return d;
}

// Group g of all: does it start and end in order within the batch?  The lengths
// must lie within the table too, but are clamped; starts that do not rise would
// give sequences to several groups, so then no group's prefix is attended.
__device__ __forceinline__ bool group_ok(const SharedParams& p, int g, bool report) {
  const int s0 = __ldg(p.group_starts + g), s1 = __ldg(p.group_starts + g + 1);
  const bool ok = s0 >= 0 && s1 >= s0 && s1 <= p.batch;
  if (report && p.err) {
    const int len = __ldg(p.prefix_lens + g);
    if (!ok || len < 0 || len > p.prefix_pages * kPageKeys) atomicOr(p.err, kErrBadArgs);
  }
  return ok;
}
constexpr int kBadPlan = INT_MIN;  // in part_plan[0]: as above

// Work is counted in steps of the prefix kernel's two chains: a unit of two
// tiles passes over one key block a step (one tile a chain), a unit of one
// tile over two (one block a chain).  A group's steps lie on a line in the
// order (head, chunk of key blocks, unit, step).  With one unit a head's
// blocks are one chunk; with more, chunks are about `share` blocks, so that
// the units of a head pass over the same keys at about the same time and all
// but the first find them in L2.  A (head, chunk, unit) is a segment.  Chunks
// but the last have an even number of blocks.
__device__ __forceinline__ int chunk_blocks(const GroupDims& d, int share) {
  return d.mu == 1 ? (d.nb + 1) & ~1 : min((share + 1) & ~1, (d.nb + 1) & ~1);
}
// Steps of one head over its first `blocks` blocks (even, or all of them).
__device__ __forceinline__ int head_steps(const GroupDims& d, int blocks) {
  return (d.mu - d.single) * blocks + d.single * ((blocks + 1) >> 1);
}
// What a head takes of the line: its steps, in whole shares if each head begins
// on a CTA of its own.
__device__ __forceinline__ int line_steps(const GroupDims& d, int share, int even) {
  const int n = head_steps(d, d.nb);
  return even && share > 0 ? (n + share - 1) / share * share : n;
}
// Steps of unit m over `len` blocks.
__device__ __forceinline__ int unit_steps(const GroupDims& d, int m, int len) {
  return d.single && m == d.mu - 1 ? (len + 1) >> 1 : len;
}

}  // namespace ffai

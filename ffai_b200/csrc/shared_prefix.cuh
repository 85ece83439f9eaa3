// What the two kernels of ffai_attn_shared_prefix agree on.
#pragma once

#include "common.cuh"
#include "kernels.h"

namespace ffai {

// A group's query rows per KV head, its row tiles and key blocks.  Rows are
// ordered by (sequence, token, head within the KV head's group).
struct GroupDims {
  int b0;    // first sequence
  int rows;  // sequences * q_len * G
  int mt;    // tiles of 128 rows
  int plen;  // prefix keys
  int nb;    // blocks of 128 keys; 0 without rows or keys
};
__device__ __forceinline__ GroupDims group_dims(const SharedParams& p, int g) {
  GroupDims d;
  d.b0 = min(max(__ldg(p.group_starts + g), 0), p.batch);
  const int b1 = min(max(__ldg(p.group_starts + g + 1), d.b0), p.batch);
  d.rows = (b1 - d.b0) * p.q_len * (p.heads / p.kv_heads);
  d.mt = (d.rows + 127) / 128;
  d.plen = min(max(__ldg(p.prefix_lens + g), 0), p.prefix_pages * kPageKeys);
  d.nb = d.rows > 0 ? (d.plen + 127) / 128 : 0;
  return d;
}

}  // namespace ffai

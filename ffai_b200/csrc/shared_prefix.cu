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

#include "rows.cuh"
#include "shared_prefix.cuh"

namespace ffai {

namespace {

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
  RowQ q[1];
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
  walk<F16, W, TAIL, 1>(st, q, p, kvh, table, p.max_pages, ids, len, common, see, warp, ring);
  const int group = group_of(p, b);
  if (!p.part_o && blockIdx.x == 0 && threadIdx.x < 32)  // a prefix kernel's business otherwise
    for (int gi = lane; gi < p.groups; gi += 32) group_ok(p, gi, true);
  if (!p.part_o && group >= 0) {  // the prefix too
    const int plen = min(max(__ldg(p.prefix_lens + group), 0), p.prefix_pages * kPageKeys);
    const int all[2] = {plen, plen};
    table = p.prefix_table + static_cast<size_t>(group) * p.prefix_pages;
    walk<F16, W, false, 1>(st, q, p, kvh, table, p.prefix_pages,
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
    RowQ q[1];
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
    walk<F16, W, TAIL, 1>(st, q, p, kvh, table, p.max_pages, ids, len, common, see, warp, ring);
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
  RowQ q[1];
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
  walk<F16, kSpWarps, false, 1>(st, q, p, kvh, table, mine, ids, len, len, see, warp, sp_smem + warp * kSpRing);
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

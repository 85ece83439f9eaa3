// The shared part of ffai_attn_shared_prefix on the tensor cores: all query
// rows of a group against the group's prefix, whose keys are read once for up
// to 256 rows.
//
// A group of s sequences has s * q_len * G query rows per KV head (G = query
// heads per KV head), in units of 256: two tiles of 128, the M of tcgen05.mma.
// The prefix is cut into blocks of 128 keys (two pages).  The steps of all
// units of all groups and heads are laid out on one line, W of them
// (shared_prefix.cuh), and CTA c takes the steps [c S, (c + 1) S), S = ceil(W /
// CTAs): every CTA gets the same work whatever the lengths and group sizes.
// What a CTA holds of a segment (same rows, consecutive blocks) leaves one
// partial result (running maximum, sum, unnormalised output), merged by
// shared_rows_kernel, or with own keys beside by merge_rows_kernel.  The
// partial of CTA c for segment t lies in slot c + t: along the line either c or
// t grows from one partial to the next, so slots are distinct.
//
// Per CTA: warp 16 streams the pages through a 4-stage ring of K and V blocks
// by TMA for two chains (t = 0, 1), each with an MMA warp (17, 18), scores,
// weights and an output accumulator of its own in tensor memory and 8 softmax
// warps, so one chain's softmax runs beside the other's products.  With more
// than 128 rows in the unit chain t takes tile t and both take every block;
// else both hold the one tile and take the blocks in turn (chain 0 the even
// ones), and at the end chain 1 hands its accumulator to chain 0 through shared
// memory, warp to warp.
//
// Bound by the exponentials (16 a clock and SM) and the moves between tensor
// memory and registers around them: a step, 256 rows by 128 keys, takes 1.46 us
// where its exponentials take 1.07 and its products 0.63.  Filling costs 4 us to
// the first scores, a segment's end 2.  89 GFLOP over three prefixes of up to
// 32768 keys: 150 us, tensor pipe 29 % active.  Of these the 74 to 77 steps of a
// CTA make 108 to 112; the rest goes into fills and ends, for a CTA has up to
// five segments (2.2 on average) there.
//
// Every wait is bounded (common.cuh); on a timeout the CTA raises an error
// bit, drains its copies and MMAs, frees tensor memory and exits.
#include <atomic>

#include "shared_prefix.cuh"

namespace ffai {

namespace {

constexpr int kPxStages = 4;
constexpr int kPxThreads = 608;  // 16 softmax warps, TMA warp, 2 MMA warps
constexpr int kPxProducer = 16, kPxMma0 = 17;
constexpr uint32_t kPxTile = 128 * 128;       // 128 rows of 128 bytes
constexpr uint32_t kPxPage = kPageKeys * 128; // a page's rows of one head
constexpr uint32_t kPxTmem = 512;
constexpr uint32_t kPxS = 0, kPxP = 256, kPxO = 384;  // + 128 t, + 64 t, + 64 t

// A walk over a CTA's stretch of the line, segment by segment.
struct Walk {
  GroupDims d;
  int g, h, q, m;  // group, KV head, chunk, unit
  int cl, len;     // key blocks of a chunk, and of this one
  int steps, step; // steps of this unit over the chunk, and the current one
  int left;        // steps left, the current one included
  int seg;         // index of the segment on the line
  int base;        // key blocks of this CTA before this segment
  int alt;         // one-tile segments of this CTA before this one
};
__device__ __forceinline__ bool walk_pair(const Walk& w) { return !(w.d.single && w.m == w.d.mu - 1); }
// What this CTA has of the current segment: steps, key blocks, the first block.
__device__ __forceinline__ int walk_steps(const Walk& w) { return min(w.left, w.steps - w.step); }
__device__ __forceinline__ int walk_blocks(const Walk& w) {
  const int n = walk_steps(w);
  return walk_pair(w) ? n : min(2 * n, w.len - 2 * w.step);
}
__device__ __forceinline__ int walk_first(const Walk& w) {
  return w.q * w.cl + (walk_pair(w) ? w.step : 2 * w.step);
}

struct __align__(8) PxBars {
  uint64_t q_full[2];
  uint64_t k_full[kPxStages], v_full[kPxStages], kv_empty[kPxStages];
  uint64_t s_full[2], sc_done[2], p_full[2], o_done[2];
  uint64_t mrg_full[8], mrg_empty[8];
  uint64_t drain;
  uint32_t tmem_base;
  int abort_flag;
  int share;
  Walk start;  // this CTA's stretch
};

// Shared memory, at fixed offsets from its 1024-byte aligned start (which the
// kernel checks), so that no pointer into it takes a register.
constexpr uint32_t kPxOffK = 2 * kPxTile;  // after the chains' query tiles
constexpr uint32_t kPxOffV = kPxOffK + kPxStages * kPxTile;
constexpr uint32_t kPxOffMerge = kPxOffV + kPxStages * kPxTile;
constexpr uint32_t kPxMergeFloats = 32 * 32 + 64;  // per pair of warps
constexpr uint32_t kPxOffWalks = kPxOffMerge + 8 * kPxMergeFloats * sizeof(float);
constexpr uint32_t kPxOffBars = kPxOffWalks + 16 * sizeof(Walk);
constexpr size_t kPxSmem = kPxOffBars + sizeof(PxBars);
static_assert(sizeof(Walk) % 4 == 0 && kPxOffBars % 8 == 0 && kPxSmem <= 227 * 1024, "shared memory");
extern __shared__ __align__(1024) uint8_t px_smem[];
#define PX_BARS (reinterpret_cast<PxBars*>(px_smem + kPxOffBars))

// To the next segment, if the stretch goes on.
__device__ __forceinline__ void walk_next(Walk& w, const SharedParams& p) {
  w.base += walk_blocks(w);
  w.alt += walk_pair(w) ? 0 : 1;
  w.left -= walk_steps(w);
  if (w.left <= 0) return;  // else the segment is done
  w.step = 0;
  ++w.seg;
  if (++w.m == w.d.mu) {
    w.m = 0;
    if (++w.q * w.cl >= w.d.nb) {
      w.q = 0;
      if (++w.h == p.kv_heads) {
        w.h = 0;
        do w.d = group_dims(p, ++w.g);
        while (w.d.nb == 0);
        w.cl = chunk_blocks(w.d, PX_BARS->share);
      }
    }
    w.len = min(w.cl, w.d.nb - w.q * w.cl);
  }
  w.steps = unit_steps(w.d, w.m, w.len);
}

__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                                          unsigned* err, unsigned code) {
  const bool ok = mbar_wait(bar, parity, abort_flag, err, code);
  return __all_sync(0xffffffffu, ok);
}

// One warp: the length of the line and where this CTA starts on it.  CTA 0
// also leaves each group's first step and segment, and S, for the merge.
__device__ __forceinline__ void find_stretch(const SharedParams& p) {
  PxBars* bars = PX_BARS;
  const int lane = threadIdx.x % 32;
  int total = 0;
  bool bad = false;
#pragma unroll 1
  for (int base = 0; base < p.groups; base += 32) {
    const int g = base + lane;
    int n = 0;
    if (g < p.groups) {
      const GroupDims d = group_dims(p, g);
      n = p.kv_heads * head_steps(d, d.nb);
      bad = bad || !group_ok(p, g, blockIdx.x == 0);
    }
    total += __reduce_add_sync(0xffffffffu, n);
  }
  if (__any_sync(0xffffffffu, bad)) {
    if (lane == 0) {
      bars->share = bars->start.left = bars->start.base = 0;
      if (blockIdx.x == 0) p.part_plan[0] = kBadPlan;
    }
    return;
  }
  int share = (total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x);
  // A CTA that goes from one head to the next drains and fills its pipelines
  // once more, about the time of three steps.  So where shares at most one step
  // longer let every head begin on a CTA of its own (its steps padded to whole
  // shares), they do: 64 sequences over 8200 keys 30.3 -> 27.6 us, 48 of two
  // queries over 20000 59.6 -> 52.7, long lines alike.
  int even = 0;
#pragma unroll 1
  for (int longer = 0; longer < 2 && !even; ++longer) {
    int ctas = 0;
#pragma unroll 1
    for (int base = 0; base < p.groups; base += 32) {
      const int g = base + lane;
      int n = 0;
      if (g < p.groups) {
        const GroupDims d = group_dims(p, g);
        n = p.kv_heads * (line_steps(d, share + longer, 1) / max(share + longer, 1));
      }
      ctas += __reduce_add_sync(0xffffffffu, n);
    }
    if (ctas <= static_cast<int>(gridDim.x)) {
      even = 1;
      share += longer;
      total = ctas * share;
    }
  }
  const int first = static_cast<int>(blockIdx.x) * share;
  const int left = min(total, first + share) - first;
  if (lane == 0) {
    bars->share = share;
    bars->start.left = left;
    bars->start.base = 0;  // all that is read of a stretch without steps
    if (blockIdx.x == 0) p.part_plan[0] = even ? -share : share;
  }
  __syncwarp();
  int lin = 0, segs = 0;
#pragma unroll 1
  for (int base = 0; base < p.groups; base += 32) {
    const int g = base + lane;
    int n = 0, t = 0, cl = 1;
    GroupDims d{};
    if (g < p.groups) {
      d = group_dims(p, g);
      if (d.nb > 0) {
        cl = chunk_blocks(d, share);
        t = p.kv_heads * d.mu * ((d.nb + cl - 1) / cl);
        n = p.kv_heads * line_steps(d, share, even);
      }
    }
    int ni = n, ti = t;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, ni, o), b = __shfl_up_sync(0xffffffffu, ti, o);
      if (lane >= o) {
        ni += a;
        ti += b;
      }
    }
    const int l0 = lin + ni - n, t0 = segs + ti - t;
    if (g < p.groups && blockIdx.x == 0) {
      p.part_plan[1 + 2 * g] = l0;
      p.part_plan[2 + 2 * g] = t0;
    }
    if (left > 0 && l0 <= first && first < l0 + n) {  // one lane, once
      Walk w;
      w.d = d;
      w.g = g;
      w.cl = cl;
      int rest = first - l0;
      const int per_head = line_steps(d, share, even), per_chunk = head_steps(d, cl);
      w.h = rest / per_head;
      rest -= w.h * per_head;
      w.left = even ? min(left, head_steps(d, d.nb) - rest) : left;
      w.q = rest / per_chunk;
      rest -= w.q * per_chunk;
      w.len = min(cl, d.nb - w.q * cl);
      w.m = min(rest / w.len, d.mu - 1);
      w.step = rest - w.m * w.len;
      w.steps = unit_steps(d, w.m, w.len);
      w.base = w.alt = 0;
      w.seg = t0 + (w.h * ((d.nb + cl - 1) / cl) + w.q) * d.mu + w.m;
      bars->start = w;
    }
    lin += __shfl_sync(0xffffffffu, ni, 31);
    segs += __shfl_sync(0xffffffffu, ti, 31);
  }
}

// ---------------------------------------------------------------- producer
__device__ __forceinline__ void px_producer(const CUtensorMap* tmK, const CUtensorMap* tmV,
                                            const SharedParams& p) {
  PxBars* bars = PX_BARS;
  uint8_t* sK = px_smem + kPxOffK;
  uint8_t* sV = px_smem + kPxOffV;
  volatile int* abort_flag = &bars->abort_flag;
  const int lane = threadIdx.x % 32;
  Walk w = bars->start;
  uint32_t it = 0;
  bool ok = true;
  while (ok && w.left > 0) {
    const int* table = p.prefix_table + static_cast<size_t>(w.g) * p.prefix_pages;
    const int n_pages = (w.d.plen + kPageKeys - 1) / kPageKeys;
    const int b0 = walk_first(w), b1 = b0 + walk_blocks(w);
    for (int base = b0; ok && base < b1; base += 16) {
      // the page ids of the next 16 blocks, one per lane
      const int pg = 2 * base + lane;
      int id = pg < n_pages ? __ldg(table + pg) : 0;
      if (id < 0 || id >= p.num_pages) {  // reported; page 0 is read in its place
        if (p.err) atomicOr(p.err, kErrBadArgs);
        id = 0;
      }
      for (int j = base; j < min(b1, base + 16); ++j, ++it) {
        const uint32_t s = it % kPxStages;
        if (it >= static_cast<uint32_t>(kPxStages) &&
            !warp_wait(&bars->kv_empty[s], ((it / kPxStages) - 1) & 1, abort_flag, p.err,
                       kErrTimeoutProducer)) {
          ok = false;
          break;
        }
        const int p0 = __shfl_sync(0xffffffffu, id, 2 * (j - base));
        const int p1 = __shfl_sync(0xffffffffu, id, 2 * (j - base) + 1);
        const bool two = 2 * j + 1 < n_pages;
        const uint32_t bytes = two ? 2 * kPxPage : kPxPage;
        mbar_arrive_expect_tx_w(&bars->k_full[s], bytes);
        tma_load_3d_w(sK + s * kPxTile, tmK, &bars->k_full[s], 0, 0, p0 * p.kv_heads + w.h);
        if (two)
          tma_load_3d_w(sK + s * kPxTile + kPxPage, tmK, &bars->k_full[s], 0, 0,
                        p1 * p.kv_heads + w.h);
        mbar_arrive_expect_tx_w(&bars->v_full[s], bytes);
        tma_load_3d_w(sV + s * kPxTile, tmV, &bars->v_full[s], 0, 0, p0 * p.kv_heads + w.h);
        if (two)
          tma_load_3d_w(sV + s * kPxTile + kPxPage, tmV, &bars->v_full[s], 0, 0,
                        p1 * p.kv_heads + w.h);
      }
    }
    walk_next(w, p);
  }
  if (!ok || *abort_flag) {  // every copy lands before the CTA exits
    int none = 0;
    for (uint32_t s = 0; s < static_cast<uint32_t>(kPxStages) && s < it; ++s) {
      const uint32_t arms = (it - 1 - s) / kPxStages + 1;
      mbar_wait(&bars->k_full[s], (arms - 1) & 1, &none, p.err, kErrTimeoutDrain);
      mbar_wait(&bars->v_full[s], (arms - 1) & 1, &none, p.err, kErrTimeoutDrain);
    }
  }
}

// ---------------------------------------------------------------- MMA issuers
// The key blocks of chain t, `it` counted over the CTA's stretch: in a pair
// unit every block, else every second.  The scores of its next block are
// issued before the second product of the current one within a segment.
struct ChainBlock {
  uint32_t it;
  bool first;  // of this chain's blocks in the segment
};

struct ChainWalk {
  const SharedParams& p;
  Walk w;
  int t, pos;  // pos: this chain's blocks of the current segment so far
  __device__ __forceinline__ ChainWalk(const SharedParams& params, int chain)
      : p(params), w(PX_BARS->start), t(chain), pos(0) {}
  // The chain's next block, or false at the end of the stretch.
  __device__ __forceinline__ bool next(ChainBlock& b) {
    while (w.left > 0) {
      const bool pair = walk_pair(w);
      const int j = pair ? pos : 2 * pos + t;
      if (j < walk_blocks(w)) {
        b.it = static_cast<uint32_t>(w.base + j);
        b.first = pos == 0;
        ++pos;
        return true;
      }
      walk_next(w, p);
      pos = 0;
    }
    return false;
  }
};

template <int F16>
__device__ __forceinline__ void px_mma(const SharedParams& p, int t, uint32_t tmem) {
  PxBars* bars = PX_BARS;
  uint8_t* sQ = px_smem;
  uint8_t* sK = px_smem + kPxOffK;
  uint8_t* sV = px_smem + kPxOffV;
  volatile int* abort_flag = &bars->abort_flag;
  constexpr uint32_t idesc_s = idesc_f16(F16 ? 0u : 1u, 128, 128, 0, 0);
  constexpr uint32_t idesc_o = idesc_f16(F16 ? 0u : 1u, 128, 64, 0, 1);
  ChainWalk walk(p, t);
  uint32_t n_s = 0, n_pv = 0;
  uint32_t n_q = 0;   // segments of this chain
  uint32_t seen = 0;  // blocks taken or passed
  // Blocks of the other chain alone are passed, not skipped: a wait by parity
  // holds only for who has seen the barrier's every phase, and a stage is
  // loaded again once both chains have seen it.
  auto pass = [&](uint32_t to) -> bool {
    for (; seen < to; ++seen) {
      const uint32_t s = seen % kPxStages, parity = (seen / kPxStages) & 1;
      if (!warp_wait(&bars->k_full[s], parity, abort_flag, p.err, kErrTimeoutMma) ||
          !warp_wait(&bars->v_full[s], parity, abort_flag, p.err, kErrTimeoutMma))
        return false;
      mbar_arrive_w(&bars->kv_empty[s]);
    }
    return true;
  };
  auto issue_s = [&](const ChainBlock& b) -> bool {
    const uint32_t s = b.it % kPxStages;
    if (!pass(b.it)) return false;
    ++seen;
    if (!warp_wait(&bars->k_full[s], (b.it / kPxStages) & 1, abort_flag, p.err, kErrTimeoutMma))
      return false;
    if (b.first && !warp_wait(&bars->q_full[t], n_q++ & 1, abort_flag, p.err, kErrTimeoutMma))
      return false;
    if (n_s > 0 &&
        !warp_wait(&bars->sc_done[t], (n_s - 1) & 1, abort_flag, p.err, kErrTimeoutMma))
      return false;
    tc_fence_after();
    const uint64_t dq = smem_desc_sw128(smem_u32(sQ + t * kPxTile), 16, 1024);
    const uint64_t dk = smem_desc_sw128(smem_u32(sK + s * kPxTile), 16, 1024);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      mma_ss_w(tmem + kPxS + t * 128, dq + 2 * k, dk + 2 * k, idesc_s, k > 0 ? 1u : 0u);
    mma_commit_w(&bars->s_full[t]);
    ++n_s;
    return true;
  };
  ChainBlock cur, nxt;
  bool more = walk.next(cur);
  if (more && !issue_s(cur)) return;
  while (more) {
    more = walk.next(nxt);
    // Within a segment the next scores go first; across segments the last
    // product does, since the segment's epilogue waits for it.
    const bool ahead = more && !nxt.first;
    if (ahead && !issue_s(nxt)) return;
    const uint32_t s = cur.it % kPxStages;
    if (!warp_wait(&bars->v_full[s], (cur.it / kPxStages) & 1, abort_flag, p.err, kErrTimeoutMma))
      return;
    if (!warp_wait(&bars->p_full[t], n_pv & 1, abort_flag, p.err, kErrTimeoutMma)) return;
    tc_fence_after();
    const uint64_t dv = smem_desc_sw128(smem_u32(sV + s * kPxTile), 8192, 1024);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      mma_ts_w(tmem + kPxO + t * 64, tmem + kPxP + t * 64 + k * 8, dv + k * (2048 >> 4), idesc_o,
               (!cur.first || k > 0) ? 1u : 0u);
    mma_commit_w(&bars->o_done[t]);
    mma_commit_w(&bars->kv_empty[s]);
    ++n_pv;
    if (more && !ahead && !issue_s(nxt)) return;
    cur = nxt;
  }
  pass(static_cast<uint32_t>(walk.w.base));
}

// ---------------------------------------------------------------- softmax
// Rows of a tile: row r (0..127) sits at MMA row 32 (c % 4) + 16 (c / 4) + r %
// 16 with c = r / 16, so softmax warp c of a chain owns rows 16 c .. and few
// rows spread over the four scheduler quarters.
__device__ __forceinline__ int mma_row(int r) {
  const int c = r >> 4;
  return 32 * (c & 3) + 16 * (c >> 2) + (r & 15);
}

// Query rows [row0, row0 + rows) of the unit's group and head into swizzled
// shared memory, zeros behind them: 256 threads, four 16-byte pieces (8 head
// dims) each.  Rolled, with copies that hold no register: the code runs once a
// segment, and what it costs is fetching its instructions.
__device__ __forceinline__ void load_q(const SharedParams& p, const Walk& w, int row0, int rows,
                                       uint8_t* dst) {
  const int G = p.heads / p.kv_heads, R = p.q_len * G;
  const int c = threadIdx.x & 7;
#pragma unroll 1
  for (int r = (threadIdx.x & 255) >> 3; r < 128; r += 32) {
    const bool have = r < rows;
    const int row = have ? row0 + r : row0;
    const int b = row / R, rr = row - b * R, tok = rr / G, h = w.h * G + rr - tok * G;
    const size_t off = static_cast<size_t>(w.d.b0 + b) * p.q_sb + static_cast<size_t>(tok) * p.q_st +
                       static_cast<size_t>(h) * p.q_sh + c * 8;
    const int mr = mma_row(r);
    uint8_t* to = dst + mr * 128 + ((c ^ (mr & 7)) << 4);
    if (p.q_dtype == 0) {  // f32 queries are rounded to the cache's type
      const float4* src = reinterpret_cast<const float4*>(static_cast<const float*>(p.q) + off);
      const float4 a = __ldg(src), e = __ldg(src + 1);
      uint4 x = p.kv_dtype == 2 ? make_uint4(pack_f16x2(a.x, a.y), pack_f16x2(a.z, a.w),
                                             pack_f16x2(e.x, e.y), pack_f16x2(e.z, e.w))
                                : make_uint4(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w),
                                             pack_bf16x2(e.x, e.y), pack_bf16x2(e.z, e.w));
      *reinterpret_cast<uint4*>(to) = have ? x : make_uint4(0, 0, 0, 0);
    } else {
      cp_async16(to, static_cast<const uint16_t*>(p.q) + off, have);
    }
  }
  cp_async_wait_all();
}

template <int F16>
__device__ __forceinline__ void px_softmax(const SharedParams& p, uint32_t tmem) {
  PxBars* bars = PX_BARS;
  uint8_t* sQ = px_smem;
  uint8_t* sV = px_smem + kPxOffV;
  float* s_merge = reinterpret_cast<float*>(px_smem + kPxOffMerge);
  Walk& w = *(reinterpret_cast<Walk*>(px_smem + kPxOffWalks) + threadIdx.x / 32);
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int t = warp / 8, c = warp % 8;
  const int lb = 32 * (c % 4) + 16 * (c / 4);
  const int t0 = lane & 3, t1 = lane >> 2;
  // this warp's lanes and chain: weights at tP, scores and accumulator from it
  const uint32_t tP = tmem + (static_cast<uint32_t>(lb) << 16) + kPxP + t * 64;
  const uint32_t tS = tP + kPxS - kPxP + t * 64;
  const uint32_t tO = tP + kPxO - kPxP;
  float* mbuf = s_merge + c * kPxMergeFloats;
  uint32_t n_s = 0;    // blocks of this chain so far
  for (uint32_t i = lane; i < sizeof(Walk) / 4; i += 32)
    reinterpret_cast<int*>(&w)[i] = reinterpret_cast<const int*>(&bars->start)[i];
  __syncwarp();

  while (w.left > 0) {
    const bool pair = walk_pair(w);
    // this chain's blocks: all, or every second one (none of a single one for chain 1)
    const int cnt = pair ? walk_blocks(w) : (walk_blocks(w) + 1 - t) >> 1;
    const bool any = cnt > 0;
    const int row0 = w.m * kPxRows + (pair ? 128 * t : 0);
    const int rows = min(128, w.d.rows - row0);  // of this chain's tile
    if (any) {
      // The chain's last segment is done (its last product was waited for), so
      // its query buffer is free.
      load_q(p, w, row0, rows, sQ + t * kPxTile);
      fence_proxy_async_smem();
      mbar_arrive(&bars->q_full[t]);
    }
    const bool active = 16 * c < rows;  // warp-uniform: some row of this warp is real
    float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
#pragma unroll 1
    for (int i = 0; i < cnt; ++i, ++n_s) {
      if (!warp_wait(&bars->s_full[t], n_s & 1, abort_flag, p.err, kErrTimeoutSoftmax)) return;
      tc_fence_after();
      int live = kPxKeys;  // keys of this block that exist; fewer in a prefix's last block only
      if (i == cnt - 1) {
        const int j = pair ? i : 2 * i + t;
        live = w.d.plen - (walk_first(w) + j) * kPxKeys;
        if (live < kPxKeys) {
          // Value rows behind the last live key may hold anything (a weight
          // of 0 times a NaN is a NaN): the chain's 256 threads zero them
          // before the second product.
          const uint32_t it = static_cast<uint32_t>(w.base + j), st = it % kPxStages;
          if (!warp_wait(&bars->v_full[st], (it / kPxStages) & 1, abort_flag, p.err,
                         kErrTimeoutSoftmax))
            return;
          uint4* v = reinterpret_cast<uint4*>(sV + st * kPxTile);
          for (int k = live * 8 + (threadIdx.x & 255); k < kPxKeys * 8; k += 256)
            v[k] = make_uint4(0, 0, 0, 0);
          fence_proxy_async_smem();
        }
      }
      if (!active) {
        tc_fence_before();
        mbar_arrive(&bars->sc_done[t]);
        // the previous product must have left P before it is declared full again
        if (n_s > 0 &&
            !warp_wait(&bars->o_done[t], (n_s - 1) & 1, abort_flag, p.err, kErrTimeoutSoftmax))
          return;
        mbar_arrive(&bars->p_full[t]);
        continue;
      }
      uint32_t sr[64];
      tmem_ld_16x256b_x16(tS, sr);
      tmem_wait_ld();
      tc_fence_before();
      mbar_arrive(&bars->sc_done[t]);
      float* sf = reinterpret_cast<float*>(sr);
      if (live < kPxKeys) {
#pragma unroll
        for (int k = 0; k < 16; ++k)
#pragma unroll
          for (int x = 0; x < 2; ++x)
            if (8 * k + 2 * t0 + x >= live) sf[4 * k + x] = sf[4 * k + 2 + x] = -INFINITY;
      }
      float mx[2];
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        float a = fmaxf(sf[2 * v], sf[2 * v + 1]), b = fmaxf(sf[4 + 2 * v], sf[4 + 2 * v + 1]);
#pragma unroll
        for (int k = 2; k < 16; k += 2) {
          a = max3f(a, sf[4 * k + 2 * v], sf[4 * k + 2 * v + 1]);
          b = max3f(b, sf[4 * k + 4 + 2 * v], sf[4 * k + 4 + 2 * v + 1]);
        }
        mx[v] = fmaxf(a, b);
      }
      // The reference value of a row moves only when the maximum outgrows it
      // by 2^8: weights stay below 2^8 and most blocks never rescale.
      if (__any_sync(0xffffffffu, mx[0] * p.scale_log2 > m_run[0] + 8.0f ||
                                      mx[1] * p.scale_log2 > m_run[1] + 8.0f)) {
        float corr[2] = {1.f, 1.f};
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          mx[v] = fmaxf(mx[v], __shfl_xor_sync(0xffffffffu, mx[v], 1));
          mx[v] = fmaxf(mx[v], __shfl_xor_sync(0xffffffffu, mx[v], 2));
          const float m_blk = mx[v] * p.scale_log2;
          if (m_blk > m_run[v] + 8.0f) {
            const float m_new = ceilf(m_blk);
            corr[v] = ex2_approx(m_run[v] - m_new);
            m_run[v] = m_new;
            l_run[v] *= corr[v];
          }
        }
        if (i > 0) {  // the accumulator so far, once the last product is in it
          if (!warp_wait(&bars->o_done[t], (n_s - 1) & 1, abort_flag, p.err, kErrTimeoutSoftmax))
            return;
          tc_fence_after();
#pragma unroll 1
          for (int h = 0; h < 8; ++h) {
            uint32_t o4[4];
            tmem_ld_16x256b_x1(tO + 8 * h, o4);
            tmem_wait_ld_regs4(o4);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              o4[e] = __float_as_uint(__uint_as_float(o4[e]) * corr[e >> 1]);
            tmem_st_16x256b_x1(tO + 8 * h, o4);
          }
          tmem_wait_st();
        }
      }
      // weights in pairs; the sum takes them unrounded, the product in 16 bits
      uint32_t pk[32];
      {
        const uint64_t c2 = f2_pack(p.scale_log2, p.scale_log2);
        uint64_t neg_m[2];  // (0 while every score was -inf)
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          const float n = m_run[v] == -INFINITY ? 0.f : -m_run[v];
          neg_m[v] = f2_pack(n, n);
        }
        uint64_t acc[2];
#pragma unroll
        for (int v = 0; v < 2; ++v) acc[v] = f2_pack(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < 16; ++k) {
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            float x0, x1;
            f2_unpack(f2_fma(f2_pack(sf[4 * k + 2 * v], sf[4 * k + 2 * v + 1]), c2, neg_m[v]), x0,
                      x1);
            const float p0 = ex2_approx(x0), p1 = ex2_approx(x1);
            pk[2 * k + v] = F16 ? pack_f16x2(p0, p1) : pack_bf16x2(p0, p1);
            acc[v] = f2_add(acc[v], f2_pack(p0, p1));
          }
        }
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          float a, b;
          f2_unpack(acc[v], a, b);
          l_run[v] += a + b;
        }
      }
      // P is free once the previous product has read it
      if (n_s > 0 &&
          !warp_wait(&bars->o_done[t], (n_s - 1) & 1, abort_flag, p.err, kErrTimeoutSoftmax))
        return;
      tc_fence_after();
      tmem_st_16x128b_x16(tP, pk);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&bars->p_full[t]);
    }

    // ---- end of the segment's stretch
    if (any && !warp_wait(&bars->o_done[t], (n_s - 1) & 1, abort_flag, p.err, kErrTimeoutSoftmax))
      return;
    tc_fence_after();
    if (active) {
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        l_run[v] += __shfl_xor_sync(0xffffffffu, l_run[v], 1);
        l_run[v] += __shfl_xor_sync(0xffffffffu, l_run[v], 2);
      }
    }
    // One tile for both chains: chain 1 hands over to chain 0.  (A pair of
    // warps without rows hands over nothing, but keeps the barriers' count.)
    // The accumulator is moved eight registers (16 columns) at a time.
    if (!pair && t == 1) {
      if (w.alt >= 1 && !warp_wait(&bars->mrg_empty[c], (w.alt - 1) & 1, abort_flag, p.err,
                                   kErrTimeoutSoftmax))
        return;
      if (active) {
        if (any) {
#pragma unroll 1
          for (int h = 0; h < 4; ++h) {
            uint32_t o8[8];
            tmem_ld_16x256b_x2(tO + 16 * h, o8);
            tmem_wait_ld_regs8(o8);
#pragma unroll
            for (int e = 0; e < 8; ++e) mbuf[(8 * h + e) * 32 + lane] = __uint_as_float(o8[e]);
          }
        }
        if (t0 == 0) {
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            mbuf[32 * 32 + 2 * (t1 + 8 * v)] = m_run[v];
            mbuf[32 * 32 + 2 * (t1 + 8 * v) + 1] = l_run[v];
          }
        }
      }
      mbar_arrive(&bars->mrg_full[c]);
    } else {
      float f0[2] = {1.f, 1.f}, f1[2] = {0.f, 0.f};
      if (!pair) {
        if (!warp_wait(&bars->mrg_full[c], w.alt & 1, abort_flag, p.err, kErrTimeoutSoftmax)) return;
        if (active) {
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            const int r = t1 + 8 * v;
            const float m1 = mbuf[32 * 32 + 2 * r], l1 = mbuf[32 * 32 + 2 * r + 1];
            const float M = fmaxf(m_run[v], m1);
            // a chain without blocks here has m = -inf: its accumulator is
            // stale and its factor, 0, marks it as not used
            f0[v] = m_run[v] == -INFINITY ? 0.f : ex2_approx(m_run[v] - M);
            f1[v] = m1 == -INFINITY ? 0.f : ex2_approx(m1 - M);
            m_run[v] = M;
            l_run[v] = l_run[v] * f0[v] + l1 * f1[v];
          }
        }
      }
      const int slot = static_cast<int>(blockIdx.x) + w.seg;
      if (active && slot >= p.part_slots) {  // the workspace's size rules it out
        if (p.err && lane == 0) atomicOr(p.err, kErrNoSlot);
      } else if (active) {
        const size_t at = static_cast<size_t>(slot) * kPxRows + (pair ? 128 * t : 0) + 16 * c + t1;
        float* dst = p.part_o + at * 64 + 2 * t0;
#pragma unroll 1
        for (int h = 0; h < 4; ++h) {
          uint32_t o8[8];
          if (any) {
            tmem_ld_16x256b_x2(tO + 16 * h, o8);
            tmem_wait_ld_regs8(o8);
          }
#pragma unroll
          for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int v = 0; v < 2; ++v) {
              float o[2];
#pragma unroll
              for (int x = 0; x < 2; ++x) {
                const int e = 4 * k + 2 * v + x;
                o[x] = f0[v] > 0.f ? __uint_as_float(o8[e]) * f0[v] : 0.f;
                if (f1[v] > 0.f) o[x] = fmaf(mbuf[(8 * h + e) * 32 + lane], f1[v], o[x]);
              }
              if (16 * c + t1 + 8 * v < rows)
                *reinterpret_cast<float2*>(dst + 8 * v * 64 + 16 * h + 8 * k) = make_float2(o[0], o[1]);
            }
        }
        if (t0 == 0) {
#pragma unroll
          for (int v = 0; v < 2; ++v)
            if (16 * c + t1 + 8 * v < rows)
              *reinterpret_cast<float2*>(p.part_ml + 2 * (at + 8 * v)) = make_float2(m_run[v], l_run[v]);
        }
      }
      if (!pair) mbar_arrive(&bars->mrg_empty[c]);
    }
    tc_fence_before();
    __syncwarp();
    if (lane == 0) walk_next(w, p);
    __syncwarp();
  }
}

template <int F16>
__global__ void __launch_bounds__(kPxThreads, 1)
    prefix_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                     const SharedParams p) {
  if (smem_u32(px_smem) % 1024 != 0) {  // the whole grid alike
    if (threadIdx.x == 0 && p.err) atomicOr(p.err, kErrBadArgs);
    return;
  }
  PxBars* bars = PX_BARS;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  if (warp == kPxMma0) {
    find_stretch(p);
  } else if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&bars->q_full[t], 256);
      mbar_init(&bars->s_full[t], 1);
      mbar_init(&bars->sc_done[t], 256);
      mbar_init(&bars->p_full[t], 256);
      mbar_init(&bars->o_done[t], 1);
    }
    for (int s = 0; s < kPxStages; ++s) {
      mbar_init(&bars->k_full[s], 1);
      mbar_init(&bars->v_full[s], 1);
      mbar_init(&bars->kv_empty[s], 2);
    }
    for (int c = 0; c < 8; ++c) {
      mbar_init(&bars->mrg_full[c], 32);
      mbar_init(&bars->mrg_empty[c], 32);
    }
    mbar_init(&bars->drain, 2);
    bars->abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == kPxProducer) {
    tmem_alloc(&bars->tmem_base, kPxTmem);
    tmem_relinquish();
  }
  if (warp == kPxMma0 + 1 && lane == 0) {
    prefetch_tensormap(&tmK);
    prefetch_tensormap(&tmV);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;
  // every CTA is resident: the rows kernel may start on what this one leaves
  griddep_launch_dependents();

  if (warp == kPxProducer) {
    px_producer(&tmK, &tmV, p);
  } else if (warp >= kPxMma0) {
    px_mma<F16>(p, warp - kPxMma0, tmem);
    int none = 0;  // every MMA issued has finished before tensor memory is freed
    mma_commit_w(&bars->drain);
    mbar_wait(&bars->drain, 0, &none, p.err, kErrTimeoutDrain);
  } else {
    px_softmax<F16>(p, tmem);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == kPxProducer) {
    tc_fence_after();
    tmem_dealloc(tmem, kPxTmem);
  }
}

}  // namespace

cudaError_t launch_prefix_tc(const CUtensorMap& tmK, const CUtensorMap& tmV, const SharedParams& p,
                             int grid, cudaStream_t s) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  static std::atomic<bool> configured[2][64];
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  const int which = p.kv_dtype == 2;
  auto kern = which ? prefix_tc_kernel<1> : prefix_tc_kernel<0>;
  if (!configured[which][dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(kPxSmem));
    if (e != cudaSuccess) return e;
    configured[which][dev].store(true, std::memory_order_release);
  }
  kern<<<grid, kPxThreads, kPxSmem, s>>>(tmK, tmV, p);
  return cudaGetLastError();
}

}  // namespace ffai

// Attention of a chunk of new tokens over a paged KV cache on the tensor cores:
// sequences with many query rows (the mathematics: chunk_rows.cu).
//
// A unit is 256 of a (sequence, KV head)'s rows, ordered by (token, head within
// the group): two tiles of 128, the M of tcgen05.mma, that share every block of
// 128 keys (two pages), so a page is fetched once for 256 rows.  A unit passes over the
// blocks its last row sees.  The steps of all units lie on one line (chunk.cuh),
// and CTA c takes an equal stretch of it, whatever the lengths and however the
// chunks and the single tokens mix.  What a CTA holds of a unit is finished there
// if it is all of it, else left as a partial result for the last of the unit's CTAs
// to come.
//
// Per CTA: warp 16 streams the pages through a 4-stage ring of K and V blocks by TMA
// for two chains (t = 0, 1), each with an MMA warp (17, 18), scores, weights and an
// output accumulator of its own in tensor memory and 8 softmax warps, so one
// chain's softmax runs beside the other's products.  With more than 128 rows in the
// unit chain t takes tile t and both take every block; else both hold the one tile
// and take the blocks in turn (chain 0 the even ones), and at the end chain 1 hands
// its accumulator to chain 0 through shared memory, warp to warp.
//
// The blocks at the diagonal hold values that some rows of a tile see and others do
// not.  A weight of 0 would turn a value that is not finite into a NaN, so the chain
// looks at those rows of V first; if there is one, it is added to the rows that see
// it, and the product takes a copy of the block with zeros in its place.
//
// Bound by the exponentials, one a score on the 16-lane unit, and the moves between
// tensor memory and registers around them: chunks of prompts, 32 / 8 heads,
// bf16: one of 8192 behind 24000 keys 2.53 ms, 748 TFLOP/s, 1.66 us a step of
// 256 rows and 128 keys (1.07 of it the exponentials, 0.8 the products); one of 8192 behind
// 3000 and one of 2731 behind 24000 1.59 ms, 655 TFLOP/s.
//
// Every wait is bounded (common.cuh); on a timeout the CTA raises an error bit,
// drains its copies and MMAs, takes the tickets it has not come to, frees tensor
// memory and exits.
#include <atomic>

#include "chunk.cuh"

namespace ffai {

namespace {

constexpr int kCtStages = 4;
constexpr int kCtThreads = 608;  // 16 softmax warps, TMA warp, 2 MMA warps
constexpr int kCtProducer = 16, kCtMma0 = 17;
constexpr uint32_t kCtTile = 128 * 128;        // 128 rows of 128 bytes
constexpr uint32_t kCtPage = kPageKeys * 128;  // a page's rows of one head
constexpr uint32_t kCtTmem = 512;
constexpr uint32_t kCtS = 0, kCtP = 256, kCtO = 384;  // + 128 t, + 64 t, + 64 t

// A walk over a CTA's stretch of the line, unit by unit.
struct Walk {
  ChunkSeq s;
  int b, h, m;      // sequence, KV head, unit
  int rows, nb;     // of the unit: rows, key blocks
  int steps, step;  // of the unit, and the current one
  int left;         // steps left, the current one included
  int unit0;        // the unit's first step on the line
  int base;         // key blocks of this CTA before this unit
  int alt;          // one-tile units of this CTA before this one
};
__device__ __forceinline__ bool walk_pair(const Walk& w) { return w.rows > 128; }
// What this CTA has of the current unit: steps, key blocks, the first block.
__device__ __forceinline__ int walk_steps(const Walk& w) { return min(w.left, w.steps - w.step); }
__device__ __forceinline__ int walk_blocks(const Walk& w) {
  const int n = walk_steps(w);
  return walk_pair(w) ? n : min(2 * n, w.nb - 2 * w.step);
}
__device__ __forceinline__ int walk_first(const Walk& w) { return walk_pair(w) ? w.step : 2 * w.step; }
// The unit's sizes.
__device__ __forceinline__ void walk_unit(Walk& w, const ChunkParams& p) {
  const int G = p.heads / p.kv_heads, end = min((w.m + 1) * kPxRows, w.s.n * G);
  w.rows = end - w.m * kPxRows;
  w.nb = chunk_blocks<kChKeys>(chunk_limit(p, w.s, (end - 1) / G));
  w.steps = walk_pair(w) ? w.nb : (w.nb + 1) >> 1;
}
// To the next unit, if the stretch goes on.
__device__ __forceinline__ void walk_next(Walk& w, const ChunkParams& p) {
  w.base += walk_blocks(w);
  w.alt += walk_pair(w) ? 0 : 1;
  w.left -= walk_steps(w);
  if (w.left <= 0) return;  // else the unit is done
  w.unit0 += w.steps;
  w.step = 0;
  if (++w.m == chunk_units<kPxRows>(w.s, p.heads / p.kv_heads)) {
    w.m = 0;
    if (++w.h == p.kv_heads) {
      w.h = 0;
      w.s.n = 0;
      bool bad = false;
      while (w.s.n == 0 && ++w.b < p.batch) w.s = chunk_seq(p, w.b, bad);
      if (w.s.n == 0) {  // (never, unless the lengths are written meanwhile)
        w.left = 0;
        return;
      }
    }
  }
  walk_unit(w, p);
}

// The first and the last CTA that have a part of the unit; it is one's whole where they
// are the same.  Else each takes a ticket for each of its tiles (one chain's, if there is
// one tile), and the last to take it merges the parts.
struct UnitTeams {
  int c0, c1;
};
__device__ __forceinline__ UnitTeams walk_teams(const Walk& w, int share) {
  return {w.unit0 / share, min((w.unit0 + w.steps - 1) / share, static_cast<int>(gridDim.x) - 1)};
}
__device__ __forceinline__ bool walk_whole(const Walk& w) { return walk_steps(w) == w.steps; }
__device__ __forceinline__ bool take_ticket(const ChunkParams& p, const Walk& w, const UnitTeams& u, int t) {
  const unsigned n = static_cast<unsigned>(u.c1 - u.c0);
  return atomicInc(p.tickets + 2 * u.c0 + (walk_pair(w) ? t : 0), n) == n;
}
// A wait of chain t ran out: one of its threads takes the tickets that it has not come
// to (not the current unit's, if `taken`), since those of the other CTAs would stay in
// the words and mislead the calls behind this one.  (Whoever is the last now merges what
// this CTA never wrote: the call is reported.)
__device__ __noinline__ void take_the_rest(const ChunkParams& p, Walk& w, int share, int t, bool taken) {
  for (; w.left > 0; walk_next(w, p), taken = false)
    if (!taken && !walk_whole(w) && (walk_pair(w) || t == 0)) take_ticket(p, w, walk_teams(w, share), t);
}

struct __align__(8) CtBars {
  uint64_t q_full[2];
  uint64_t k_full[kCtStages], v_full[kCtStages], kv_empty[kCtStages];
  uint64_t s_full[2], sc_done[2], p_full[2], o_done[2];
  uint64_t sync[2];  // a chain's softmax warps among themselves
  uint64_t mrg_full[8], mrg_empty[8];
  uint64_t drain;
  uint32_t tmem_base;
  int abort_flag;
  int share;
  int odd[2];   // the chain's block (counted from 1) that holds values that are not finite
  int copy[2];  // 1: the product takes the chain's copy of V
  int keep[2];  // 1: it adds to the accumulator although it is the unit's first
  int last[2];  // 1: this CTA merges the tile
  Walk start;   // this CTA's stretch
};

// Shared memory, at fixed offsets from its 1024-byte aligned start (which the
// kernel checks), so that no pointer into it takes a register.
constexpr uint32_t kCtOffK = 2 * kCtTile;  // after the chains' query tiles
constexpr uint32_t kCtOffV = kCtOffK + kCtStages * kCtTile;
constexpr uint32_t kCtOffCopy = kCtOffV + kCtStages * kCtTile;  // a copy of V per chain
constexpr uint32_t kCtOffMerge = kCtOffCopy + 2 * kCtTile;
constexpr uint32_t kCtMergeFloats = 32 * 32 + 32;  // per pair of warps
constexpr uint32_t kCtOffWalks = kCtOffMerge + 8 * kCtMergeFloats * sizeof(float);
constexpr uint32_t kCtOffBars = (kCtOffWalks + 16 * sizeof(Walk) + 7) / 8 * 8;
constexpr size_t kCtSmem = kCtOffBars + sizeof(CtBars);
static_assert(sizeof(Walk) % 4 == 0 && kCtSmem <= 227 * 1024, "shared memory");
extern __shared__ __align__(1024) uint8_t ct_smem[];
#define CT_BARS (reinterpret_cast<CtBars*>(ct_smem + kCtOffBars))

__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                                          unsigned* err, unsigned code) {
  const bool ok = mbar_wait(bar, parity, abort_flag, err, code);
  return __all_sync(0xffffffffu, ok);
}

// ---------------------------------------------------------------- producer
__device__ __forceinline__ void ct_producer(const CUtensorMap* tmK, const CUtensorMap* tmV,
                                            const ChunkParams& p) {
  CtBars* bars = CT_BARS;
  uint8_t* sK = ct_smem + kCtOffK;
  uint8_t* sV = ct_smem + kCtOffV;
  volatile int* abort_flag = &bars->abort_flag;
  const int lane = threadIdx.x % 32;
  Walk w = bars->start;
  uint32_t it = 0;
  bool ok = true;
  while (ok && w.left > 0) {
    const int* table = p.block_table + static_cast<size_t>(w.b) * p.max_pages;
    const int n_pages = (w.s.len + kPageKeys - 1) / kPageKeys;
    const int b0 = walk_first(w), b1 = b0 + walk_blocks(w);
    for (int base = b0; ok && base < b1; base += 16) {
      // the page ids of the next 16 blocks, one per lane
      const int pg = 2 * base + lane;
      int id = pg < n_pages && pg < 2 * b1 ? __ldg(table + pg) : 0;
      if (id < 0 || id >= p.num_pages) {  // reported; page 0 is read in its place
        if (p.err) atomicOr(p.err, kErrBadArgs);
        id = 0;
      }
      for (int j = base; j < min(b1, base + 16); ++j, ++it) {
        const uint32_t s = it % kCtStages;
        if (it >= static_cast<uint32_t>(kCtStages) &&
            !warp_wait(&bars->kv_empty[s], ((it / kCtStages) - 1) & 1, abort_flag, p.err,
                       kErrTimeoutProducer)) {
          ok = false;
          break;
        }
        const int p0 = __shfl_sync(0xffffffffu, id, 2 * (j - base));
        const int p1 = __shfl_sync(0xffffffffu, id, 2 * (j - base) + 1);
        const bool two = 2 * j + 1 < n_pages;
        const uint32_t bytes = two ? 2 * kCtPage : kCtPage;
        mbar_arrive_expect_tx_w(&bars->k_full[s], bytes);
        tma_load_3d_w(sK + s * kCtTile, tmK, &bars->k_full[s], 0, 0, p0 * p.kv_heads + w.h);
        if (two)
          tma_load_3d_w(sK + s * kCtTile + kCtPage, tmK, &bars->k_full[s], 0, 0,
                        p1 * p.kv_heads + w.h);
        mbar_arrive_expect_tx_w(&bars->v_full[s], bytes);
        tma_load_3d_w(sV + s * kCtTile, tmV, &bars->v_full[s], 0, 0, p0 * p.kv_heads + w.h);
        if (two)
          tma_load_3d_w(sV + s * kCtTile + kCtPage, tmV, &bars->v_full[s], 0, 0,
                        p1 * p.kv_heads + w.h);
      }
    }
    walk_next(w, p);
  }
  // Every copy lands before the CTA exits, whether a wait has run out by now, will
  // run out yet, or none does.
  int none = 0;
  for (uint32_t s = 0; s < static_cast<uint32_t>(kCtStages) && s < it; ++s) {
    const uint32_t arms = (it - 1 - s) / kCtStages + 1;
    mbar_wait(&bars->k_full[s], (arms - 1) & 1, &none, p.err, kErrTimeoutDrain);
    mbar_wait(&bars->v_full[s], (arms - 1) & 1, &none, p.err, kErrTimeoutDrain);
  }
}

// ---------------------------------------------------------------- MMA issuers
// The key blocks of chain t, `it` counted over the CTA's stretch: in a pair
// unit every block, else every second.  The scores of its next block are
// issued before the second product of the current one within a unit.
struct ChainBlock {
  uint32_t it;
  bool first;  // of this chain's blocks in the unit
};

struct ChainWalk {
  const ChunkParams& p;
  Walk w;
  int t, pos;  // pos: this chain's blocks of the current unit so far
  __device__ __forceinline__ ChainWalk(const ChunkParams& params, int chain)
      : p(params), w(CT_BARS->start), t(chain), pos(0) {}
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
__device__ __forceinline__ void ct_mma(const ChunkParams& p, int t, uint32_t tmem) {
  CtBars* bars = CT_BARS;
  uint8_t* sQ = ct_smem;
  uint8_t* sK = ct_smem + kCtOffK;
  uint8_t* sV = ct_smem + kCtOffV;
  volatile int* abort_flag = &bars->abort_flag;
  constexpr uint32_t idesc_s = idesc_f16(F16 ? 0u : 1u, 128, 128, 0, 0);
  constexpr uint32_t idesc_o = idesc_f16(F16 ? 0u : 1u, 128, 64, 0, 1);
  ChainWalk walk(p, t);
  uint32_t n_s = 0, n_pv = 0;
  uint32_t n_q = 0;   // units of this chain
  uint32_t seen = 0;  // blocks taken or passed
  // Blocks of the other chain alone are passed, not skipped: a wait by parity
  // holds only for who has seen the barrier's every phase, and a stage is
  // loaded again once both chains have seen it.
  auto pass = [&](uint32_t to) -> bool {
    for (; seen < to; ++seen) {
      const uint32_t s = seen % kCtStages, parity = (seen / kCtStages) & 1;
      if (!warp_wait(&bars->k_full[s], parity, abort_flag, p.err, kErrTimeoutMma) ||
          !warp_wait(&bars->v_full[s], parity, abort_flag, p.err, kErrTimeoutMma))
        return false;
      mbar_arrive_w(&bars->kv_empty[s]);
    }
    return true;
  };
  auto issue_s = [&](const ChainBlock& b) -> bool {
    const uint32_t s = b.it % kCtStages;
    if (!pass(b.it)) return false;
    ++seen;
    if (!warp_wait(&bars->k_full[s], (b.it / kCtStages) & 1, abort_flag, p.err, kErrTimeoutMma))
      return false;
    if (b.first && !warp_wait(&bars->q_full[t], n_q++ & 1, abort_flag, p.err, kErrTimeoutMma))
      return false;
    if (n_s > 0 &&
        !warp_wait(&bars->sc_done[t], (n_s - 1) & 1, abort_flag, p.err, kErrTimeoutMma))
      return false;
    tc_fence_after();
    const uint64_t dq = smem_desc_sw128(smem_u32(sQ + t * kCtTile), 16, 1024);
    const uint64_t dk = smem_desc_sw128(smem_u32(sK + s * kCtTile), 16, 1024);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      mma_ss_w(tmem + kCtS + t * 128, dq + 2 * k, dk + 2 * k, idesc_s, k > 0 ? 1u : 0u);
    mma_commit_w(&bars->s_full[t]);
    ++n_s;
    return true;
  };
  ChainBlock cur, nxt;
  bool more = walk.next(cur);
  if (more && !issue_s(cur)) return;
  while (more) {
    more = walk.next(nxt);
    // Within a unit the next scores go first; across units the last product
    // does, since the unit's epilogue waits for it.
    const bool ahead = more && !nxt.first;
    if (ahead && !issue_s(nxt)) return;
    const uint32_t s = cur.it % kCtStages;
    if (!warp_wait(&bars->v_full[s], (cur.it / kCtStages) & 1, abort_flag, p.err, kErrTimeoutMma))
      return;
    if (!warp_wait(&bars->p_full[t], n_pv & 1, abort_flag, p.err, kErrTimeoutMma)) return;
    tc_fence_after();
    const uint8_t* v = *static_cast<volatile int*>(&bars->copy[t]) ? ct_smem + kCtOffCopy + t * kCtTile
                                                                   : sV + s * kCtTile;
    const bool add = !cur.first || *static_cast<volatile int*>(&bars->keep[t]);
    const uint64_t dv = smem_desc_sw128(smem_u32(v), 8192, 1024);
#pragma unroll
    for (int k = 0; k < 8; ++k)
      mma_ts_w(tmem + kCtO + t * 64, tmem + kCtP + t * 64 + k * 8, dv + k * (2048 >> 4), idesc_o,
               (add || k > 0) ? 1u : 0u);
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

// Query rows [row0, row0 + rows) of the unit's sequence and head into swizzled
// shared memory, zeros behind them: 256 threads, four 16-byte pieces (8 head
// dims) each.
__device__ __forceinline__ void load_q(const ChunkParams& p, const Walk& w, int row0, int rows,
                                       uint8_t* dst) {
  const int G = p.heads / p.kv_heads;
  const int c = threadIdx.x & 7;
#pragma unroll 1
  for (int r = (threadIdx.x & 255) >> 3; r < 128; r += 32) {
    const bool have = r < rows;
    const int row = have ? row0 + r : row0;
    const int tok = row / G, h = w.h * G + row - tok * G;
    const size_t off = static_cast<size_t>(w.s.t0 + tok) * p.q_st + static_cast<size_t>(h) * p.q_sh + c * 8;
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

// The rest of a chain meets here (bounded, like every wait): its 256 threads.
__device__ __forceinline__ bool chain_sync(uint64_t* bar, uint32_t& n, volatile int* abort_flag, unsigned* err) {
  mbar_arrive(bar);
  return warp_wait(bar, n++ & 1, abort_flag, err, kErrTimeoutSoftmax);
}

// Where a wait runs out it returns at once: whether the current unit's ticket is taken.
template <int F16>
__device__ __forceinline__ bool ct_softmax(const ChunkParams& p, uint32_t tmem) {
  CtBars* bars = CT_BARS;
  uint8_t* sQ = ct_smem;
  uint8_t* sV = ct_smem + kCtOffV;
  float* s_merge = reinterpret_cast<float*>(ct_smem + kCtOffMerge);
  Walk& w = *(reinterpret_cast<Walk*>(ct_smem + kCtOffWalks) + threadIdx.x / 32);
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int t = warp / 8, c = warp % 8;
  const int lb = 32 * (c % 4) + 16 * (c / 4);
  const int t0 = lane & 3, t1 = lane >> 2;
  // this warp's lanes and chain: weights at tP, scores and accumulator from it
  const uint32_t tP = tmem + (static_cast<uint32_t>(lb) << 16) + kCtP + t * 64;
  const uint32_t tS = tP + kCtS - kCtP + t * 64;
  const uint32_t tO = tP + kCtO - kCtP;
  float* mbuf = s_merge + c * kCtMergeFloats;
  uint32_t n_s = 0;     // blocks of this chain so far
  uint32_t n_sync = 0;  // meetings of its warps
  for (uint32_t i = lane; i < sizeof(Walk) / 4; i += 32)
    reinterpret_cast<int*>(&w)[i] = reinterpret_cast<const int*>(&bars->start)[i];
  __syncwarp();

  while (w.left > 0) {
    const bool pair = walk_pair(w);
    // this chain's blocks: all, or every second one (none of a single one for chain 1)
    const int cnt = pair ? walk_blocks(w) : (walk_blocks(w) + 1 - t) >> 1;
    const bool any = cnt > 0;
    const int row0 = w.m * kPxRows + (pair ? 128 * t : 0);
    const int rows = min(128, w.rows - (pair ? 128 * t : 0));  // of this chain's tile
    if (any) {
      // The chain's last unit is done (its last product was waited for), so
      // its query buffer is free.
      load_q(p, w, row0, rows, sQ + t * kCtTile);
      fence_proxy_async_smem();
      mbar_arrive(&bars->q_full[t]);
    }
    const bool active = 16 * c < rows;  // warp-uniform: some row of this warp is real
    // Keys that the tile's first row sees, so the whole tile, counted from the chain's
    // next block; and how many more this thread's two rows see (rows behind the last see
    // what it does), in 16 bits each: registers are short.
    int common;
    uint32_t more = 0;
    {
      const int G = p.heads / p.kv_heads, tok0 = row0 / G;
      common = (p.causal ? w.s.len - (w.s.n - 1 - tok0) : w.s.len) - (walk_first(w) + (pair ? 0 : t)) * kChKeys;
      if (p.causal)
#pragma unroll
        for (int v = 0; v < 2; ++v)
          more |= static_cast<uint32_t>((row0 + min(16 * c + t1 + 8 * v, rows - 1)) / G - tok0) << 16 * v;
    }
    float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
#pragma unroll 1
    for (int i = 0; i < cnt; ++i, ++n_s, common -= pair ? kChKeys : 2 * kChKeys) {
      if (!warp_wait(&bars->s_full[t], n_s & 1, abort_flag, p.err, kErrTimeoutSoftmax)) return false;
      tc_fence_after();
      if (common < kChKeys) {
        // Some row of the tile does not see some key of this block.  Value rows
        // behind the sequence's last key may hold anything (a weight of 0 times a
        // NaN is a NaN): the chain's 256 threads zero them.
        const int j = pair ? i : 2 * i + t;
        const uint32_t it = static_cast<uint32_t>(w.base + j), st = it % kCtStages;
        const int live = min(kChKeys, max(0, w.s.len - (walk_first(w) + j) * kChKeys));
        const int lo = max(0, min(common, live));
        if (!warp_wait(&bars->v_full[st], (it / kCtStages) & 1, abort_flag, p.err,
                       kErrTimeoutSoftmax))
          return false;
        uint4* v = reinterpret_cast<uint4*>(sV + st * kCtTile);
        for (int k = live * 8 + (threadIdx.x & 255); k < kChKeys * 8; k += 256)
          v[k] = make_uint4(0, 0, 0, 0);
        // the last product is done with the chain's copy, flags and accumulator
        if (n_s > 0 &&
            !warp_wait(&bars->o_done[t], (n_s - 1) & 1, abort_flag, p.err, kErrTimeoutSoftmax))
          return false;
        bool odd = false;
        for (int k = lo * 8 + (threadIdx.x & 255); k < live * 8; k += 256) {
          const uint4 x = v[k];
          odd = odd || (odd_halves<F16>(x.x) | odd_halves<F16>(x.y) | odd_halves<F16>(x.z) |
                        odd_halves<F16>(x.w));
        }
        if (odd) bars->odd[t] = static_cast<int>(n_s) + 1;
        if (!chain_sync(&bars->sync[t], n_sync, abort_flag, p.err)) return false;
        const bool fix = *static_cast<volatile int*>(&bars->odd[t]) == static_cast<int>(n_s) + 1;
        if (fix) {
          tc_fence_after();
          if (active) {
            // such values into the accumulators of the rows that see them
#pragma unroll 1
            for (int h = 0; h < 8; ++h) {
              uint32_t o4[4] = {0, 0, 0, 0};
              if (i > 0) {
                tmem_ld_16x256b_x1(tO + 8 * h, o4);
                tmem_wait_ld_regs4(o4);
              }
#pragma unroll 1
              for (int key = lo; key < live; ++key) {
                const uint32_t x = *reinterpret_cast<const uint32_t*>(
                    sV + st * kCtTile + key * 128 + ((h ^ (key & 7)) << 4) + 4 * t0);
                const uint32_t o = odd_halves<F16>(x);
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                  if (key >= common + static_cast<int>(more >> 16 * r & 0xffffu)) continue;
                  if (o & 0xffffu)
                    o4[2 * r] = __float_as_uint(__uint_as_float(o4[2 * r]) + lo_half(x, F16));
                  if (o >> 16)
                    o4[2 * r + 1] = __float_as_uint(__uint_as_float(o4[2 * r + 1]) + hi_half(x, F16));
                }
              }
              tmem_st_16x256b_x1(tO + 8 * h, o4);
            }
            tmem_wait_st();
          }
          if (!chain_sync(&bars->sync[t], n_sync, abort_flag, p.err)) return false;
          // zeros in their places: in a copy if the other chain reads the block too
          uint4* to = pair ? reinterpret_cast<uint4*>(ct_smem + kCtOffCopy + t * kCtTile) : v;
          for (int k = threadIdx.x & 255; k < kChKeys * 8; k += 256) {
            uint4 x = v[k];
            const int key = k >> 3;
            if (key >= lo)
              x = key < live ? make_uint4(x.x & ~odd_halves<F16>(x.x), x.y & ~odd_halves<F16>(x.y),
                                          x.z & ~odd_halves<F16>(x.z), x.w & ~odd_halves<F16>(x.w))
                             : make_uint4(0, 0, 0, 0);
            to[k] = x;
          }
        }
        if ((threadIdx.x & 255) == 0) {
          bars->copy[t] = fix && pair;
          bars->keep[t] = fix && i == 0;
        }
        fence_proxy_async_smem();
      }
      if (!active) {
        tc_fence_before();
        mbar_arrive(&bars->sc_done[t]);
        // the previous product must have left P before it is declared full again
        if (n_s > 0 &&
            !warp_wait(&bars->o_done[t], (n_s - 1) & 1, abort_flag, p.err, kErrTimeoutSoftmax))
          return false;
        mbar_arrive(&bars->p_full[t]);
        continue;
      }
      uint32_t sr[64];
      tmem_ld_16x256b_x16(tS, sr);
      tmem_wait_ld();
      tc_fence_before();
      mbar_arrive(&bars->sc_done[t]);
      float* sf = reinterpret_cast<float*>(sr);
      if (common < kChKeys) {
        const int rel[2] = {common + static_cast<int>(more & 0xffffu), common + static_cast<int>(more >> 16)};
#pragma unroll
        for (int k = 0; k < 16; ++k)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            if (8 * k + 2 * t0 + x >= rel[0]) sf[4 * k + x] = -INFINITY;
            if (8 * k + 2 * t0 + x >= rel[1]) sf[4 * k + 2 + x] = -INFINITY;
          }
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
      // The reference value of a row moves only when the maximum outgrows it by 2^8, so
      // that most blocks never rescale.  Weights stay below 2^8; in f16 below 2^15, and
      // the largest is 2^6 at least, so that none above 2^-20 of it is a subnormal number.
      constexpr float kLift = F16 ? 7.f : 0.f, kLag = 8.f + kLift;
      float corr[2] = {1.f, 1.f};
      const bool moves = __any_sync(0xffffffffu, mx[0] * p.scale_log2 > m_run[0] + kLag ||
                                                     mx[1] * p.scale_log2 > m_run[1] + kLag);
      if (moves) {
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          mx[v] = fmaxf(mx[v], __shfl_xor_sync(0xffffffffu, mx[v], 1));
          mx[v] = fmaxf(mx[v], __shfl_xor_sync(0xffffffffu, mx[v], 2));
          const float m_blk = mx[v] * p.scale_log2;
          if (m_blk > m_run[v] + kLag) {
            const float m_new = ceilf(m_blk) - kLift;
            corr[v] = ex2_approx(m_run[v] - m_new);
            m_run[v] = m_new;
            l_run[v] *= corr[v];
          }
        }
      }
      // weights in pairs; the sum takes them unrounded, the product in 16 bits (off by
      // 2^-8 or 2^-11 of them, in f16 by 2^-31 of the largest where that is more)
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
        return false;
      tc_fence_after();
      // The accumulator so far, which that product was the last to add to: here, where
      // the scores are no more, since with them the registers did not suffice (2.1 us a
      // step of 256 rows and 128 keys instead of 1.6).
      if (moves && i > 0) {
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
      }
      tmem_st_16x128b_x16(tP, pk);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&bars->p_full[t]);
    }

    // ---- end of the unit's stretch
    if (any && !warp_wait(&bars->o_done[t], (n_s - 1) & 1, abort_flag, p.err, kErrTimeoutSoftmax))
      return false;
    tc_fence_after();
    if (any && (threadIdx.x & 255) == 0) bars->copy[t] = bars->keep[t] = 0;  // (seen by the next unit's p_full)
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
        return false;
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
        if (!warp_wait(&bars->mrg_full[c], w.alt & 1, abort_flag, p.err, kErrTimeoutSoftmax)) return false;
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
      const int G = p.heads / p.kv_heads;
      const bool whole = walk_whole(w);
      const UnitTeams teams = walk_teams(w, bars->share);
      const int cta = static_cast<int>(blockIdx.x);
      const UnitParts u{teams.c0, teams.c1, kPxRows, pair ? 128 * t : 0, row0, rows, w.s.t0, w.h};
      if (active) {
        float inv[2];
        size_t at[2];
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          const int r = 16 * c + t1 + 8 * v, row = row0 + min(r, rows - 1), tok = row / G;
          const int h = w.h * G + row - tok * G;
          if (whole) {
            inv[v] = l_run[v] == 0.f ? 0.f : 1.f / l_run[v];
            f0[v] *= inv[v];
            f1[v] *= inv[v];
            at[v] = (static_cast<size_t>(w.s.t0 + tok) * p.heads + h) * 64 + 2 * t0;
            if (p.lse && t0 == 0 && r < rows)
              p.lse[static_cast<size_t>(h) * p.tokens + w.s.t0 + tok] =
                  l_run[v] == 0.f ? -INFINITY : (m_run[v] + log2f(l_run[v])) * 0.69314718055994530942f;
          } else {
            at[v] = part_row(u, cta, r) * 64 + 2 * t0;
            if (t0 == 0 && r < rows)
              __stcg(reinterpret_cast<float2*>(p.part_ml + 2 * part_row(u, cta, r)),
                     make_float2(m_run[v], l_run[v]));
          }
        }
        const int kind = whole ? p.out_dtype : 3;
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
                // (0: not used; a NaN is one of a row that sees one)
                o[x] = f0[v] != 0.f ? __uint_as_float(o8[e]) * f0[v] : 0.f;
                if (f1[v] != 0.f) o[x] = fmaf(mbuf[(8 * h + e) * 32 + lane], f1[v], o[x]);
              }
              if (16 * c + t1 + 8 * v < rows) {
                const size_t to = at[v] + 16 * h + 8 * k;
                if (kind == 3)
                  __stcg(reinterpret_cast<float2*>(p.part_o + to), make_float2(o[0], o[1]));
                else if (kind == 0)
                  *reinterpret_cast<float2*>(static_cast<float*>(p.out) + to) = make_float2(o[0], o[1]);
                else
                  *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.out) + to) =
                      kind == 2 ? pack_f16x2(o[0], o[1]) : pack_bf16x2(o[0], o[1]);
              }
            }
        }
      }
      if (!pair) mbar_arrive(&bars->mrg_empty[c]);
      if (!whole) {
        // ---- the last of the unit's CTAs merges the parts of this tile, in their order
        __threadfence();
        if (!chain_sync(&bars->sync[t], n_sync, abort_flag, p.err)) return false;
        if ((threadIdx.x & 255) == 0) {
          bars->last[t] = take_ticket(p, w, teams, t);
          __threadfence();
        }
        if (!chain_sync(&bars->sync[t], n_sync, abort_flag, p.err)) return true;
        if (*static_cast<volatile int*>(&bars->last[t])) {
          const int part = threadIdx.x & 7;
#pragma unroll 1
          for (int r = (threadIdx.x & 255) >> 3; r < rows; r += 32) {
            Merged acc{-INFINITY, 0.f, {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}};
#pragma unroll 2
            for (int x = teams.c0; x <= teams.c1; ++x) {
              const size_t from = part_row(u, x, r);
              const float4* o = reinterpret_cast<const float4*>(p.part_o + from * 64 + 8 * part);
              acc.add(__ldcg(reinterpret_cast<const float2*>(p.part_ml + 2 * from)), __ldcg(o), __ldcg(o + 1));
            }
            store_unit_row(p, u, acc, r, part);
          }
        }
      }
    }
    tc_fence_before();
    __syncwarp();
    if (lane == 0) walk_next(w, p);
    __syncwarp();
  }
  return false;
}

template <int F16>
__global__ void __launch_bounds__(kCtThreads, 1)
    chunk_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                    const __grid_constant__ ChunkParams p) {
  if (smem_u32(ct_smem) % 1024 != 0) {  // the whole grid alike
    if (threadIdx.x == 0 && p.err) atomicOr(p.err, kErrBadArgs);
    return;
  }
  CtBars* bars = CT_BARS;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&bars->q_full[t], 256);
      mbar_init(&bars->s_full[t], 1);
      mbar_init(&bars->sc_done[t], 256);
      mbar_init(&bars->p_full[t], 256);
      mbar_init(&bars->o_done[t], 1);
      mbar_init(&bars->sync[t], 256);
      bars->odd[t] = bars->copy[t] = bars->keep[t] = 0;
    }
    for (int s = 0; s < kCtStages; ++s) {
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
  if (warp == kCtProducer) {
    tmem_alloc(&bars->tmem_base, kCtTmem);
    tmem_relinquish();
  }
  if (warp == kCtMma0 + 1 && lane == 0) {
    prefetch_tensormap(&tmK);
    prefetch_tensormap(&tmV);
  }
  // (the walks' place serves before they are)
  Stretch* start = reinterpret_cast<Stretch*>(ct_smem + kCtOffWalks);
  find_stretch<kPxRows, kChKeys, kCtThreads, 1>(p, start, reinterpret_cast<int2*>(start + 2));
  if (threadIdx.x == 0) {
    const Stretch x = *start;
    Walk w{};
    w.left = x.left;
    if (x.left > 0) {
      bool bad = false;
      w.s = chunk_seq(p, x.b, bad);
      w.b = x.b, w.h = x.h, w.m = x.m;
      w.step = x.step;
      w.unit0 = x.unit0;
      walk_unit(w, p);
      bars->share = x.share;
    }
    bars->start = w;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem_base;

  if (warp == kCtProducer) {
    ct_producer(&tmK, &tmV, p);
  } else if (warp >= kCtMma0) {
    ct_mma<F16>(p, warp - kCtMma0, tmem);
    int none = 0;  // every MMA issued has finished before tensor memory is freed
    mma_commit_w(&bars->drain);
    mbar_wait(&bars->drain, 0, &none, p.err, kErrTimeoutDrain);
  } else {
    const bool taken = ct_softmax<F16>(p, tmem);
    if ((threadIdx.x & 255) == 0)
      take_the_rest(p, *(reinterpret_cast<Walk*>(ct_smem + kCtOffWalks) + warp), bars->share, warp / 8, taken);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == kCtProducer) {
    tc_fence_after();
    tmem_dealloc(tmem, kCtTmem);
  }
}

}  // namespace

cudaError_t launch_chunk_tc(const CUtensorMap& tmK, const CUtensorMap& tmV, const ChunkParams& p,
                            int grid, cudaStream_t s) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  static std::atomic<bool> configured[2][64];
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  const int which = p.kv_dtype == 2;
  auto kern = which ? chunk_tc_kernel<1> : chunk_tc_kernel<0>;
  if (!configured[which][dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(kCtSmem));
    if (e != cudaSuccess) return e;
    configured[which][dev].store(true, std::memory_order_release);
  }
  kern<<<grid, kCtThreads, kCtSmem, s>>>(tmK, tmV, p);
  return cudaGetLastError();
}

}  // namespace ffai

// The shared part of ffai_attn_shared_prefix on the tensor cores: all query
// rows of a group against the group's prefix, read once per 128 rows.
//
// A group of s sequences has s * q_len * G query rows per KV head (G = query
// heads per KV head); they form tiles of 128 rows, the M of tcgen05.mma.  The
// prefix is cut into blocks of 128 keys (two pages).  All (tile, block) pairs
// of all groups and heads are laid out on one line, W of them, tile after
// tile, and CTA c takes the pairs [c S, (c + 1) S), S = ceil(W / CTAs): every
// CTA gets the same number of key blocks whatever the lengths and group
// sizes, and a tile that spans CTAs leaves one partial result (running
// maximum, sum, unnormalised output) per CTA, merged by shared_rows_kernel.
// The partial of CTA c for tile t lies in slot c + t: along the line either
// c or t grows from one partial to the next, so slots are distinct.
//
// Per CTA: warp 16 streams the pages through a 4-stage ring of K and V
// blocks by TMA; blocks alternate between two chains (t = 0, 1), each with an
// MMA warp (17, 18), scores, weights and an output accumulator of its own in
// tensor memory and 8 softmax warps, so one chain's softmax runs beside the
// other's products.  At the end of a tile chain 1 hands its accumulator to
// chain 0 through shared memory, warp to warp.
//
// Bound: a block is 32 KB of HBM traffic for up to 128 rows; at 1/148 of the
// measured copy rate that is 0.75 us, and a chain pair needs about as long for
// two 128 x 128 softmax blocks, so up to 128 rows the kernel streams.
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

struct __align__(8) PxBars {
  uint64_t q_full[2];
  uint64_t k_full[kPxStages], v_full[kPxStages], kv_empty[kPxStages];
  uint64_t s_full[2], sc_done[2], p_full[2], o_done[2];
  uint64_t mrg_full[8], mrg_empty[8];
  uint64_t drain;
  uint32_t tmem_base;
  int abort_flag;
  // this CTA's stretch of the line
  long long total;
  int start_group, left;
  long long start_off, start_tile;
};

constexpr size_t kPxTiles = (2 + 2 * kPxStages) * kPxTile;
constexpr size_t kPxMerge = 8 * (32 * 32 + 64) * sizeof(float);
constexpr size_t kPxSmem = kPxTiles + kPxMerge + sizeof(PxBars) + 1024;

// The pairs of a CTA's stretch, one after another.  Every role walks its own.
struct Walker {
  const SharedParams& p;
  GroupDims d;
  int g, h, m, blk;  // group, KV head, row tile, key block
  int left;          // pairs left, the current one included
  int seg;           // tiles entered before this one (of this CTA)
  long long tile;    // index of the tile on the line
  __device__ __forceinline__ Walker(const SharedParams& params, const PxBars* bars) : p(params) {
    g = bars->start_group;
    left = bars->left;
    seg = 0;
    tile = bars->start_tile;
    if (left > 0) {
      d = group_dims(p, g);
      const long long t = bars->start_off / d.nb;
      blk = static_cast<int>(bars->start_off - t * d.nb);
      h = static_cast<int>(t / d.mt);
      m = static_cast<int>(t - static_cast<long long>(h) * d.mt);
    }
  }
  __device__ __forceinline__ int stretch() const { return min(left, d.nb - blk); }
  // Step over `n` pairs of the current tile.
  __device__ __forceinline__ void skip(int n) {
    left -= n;
    blk += n;
    if (left <= 0 || blk < d.nb) return;
    blk = 0;
    ++seg;
    ++tile;
    if (++m < d.mt) return;
    m = 0;
    if (++h < p.kv_heads) return;
    h = 0;
    do d = group_dims(p, ++g);
    while (d.nb == 0);
  }
};

__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag,
                                          unsigned* err, unsigned code) {
  const bool ok = mbar_wait(bar, parity, abort_flag, err, code);
  return __all_sync(0xffffffffu, ok);
}

// One warp: lengths of the line and where this CTA starts on it.  CTA 0 also
// leaves each group's first pair and tile, and S, for the merge.
__device__ __forceinline__ void find_stretch(const SharedParams& p, PxBars* bars) {
  const int lane = threadIdx.x % 32;
  long long total = 0;
  for (int base = 0; base < p.groups; base += 32) {
    const int g = base + lane;
    long long n = 0;
    if (g < p.groups) {
      const GroupDims d = group_dims(p, g);
      n = static_cast<long long>(p.kv_heads) * d.mt * d.nb;
      if (blockIdx.x == 0 && p.err) {
        const int raw = __ldg(p.prefix_lens + g);
        const int s0 = __ldg(p.group_starts + g), s1 = __ldg(p.group_starts + g + 1);
        if (raw < 0 || raw > p.prefix_pages * kPageKeys || s0 < 0 || s1 < s0 || s1 > p.batch)
          atomicOr(p.err, kErrBadArgs);
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    total += n;
  }
  const long long share = (total + gridDim.x - 1) / gridDim.x;
  const long long first = blockIdx.x * share;
  const long long end = min(total, first + share);
  if (lane == 0) {
    bars->left = first < end ? static_cast<int>(end - first) : 0;
    if (blockIdx.x == 0) p.part_plan[0] = share;
  }
  long long lin = 0, tiles = 0;
  for (int base = 0; base < p.groups; base += 32) {
    const int g = base + lane;
    long long n = 0, t = 0;
    if (g < p.groups) {
      const GroupDims d = group_dims(p, g);
      t = d.nb > 0 ? static_cast<long long>(p.kv_heads) * d.mt : 0;
      n = t * d.nb;
    }
    long long ni = n, ti = t;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long a = __shfl_up_sync(0xffffffffu, ni, o), b = __shfl_up_sync(0xffffffffu, ti, o);
      if (lane >= o) {
        ni += a;
        ti += b;
      }
    }
    const long long l0 = lin + ni - n, t0 = tiles + ti - t;
    if (g < p.groups && blockIdx.x == 0) {
      p.part_plan[1 + 2 * g] = l0;
      p.part_plan[2 + 2 * g] = t0;
    }
    if (first < end && n > 0 && l0 <= first && first < l0 + n) {  // one lane, once
      bars->start_group = g;
      bars->start_off = first - l0;
      bars->start_tile = t0 + (first - l0) / (n / t);
    }
    lin += __shfl_sync(0xffffffffu, ni, 31);
    tiles += __shfl_sync(0xffffffffu, ti, 31);
  }
}

// ---------------------------------------------------------------- producer
__device__ __forceinline__ void px_producer(const CUtensorMap* tmK, const CUtensorMap* tmV,
                                            const SharedParams& p, uint8_t* sK, uint8_t* sV,
                                            PxBars* bars) {
  volatile int* abort_flag = &bars->abort_flag;
  const int lane = threadIdx.x % 32;
  Walker w(p, bars);
  uint32_t it = 0;
  bool ok = true;
  while (ok && w.left > 0) {
    const int* table = p.prefix_table + static_cast<size_t>(w.g) * p.prefix_pages;
    const int n_pages = (w.d.plen + kPageKeys - 1) / kPageKeys;
    const int b0 = w.blk, b1 = w.blk + w.stretch();
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
    w.skip(b1 - b0);
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
// Chain t takes the blocks it (counted over the CTA's stretch) with it % 2 ==
// t.  The scores of its next block are issued before the second product of
// the current one, within a tile and across tiles.
struct ChainBlock {
  uint32_t it;
  int seg;
  bool first;  // of this chain's blocks in the tile
};

struct ChainWalk {
  Walker w;
  int t, pos;    // pos: blocks of the current tile's stretch passed by this chain
  uint32_t base; // it of the current tile's first block
  __device__ __forceinline__ ChainWalk(const SharedParams& p, const PxBars* bars, int chain)
      : w(p, bars), t(chain), pos(0), base(0) {}
  // The chain's next block, or false at the end of the stretch.
  __device__ __forceinline__ bool next(ChainBlock& b) {
    while (w.left > 0) {
      const int n = w.stretch();
      const int off = static_cast<int>((base ^ static_cast<uint32_t>(t)) & 1u);  // first of this chain
      const int j = off + 2 * pos;
      if (j < n) {
        b.it = base + j;
        b.seg = w.seg;
        b.first = pos == 0;
        ++pos;
        return true;
      }
      w.skip(n);
      base += n;
      pos = 0;
    }
    return false;
  }
};

template <int F16>
__device__ __forceinline__ void px_mma(const SharedParams& p, int t, uint8_t* sQ, uint8_t* sK,
                                       uint8_t* sV, uint32_t tmem, PxBars* bars) {
  volatile int* abort_flag = &bars->abort_flag;
  constexpr uint32_t idesc_s = idesc_f16(F16 ? 0u : 1u, 128, 128, 0, 0);
  constexpr uint32_t idesc_o = idesc_f16(F16 ? 0u : 1u, 128, 64, 0, 1);
  ChainWalk walk(p, bars, t);
  uint32_t n_s = 0, n_pv = 0;
  auto issue_s = [&](const ChainBlock& b) -> bool {
    const uint32_t s = b.it % kPxStages;
    if (!warp_wait(&bars->k_full[s], (b.it / kPxStages) & 1, abort_flag, p.err, kErrTimeoutMma))
      return false;
    if (b.first && !warp_wait(&bars->q_full[b.seg & 1], (b.seg >> 1) & 1, abort_flag, p.err,
                              kErrTimeoutMma))
      return false;
    if (n_s > 0 &&
        !warp_wait(&bars->sc_done[t], (n_s - 1) & 1, abort_flag, p.err, kErrTimeoutMma))
      return false;
    tc_fence_after();
    const uint64_t dq = smem_desc_sw128(smem_u32(sQ + (b.seg & 1) * kPxTile), 16, 1024);
    const uint64_t dk = smem_desc_sw128(smem_u32(sK + s * kPxTile), 16, 1024);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      mma_ss_w(tmem + kPxS + t * 128, dq + 2 * k, dk + 2 * k, idesc_s, k > 0 ? 1u : 0u);
    mma_commit_w(&bars->s_full[t]);
    ++n_s;
    return true;
  };
  ChainBlock cur, nxt;
  if (!walk.next(cur)) return;
  if (!issue_s(cur)) return;
  while (true) {
    const bool more = walk.next(nxt);
    // Within a tile the next scores go first; across tiles the last product
    // does, since the tile's epilogue waits for it.
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
    if (!more) return;
    if (!ahead && !issue_s(nxt)) return;
    cur = nxt;
  }
}

// ---------------------------------------------------------------- softmax
// Rows of a tile: row r (0..127) sits at MMA row 32 (c % 4) + 16 (c / 4) + r %
// 16 with c = r / 16, so softmax warp c of a chain owns rows 16 c .. and few
// rows spread over the four scheduler quarters.
__device__ __forceinline__ int mma_row(int r) {
  const int c = r >> 4;
  return 32 * (c & 3) + 16 * (c >> 2) + (r & 15);
}

// The tile's query rows into swizzled shared memory: 512 threads, each two
// 16-byte pieces (8 head dims).  Rows past the tile's end are zero.
__device__ __forceinline__ void load_q(const SharedParams& p, const Walker& w, uint8_t* dst) {
  const int G = p.heads / p.kv_heads, R = p.q_len * G;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int piece = threadIdx.x + i * 512;
    const int r = piece >> 3, c = piece & 7;
    const int row = w.m * 128 + r;
    uint4 x = make_uint4(0, 0, 0, 0);
    if (row < w.d.rows) {
      const int b = w.d.b0 + row / R, rr = row % R;
      const int tok = rr / G, h = w.h * G + rr % G;
      const size_t off = static_cast<size_t>(b) * p.q_sb + static_cast<size_t>(tok) * p.q_st +
                         static_cast<size_t>(h) * p.q_sh + c * 8;
      if (p.q_dtype == 0) {  // f32 queries are rounded to the cache's type
        const float4* src = reinterpret_cast<const float4*>(static_cast<const float*>(p.q) + off);
        const float4 a = __ldg(src), e = __ldg(src + 1);
        x = p.kv_dtype == 2 ? make_uint4(pack_f16x2(a.x, a.y), pack_f16x2(a.z, a.w),
                                         pack_f16x2(e.x, e.y), pack_f16x2(e.z, e.w))
                            : make_uint4(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w),
                                         pack_bf16x2(e.x, e.y), pack_bf16x2(e.z, e.w));
      } else {
        x = __ldg(reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.q) + off));
      }
    }
    const int mr = mma_row(r);
    *reinterpret_cast<uint4*>(dst + mr * 128 + ((c ^ (mr & 7)) << 4)) = x;
  }
}

template <int F16>
__device__ __forceinline__ void px_softmax(const SharedParams& p, uint32_t tmem, uint8_t* sQ,
                                           uint8_t* sV, float* s_merge, PxBars* bars) {
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int t = warp / 8, c = warp % 8;
  const int lb = 32 * (c % 4) + 16 * (c / 4);
  const int t0 = lane & 3, t1 = lane >> 2;
  const uint32_t lane_addr = static_cast<uint32_t>(lb) << 16;
  const uint32_t tS = tmem + lane_addr + kPxS + t * 128;
  const uint32_t tP = tmem + lane_addr + kPxP + t * 64;
  const uint32_t tO = tmem + lane_addr + kPxO + t * 64;
  const float sl2 = p.scale_log2;
  float* mbuf = s_merge + c * (32 * 32 + 64);
  uint32_t n_s = 0;   // blocks of this chain so far
  uint32_t base = 0;  // it of the current tile's first block
  Walker w(p, bars);

  while (w.left > 0) {
    const int n = w.stretch();
    const int seg = w.seg;
    // The buffer's last tile, seg - 2, is done with in both chains: a chain 0
    // warp has met chain 1's hand-over of seg - 1, a chain 1 warp chain 0's
    // release of seg - 2, and either follows that chain's last product.
    load_q(p, w, sQ + (seg & 1) * kPxTile);
    fence_proxy_async_smem();
    mbar_arrive(&bars->q_full[seg & 1]);

    const int rows = min(128, w.d.rows - w.m * 128);
    const bool active = 16 * c < rows;  // warp-uniform: some row of this warp is real
    const int off = static_cast<int>((base ^ static_cast<uint32_t>(t)) & 1u);
    float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
    bool any = false;
    for (int j = off; j < n; j += 2) {
      if (!warp_wait(&bars->s_full[t], n_s & 1, abort_flag, p.err, kErrTimeoutSoftmax)) return;
      tc_fence_after();
      const int live = w.d.plen - (w.blk + j) * 128;  // keys of this block that exist
      const uint32_t it = base + j;
      if (live < 128) {
        // Value rows behind the last live key may hold anything (a weight of
        // 0 times a NaN is a NaN): the chain's 256 threads zero them before
        // the second product.
        const uint32_t st = it % kPxStages;
        if (!warp_wait(&bars->v_full[st], (it / kPxStages) & 1, abort_flag, p.err,
                       kErrTimeoutSoftmax))
          return;
        uint4* v = reinterpret_cast<uint4*>(sV + st * kPxTile);
        for (int i = live * 8 + (threadIdx.x & 255); i < 128 * 8; i += 256)
          v[i] = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
      }
      if (!active) {
        tc_fence_before();
        mbar_arrive(&bars->sc_done[t]);
        // the previous product must have left P before it is declared full again
        if (n_s > 0 &&
            !warp_wait(&bars->o_done[t], (n_s - 1) & 1, abort_flag, p.err, kErrTimeoutSoftmax))
          return;
        mbar_arrive(&bars->p_full[t]);
        ++n_s;
        any = true;
        continue;
      }
      uint32_t sr[64];
      tmem_ld_16x256b_x16(tS, sr);
      tmem_wait_ld();
      tc_fence_before();
      mbar_arrive(&bars->sc_done[t]);
      float* sf = reinterpret_cast<float*>(sr);
      if (live < 128) {
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
      float corr[2] = {1.f, 1.f};
      bool grow = false;
      if (__any_sync(0xffffffffu,
                     mx[0] * sl2 > m_run[0] + 8.0f || mx[1] * sl2 > m_run[1] + 8.0f)) {
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          mx[v] = fmaxf(mx[v], __shfl_xor_sync(0xffffffffu, mx[v], 1));
          mx[v] = fmaxf(mx[v], __shfl_xor_sync(0xffffffffu, mx[v], 2));
          const float m_blk = mx[v] * sl2;
          if (m_blk > m_run[v] + 8.0f) {
            const float m_new = ceilf(m_blk);
            corr[v] = ex2_approx(m_run[v] - m_new);
            m_run[v] = m_new;
            grow = true;
          }
        }
      }
      // weights in pairs; the sum takes them unrounded, the product in 16 bits
      uint32_t pk[32];
      float bsum[2];
      const uint64_t c2 = f2_pack(sl2, sl2);
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        const float neg = m_run[v] == -INFINITY ? 0.f : -m_run[v];
        const uint64_t n2 = f2_pack(neg, neg);
        uint64_t acc0 = f2_pack(0.f, 0.f), acc1 = acc0;
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          float x0, x1;
          f2_unpack(f2_fma(f2_pack(sf[4 * k + 2 * v], sf[4 * k + 2 * v + 1]), c2, n2), x0, x1);
          const float p0 = ex2_approx(x0), p1 = ex2_approx(x1);
          pk[2 * k + v] = F16 ? pack_f16x2(p0, p1) : pack_bf16x2(p0, p1);
          if (k & 1)
            acc1 = f2_add(acc1, f2_pack(p0, p1));
          else
            acc0 = f2_add(acc0, f2_pack(p0, p1));
        }
        float a, b;
        f2_unpack(f2_add(acc0, acc1), a, b);
        bsum[v] = a + b;
      }
      l_run[0] = fmaf(l_run[0], corr[0], bsum[0]);
      l_run[1] = fmaf(l_run[1], corr[1], bsum[1]);
      if (n_s > 0 &&
          !warp_wait(&bars->o_done[t], (n_s - 1) & 1, abort_flag, p.err, kErrTimeoutSoftmax))
        return;
      tc_fence_after();
      if (__any_sync(0xffffffffu, grow && any)) {
#pragma unroll 1
        for (int h = 0; h < 4; ++h) {
          uint32_t orr[8];
          tmem_ld_16x256b_x2(tO + 16 * h, orr);
          tmem_wait_ld_regs8(orr);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            orr[e] = __float_as_uint(__uint_as_float(orr[e]) * corr[(e >> 1) & 1]);
          tmem_st_16x256b_x2(tO + 16 * h, orr);
        }
      }
      tmem_st_16x128b_x16(tP, pk);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(&bars->p_full[t]);
      ++n_s;
      any = true;
    }

    // ---- end of the tile's stretch: chain 1 hands over to chain 0
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
    // (an inactive pair has nothing to hand over, but keeps the barriers' count)
    uint32_t orr[32];
    if (t == 1) {
      if (seg >= 1 && !warp_wait(&bars->mrg_empty[c], (seg - 1) & 1, abort_flag, p.err,
                                 kErrTimeoutSoftmax))
        return;
      if (active) {
        if (any) {
          tmem_ld_16x256b_x8(tO, orr);
          tmem_wait_ld_regs(orr);
#pragma unroll
          for (int e = 0; e < 32; ++e) mbuf[e * 32 + lane] = __uint_as_float(orr[e]);
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
      if (active && any) {
        tmem_ld_16x256b_x8(tO, orr);
        tmem_wait_ld_regs(orr);
      }
      if (!warp_wait(&bars->mrg_full[c], seg & 1, abort_flag, p.err, kErrTimeoutSoftmax)) return;
      // (group_starts that do not rise can give more tiles than there is room for)
      if (active && blockIdx.x + w.tile < p.part_slots) {
        const size_t slot = static_cast<size_t>(blockIdx.x + w.tile) * 128 + 16 * c;
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          const int r = t1 + 8 * v;
          const float m1 = mbuf[32 * 32 + 2 * r], l1 = mbuf[32 * 32 + 2 * r + 1];
          const float M = fmaxf(m_run[v], m1);
          // a chain without blocks in this stretch has m = -inf: its
          // accumulator is stale and not used
          const float f0 = m_run[v] == -INFINITY ? 0.f : ex2_approx(m_run[v] - M);
          const float f1 = m1 == -INFINITY ? 0.f : ex2_approx(m1 - M);
          if (16 * c + r < rows) {
            float* dst = p.part_o + (slot + r) * 64 + 2 * t0;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              float2 o = make_float2(0.f, 0.f);
              if (m_run[v] != -INFINITY) {
                o.x = __uint_as_float(orr[4 * k + 2 * v]) * f0;
                o.y = __uint_as_float(orr[4 * k + 2 * v + 1]) * f0;
              }
              if (m1 != -INFINITY) {
                o.x = fmaf(mbuf[(4 * k + 2 * v) * 32 + lane], f1, o.x);
                o.y = fmaf(mbuf[(4 * k + 2 * v + 1) * 32 + lane], f1, o.y);
              }
              *reinterpret_cast<float2*>(dst + 8 * k) = o;
            }
            if (t0 == 0)
              *reinterpret_cast<float2*>(p.part_ml + 2 * (slot + r)) =
                  make_float2(M, l_run[v] * f0 + l1 * f1);
          }
        }
      }
      mbar_arrive(&bars->mrg_empty[c]);
    }
    tc_fence_before();
    base += n;
    w.skip(n);
  }
}

template <int F16>
__global__ void __launch_bounds__(kPxThreads, 1)
    prefix_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                     const SharedParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + 2 * kPxTile;
  uint8_t* sV = sK + kPxStages * kPxTile;
  float* s_merge = reinterpret_cast<float*>(sV + kPxStages * kPxTile);
  PxBars* bars = reinterpret_cast<PxBars*>(reinterpret_cast<uint8_t*>(s_merge) + kPxMerge);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

  if (warp == kPxMma0) {
    find_stretch(p, bars);
  } else if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&bars->q_full[t], 512);
      mbar_init(&bars->s_full[t], 1);
      mbar_init(&bars->sc_done[t], 256);
      mbar_init(&bars->p_full[t], 256);
      mbar_init(&bars->o_done[t], 1);
    }
    for (int s = 0; s < kPxStages; ++s) {
      mbar_init(&bars->k_full[s], 1);
      mbar_init(&bars->v_full[s], 1);
      mbar_init(&bars->kv_empty[s], 1);
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
    px_producer(&tmK, &tmV, p, sK, sV, bars);
  } else if (warp >= kPxMma0) {
    px_mma<F16>(p, warp - kPxMma0, sQ, sK, sV, tmem, bars);
    int none = 0;  // every MMA issued has finished before tensor memory is freed
    mma_commit_w(&bars->drain);
    mbar_wait(&bars->drain, 0, &none, p.err, kErrTimeoutDrain);
  } else {
    px_softmax<F16>(p, tmem, sQ, sV, s_merge, bars);
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

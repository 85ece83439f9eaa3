// Requests that take over each other's pages (beams that fork, requests that are
// cut back or end), a pool made dense, and the copies both ask for.
//
// Fork: row b of the new table continues row s = src[b] of the old one with its
// first n_b = min(lens[s], keep[b]) keys.  With R(p) the number of new entries
// that name page p, and W(p) the rows whose last page p is while n_b is no
// multiple of 64 -- who append into it next --, row b in W(p) takes a page of
// its own and a copy of n_b mod 64 keys, unless it is alone (R(p) = 1) or the
// first of W(p) while all of R(p) write (R(p) = |W(p)|).  Pages of the old
// table with R(p) = 0 go back to the stack first, in the order of their
// numbers; then the copies take theirs off it in row order.
//
// Compact: of the U pages that the table or the stack names, the live ones
// belong on the lowest numbers: with r(p) the rank of p among the U and L the
// live ones, the live p with r(p) >= L move to the idle ones with r(p) < L, in
// order.  One scan over the pages gives all ranks: the j-th mover is j = (live
// before p) - (live below rank L), the j-th hole j = (idle before p).
//
// The table is the only record of who shares what: the counts are made anew by
// every call, in words per page that are zero between calls.  Whole numbers
// throughout; atomics only add, or take a maximum, so their order is of no
// matter.
//
// Both are one cluster of CTAs (one launch; the phases meet at the cluster's
// barrier), bound by a chain of dependent loads and two to five barriers: a fork of
// 60 rows of 7 pages takes 9 us, of 1000 rows of 32 pages in a pool of 13209 18 (22
// before a warp had four rows' pages on their way); a compaction of 16 rows 9, of 300
// rows of 32 pages in a pool of 13139 20.  The copies are bound by HBM: 3000 pages of
// 8 heads, 784 MB read and written, 128 us = 6.1 TB/s (150 before the copies at the
// front of a list were dealt to all warps); 1000 ends of pages 4.
#include "common.cuh"
#include "kernels.h"

namespace ffai {

namespace {

constexpr int kMvThreads = 512;
constexpr int kMvWarps = kMvThreads / 32;
constexpr int kMvCluster = 8;
constexpr int kMvAhead = 4;  // rows whose pages a warp has on their way

__device__ __forceinline__ int pages_of(int keys) { return (keys + kPageKeys - 1) / kPageKeys; }

struct Pair {
  int a, b;
};

// Exclusive prefix sums of two numbers per thread over the CTA, and their totals.
__device__ __forceinline__ Pair block_scan(Pair v, Pair* s_warp, Pair* total) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  Pair in = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int a = __shfl_up_sync(0xffffffffu, in.a, o), b = __shfl_up_sync(0xffffffffu, in.b, o);
    if (lane >= o) {
      in.a += a;
      in.b += b;
    }
  }
  if (lane == 31) s_warp[warp] = in;
  __syncthreads();
  Pair base{0, 0}, all{0, 0};
#pragma unroll
  for (int w = 0; w < kMvWarps; ++w) {
    if (w < warp) {
      base.a += s_warp[w].a;
      base.b += s_warp[w].b;
    }
    all.a += s_warp[w].a;
    all.b += s_warp[w].b;
  }
  __syncthreads();
  *total = all;
  return {base.a + in.a - v.a, base.b + in.b - v.b};
}

// What each CTA of the cluster tells the others: through global memory, at L2.
__device__ __forceinline__ void cluster_sync() {
  __threadfence();
  cluster_arrive();
  cluster_wait();
}

// Keys of new row b, and the old row they come from (-1: none).
struct NewRow {
  int src, n;
};
__device__ __forceinline__ NewRow new_row(const ForkParams& p, int b, bool& bad) {
  NewRow r{__ldg(p.src + b), 0};
  if (r.src >= p.batch) {
    bad = true;
    r.src = -1;
  }
  if (r.src < 0) return {-1, 0};
  const int len = __ldg(p.lens + r.src);
  // (a length outside the table counts as none; reported where the old rows are read)
  r.n = len < 0 || len > p.max_pages * kPageKeys ? 0 : len;
  if (p.keep) r.n = min(r.n, max(0, __ldg(p.keep + b)));
  return r;
}

// Copy of row b's last page: 0 none, else the keys; `page` that page.
__device__ __forceinline__ int copy_keys(const ForkParams& p, int b, const NewRow& r, int& page) {
  const int part = r.n % kPageKeys;
  if (part == 0) return 0;
  page = __ldg(p.block_table + static_cast<size_t>(r.src) * p.max_pages + r.n / kPageKeys);
  if (page < 0 || page >= p.num_pages) return 0;
  const int4 w = __ldcg(p.words + page);  // references, writers, new_batch - first writer
  const bool mine = w.x == 1 || (w.x == w.y && w.z == p.new_batch - b);
  return mine ? 0 : part;
}

__global__ void __launch_bounds__(kMvThreads) page_fork_kernel(ForkParams p) {
  __shared__ Pair s_warp[kMvWarps];
  const int ctas = gridDim.x, cta = blockIdx.x;  // one cluster
  const int threads = ctas * kMvThreads, t = cta * kMvThreads + threadIdx.x;
  const int mp = p.max_pages;
  bool bad = false;

  // ---- references of the new table, and the old table's pages: a warp looks at 32 rows'
  // lengths at once and takes their entries 32 by 32
  const int lane = threadIdx.x % 32, warps = threads / 32;
  const int most = max(p.new_batch, p.batch);
  const int per = min(32, (most + warps - 1) / warps);  // rows of a warp at a time
  for (int b0 = t / 32 * per; b0 < most; b0 += warps * per) {
    NewRow mine{-1, 0};
    int old = 0;
    if (lane < per && b0 + lane < p.new_batch) mine = new_row(p, b0 + lane, bad);
    if (lane < per && b0 + lane < p.batch) {
      old = __ldg(p.lens + b0 + lane);
      if (old < 0 || old > mp * kPageKeys) {
        bad = true;
        old = 0;
      }
    }
    const int rows = min(per, most - b0);
    for (int i0 = 0; i0 < mp; i0 += 32) {
      const int i = i0 + lane;
      for (int k0 = 0; k0 < rows; k0 += kMvAhead) {
        int page[kMvAhead], was[kMvAhead], n[kMvAhead], len[kMvAhead];
#pragma unroll
        for (int k = 0; k < kMvAhead; ++k) {  // (rows behind the last have no keys)
          const int at = min(k0 + k, 31), b = b0 + at;
          const int src = __shfl_sync(0xffffffffu, mine.src, at);
          n[k] = k0 + k < rows ? __shfl_sync(0xffffffffu, mine.n, at) : 0;
          len[k] = k0 + k < rows ? __shfl_sync(0xffffffffu, old, at) : 0;
          page[k] = was[k] = 0;
          if (i < pages_of(n[k])) page[k] = __ldg(p.block_table + static_cast<size_t>(src) * mp + i);
          if (i < pages_of(len[k])) was[k] = __ldg(p.block_table + static_cast<size_t>(b) * mp + i);
        }
#pragma unroll
        for (int k = 0; k < kMvAhead; ++k) {
          const int b = b0 + k0 + k;
          if (i < pages_of(len[k])) {
            if (was[k] < 0 || was[k] >= p.num_pages)
              bad = true;
            else
              __stcg(reinterpret_cast<int*>(p.words + was[k]) + 3, 1);
          }
          int g = -1;
          if (i < pages_of(n[k])) {
            g = page[k];
            if (g < 0 || g >= p.num_pages) {
              bad = true;
              g = -1;
            } else {
              int* w = reinterpret_cast<int*>(p.words + g);
              atomicAdd(w, 1);
              if ((i + 1) * kPageKeys > n[k]) {
                atomicAdd(w + 1, 1);
                atomicMax(w + 2, p.new_batch - b);
              }
            }
          }
          if (i < mp && k0 + k < rows && b < p.new_batch) p.table_out[static_cast<size_t>(b) * mp + i] = g;
        }
      }
    }
  }
  cluster_sync();

  // ---- pages that no row names any more, and rows that need a copy
  const int pper = (p.num_pages + threads - 1) / threads, rper = (p.new_batch + threads - 1) / threads;
  const int p0 = min(p.num_pages, t * pper), p1 = min(p.num_pages, p0 + pper);
  const int r0 = min(p.new_batch, t * rper), r1 = min(p.new_batch, r0 + rper);
  Pair sum{0, 0};
#pragma unroll 4
  for (int g = p0; g < p1; ++g) {
    const int4 w = __ldcg(p.words + g);
    sum.a += w.w != 0 && w.x == 0;
  }
  for (int b = r0; b < r1; ++b) {  // (what this thread finds here it reads again below)
    const NewRow r = new_row(p, b, bad);
    int page = -1;
    const int keys = copy_keys(p, b, r, page);
    sum.b += keys > 0;
    p.lens_out[b] = r.n;
    p.copy_src[b] = keys > 0 ? page : -1;
    p.copy_keys[b] = keys;
  }
  Pair total;
  Pair at = block_scan(sum, s_warp, &total);
  if (ctas > 1) {
    if (threadIdx.x == 0) __stcg(p.totals + cta, make_int2(total.a, total.b));
    cluster_sync();
    total = {0, 0};
    for (int c = 0; c < ctas; ++c) {
      const int2 x = __ldcg(p.totals + c);
      if (c < cta) {
        at.a += x.x;
        at.b += x.y;
      }
      total.a += x.x;
      total.b += x.y;
    }
  }
  int count = __ldg(p.free_count);
  bad |= count < 0 || count > p.free_cap;
  count = min(max(count, 0), p.free_cap);
  bad |= total.a > p.free_cap - count;
#pragma unroll 4
  for (int g = p0; g < p1; ++g) {
    const int4 w = __ldcg(p.words + g);
    if (w.w != 0 && w.x == 0) {
      if (at.a < p.free_cap - count) __stcg(p.free_pages + count + at.a, g);
      ++at.a;
    }
    __stcg(p.words + g, make_int4(0, 0, 0, 0));  // for the next call
  }
  count = min(count + total.a, p.free_cap);
  if (ctas > 1)
    cluster_sync();
  else
    __syncthreads();

  // ---- rows: their copies, their last pages, their lengths
  for (int b = r0; b < r1; ++b) {
    const int keys = p.copy_keys[b];
    int fresh = -1;
    if (keys > 0) {
      if (at.b < count) {
        fresh = __ldcg(p.free_pages + (count - 1 - at.b));
        if (fresh < 0 || fresh >= p.num_pages) {
          bad = true;
          fresh = -1;
        }
      }
      ++at.b;
      const int n = p.lens_out[b];
      p.table_out[static_cast<size_t>(b) * mp + n / kPageKeys] = fresh;
      if (fresh < 0) {  // no page: the whole pages stay
        p.lens_out[b] = n - keys;
        p.copy_src[b] = -1;
        p.copy_keys[b] = 0;
      }
    }
    p.copy_dst[b] = fresh;
  }
  if (t == 0) *p.free_count_out = count - min(total.b, count);
  if (__syncthreads_or(bad) && threadIdx.x == 0 && p.err) atomicOr(p.err, kErrBadArgs);
}

__global__ void __launch_bounds__(kMvThreads) page_compact_kernel(CompactParams p) {
  __shared__ Pair s_warp[kMvWarps];
  const int ctas = gridDim.x, cta = blockIdx.x;
  const int threads = ctas * kMvThreads, t = cta * kMvThreads + threadIdx.x;
  const int mp = p.max_pages, entries = p.batch * mp;
  int count = __ldg(p.free_count);
  bool bad = count < 0 || count > p.free_cap;
  count = min(max(count, 0), p.free_cap);

  // ---- words of a page: live, times on the stack, number as a mover
  const auto used = [&](int e) {
    const int b = e / mp, len = __ldg(p.lens + b);
    if (len < 0 || len > mp * kPageKeys) {
      bad = true;
      return false;
    }
    return e - b * mp < pages_of(len);
  };
#pragma unroll 4
  for (int e = t; e < entries; e += threads) {
    if (!used(e)) continue;
    const int page = __ldg(p.block_table + e);
    if (page < 0 || page >= p.num_pages)
      bad = true;
    else
      __stcg(reinterpret_cast<int*>(p.words + page), 1);
  }
#pragma unroll 4
  for (int i = t; i < count; i += threads) {
    const int page = __ldg(p.free_pages + i);
    if (page < 0 || page >= p.num_pages)
      bad = true;
    else
      atomicAdd(reinterpret_cast<int*>(p.words + page) + 1, 1);
  }
  cluster_sync();

  // ---- ranks: live and idle pages before this thread's
  const int pper = (p.num_pages + threads - 1) / threads;
  const int p0 = min(p.num_pages, t * pper), p1 = min(p.num_pages, p0 + pper);
  Pair sum{0, 0};
#pragma unroll 4
  for (int g = p0; g < p1; ++g) {
    const int4 w = __ldcg(p.words + g);
    sum.a += w.x;
    sum.b += w.y;
    bad |= w.x + w.y > 1;
  }
  const int any_bad = __syncthreads_or(bad);
  Pair total;
  Pair at = block_scan(sum, s_warp, &total);
  bool stop = any_bad != 0;
  if (ctas > 1) {
    // (the sign carries the verdict: live pages and 1, negative, from a CTA that met one)
    if (threadIdx.x == 0) __stcg(p.totals + cta, make_int2(stop ? -total.a - 1 : total.a, total.b));
    cluster_sync();
    total = {0, 0};
    for (int c = 0; c < ctas; ++c) {
      int2 x = __ldcg(p.totals + c);
      if (x.x < 0) {
        stop = true;
        x.x = -x.x - 1;
      }
      if (c < cta) {
        at.a += x.x;
        at.b += x.y;
      }
      total.a += x.x;
      total.b += x.y;
    }
  }
  const int live = total.a;
  // live pages below rank `live`: known to the thread whose pages pass it
  {
    Pair x = at;
    if (x.a + x.b < live || (t == 0 && live == 0)) {
      for (int g = p0; g < p1 && x.a + x.b < live; ++g) {
        const int4 w = __ldcg(p.words + g);
        x.a += w.x;
        x.b += w.y;
      }
      if (x.a + x.b >= live) __stcg(p.below, x.a);
    }
  }
  cluster_sync();
  const int below = __ldcg(p.below), moves = stop ? 0 : live - below;

  // ---- the lists, and the stack
  if (!stop) {
    Pair x = at;
    for (int g = p0; g < p1; ++g) {
      const int4 w = __ldcg(p.words + g);
      const int rank = x.a + x.b;
      if (w.x && rank >= live) {
        const int j = x.a - below;
        __stcg(p.copy_src + j, g);
        __stcg(reinterpret_cast<int*>(p.words + g) + 2, j + 1);
      }
      if (w.y && rank < live) __stcg(p.copy_dst + x.b, g);
      if (w.x + w.y > 0 && rank >= live) p.free_out[live + total.b - 1 - rank] = g;
      x.a += w.x;
      x.b += w.y;
    }
  }
  for (int i = t; i < p.cap; i += threads)
    if (i >= moves) p.copy_src[i] = p.copy_dst[i] = -1;
  for (int i = (stop ? 0 : count) + t; i < p.free_cap; i += threads) p.free_out[i] = __ldg(p.free_pages + i);
  cluster_sync();

  // ---- the table
#pragma unroll 4
  for (int e = t; e < entries; e += threads) {
    int page = __ldg(p.block_table + e);
    if (!stop && used(e)) {
      const int j = __ldcg(reinterpret_cast<const int*>(p.words + page) + 2);
      if (j > 0) page = __ldcg(p.copy_dst + (j - 1));
    }
    p.table_out[e] = page;
  }
  if (stop && t == 0 && p.err) atomicOr(p.err, kErrBadArgs);
  cluster_sync();
#pragma unroll 4
  for (int g = p0; g < p1; ++g) __stcg(p.words + g, make_int4(0, 0, 0, 0));  // for the next call
}

// One warp per (entry, KV head, pool): `keys` rows of a page, contiguous.  A warp
// looks at `per` items at once, so that entries without a copy cost little; they lie
// a grid apart, since those with a copy lie together.
__global__ void __launch_bounds__(256) kv_copy_keys_kernel(CopyParams p, long long items, int per) {
  const int lane = threadIdx.x % 32;
  const long long warps = static_cast<long long>(gridDim.x) * (blockDim.x / 32);
  const long long w0 = blockIdx.x * static_cast<long long>(blockDim.x / 32) + threadIdx.x / 32;
  for (long long base = w0; base < items; base += warps * per) {
    int src = -1, dst = -1, keys = 0, part = 0;
    const long long item = base + lane * warps;
    if (lane < per && item < items) {
      part = static_cast<int>(item / p.n);
      const int e = static_cast<int>(item - static_cast<long long>(part) * p.n);
      src = __ldg(p.src + e);
      dst = __ldg(p.dst + e);
      keys = p.keys ? __ldg(p.keys + e) : kPageKeys;
      if (src >= p.num_pages || dst >= p.num_pages || keys < 0 || keys > kPageKeys) {
        if (p.err) atomicOr(p.err, kErrBadArgs);
        src = -1;
      }
    }
    unsigned todo = __ballot_sync(0xffffffffu, src >= 0 && dst >= 0 && keys > 0);
    while (todo) {
      const int l = __ffs(todo) - 1;
      todo &= todo - 1;
      const int a = __shfl_sync(0xffffffffu, src, l), b = __shfl_sync(0xffffffffu, dst, l);
      const int n = __shfl_sync(0xffffffffu, keys, l) * p.row_vecs;
      const int q = __shfl_sync(0xffffffffu, part, l);
      const int head = q >> 1;
      uint4* pool = static_cast<uint4*>(q & 1 ? p.v_pool : p.k_pool);
      const size_t page = static_cast<size_t>(kPageKeys) * p.row_vecs;
      const uint4* from = pool + (static_cast<size_t>(a) * p.heads + head) * page;
      uint4* to = pool + (static_cast<size_t>(b) * p.heads + head) * page;
      constexpr int kFlight = 8;
      for (int i = lane; i < n; i += 32 * kFlight) {
        uint4 x[kFlight];
#pragma unroll
        for (int k = 0; k < kFlight; ++k)
          if (i + 32 * k < n) x[k] = from[i + 32 * k];
#pragma unroll
        for (int k = 0; k < kFlight; ++k)
          if (i + 32 * k < n) to[i + 32 * k] = x[k];
      }
    }
  }
}

// One cluster: a single CTA where that has at most a few entries a thread.
template <typename P>
cudaError_t launch_cluster(void (*kernel)(P), const P& p, long long items, cudaStream_t s) {
  const int ctas = items <= 4LL * kMvThreads ? 1 : kMvCluster;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kMvThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

}  // namespace

cudaError_t launch_page_fork(const ForkParams& p, cudaStream_t s) {
  const long long rows = static_cast<long long>(p.batch > p.new_batch ? p.batch : p.new_batch);
  const long long entries = rows * p.max_pages;
  return launch_cluster(page_fork_kernel, p, entries > p.num_pages ? entries : p.num_pages, s);
}

cudaError_t launch_page_compact(const CompactParams& p, cudaStream_t s) {
  const long long entries = static_cast<long long>(p.batch) * p.max_pages;
  return launch_cluster(page_compact_kernel, p, entries > p.num_pages ? entries : p.num_pages, s);
}

cudaError_t launch_kv_copy_keys(const CopyParams& p, int sms, cudaStream_t s) {
  if (p.n <= 0) return cudaSuccess;
  const long long items = 2LL * p.n * p.heads;
  const long long room = 8LL * 8 * sms;  // warps in flight
  int per = 1;
  while (per < 32 && items > 2 * per * room) per *= 2;
  const long long ctas = ((items + per - 1) / per + 7) / 8;
  kv_copy_keys_kernel<<<static_cast<unsigned>(ctas < 8LL * sms ? ctas : 8LL * sms), 256, 0, s>>>(
      p, items, per);
  return cudaGetLastError();
}

}  // namespace ffai

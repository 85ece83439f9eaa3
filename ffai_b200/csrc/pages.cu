// Page tables and slot maps of a paged KV cache built on the device from
// request lengths, the release of finished requests' pages, and the scatter of
// new keys and values into the pages by slot.
//
// Request b holds ceil(L_b / 64) pages and asks for n_b new keys, so it needs
//   need_b = ceil((L_b + n_b) / 64) - ceil(L_b / 64)
// pages more.  With first_b the sum of the needs before it, its j-th new page
// is free_pages[free_count - 1 - (first_b + j)]: the free list is a stack, and
// pages go out in request order.  The slot of key position i of b is
// table[b][i / 64] * 64 + i % 64.  Whole numbers throughout, no atomics whose
// order matters: the result depends on the inputs alone.
//
// Bounds and device time on one B200: plans and releases are a chain of
// dependent loads and two scans, 3.8 us for 32 requests, 7.7 for 2000 with 130000
// tokens (1.2 of it for the looks at page ids), 3.1 for the release of 500 (a
// launch alone is about 2).  The scatter is bound by its bytes: 20001 tokens of
// 8 heads, f32 to bf16, move 123 MB in 23 us (5.3 TB/s, measured copies reach
// 6.46); 60 tokens of 20 heads take 2.1.
#include "common.cuh"
#include "kernels.h"

namespace ffai {

namespace {

constexpr int kPlThreads = 512;
constexpr int kPlWarps = kPlThreads / 32;

// Exclusive prefix sums of two 64-bit numbers per thread over the CTA.
struct Sum2 {
  long long a, b;
};
__device__ __forceinline__ Sum2 block_exclusive(Sum2 v, Sum2* s_warp) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  Sum2 inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long a = __shfl_up_sync(0xffffffffu, inc.a, o);
    const long long b = __shfl_up_sync(0xffffffffu, inc.b, o);
    if (lane >= o) {
      inc.a += a;
      inc.b += b;
    }
  }
  if (lane == 31) s_warp[warp] = inc;
  __syncthreads();
  Sum2 base{0, 0};
  for (int w = 0; w < warp; ++w) {
    base.a += s_warp[w].a;
    base.b += s_warp[w].b;
  }
  __syncthreads();
  return {base.a + inc.a - v.a, base.b + inc.b - v.b};
}

__device__ __forceinline__ int pages_of(long long keys) {
  return static_cast<int>((keys + kPageKeys - 1) / kPageKeys);
}

// Every CTA scans all requests (a few loads and two shuffle scans, cheaper
// than a second launch or a grid-wide exchange) and then maps its own stretch
// of the packed tokens.  Shared memory per request: the packed row of its
// first token, its length, and the stack offset of its first new page, or
// -1 when it is refused.  Page ids are looked at before anything is promised:
// the stack ends at its first bad id, and a request whose last page is bad
// and still has room takes part as if it outgrew the table.
__global__ void __launch_bounds__(kPlThreads) page_plan_kernel(PlanParams p) {
  extern __shared__ int s_plan[];
  int* s_cu = s_plan;                 // batch + 1
  int* s_len = s_plan + p.batch + 1;  // batch
  int* s_first = s_len + p.batch;     // batch; before that the pages needed, or -1
  __shared__ Sum2 s_warp[kPlWarps];
  __shared__ int s_taken, s_usable;
  const int per = (p.batch + kPlThreads - 1) / kPlThreads;
  const int b0 = min(p.batch, static_cast<int>(threadIdx.x) * per), b1 = min(p.batch, b0 + per);
  const int reach = p.max_pages * kPageKeys;  // host: fits 30 bits
  const int held_count = __ldg(p.free_count);
  bool bad = held_count < 0 || held_count > p.free_cap;
  const int count = bad ? 0 : held_count;
  if (threadIdx.x == 0) {
    s_taken = 0;
    s_usable = count;
  }
  __syncthreads();
  // The pages that requests within the rows can ask for: one a request and one
  // for every 64 rows.  Behind the first bad id the stack is not used.
  const int asked = min(count, p.slot_cap / kPageKeys + min(p.batch, p.slot_cap));
  int first_bad = INT32_MAX;
#pragma unroll 4
  for (int i = threadIdx.x; i < asked; i += kPlThreads) {
    const int id = __ldg(p.free_pages + (count - 1 - i));
    if (id < 0 || id >= p.num_pages) first_bad = min(first_bad, i);
  }
  if (first_bad != INT32_MAX) atomicMin(&s_usable, first_bad);

  Sum2 sum{0, 0};
  constexpr int kTogether = 4;  // requests whose loads are in flight together
  for (int bb = b0; bb < b1; bb += kTogether) {
    int len[kTogether], want[kTogether], id[kTogether];
#pragma unroll
    for (int k = 0; k < kTogether; ++k) {
      const int b = min(bb + k, b1 - 1);
      len[k] = __ldg(p.lens + b);
      want[k] = __ldg(p.new_tokens + b);
    }
#pragma unroll
    for (int k = 0; k < kTogether; ++k) {
      const int b = min(bb + k, b1 - 1);
      id[k] = 0;
      if (len[k] > 0 && len[k] < reach && len[k] % kPageKeys != 0 && want[k] > 0)
        // (an entry that no thread writes: new ones lie behind it)
        id[k] = p.block_table[static_cast<size_t>(b) * p.max_pages + len[k] / kPageKeys];
    }
#pragma unroll
    for (int k = 0; k < kTogether; ++k) {
      if (bb + k >= b1) break;
      bool ok = len[k] >= 0 && want[k] >= 0 && static_cast<long long>(len[k]) + want[k] <= reach;
      bad |= len[k] < 0 || want[k] < 0;
      if (ok && (id[k] < 0 || id[k] >= p.num_pages)) {
        ok = false;
        bad = true;
      }
      const int need = ok ? pages_of(len[k] + want[k]) - pages_of(len[k]) : -1;
      s_len[bb + k] = len[k];
      s_first[bb + k] = need;
      sum.a += max(want[k], 0);
      sum.b += max(need, 0);
    }
  }
  Sum2 at = block_exclusive(sum, s_warp);
  const int usable = s_usable;
  int taken = 0;
  for (int b = b0; b < b1; ++b) {
    const int len = s_len[b], want = __ldg(p.new_tokens + b), need = s_first[b];
    s_cu[b] = static_cast<int>(min(at.a, static_cast<long long>(INT32_MAX)));
    const long long first = at.b;
    at.a += max(want, 0);
    at.b += max(need, 0);
    const bool fits = need >= 0 && at.a <= p.slot_cap;
    const bool served = fits && (need == 0 || at.b <= usable);
    bad |= fits && !served && at.b <= count;  // for a bad id on the stack alone
    s_first[b] = served ? static_cast<int>(need == 0 ? 0 : first) : -1;
    if (served && need > 0) taken = static_cast<int>(at.b);
    if (blockIdx.x == 0) {
      p.cu_new[b] = s_cu[b];
      p.lens_out[b] = served ? len + want : len;
    }
  }
  if (b1 == p.batch && b0 < p.batch) {
    s_cu[p.batch] = static_cast<int>(min(at.a, static_cast<long long>(INT32_MAX)));
    if (blockIdx.x == 0) p.cu_new[p.batch] = s_cu[p.batch];
  }
  if (taken > 0) atomicMax(&s_taken, taken);
  __syncthreads();
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.free_count_out = held_count - s_taken;
  if (bad && blockIdx.x == 0 && p.err) atomicOr(p.err, kErrBadArgs);

  const int total = s_cu[p.batch];
  for (int t = blockIdx.x * kPlThreads + threadIdx.x; t < p.slot_cap; t += gridDim.x * kPlThreads) {
    int slot = -1, pos = 0;
    if (t < total) {
      // the request whose rows hold t: the last b with cu[b] <= t
      int lo = 0, hi = p.batch;  // cu[lo] <= t < cu[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_cu[mid] <= t)
          lo = mid;
        else
          hi = mid;
      }
      const int b = lo, first = s_first[b];
      if (first >= 0) {
        const int len = s_len[b], at_key = len + (t - s_cu[b]);
        const int held = pages_of(len), pg = at_key / kPageKeys;
        int* row = p.block_table + static_cast<size_t>(b) * p.max_pages;
        int id;
        if (pg < held) {
          id = row[pg];  // entries below `held` are written by no thread
        } else {
          id = __ldg(p.free_pages + (count - 1 - (first + pg - held)));
          // the page's first key of this request writes its table entry
          if (at_key % kPageKeys == 0) row[pg] = id;
        }
        slot = id * kPageKeys + at_key % kPageKeys;
        pos = at_key + (p.pos_base ? __ldg(p.pos_base + b) : 0);
      }
    }
    p.slots[t] = slot;
    if (p.positions) p.positions[t] = pos;
  }
}

// The pages of requests with done != 0 are pushed on the stack in request
// order, each request's in key order, as far as the stack reaches.  Every CTA
// scans all requests, then its warps copy the pages of every gridDim-th request.
__global__ void __launch_bounds__(kPlThreads) page_release_kernel(ReleaseParams p) {
  extern __shared__ int s_at[];  // batch: stack position of a request's first page, or -1
  __shared__ Sum2 s_warp[kPlWarps];
  const int per = (p.batch + kPlThreads - 1) / kPlThreads;
  const int b0 = min(p.batch, static_cast<int>(threadIdx.x) * per), b1 = min(p.batch, b0 + per);
  int count = __ldg(p.free_count);
  bool bad = count < 0 || count > p.free_cap;
  count = min(max(count, 0), p.free_cap);
  const int reach = p.max_pages * kPageKeys;
  auto gives = [&](int b) {
    const int len = __ldg(p.lens + b);
    if (__ldg(p.done + b) == 0) return 0;
    if (len < 0 || len > reach) {
      bad = true;
      return 0;
    }
    return pages_of(len);
  };
  Sum2 sum{0, 0};
  for (int b = b0; b < b1; ++b) sum.a += gives(b);
  Sum2 at = block_exclusive(sum, s_warp);
  for (int b = b0; b < b1; ++b) {
    const int n = gives(b);
    const long long dst = count + at.a;
    s_at[b] = n > 0 && dst < p.free_cap ? static_cast<int>(dst) : -1;
    bad |= dst + n > p.free_cap;
    at.a += n;
    if (blockIdx.x == 0) p.lens_out[b] = __ldg(p.done + b) != 0 ? 0 : __ldg(p.lens + b);
  }
  if (b1 == p.batch && b0 < p.batch && blockIdx.x == 0)
    *p.free_count_out = static_cast<int>(min(count + at.a, static_cast<long long>(p.free_cap)));
  if (bad && blockIdx.x == 0 && p.err) atomicOr(p.err, kErrBadArgs);
  __syncthreads();
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  for (int b = blockIdx.x * kPlWarps + warp; b < p.batch; b += gridDim.x * kPlWarps) {
    const int dst = s_at[b];
    if (dst < 0) continue;
    const int n = min(pages_of(__ldg(p.lens + b)), p.free_cap - dst);
    for (int i = lane; i < n; i += 32)
      p.free_pages[dst + i] = __ldg(p.block_table + static_cast<size_t>(b) * p.max_pages + i);
  }
}

// ---------------------------------------------------------------- write

template <typename T>
struct alignas(sizeof(T) * 8 < 16 ? sizeof(T) * 8 : 16) Vec8 {
  T v[8];
};

// One thread per 8 elements of a (token, head) row of both keys and values;
// 8 threads make a row, so a warp writes four whole rows of a pool.  VEC:
// 16-byte accesses (rows and base aligned), else element by element.
template <typename S, typename T, bool VEC>
__global__ void __launch_bounds__(256) kv_write_kernel(WriteParams p) {
  const long long n = static_cast<long long>(p.tokens) * p.heads * 8;
  const S* ks = static_cast<const S*>(p.k_new);
  const S* vs = static_cast<const S*>(p.v_new);
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
    const int part = static_cast<int>(i & 7);
    const long long th = i >> 3;
    const int tok = static_cast<int>(th / p.heads), h = static_cast<int>(th - static_cast<long long>(tok) * p.heads);
    const int slot = __ldg(p.slots + tok);
    if (slot < 0) continue;
    const int page = slot / kPageKeys;
    if (page >= p.num_pages) {
      if (p.err) atomicOr(p.err, kErrBadArgs);
      continue;
    }
    const long long src = tok * p.src_stride + h * 64 + part * 8;
    const long long dst =
        ((static_cast<long long>(page) * p.heads + h) * kPageKeys + slot % kPageKeys) * 64 + part * 8;
    Vec8<S> a, b;
    if constexpr (VEC) {
      a = *reinterpret_cast<const Vec8<S>*>(ks + src);
      b = *reinterpret_cast<const Vec8<S>*>(vs + src);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        a.v[e] = ks[src + e];
        b.v[e] = vs[src + e];
      }
    }
    Vec8<T> x, y;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (sizeof(S) == sizeof(T)) {  // the same type: a copy
        x.v[e] = a.v[e];
        y.v[e] = b.v[e];
      } else {
        x.v[e] = from_f32<T>(to_f32<S>(a.v[e]));
        y.v[e] = from_f32<T>(to_f32<S>(b.v[e]));
      }
    }
    // the pools are 16-byte aligned (host), and a row starts at a multiple of 64 elements
    *reinterpret_cast<Vec8<T>*>(static_cast<T*>(p.k_pool) + dst) = x;
    *reinterpret_cast<Vec8<T>*>(static_cast<T*>(p.v_pool) + dst) = y;
  }
}

template <typename S, typename T>
cudaError_t write_t(const WriteParams& p, int grid, cudaStream_t s) {
  if (p.vec)
    kv_write_kernel<S, T, true><<<grid, 256, 0, s>>>(p);
  else
    kv_write_kernel<S, T, false><<<grid, 256, 0, s>>>(p);
  return cudaGetLastError();
}

int plan_grid(long long items, int sms) {
  const long long g = (items + kPlThreads - 1) / kPlThreads;
  return static_cast<int>(g < 1 ? 1 : (g < sms ? g : sms));
}

template <typename K>
cudaError_t allow_smem(K kernel, size_t bytes) {
  if (bytes <= 48 * 1024) return cudaSuccess;
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              static_cast<int>(bytes));
}

}  // namespace

cudaError_t launch_page_plan(const PlanParams& p, int sms, cudaStream_t s) {
  const size_t smem = (3 * static_cast<size_t>(p.batch) + 1) * sizeof(int);
  cudaError_t e = allow_smem(page_plan_kernel, smem);
  if (e != cudaSuccess) return e;
  page_plan_kernel<<<plan_grid(p.slot_cap, sms), kPlThreads, smem, s>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_page_release(const ReleaseParams& p, int sms, cudaStream_t s) {
  const size_t smem = static_cast<size_t>(p.batch) * sizeof(int);
  cudaError_t e = allow_smem(page_release_kernel, smem);
  if (e != cudaSuccess) return e;
  page_release_kernel<<<plan_grid(p.batch * 32ll, sms), kPlThreads, smem, s>>>(p);
  return cudaGetLastError();
}

cudaError_t launch_kv_write(const WriteParams& p, int sms, cudaStream_t s) {
  const long long blocks = (static_cast<long long>(p.tokens) * p.heads * 8 + 255) / 256;
  const int grid = static_cast<int>(blocks < sms * 8ll ? blocks : sms * 8ll);
  switch (p.src_dtype * 3 + p.dst_dtype) {
    case 0: return write_t<float, float>(p, grid, s);
    case 1: return write_t<float, __nv_bfloat16>(p, grid, s);
    case 2: return write_t<float, __half>(p, grid, s);
    case 4: return write_t<__nv_bfloat16, __nv_bfloat16>(p, grid, s);
    case 8: return write_t<__half, __half>(p, grid, s);
  }
  return cudaErrorInvalidValue;
}

}  // namespace ffai

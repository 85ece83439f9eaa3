// Attention of a chunk of new tokens over a paged KV cache, sequences with few
// query rows: single tokens, a handful of drafted ones.
//
// Sequence b brings n_b = cu_q[b + 1] - cu_q[b] tokens, the newest of the
// len_b = seq_lens[b] keys in its pages.  Query row (token i, head h) sees the
// keys j < len_b - (n_b - 1 - i), all len_b of them without the causal mask; query
// head h reads KV head h / G, G = heads / kv_heads:
//   s_j = scale q.k_j,  o = sum_j e^(s_j - m) v_j / l,  l = sum_j e^(s_j - m).
// A row that sees no key gives zeros and an lse of -inf.
//
// A unit is 16 of a (sequence, KV head)'s n_b G rows, the matrix instruction's;
// it passes over its keys in blocks of 128, a step each, four warps with 32 keys
// apiece (rows.cuh).  The steps of all units lie on one line, W of them, and CTA
// c takes the steps [c S, (c + 1) S): a long cache is read by many CTAs, whatever
// the batch, and no length passes through the host.  A unit that lies in one
// stretch is finished there; else each CTA leaves a partial result (running
// maximum, sum, unnormalised output), and the last of the unit's CTAs to come
// (a ticket) merges all of them, in their order on the line, so equal inputs
// give equal bits.  A CTA has at most two such partials, of its first and its
// last unit.
#include <algorithm>

#include "chunk.cuh"
#include "rows.cuh"

namespace ffai {

namespace {

template <int F16, int TERMS>
__global__ void __launch_bounds__(kSpThreads, TERMS > 1 ? 2 : 3) chunk_rows_kernel(ChunkParams p) {
  extern __shared__ __align__(128) uint8_t sp_smem[];
  __shared__ Stretch s_start;
  __shared__ int s_warp[kSpWarps];
  __shared__ int s_last;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane >> 2;
  const int G = p.heads / p.kv_heads;
  RowsMerge<kSpWarps>& sm = *reinterpret_cast<RowsMerge<kSpWarps>*>(sp_smem);
  find_stretch<kChRows, kSpThreads>(p, &s_start, s_warp);
  Stretch w = s_start;
  bool bad = false;
  ChunkSeq s{};
  if (w.left > 0) s = chunk_seq(p, w.b, bad);
  while (w.left > 0) {
    // ---- the unit's rows, and the keys each sees
    const int row0 = w.m * kChRows, rows = min(kChRows, s.n * G - row0);
    const int steps = unit_steps<kChRows>(p, s, G, w.m), n = min(w.left, steps - w.step);
    const int k0 = w.step * kChKeys;
    int seq[2] = {0, 0}, tok[2], head[2], see[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int row = row0 + g + 8 * r, i = row / G;
      const bool real = g + 8 * r < rows;
      tok[r] = real ? s.t0 + i : -1;
      head[r] = w.h * G + row - i * G;
      see[r] = real ? chunk_limit(p, s, i) - k0 : 0;
    }
    const int common = max(0, chunk_limit(p, s, row0 / G) - k0);
    const int len = min(chunk_limit(p, s, (row0 + rows - 1) / G) - k0, n * kChKeys);
    const int* table = p.block_table + static_cast<size_t>(w.b) * p.max_pages + 2 * w.step;
    const int pages = p.max_pages - 2 * w.step;
    const int ids = step_page<kSpWarps>(table, pages, warp, 0);
    RowQ q[TERMS];
    RowState st;
    load_rows(q, st, p, seq, tok, head);
    walk<F16, kSpWarps, true, TERMS>(st, q, p, w.h, table, pages, ids, len, common, see, warp,
                              sp_smem + warp * kSpRing);
    cp_async_wait_all();
    __syncthreads();  // the rings are done with
    put_state(st, sm, warp);
    __syncthreads();
    const int row = threadIdx.x / 8, part = threadIdx.x % 8;
    Merged acc{-INFINITY, 0.f, {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}};
#pragma unroll 1
    for (int x = 0; x < kSpWarps; ++x) add_state(acc, sm, x, row, part);
    bool write = n == steps;
    if (!write) {
      // ---- a part of the unit: left for the last of its CTAs
      const int c0 = w.unit0 / w.share;
      const int c1 = min((w.unit0 + steps - 1) / w.share, static_cast<int>(gridDim.x) - 1);
      const int cta = static_cast<int>(blockIdx.x);
      const auto slot = [&](int c) { return (static_cast<size_t>(2 * c + (c == c0 ? 1 : 0)) * kChRows + row); };
      float4* o = reinterpret_cast<float4*>(p.part_o + slot(cta) * 64 + 8 * part);
      __stcg(o, make_float4(acc.o[0], acc.o[1], acc.o[2], acc.o[3]));
      __stcg(o + 1, make_float4(acc.o[4], acc.o[5], acc.o[6], acc.o[7]));
      if (part == 0)
        __stcg(reinterpret_cast<float2*>(p.part_ml + 2 * slot(cta)), make_float2(acc.m, acc.l));
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0)
        s_last = atomicInc(p.tickets + c0, static_cast<unsigned>(c1 - c0)) ==
                 static_cast<unsigned>(c1 - c0);
      __syncthreads();
      if (s_last) {
        __threadfence();
        write = true;
        acc = Merged{-INFINITY, 0.f, {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}};
#pragma unroll 4
        for (int c = c0; c <= c1; ++c) {
          const float4* x = reinterpret_cast<const float4*>(p.part_o + slot(c) * 64 + 8 * part);
          acc.add(__ldcg(reinterpret_cast<const float2*>(p.part_ml + 2 * slot(c))), __ldcg(x), __ldcg(x + 1));
        }
      }
    }
    if (write && row < rows) {
      const int i = (row0 + row) / G;
      store_row(p, acc, s.t0 + i, w.h * G + row0 + row - i * G, part);
    }
    __syncthreads();  // the states are read: the rings may be filled again
    // ---- on to the next unit
    w.left -= n;
    if (w.left > 0) {
      w.step = 0;
      w.unit0 += steps;
      if (++w.m == chunk_units<kChRows>(s, G)) {
        w.m = 0;
        if (++w.h == p.kv_heads) {
          w.h = 0;
          s.n = 0;
          while (s.n == 0 && ++w.b < p.batch) s = chunk_seq(p, w.b, bad);
          if (s.n == 0) break;
        }
      }
    }
  }
}

}  // namespace

cudaError_t launch_chunk_rows(const ChunkParams& p, int grid, cudaStream_t s) {
  // f16: two terms hold 22 of a query's 24 bits, bf16: three hold all
  auto kern = p.precise ? (p.kv_dtype == 2 ? chunk_rows_kernel<1, 2> : chunk_rows_kernel<0, 3>)
                        : (p.kv_dtype == 2 ? chunk_rows_kernel<1, 1> : chunk_rows_kernel<0, 1>);
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       static_cast<int>(kSpSmem));
  if (e != cudaSuccess) return e;
  kern<<<grid, kSpThreads, kSpSmem, s>>>(p);
  return cudaGetLastError();
}

}  // namespace ffai

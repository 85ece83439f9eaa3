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
// tiles of 16 (the matrix instruction's rows); each warp of a CTA takes every
// kSpWarps-th step of 32 keys with a softmax state of its own, and the warps
// merge at the end.  K and V go from global memory straight into the operand
// registers: the products' inner order is free, so it is chosen such that
// each lane's operands are whole 16-byte pieces of the key rows.
#include "shared_prefix.cuh"

namespace ffai {

namespace {

constexpr int kSpWarps = 4;
constexpr int kSpThreads = kSpWarps * 32;
constexpr int kSpKeys = 32;  // keys per warp step (divides a page)

template <int F16>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  if constexpr (F16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
        "{%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Softmax state of a warp's 16 rows: lane (g, t) = (lane / 4, lane % 4) holds
// rows g and g + 8; o[j][2 v + w] is row g + 8 v, head dim 16 t + 8 w + j.
struct RowState {
  float m[2], l[2];
  float o[8][4];
};

// The 16 query rows as A operands: k-step s (16 of the 64 head dims) holds
// dims 32 (s / 2) + 8 t + 4 (s % 2) + {0, 1} and + {2, 3}, so that the lane's
// part of a key row is the two 16-byte pieces at dims 8 t and 32 + 8 t.
struct RowQ {
  uint32_t a[4][4];
};

__device__ __forceinline__ uint4 zero4() { return make_uint4(0, 0, 0, 0); }

// One step: 32 keys of one page starting at kp / vp; `live` of them hold data
// (the rest are not read), and row v of this lane sees the first `see[v]`.
template <int F16>
__device__ __forceinline__ void step32(RowState& st, const RowQ& q, const uint16_t* kp,
                                       const uint16_t* vp, int live, const int (&see)[2],
                                       float scale_log2) {
  const int lane = threadIdx.x % 32, g = lane >> 2, t = lane & 3;
  uint4 k[4][2];  // n-tile i: key 8 i + g
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int key = 8 * i + g;
    const uint4* src = reinterpret_cast<const uint4*>(kp + key * 64);
    k[i][0] = key < live ? __ldg(src + t) : zero4();
    k[i][1] = key < live ? __ldg(src + 4 + t) : zero4();
  }
  uint4 v[2][4];  // 16-key half h: keys 16 h + 2 t + {0, 1, 8, 9}, dims 8 g ..
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int key = 16 * h + 2 * t + (e & 1) + 8 * (e >> 1);
      v[h][e] = key < live ? __ldg(reinterpret_cast<const uint4*>(vp + key * 64) + g) : zero4();
    }
  float s[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int e = 0; e < 4; ++e) s[i][e] = 0.f;
    mma16816<F16>(s[i], q.a[0], k[i][0].x, k[i][0].y);
    mma16816<F16>(s[i], q.a[1], k[i][0].z, k[i][0].w);
    mma16816<F16>(s[i], q.a[2], k[i][1].x, k[i][1].y);
    mma16816<F16>(s[i], q.a[3], k[i][1].z, k[i][1].w);
  }
  uint32_t p[2][4];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        // a key the row does not see weighs nothing, whatever it holds
        const float x = 8 * i + 2 * t + e < see[r] ? s[i][2 * r + e] * scale_log2 : -INFINITY;
        s[i][2 * r + e] = x;
        mx = fmaxf(mx, x);
      }
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    const float m_new = fmaxf(st.m[r], mx);
    const float base = m_new == -INFINITY ? 0.f : m_new;
    const float corr = ex2_approx(st.m[r] - base);
    st.m[r] = m_new;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float p0 = ex2_approx(s[i][2 * r] - base), p1 = ex2_approx(s[i][2 * r + 1] - base);
      sum += p0 + p1;
      // the weights enter the second product in the cache's 16-bit type (at
      // most 1, relative error 2^-9 or 2^-12); their sum stays unrounded f32
      p[i >> 1][(i & 1) * 2 + r] = F16 ? pack_f16x2(p0, p1) : pack_bf16x2(p0, p1);
    }
    st.l[r] = fmaf(st.l[r], corr, sum);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      st.o[j][2 * r] *= corr;
      st.o[j][2 * r + 1] *= corr;
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t e0[4] = {v[h][0].x, v[h][0].y, v[h][0].z, v[h][0].w};
    const uint32_t e1[4] = {v[h][1].x, v[h][1].y, v[h][1].z, v[h][1].w};
    const uint32_t e2[4] = {v[h][2].x, v[h][2].y, v[h][2].z, v[h][2].w};
    const uint32_t e3[4] = {v[h][3].x, v[h][3].y, v[h][3].z, v[h][3].w};
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      mma16816<F16>(st.o[2 * c], p[h], __byte_perm(e0[c], e1[c], 0x5410),
                    __byte_perm(e2[c], e3[c], 0x5410));
      mma16816<F16>(st.o[2 * c + 1], p[h], __byte_perm(e0[c], e1[c], 0x7632),
                    __byte_perm(e2[c], e3[c], 0x7632));
    }
  }
}

__device__ __forceinline__ uint32_t q_pair(const SharedParams& p, const void* row, int dim) {
  if (p.q_dtype == 0) {  // f32 queries are rounded to the cache's type
    const float2 x = __ldg(reinterpret_cast<const float2*>(static_cast<const float*>(row) + dim));
    return p.kv_dtype == 2 ? pack_f16x2(x.x, x.y) : pack_bf16x2(x.x, x.y);
  }
  return __ldg(reinterpret_cast<const uint32_t*>(static_cast<const uint16_t*>(row) + dim));
}

__device__ __forceinline__ const void* q_row(const SharedParams& p, int b, int tok, int h) {
  const size_t off = static_cast<size_t>(b) * p.q_sb + static_cast<size_t>(tok) * p.q_st +
                     static_cast<size_t>(h) * p.q_sh;
  return static_cast<const uint8_t*>(p.q) + off * (p.q_dtype == 0 ? 4 : 2);
}

// The group whose sequences hold b, or -1 (a whole warp): starts[] rises, so
// it is the last group that starts at or before b, if b is before its end.
__device__ __forceinline__ int group_of(const SharedParams& p, int b) {
  const int lane = threadIdx.x % 32;
  int n = 0;  // groups that start at or before b
  for (int base = 0; base < p.groups; base += 32) {
    const int g = base + lane;
    const bool in = g < p.groups && __ldg(p.group_starts + g) <= b;
    n += __popc(__ballot_sync(0xffffffffu, in));
  }
  if (n == 0) return -1;
  return b < __ldg(p.group_starts + n) ? n - 1 : -1;
}

// Page ids of a warp's next 32 steps, one per lane: warp w takes the steps w, w
// + kSpWarps, ... of 32 keys, and `first` counts the warp's own.
__device__ __forceinline__ int step_page(const int* table, int pages, int warp, int first) {
  const int page = (warp + kSpWarps * (first + static_cast<int>(threadIdx.x % 32))) / 2;
  return page < pages ? __ldg(table + page) : -1;
}

// Walk `len` keys of a list of pages.  `ids` holds the first 32 steps' page
// ids, loaded ahead (the table does not depend on the lengths).
template <int F16>
__device__ __forceinline__ void walk(RowState& st, const RowQ& q, const SharedParams& p, int kvh,
                                     const int* table, int pages, int ids, int len,
                                     const int (&see)[2], int warp) {
  const uint16_t* kpool = static_cast<const uint16_t*>(p.k_pool);
  const uint16_t* vpool = static_cast<const uint16_t*>(p.v_pool);
  int n = 0;
  for (int k0 = warp * kSpKeys; k0 < len; k0 += kSpWarps * kSpKeys, ++n) {
    if (n == 32) {
      ids = step_page(table, pages, warp, k0 / (kSpWarps * kSpKeys));
      n = 0;
    }
    const int page = __shfl_sync(0xffffffffu, ids, n);
    if (page < 0 || page >= p.num_pages) {  // not read; its keys weigh nothing
      if (p.err && threadIdx.x % 32 == 0) atomicOr(p.err, kErrBadArgs);
      continue;
    }
    const size_t off =
        ((static_cast<size_t>(page) * p.kv_heads + kvh) * kPageKeys + k0 % kPageKeys) * 64;
    const int rel[2] = {see[0] - k0, see[1] - k0};
    step32<F16>(st, q, kpool + off, vpool + off, len - k0, rel, p.scale_log2);
  }
}

constexpr int kSpStage = 96;  // staged (part, row) pairs: 80 floats each

// A merge of partial softmax results of one row, 8 head dims a thread.
struct Merged {
  float m, l, o[8];
  __device__ __forceinline__ void add(const float2 ml, const float4 a, const float4 b) {
    if (ml.x == -INFINITY) return;  // nothing in it
    const float M = fmaxf(m, ml.x);
    const float f0 = m == -INFINITY ? 0.f : ex2_approx(m - M), f1 = ex2_approx(ml.x - M);
    m = M;
    l = l * f0 + ml.y * f1;
    const float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = o[e] * f0 + x[e] * f1;
  }
};

// The prefix kernel's partials of this CTA's rows (thread = row, 8 head dims),
// folded into `acc`: copied to shared memory as many at a time as fit, so that
// their latencies overlap, then added in the order of the line.
__device__ __forceinline__ void fold_partials(Merged& acc, float* stage, const SharedParams& p,
                                              int group, int b, int kvh, int row, int R) {
  const int part = threadIdx.x % 8, lrow = threadIdx.x / 8;
  const GroupDims d = group_dims(p, group);
  if (d.nb == 0) return;
  // written by the preceding kernel, which may have run beside this one
  const int share = __ldcg(p.part_plan), lin0 = __ldcg(p.part_plan + 1 + 2 * group),
            seg0 = __ldcg(p.part_plan + 2 + 2 * group);
  if (row >= R) return;
  const int cl = chunk_blocks(d, share), chunks = (d.nb + cl - 1) / cl;
  const int rg = (b - d.b0) * R + row, m = rg / kPxRows;
  const size_t at = static_cast<size_t>(rg - m * kPxRows);
  const int head0 = lin0 + kvh * head_steps(d, d.nb);
  // a thread stages and reads its own pieces: no barrier
  const int rows = min(R, 16), room = kSpStage / rows;  // parts staged at a time
  float* mine = stage + (lrow * 8 + part) * 8;
  float* mine_ml = stage + kSpStage * 64 + (lrow * 8 + part) * 2;
  const int pitch = rows * 64, pitch_ml = rows * 16;
  int q = 0, c = -1, c1 = -2, seg = 0;
  bool more = true;
  while (more) {
    int n = 0;
#pragma unroll 1
    while (n < room) {
      if (c > c1 || c1 < 0) {  // next chunk
        if (q == chunks) {
          more = false;
          break;
        }
        const int len = min(cl, d.nb - q * cl);
        const int l0 = head0 + head_steps(d, q * cl) + m * len;
        seg = seg0 + (kvh * chunks + q) * d.mu + m;
        c = l0 / share;
        c1 = (l0 + unit_steps(d, m, len) - 1) / share;
        ++q;
      }
      const int slot = c + seg;
      const bool have = slot < p.part_slots;
      const size_t pr = static_cast<size_t>(have ? slot : 0) * kPxRows + at;
      cp_async16(mine + n * pitch, p.part_o + pr * 64 + 8 * part, have);
      cp_async16(mine + n * pitch + 4, p.part_o + pr * 64 + 8 * part + 4, have);
      if (have)
        cp_async8(mine_ml + n * pitch_ml, p.part_ml + 2 * pr);
      else
        *reinterpret_cast<float2*>(mine_ml + n * pitch_ml) = make_float2(-INFINITY, 0.f);
      ++c;
      ++n;
    }
    cp_async_wait_all();
#pragma unroll 1
    for (int i = 0; i < n; ++i)
      acc.add(*reinterpret_cast<const float2*>(mine_ml + i * pitch_ml),
              *reinterpret_cast<const float4*>(mine + i * pitch),
              *reinterpret_cast<const float4*>(mine + i * pitch + 4));
  }
}

constexpr int kSpPitch = 68;  // floats per merged row: m, l, then o[64]

template <int F16>
__global__ void __launch_bounds__(kSpThreads, 4) shared_rows_kernel(SharedParams p) {
  __shared__ __align__(16) float s_part[kSpWarps][16][kSpPitch];
  __shared__ __align__(16) float s_stage[kSpStage * 80];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane >> 2, t = lane & 3;
  const int G = p.heads / p.kv_heads, R = p.q_len * G;
  const int tiles = (R + 15) / 16;
  const unsigned id = blockIdx.x, job = id / tiles;
  const int tile = static_cast<int>(id - job * tiles);
  const int b = static_cast<int>(job / p.kv_heads), kvh = static_cast<int>(job - b * p.kv_heads);

  const int* table = p.block_table + static_cast<size_t>(b) * p.max_pages;
  const int ids = step_page(table, p.max_pages, warp, 0);
  int len = __ldg(p.seq_lens + b);
  RowQ q;
  RowState st;
  int tok[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = tile * 16 + g + 8 * r;
    tok[r] = row < R ? row / G : -1;
    const void* src = row < R ? q_row(p, b, tok[r], kvh * G + row % G) : nullptr;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int dim = 32 * (s / 2) + 8 * t + 4 * (s % 2);
      q.a[s][r] = row < R ? q_pair(p, src, dim) : 0u;
      q.a[s][2 + r] = row < R ? q_pair(p, src, dim + 2) : 0u;
    }
    st.m[r] = -INFINITY;
    st.l[r] = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) st.o[j][2 * r] = st.o[j][2 * r + 1] = 0.f;
  }
  if (len < 0 || len > p.max_pages * kPageKeys) {
    if (p.err && threadIdx.x == 0) atomicOr(p.err, kErrBadArgs);
    len = min(max(len, 0), p.max_pages * kPageKeys);
  }
  const int see[2] = {tok[0] < 0 ? 0 : max(0, len - (p.q_len - 1 - tok[0])),
                      tok[1] < 0 ? 0 : max(0, len - (p.q_len - 1 - tok[1]))};
  walk<F16>(st, q, p, kvh, table, p.max_pages, ids, len, see, warp);
  const int group = group_of(p, b);
  if (!p.part_o && group >= 0) {  // no prefix kernel: the prefix too
    int plen = __ldg(p.prefix_lens + group);
    if (plen < 0 || plen > p.prefix_pages * kPageKeys) {
      if (p.err && threadIdx.x == 0) atomicOr(p.err, kErrBadArgs);
      plen = min(max(plen, 0), p.prefix_pages * kPageKeys);
    }
    const int all[2] = {plen, plen};
    table = p.prefix_table + static_cast<size_t>(group) * p.prefix_pages;
    walk<F16>(st, q, p, kvh, table, p.prefix_pages, step_page(table, p.prefix_pages, warp, 0), plen,
              all, warp);
  }

#pragma unroll
  for (int r = 0; r < 2; ++r) {
    float l = st.l[r];
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    float* w = s_part[warp][g + 8 * r];
    if (t == 0) *reinterpret_cast<float2*>(w) = make_float2(st.m[r], l);
    float4* o = reinterpret_cast<float4*>(w + 4 + 16 * t);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      o[e] = make_float4(st.o[4 * e][2 * r], st.o[4 * e + 1][2 * r], st.o[4 * e + 2][2 * r],
                         st.o[4 * e + 3][2 * r]);
      o[2 + e] = make_float4(st.o[4 * e][2 * r + 1], st.o[4 * e + 1][2 * r + 1],
                             st.o[4 * e + 2][2 * r + 1], st.o[4 * e + 3][2 * r + 1]);
    }
  }
  __syncthreads();
  // merge: 8 threads a row, 8 head dims each
  const int lrow = threadIdx.x / 8, part = threadIdx.x % 8, rr = tile * 16 + lrow;
  Merged acc{-INFINITY, 0.f, {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}};
#pragma unroll 1
  for (int w = 0; w < kSpWarps; ++w) {
    const float* x = s_part[w][lrow];
    acc.add(*reinterpret_cast<const float2*>(x), *reinterpret_cast<const float4*>(x + 4 + 8 * part),
            *reinterpret_cast<const float4*>(x + 8 + 8 * part));
  }
  if (p.part_o) {
    griddep_wait();  // the prefix kernel's partials
    if (group >= 0) fold_partials(acc, s_stage, p, group, b, kvh, rr, R);
  }
  if (rr >= R) return;
  const int ti = rr / G, h = kvh * G + rr % G;
  const size_t at = static_cast<size_t>(b) * p.o_sb + static_cast<size_t>(ti) * p.o_st +
                    static_cast<size_t>(h) * p.o_sh + 8 * part;
  const float inv = acc.l > 0.f ? 1.f / acc.l : 0.f;
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
        acc.l > 0.f ? (acc.m + log2f(acc.l)) * 0.69314718055994530942f : -INFINITY;
}

}  // namespace

cudaError_t launch_shared_rows(const SharedParams& p, cudaStream_t s) {
  const int R = p.q_len * (p.heads / p.kv_heads);
  const long long ctas = static_cast<long long>(p.batch) * p.kv_heads * ((R + 15) / 16);
  // Behind the prefix kernel it is a programmatic dependent: sequences' own
  // keys are attended while the last prefix tiles finish.
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(kSpThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.part_o ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, p.kv_dtype == 2 ? shared_rows_kernel<1> : shared_rows_kernel<0>, p);
}

}  // namespace ffai

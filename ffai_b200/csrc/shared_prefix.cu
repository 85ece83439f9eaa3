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
// merge at the end.  A warp copies its steps' key and value rows two steps
// ahead into shared memory of its own (no barrier), and takes its operands
// from there in 16-byte pieces: the products' inner order is free, so it is
// chosen such that a lane's operands are whole pieces of the rows.
//
// The prefixes' share comes from one of three places, by size (shared_plan):
//  * this kernel walks them too, each sequence for itself (short prefixes: the
//    repeated reads hit L2 and a second launch costs more);
//  * prefix_rows_kernel, the same walk over a group's rows, when a group has few
//    rows: its partial results are merged here;
//  * prefix_tc_kernel (prefix_tc.cu), on the tensor cores proper, otherwise.
#include <atomic>

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

// A warp's copies: kSpDepth steps of 32 key rows, then 32 value rows.
constexpr int kSpDepth = 2;
constexpr int kSpStep = 2 * kSpKeys * 128;  // bytes
constexpr int kSpRing = kSpDepth * kSpStep;

// Piece c (16 bytes) of row `key` sits where the eight lanes that read together
// meet eight different banks: key rows are read by row pairs, four pieces each;
// value rows by the rows 0, 2, 4, 6 (or 1, 3, 5, 7), two pieces each.
__device__ __forceinline__ int k_piece(int key, int c) {
  return key * 128 + ((c ^ ((key & 1) << 2)) << 4);
}
__device__ __forceinline__ int v_piece(int key, int c) {
  return kSpKeys * 128 + key * 128 + ((c ^ (((key >> 1) & 3) << 1)) << 4);
}

// Start copying one step (32 keys of one page at kp / vp, `live` of them to be
// read, zeros behind them) into buf.
__device__ __forceinline__ void fetch32(uint8_t* buf, const uint16_t* kp, const uint16_t* vp, int live) {
  const int lane = threadIdx.x % 32, c = lane & 7;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int key = 4 * i + (lane >> 3);
    const bool have = key < live;
    const int off = have ? key * 64 + c * 8 : 0;
    cp_async16(buf + k_piece(key, c), kp + off, have);
    cp_async16(buf + v_piece(key, c), vp + off, have);
  }
}

// One step from buf; row v of this lane sees the first `see[v]` of its keys.
template <int F16>
__device__ __forceinline__ void step32(RowState& st, const RowQ& q, const uint8_t* buf,
                                       const int (&see)[2], float scale_log2) {
  const int lane = threadIdx.x % 32, g = lane >> 2, t = lane & 3;
  uint4 k[4][2];  // n-tile i: key 8 i + g
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    k[i][0] = *reinterpret_cast<const uint4*>(buf + k_piece(8 * i + g, t));
    k[i][1] = *reinterpret_cast<const uint4*>(buf + k_piece(8 * i + g, 4 + t));
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
  uint4 v[2][4];  // 16-key half h: keys 16 h + 2 t + {0, 1, 8, 9}, dims 8 g ..
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int e = 0; e < 4; ++e)
      v[h][e] = *reinterpret_cast<const uint4*>(
          buf + v_piece(16 * h + 2 * t + (e & 1) + 8 * (e >> 1), g));
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
// ids, loaded ahead (the table does not depend on the lengths).  `ring`: this
// warp's kSpRing bytes, not in use.
template <int F16>
__device__ __forceinline__ void walk(RowState& st, const RowQ& q, const SharedParams& p, int kvh,
                                     const int* table, int pages, int ids, int len,
                                     const int (&see)[2], int warp, uint8_t* ring) {
  const uint16_t* kpool = static_cast<const uint16_t*>(p.k_pool);
  const uint16_t* vpool = static_cast<const uint16_t*>(p.v_pool);
  constexpr int kStride = kSpWarps * kSpKeys;
  const int steps = (len - warp * kSpKeys + kStride - 1) / kStride;
  int first = 0;  // ids are those of steps first .. first + 31
  const auto fetch = [&](int i) {
    if (i < steps) {
      if (i - first == 32) {
        first = i;
        ids = step_page(table, pages, warp, first);
      }
      const int k0 = i * kStride + warp * kSpKeys;
      const int page = __shfl_sync(0xffffffffu, ids, i - first);
      const bool ok = page >= 0 && page < p.num_pages;
      if (!ok && p.err && threadIdx.x % 32 == 0) atomicOr(p.err, kErrBadArgs);  // not read
      const size_t off = ((static_cast<size_t>(ok ? page : 0) * p.kv_heads + kvh) * kPageKeys +
                          k0 % kPageKeys) * 64;
      fetch32(ring + i % kSpDepth * kSpStep, kpool + off, vpool + off, ok ? len - k0 : 0);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kSpDepth; ++i) fetch(i);
#pragma unroll 1
  for (int i = 0; i < steps; ++i) {
    cp_async_wait<kSpDepth - 1>();
    __syncwarp();
    const int k0 = i * kStride + warp * kSpKeys;
    const int rel[2] = {see[0] - k0, see[1] - k0};
    step32<F16>(st, q, ring + i % kSpDepth * kSpStep, rel, p.scale_log2);
    __syncwarp();
    fetch(i + kSpDepth);
  }
}

// The 16 query rows of a tile as operands: row r is token tok[r] (of a lane's
// two rows; -1: none) of sequence b[r], head h[r].
__device__ __forceinline__ void load_rows(RowQ& q, RowState& st, const SharedParams& p,
                                          const int (&b)[2], const int (&tok)[2], const int (&h)[2]) {
  const int t = threadIdx.x & 3;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const void* src = tok[r] >= 0 ? q_row(p, b[r], tok[r], h[r]) : nullptr;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int dim = 32 * (s / 2) + 8 * t + 4 * (s % 2);
      q.a[s][r] = src ? q_pair(p, src, dim) : 0u;
      q.a[s][2 + r] = src ? q_pair(p, src, dim + 2) : 0u;
    }
    st.m[r] = -INFINITY;
    st.l[r] = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) st.o[j][2 * r] = st.o[j][2 * r + 1] = 0.f;
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

// Shared memory: the warps' rings while they walk; then their states, the
// staged partials, and the threads' merges.
constexpr int kSpPitch = 68;  // floats per state row: m, l, -, -, o[64]
struct RowsMerge {
  float state[kSpWarps][16][kSpPitch];
  float stage[kSpStage * 80];
  float merged[kSpThreads][10];
};
union RowsShared {
  uint8_t ring[kSpWarps][kSpRing];
  RowsMerge m;
};
static_assert(sizeof(RowsShared) <= 75 * 1024, "three CTAs per SM");

// The warps' states of the tile into shared memory.
__device__ __forceinline__ void put_state(const RowState& st, RowsMerge& m, int warp) {
  const int lane = threadIdx.x % 32, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    float l = st.l[r];
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    float* w = m.state[warp][g + 8 * r];
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
}
__device__ __forceinline__ void add_state(Merged& acc, const RowsMerge& m, int w, int row, int part) {
  const float* x = m.state[w][row];
  acc.add(*reinterpret_cast<const float2*>(x), *reinterpret_cast<const float4*>(x + 4 + 8 * part),
          *reinterpret_cast<const float4*>(x + 8 + 8 * part));
}

// The partials of one row, in order: at(part) is where its row lies (in rows of
// part_o), or -1 behind the last.
struct Parts {
  const SharedParams& p;
  GroupDims d;
  int kvh, rg;
  // prefix_tc_kernel's: segments of the line, each over the CTAs that have a
  // share of it
  int share, head0, seg0, cl, chunks, m, q, c, c1, seg;
  // prefix_rows_kernel's: one per split
  int slot, last;
  __device__ __forceinline__ Parts(const SharedParams& params, int group, int b, int kv, int row, int R)
      : p(params), d(group_dims(params, group)), kvh(kv), rg((b - d.b0) * R + row) {
    // written by the preceding kernel, which may have run beside this one
    if (p.splits > 0) {
      const int tiles = (d.rows + 15) / 16, pages = (d.plen + kPageKeys - 1) / kPageKeys;
      slot = (__ldcg(p.part_plan + group) + kvh * tiles + rg / 16) * p.splits;
      const int per = (pages + p.splits - 1) / p.splits;
      last = pages > 0 ? slot + (pages + per - 1) / per - 1 : slot - 1;
      return;
    }
    share = __ldcg(p.part_plan);
    const int lin0 = __ldcg(p.part_plan + 1 + 2 * group);
    seg0 = __ldcg(p.part_plan + 2 + 2 * group);
    cl = chunk_blocks(d, share);
    chunks = d.nb > 0 ? (d.nb + cl - 1) / cl : 0;
    head0 = lin0 + kvh * head_steps(d, d.nb);
    m = rg / kPxRows;
    q = 0;
    c = 0;
    c1 = -1;
  }
  __device__ __forceinline__ long long next() {
    if (p.splits > 0) {
      if (slot > last || slot >= p.part_slots) return -1;
      return static_cast<long long>(slot++) * 16 + rg % 16;
    }
    if (c > c1) {
      if (q == chunks) return -1;
      const int len = min(cl, d.nb - q * cl);
      const int l0 = head0 + head_steps(d, q * cl) + m * len;
      seg = seg0 + (kvh * chunks + q) * d.mu + m;
      c = l0 / share;
      c1 = (l0 + unit_steps(d, m, len) - 1) / share;
      ++q;
    }
    const int at = c++ + seg;
    return at < p.part_slots ? static_cast<long long>(at) * kPxRows + rg % kPxRows : -1;
  }
};

// A row's partials folded into `acc` by the threads (row, copy, 8 head dims):
// copy k of `copies` takes every copies-th.  They are copied to shared memory as
// many at a time as fit, so that their latencies overlap.  A thread stages and
// reads its own pieces: no barrier.
__device__ __forceinline__ void fold_partials(Merged& acc, RowsMerge& sm, Parts& parts, int copy,
                                              int copies, int part) {
  const SharedParams& p = parts.p;
  constexpr int room = kSpStage / 16;  // partials a thread stages at a time
  float* mine = sm.stage + threadIdx.x * 8;
  float* mine_ml = sm.stage + kSpStage * 64 + threadIdx.x * 2;
  constexpr int pitch = 16 * 64, pitch_ml = 16 * 16;
  int nth = 0;
  bool more = true;
  while (more) {
    int n = 0;
#pragma unroll 1
    while (n < room) {
      const long long pr = parts.next();
      if (pr < 0) {
        more = false;
        break;
      }
      if (nth++ % copies != copy) continue;
      cp_async16(mine + n * pitch, p.part_o + pr * 64 + 8 * part, true);
      cp_async16(mine + n * pitch + 4, p.part_o + pr * 64 + 8 * part + 4, true);
      cp_async8(mine_ml + n * pitch_ml, p.part_ml + 2 * pr);
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

template <int F16>
__global__ void __launch_bounds__(kSpThreads, 3) shared_rows_kernel(SharedParams p) {
  extern __shared__ __align__(128) uint8_t sp_smem[];
  RowsShared& sh = *reinterpret_cast<RowsShared*>(sp_smem);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane >> 2;
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
    if (p.err && threadIdx.x == 0) atomicOr(p.err, kErrBadArgs);
    len = min(max(len, 0), p.max_pages * kPageKeys);
  }
  const int see[2] = {tok[0] < 0 ? 0 : max(0, len - (p.q_len - 1 - tok[0])),
                      tok[1] < 0 ? 0 : max(0, len - (p.q_len - 1 - tok[1]))};
  walk<F16>(st, q, p, kvh, table, p.max_pages, ids, len, see, warp, sh.ring[warp]);
  const int group = group_of(p, b);
  if (!p.part_o && group >= 0) {  // the prefix too
    int plen = __ldg(p.prefix_lens + group);
    if (plen < 0 || plen > p.prefix_pages * kPageKeys) {
      if (p.err && threadIdx.x == 0) atomicOr(p.err, kErrBadArgs);
      plen = min(max(plen, 0), p.prefix_pages * kPageKeys);
    }
    const int all[2] = {plen, plen};
    table = p.prefix_table + static_cast<size_t>(group) * p.prefix_pages;
    walk<F16>(st, q, p, kvh, table, p.prefix_pages, step_page(table, p.prefix_pages, warp, 0), plen,
              all, warp, sh.ring[warp]);
  }

  cp_async_wait_all();
  __syncthreads();  // the rings are done with
  put_state(st, sh.m, warp);
  __syncthreads();
  // Merge: 8 threads a row, 8 head dims each; with at most 8, 4, .. rows in the
  // tile, 2, 4, .. copies of them share the work.
  const int part = threadIdx.x % 8;
  const int rows2 = R <= 1 ? 1 : 1 << (32 - __clz(min(16, R) - 1));  // a power of two
  const int copies = 16 / rows2;
  const int lrow = (threadIdx.x / 8) % rows2, copy = threadIdx.x / 8 / rows2;
  const int rr = tile * 16 + lrow;
  Merged acc{-INFINITY, 0.f, {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}};
#pragma unroll 1
  for (int w = copy; w < kSpWarps; w += copies) add_state(acc, sh.m, w, lrow, part);
  if (p.part_o) {
    griddep_wait();  // the prefix kernel's partials
    if (group >= 0 && rr < R) {
      Parts parts(p, group, b, kvh, rr, R);
      fold_partials(acc, sh.m, parts, copy, copies, part);
    }
  }
  if (copies > 1) {
    float* mine = sh.m.merged[threadIdx.x];
    mine[0] = acc.m;
    mine[1] = acc.l;
#pragma unroll
    for (int e = 0; e < 8; ++e) mine[2 + e] = acc.o[e];
    __syncthreads();
    if (copy > 0) return;
#pragma unroll 1
    for (int k = 1; k < copies; ++k) {
      const float* x = sh.m.merged[threadIdx.x + k * rows2 * 8];
      acc.add(make_float2(x[0], x[1]), make_float4(x[2], x[3], x[4], x[5]),
              make_float4(x[6], x[7], x[8], x[9]));
    }
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

// The prefixes of groups with few rows: CTA (unit, split) takes split `split` of
// p.splits of the pages for unit `unit`, 16 rows of a (group, KV head), and
// leaves one partial per row in slot unit * splits + split.
template <int F16>
__global__ void __launch_bounds__(kSpThreads, 3) prefix_rows_kernel(SharedParams p) {
  extern __shared__ __align__(128) uint8_t sp_smem[];
  RowsShared& sh = *reinterpret_cast<RowsShared*>(sp_smem);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane >> 2;
  griddep_launch_dependents();
  const int G = p.heads / p.kv_heads, R = p.q_len * G;
  const int unit = blockIdx.x / p.splits, split = blockIdx.x - unit * p.splits;
  // ---- the unit's group: every warp scans the groups' unit counts
  int group = -1, unit0 = 0, before = 0;
#pragma unroll 1
  for (int base = 0; base < p.groups; base += 32) {
    const int gi = base + lane;
    int n = 0;
    if (gi < p.groups) {
      n = p.kv_heads * ((group_dims(p, gi).rows + 15) / 16);
      if (blockIdx.x == 0 && warp == 0 && p.err) {
        const int raw = __ldg(p.prefix_lens + gi);
        const int s0 = __ldg(p.group_starts + gi), s1 = __ldg(p.group_starts + gi + 1);
        if (raw < 0 || raw > p.prefix_pages * kPageKeys || s0 < 0 || s1 < s0 || s1 > p.batch)
          atomicOr(p.err, kErrBadArgs);
      }
    }
    int upto = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const int from = before + upto - n;
    if (blockIdx.x == 0 && warp == 0 && gi < p.groups) p.part_plan[gi] = from;
    const unsigned hit = __ballot_sync(0xffffffffu, from <= unit && unit < from + n);
    if (hit) {
      group = base + __ffs(hit) - 1;
      unit0 = __shfl_sync(0xffffffffu, from, __ffs(hit) - 1);
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  if (group < 0 || static_cast<int>(blockIdx.x) >= p.part_slots) return;
  const GroupDims d = group_dims(p, group);
  const int tiles = (d.rows + 15) / 16, kvh = (unit - unit0) / tiles;
  const int row0 = (unit - unit0 - kvh * tiles) * 16;
  const int pages = (d.plen + kPageKeys - 1) / kPageKeys, per = (pages + p.splits - 1) / p.splits;
  const int len = min(d.plen - split * per * kPageKeys, per * kPageKeys);
  if (len <= 0) return;
  const int* table = p.prefix_table + static_cast<size_t>(group) * p.prefix_pages + split * per;
  const int mine = min(per, pages - split * per);
  const int ids = step_page(table, mine, warp, 0);
  RowQ q;
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
  walk<F16>(st, q, p, kvh, table, mine, ids, len, see, warp, sh.ring[warp]);
  cp_async_wait_all();
  __syncthreads();
  put_state(st, sh.m, warp);
  __syncthreads();
  const int part = threadIdx.x % 8, row = threadIdx.x / 8;
  if (row0 + row >= d.rows) return;
  Merged acc{-INFINITY, 0.f, {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}};
#pragma unroll 1
  for (int w = 0; w < kSpWarps; ++w) add_state(acc, sh.m, w, row, part);
  const size_t pr = static_cast<size_t>(blockIdx.x) * 16 + row;
  float4* o = reinterpret_cast<float4*>(p.part_o + pr * 64 + 8 * part);
  o[0] = make_float4(acc.o[0], acc.o[1], acc.o[2], acc.o[3]);
  o[1] = make_float4(acc.o[4], acc.o[5], acc.o[6], acc.o[7]);
  if (part == 0) *reinterpret_cast<float2*>(p.part_ml + 2 * pr) = make_float2(acc.m, acc.l);
}

template <typename K>
cudaError_t launch_rows(K kernel, const SharedParams& p, long long ctas, bool dependent, cudaStream_t s) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  static std::atomic<bool> configured[64];
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[dev].load(std::memory_order_acquire)) {
    for (auto k : {shared_rows_kernel<0>, shared_rows_kernel<1>, prefix_rows_kernel<0>,
                   prefix_rows_kernel<1>}) {
      e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(RowsShared));
      if (e != cudaSuccess) return e;
    }
    configured[dev].store(true, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(kSpThreads);
  cfg.dynamicSmemBytes = sizeof(RowsShared);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dependent ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

}  // namespace

// Behind a prefix kernel the rows kernel is a programmatic dependent: sequences'
// own keys are attended while the last of the prefix finishes.
cudaError_t launch_shared_rows(const SharedParams& p, cudaStream_t s) {
  const int R = p.q_len * (p.heads / p.kv_heads);
  const long long ctas = static_cast<long long>(p.batch) * p.kv_heads * ((R + 15) / 16);
  return launch_rows(p.kv_dtype == 2 ? shared_rows_kernel<1> : shared_rows_kernel<0>, p, ctas,
                     p.part_o != nullptr, s);
}

cudaError_t launch_prefix_rows(const SharedParams& p, int units, cudaStream_t s) {
  return launch_rows(p.kv_dtype == 2 ? prefix_rows_kernel<1> : prefix_rows_kernel<0>, p,
                     static_cast<long long>(units) * p.splits, false, s);
}

}  // namespace ffai

// Verification of drafted tokens against the target's distribution, from given
// uniform numbers.
//
// Request b has the rows cu[b] .. cu[b + 1] - 1: its last token and its drafts.
// Row i's target distribution p is the softmax of its logits over the
// temperature T; the token of row i + 1 was drafted from q, likewise of the draft
// model's logits of row i, or given (q is 1 there).  The draft x of row i stands if
//   u_i q(x) < p(x),
// and with the first that does not the request takes a token from the
// distribution max(0, p - q) / sum of it, or, if all stand, from the last row's p:
// what is emitted is distributed as if the target alone had been sampled.
//
// In whole weights w = floor(2^36 e^d) (weights.cuh) of sum W, v and V for the
// draft's, all sums are exact and the tokens depend on the inputs alone:
//   x stands if  fl(fl(u v_x) W) < fl(w_x V)                        (f64 products)
//   r_i = max(0, w_i - floor(fl(v_i fl(W / V)))),  R their sum
//   the token is the first i with r_0 + .. + r_i > floor(fl(u' R)),
// with w in r's place if R is 0.  T = 0 puts all weight on the first maximum.
//
// Two launches.  The first, a cluster of CTAs per row of target and draft, keeps
// its stretch of the logits in registers between the maximum and the sum, so
// every logit is read once; the second, a cluster per request, finds the first
// row that fails and walks it again.
#include "common.cuh"
#include "kernels.h"
#include "weights.cuh"

namespace ffai {

namespace {

constexpr int kVfThreads = 512;
constexpr int kVfWarps = kVfThreads / 32;
constexpr int kVfCluster = 8;  // CTAs per row, at most

template <typename V, typename Op>
__device__ __forceinline__ V block_reduce(V v, V* s_red, Op op) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (lane == 0) s_red[warp] = v;
  __syncthreads();
  v = s_red[lane % kVfWarps];
#pragma unroll
  for (int o = kVfWarps / 2; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  return v;
}

__device__ __forceinline__ void st_cluster_u64(uint32_t caddr, unsigned long long v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(caddr), "l"(v) : "memory");
}
// v into mine[rank of this CTA] of every CTA of the cluster; complete after the
// cluster's next barrier.  One thread per target CTA.
__device__ __forceinline__ void tell_all(unsigned long long* mine, unsigned long long v, int ctas, int rank) {
  if (static_cast<int>(threadIdx.x) < ctas)
    st_cluster_u64(mapa_shared(smem_u32(mine + rank), threadIdx.x), v);
}

struct Request {
  int b, r0, n;  // request, its first row, rows; b -1: none
};
// Rows of request b; those that cannot be told are none.
__device__ __forceinline__ Request request(const VerifyParams& p, int b, bool& bad) {
  const int r0 = __ldg(p.cu_rows + b), r1 = __ldg(p.cu_rows + b + 1);
  if (r0 < 0 || r1 < r0 || r1 > p.rows) {
    bad = true;
    return {b, 0, 0};
  }
  return {b, r0, r1 - r0};
}
// The request that holds a row (a whole warp): the last one that starts at or before it.
__device__ __forceinline__ Request request_of(const VerifyParams& p, int row) {
  const int lane = threadIdx.x % 32;
  int n = 0;
  for (int base = 0; base < p.batch; base += 128) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int b = base + 32 * k + lane;
      const bool in = b < p.batch && __ldg(p.cu_rows + min(b, p.batch - 1)) <= row;
      n += __popc(__ballot_sync(0xffffffffu, in));
    }
  }
  bool bad = false;
  const Request r = request(p, max(n - 1, 0), bad);
  return n > 0 && row < r.r0 + r.n && row >= r.r0 ? r : Request{-1, 0, 0};
}

__device__ __forceinline__ float inverse(const float* temperature, int b) {
  const float t = temperature ? __ldg(temperature + b) : 1.0f;
  const float inv = t > 0.0f ? __fdiv_rn(1.0f, t) : INFINITY;
  return isinf(inv) ? 0.0f : inv;  // 0: the first maximum alone
}

// Weight of logit x at index i under a row's maximum.
struct Dist {
  float xmax, inv;
  int first;  // index of the first maximum, for inv = 0
  __device__ __forceinline__ unsigned long long at(float x, int i) const {
    if (xmax == -INFINITY) return 0;
    if (inv == 0.0f) return i == first ? 1ull << 36 : 0;
    return weight(__fmul_rn(delta(clean(x), xmax), inv));
  }
};

// Sums of weights, as sums of their halves with the magic numbers' bits in them:
// fma and add towards zero leave the whole part in the low mantissa bits.
struct WeightSum {
  uint32_t hi = 0, lo = 0, n = 0;
  __device__ __forceinline__ void add(float e) {
    const float t = __fmaf_rz(e, 262144.0f, 8388608.0f);
    const float r = __fmaf_rn(e, 262144.0f, -__fadd_rn(t, -8388608.0f));
    hi += __float_as_uint(t);
    lo += __float_as_uint(__fmaf_rz(r, 262144.0f, 8388608.0f));
  }
  __device__ __forceinline__ unsigned long long total(uint32_t added) const {
    const uint32_t bias = added * 0x4b000000u;
    return (static_cast<unsigned long long>(hi - bias) << 18) + (lo - bias);
  }
};

// The 16-byte pieces that hold a row, from the one its first logit lies in.
template <typename T>
struct RowPieces {
  static constexpr int kVec = 16 / sizeof(T);
  const T* row;
  int skew, vocab, pieces;
  __device__ __forceinline__ RowPieces(const void* base, long long ld, int r, int v)
      : row(static_cast<const T*>(base) + r * ld), vocab(v) {
    skew = static_cast<int>(reinterpret_cast<uintptr_t>(row) % 16 / sizeof(T));
    pieces = (skew + v + kVec - 1) / kVec;
  }
  __device__ __forceinline__ int index(int piece) const { return piece * kVec - skew; }
  // Piece i; -inf in the places outside the row, which are not read.
  __device__ __forceinline__ uint4 load(int i) const {
    const int at = index(i);
    if (i < pieces && at >= 0 && at + kVec <= vocab)
      return __ldg(reinterpret_cast<const uint4*>(row + at));
    constexpr uint32_t kNone = std::is_same<T, float>::value ? 0xff800000u
                               : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
    uint4 w = make_uint4(kNone, kNone, kNone, kNone);
    if (i < pieces) {
      T x[kVec];
#pragma unroll
      for (int e = 0; e < kVec; ++e)
        x[e] = at + e >= 0 && at + e < vocab ? row[at + e] : from_f32<T>(-INFINITY);
      memcpy(&w, x, 16);
    }
    return w;
  }
};

template <typename T, int N>  // N pieces a thread
__global__ void __launch_bounds__(kVfThreads) verify_rows_kernel(VerifyParams p) {
  constexpr int kVec = 16 / sizeof(T);
  __shared__ unsigned long long s_red[kVfWarps];
  __shared__ unsigned long long s_all[4][kVfCluster];
  griddep_launch_dependents();
  const int ctas = p.row_ctas, job = blockIdx.x / ctas, rank = blockIdx.x - job * ctas;
  const bool is_draft = job >= p.rows;
  const int row = is_draft ? job - p.rows : job;
  const Request req = request_of(p, row);
  if (req.b < 0) {  // no request's: nothing is emitted there
    if (!is_draft && rank == 0 && threadIdx.x == 0) {
      p.tokens_out[row] = -1;
      if (p.logprobs) p.logprobs[row] = 0.0f;
    }
    return;
  }
  const bool drafted = row + 1 < req.r0 + req.n;
  if (is_draft && !drafted) return;  // (the whole cluster)

  if (ctas > 1) cluster_arrive_relaxed();  // waited for below: every CTA of the row runs

  const RowPieces<T> src(is_draft ? p.draft : p.logits, is_draft ? p.draft_ld : p.ld, row, p.vocab);
  const int per = (src.pieces + ctas - 1) / ctas, first = rank * per;
  const int mine = min(per, src.pieces - first);  // may be negative
  uint4 w[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const int i = k * kVfThreads + threadIdx.x;
    w[k] = src.load(i < mine ? first + i : src.pieces);
  }
  const float inv = inverse(is_draft ? p.draft_temperature : p.temperature, req.b);

  // ---- the maximum (NaN counts as -inf: fmaxf passes it over)
  float top = -INFINITY;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    float x[kVec];
    unpack<T>(w[k], x);
#pragma unroll
    for (int e = 0; e < kVec; ++e) top = fmaxf(top, x[e]);
  }
  top += 0.0f;  // -0 as 0
  top = block_reduce(top, reinterpret_cast<float*>(s_red), [](float a, float b) { return fmaxf(a, b); });
  if (ctas > 1) {
    cluster_wait();
    tell_all(s_all[0], __float_as_uint(top), ctas, rank);
    cluster_arrive();
    cluster_wait();
    for (int c = 0; c < ctas; ++c) top = fmaxf(top, __uint_as_float(static_cast<uint32_t>(s_all[0][c])));
  }

  // ---- the weights' sum, the first maximum, the sum for log-probabilities
  unsigned long long mass = 0, where = ~0ull;
  float z = 0.0f;
  if (inv == 0.0f) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      float x[kVec];
      unpack<T>(w[k], x);
      const int at = src.index(first + k * kVfThreads + threadIdx.x);
#pragma unroll
      for (int e = 0; e < kVec; ++e)
        if (x[e] == top && at + e >= 0 && at + e < p.vocab && k * kVfThreads + static_cast<int>(threadIdx.x) < mine)
          where = min(where, static_cast<unsigned long long>(at + e));
    }
    mass = 1ull << 36;
  } else if (isinf(top)) {  // one weight for each infinite logit, or none at all
    uint32_t n = 0;
    if (top > 0.0f) {
#pragma unroll
      for (int k = 0; k < N; ++k) {
        float x[kVec];
        unpack<T>(w[k], x);
#pragma unroll
        for (int e = 0; e < kVec; ++e) n += x[e] == top;
      }
    }
    mass = static_cast<unsigned long long>(n) << 36;
  } else {
    WeightSum sum;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      float x[kVec];
      unpack<T>(w[k], x);
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const float d = __fmul_rn(__fadd_rn(x[e], -top), inv);
        sum.add(d >= -25.0f ? expf(d) : 0.0f);
      }
    }
    mass = sum.total(N * kVec);
  }
  if (p.logprobs && !is_draft) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      float x[kVec];
      unpack<T>(w[k], x);
#pragma unroll
      for (int e = 0; e < kVec; ++e) z += x[e] == x[e] ? expf(delta(x[e], top)) : 0.0f;
    }
  }
  const auto add = [](auto a, auto b) { return a + b; };
  if (inv != 0.0f) mass = block_reduce(mass, s_red, add);
  else where = block_reduce(where, s_red, [](unsigned long long a, unsigned long long b) { return min(a, b); });
  double zd = 0.0;
  if (p.logprobs && !is_draft)
    zd = block_reduce(static_cast<double>(z), reinterpret_cast<double*>(s_red), add);
  if (ctas > 1) {
    if (threadIdx.x == 0) {
      st_cluster_u64(mapa_shared(smem_u32(&s_all[1][rank]), 0), mass);
      st_cluster_u64(mapa_shared(smem_u32(&s_all[2][rank]), 0), where);
      st_cluster_u64(mapa_shared(smem_u32(&s_all[3][rank]), 0), __double_as_longlong(zd));
    }
    cluster_arrive();
    cluster_wait();
    if (rank > 0) return;
    if (inv != 0.0f) mass = 0;
    zd = 0.0;
    for (int c = 0; c < ctas; ++c) {
      if (inv != 0.0f) mass += s_all[1][c];
      where = min(where, s_all[2][c]);
      zd += __longlong_as_double(s_all[3][c]);
    }
  }
  if (threadIdx.x != 0) return;
  if (top == -INFINITY) mass = 0;
  VerifyRow out;
  out.mass = mass;
  out.xmax = top;
  out.first = static_cast<int>(where);
  out.log_z = p.logprobs && !is_draft ? static_cast<float>(log(zd)) : 0.0f;
  // the weight of the token that row's distribution is asked about
  out.at = 0;
  if (drafted) {
    const int x = __ldg(p.tokens + row + 1);
    if (x >= 0 && x < p.vocab)
      out.at = Dist{top, inv, out.first}.at(to_f32<T>(src.row[x]), x);
  }
  p.stats[job] = out;
}

template <typename T>
__global__ void __launch_bounds__(kVfThreads) verify_pick_kernel(VerifyParams p) {
  constexpr int kVec = 16 / sizeof(T);
  __shared__ unsigned long long s_red[kVfWarps], s_warp[kVfWarps];
  __shared__ unsigned long long s_all[2][kVfCluster];
  const int ctas = p.pick_ctas, b = blockIdx.x / ctas, rank = blockIdx.x - b * ctas;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  bool bad = false;
  const Request req = request(p, b, bad);
  griddep_wait();
  if (req.n == 0) {
    if (rank == 0 && threadIdx.x == 0) {
      p.accepted[b] = 0;
      p.next[b] = -1;
      if (bad && p.err) atomicOr(p.err, kErrBadArgs);
    }
    return;
  }
  if (ctas > 1) cluster_arrive_relaxed();  // waited for below: every CTA of the request runs
  // ---- the first draft that does not stand
  int fail = req.n - 1;  // the last row has none
  for (int i = threadIdx.x; i < req.n - 1; i += kVfThreads) {
    const int row = req.r0 + i;
    const VerifyRow t = p.stats[row];
    double v = 1.0, total = 1.0;
    if (p.draft) {
      const VerifyRow d = p.stats[p.rows + row];
      v = __ull2double_rn(d.at);
      total = __ull2double_rn(d.mass);
    }
    const double left = __dmul_rn(__dmul_rn(static_cast<double>(__ldg(p.u + row)), v), __ull2double_rn(t.mass));
    if (!(left < __dmul_rn(__ull2double_rn(t.at), total))) fail = min(fail, i);
  }
  fail = block_reduce(fail, reinterpret_cast<int*>(s_red), [](int x, int y) { return min(x, y); });
  const int row = req.r0 + fail;
  const VerifyRow t = p.stats[row];
  const Dist target{t.xmax, inverse(p.temperature, b), t.first};
  const bool rejected = fail < req.n - 1;
  const int drafted = rejected ? __ldg(p.tokens + row + 1) : -1;
  Dist draft{-INFINITY, 0.0f, 0};
  double rho = 0.0;
  if (rejected && p.draft) {
    const VerifyRow d = p.stats[p.rows + row];
    draft = Dist{d.xmax, inverse(p.draft_temperature, b), d.first};
    rho = d.mass ? __ddiv_rn(__ull2double_rn(t.mass), __ull2double_rn(d.mass)) : 0.0;
  }

  // ---- its weights once more: a warp takes a run of pieces
  const RowPieces<T> src(p.logits, p.ld, row, p.vocab);
  const T* draft_row = p.draft ? static_cast<const T*>(p.draft) + row * p.draft_ld : nullptr;
  const int per = (src.pieces + ctas * kVfWarps - 1) / (ctas * kVfWarps);
  const int i0 = (rank * kVfWarps + warp) * per, i1 = min(src.pieces, i0 + per);
  bool rest = rejected;  // what the draft leaves
  const auto one = [&](float x, int i) -> unsigned long long {
    unsigned long long w = target.at(x, i);
    if (!rest || w == 0) return w;
    if (!p.draft) return i == drafted ? 0 : w;
    const unsigned long long v = draft.at(to_f32<T>(draft_row[i]), i);
    if (v == 0) return w;
    const unsigned long long less =
        static_cast<unsigned long long>(__double2ll_rd(__dmul_rn(__ull2double_rn(v), rho)));
    return w > less ? w - less : 0;
  };
  const auto piece = [&](int i, unsigned long long (&r)[kVec]) {
    float x[kVec];
    const uint4 raw = src.load(i < i1 ? i : src.pieces);
    unpack<T>(raw, x);
    const int at = src.index(i);
    unsigned long long sum = 0;
#pragma unroll
    for (int e = 0; e < kVec; ++e) {
      r[e] = i < i1 && at + e >= 0 && at + e < p.vocab ? one(x[e], at + e) : 0;
      sum += r[e];
    }
    return sum;
  };
  unsigned long long total = 0, base = 0, mine = 0;
  for (int round = 0; round < 2; ++round) {
    unsigned long long sum = 0;
    for (int i = i0 + lane; i < i1; i += 32) {
      unsigned long long r[kVec];
      sum += piece(i, r);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s_warp[warp] = sum;
    __syncthreads();
    mine = 0;
    for (int w = 0; w < kVfWarps; ++w) mine += s_warp[w];
    total = mine;
    base = 0;
    if (ctas > 1) {
      if (round == 0) cluster_wait();
      tell_all(s_all[round], mine, ctas, rank);
      cluster_arrive();
      cluster_wait();
      total = 0;
      for (int c = 0; c < ctas; ++c) {
        if (c < rank) base += s_all[round][c];
        total += s_all[round][c];
      }
    }
    if (total > 0 || !rest) break;
    rest = false;  // the draft's distribution was the target's, as far as weights tell
    __syncthreads();
  }
  if (rank == 0) {
    if (threadIdx.x == 0) {
      p.accepted[b] = fail;
      if (total == 0) {
        p.next[b] = p.tokens_out[row] = -1;
        if (p.logprobs) p.logprobs[row] = 0.0f;
      }
    }
    for (int i = threadIdx.x; i < req.n; i += kVfThreads) {
      if (i == fail) continue;
      const int r = req.r0 + i, x = i < fail ? __ldg(p.tokens + r + 1) : -1;
      p.tokens_out[r] = x;
      if (p.logprobs) {
        float lp = 0.0f;
        if (x >= 0) {
          const VerifyRow s = p.stats[r];
          lp = delta(clean(to_f32<T>(static_cast<const T*>(p.logits)[r * p.ld + x])), s.xmax) - s.log_z;
        }
        p.logprobs[r] = lp;
      }
    }
  }
  if (total == 0) return;
  // ---- the token: CTA, warp, 32 pieces, piece, place
  long long goal_s = __double2ll_rd(__dmul_rn(static_cast<double>(__ldg(p.u_last + b)), __ull2double_rn(total)));
  unsigned long long goal = goal_s < 0 ? 0 : static_cast<unsigned long long>(goal_s);
  goal = min(goal, total - 1);
  if (goal < base || goal >= base + mine) return;
  unsigned long long before = base;
  for (int w = 0; w < warp; ++w) before += s_warp[w];
  if (goal < before || goal >= before + s_warp[warp]) return;
  for (int i = i0; i < i1; i += 32) {
    unsigned long long r[kVec];
    const unsigned long long sum = piece(i + lane, r);
    unsigned long long upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + upto > goal);
    if (hit) {
      if (lane == __ffs(hit) - 1) {
        unsigned long long c = before + upto - sum;
        int token = -1;
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          c += r[e];
          if (token < 0 && c > goal) token = src.index(i + lane) + e;
        }
        p.next[b] = p.tokens_out[row] = token;
        if (p.logprobs)
          p.logprobs[row] = delta(clean(to_f32<T>(src.row[token])), t.xmax) - t.log_z;
      }
      return;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
}

template <typename K>
cudaError_t launch_clusters(K kernel, const VerifyParams& p, long long jobs, int ctas, bool dependent,
                            cudaStream_t s) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(jobs * ctas));
  cfg.blockDim = dim3(kVfThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = dependent ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <typename T>
cudaError_t launch_t(VerifyParams p, int sms, cudaStream_t s) {
  constexpr int kVec = 16 / sizeof(T);
  const int pieces = (p.vocab + kVec - 1) / kVec + 1;
  const long long jobs = p.draft ? 2LL * p.rows : p.rows;
  const auto per = [&](int ctas) { return (pieces + ctas * kVfThreads - 1) / (ctas * kVfThreads); };
  if (jobs > 0) {
    // as many CTAs a row as fill the GPU, and as its pieces need
    int ctas = 1;
    while (ctas < kVfCluster && (per(ctas) > 8 || (jobs * ctas < 2 * sms && per(ctas) > 1))) ctas *= 2;
    p.row_ctas = ctas;
    const int n = per(ctas);
    auto kernel = n <= 1 ? verify_rows_kernel<T, 1>
                  : n <= 2 ? verify_rows_kernel<T, 2>
                  : n <= 4 ? verify_rows_kernel<T, 4>
                  : n <= 8 ? verify_rows_kernel<T, 8> : verify_rows_kernel<T, 17>;
    cudaError_t e = launch_clusters(kernel, p, jobs, ctas, false, s);
    if (e != cudaSuccess) return e;
  }
  int ctas = 1;
  while (ctas < kVfCluster && p.batch * ctas < 2 * sms && per(ctas) > 1) ctas *= 2;
  p.pick_ctas = ctas;
  return launch_clusters(verify_pick_kernel<T>, p, p.batch, ctas, jobs > 0, s);
}

}  // namespace

cudaError_t launch_verify(const VerifyParams& p, int sms, cudaStream_t s) {
  switch (p.dtype) {
    case 0: return launch_t<float>(p, sms, s);
    case 1: return launch_t<__nv_bfloat16>(p, sms, s);
    case 2: return launch_t<__half>(p, sms, s);
  }
  return cudaErrorInvalidValue;
}

}  // namespace ffai

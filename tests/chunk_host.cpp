// The walk of a chunk's attention over its line of steps, run on the host: parts.inc
// holds pieces of the kernels' sources, whose warp functions are played by 32 threads
// (a CTA of one warp, as find_stretch is told).  Prints what does not hold.
#include <algorithm>
#include <atomic>
#include <barrier>
#include <cstdio>
#include <cstring>
#include <map>
#include <random>
#include <thread>
#include <vector>

#include <cuda.h>
#include <cuda_runtime.h>
#include <limits.h>
#include <stdint.h>

#include "kernels.h"

#undef __noinline__
#define __noinline__

namespace {
struct Index {
  unsigned x;
};
thread_local Index threadIdx;
Index blockIdx, gridDim;
std::barrier<> warp_meets(32);
long long lanes[32];

// Every lane's value, read by f once all are there.
template <typename F>
auto exchange(long long v, F f) {
  lanes[threadIdx.x] = v;
  warp_meets.arrive_and_wait();
  auto r = f();
  warp_meets.arrive_and_wait();
  return r;
}
int __shfl_sync(unsigned, int v, int from) { return exchange(v, [=] { return static_cast<int>(lanes[from & 31]); }); }
int __shfl_up_sync(unsigned, int v, int by) {
  const int lane = threadIdx.x;
  return exchange(v, [=] { return static_cast<int>(lanes[lane < by ? lane : lane - by]); });
}
bool __all_sync(unsigned, bool v) {
  return exchange(v, [] { return std::all_of(lanes, lanes + 32, [](long long x) { return x != 0; }); });
}
void __syncthreads() { exchange(0, [] { return 0; }); }
int __syncthreads_or(int v) {
  return exchange(v, [] { return std::any_of(lanes, lanes + 32, [](long long x) { return x != 0; }) ? 1 : 0; });
}
template <typename T>
T __ldg(const T* p) {
  return *p;
}
int min(int a, int b) { return a < b ? a : b; }
int max(int a, int b) { return a > b ? a : b; }
unsigned atomicOr(unsigned* p, unsigned v) { return *p |= v; }
unsigned atomicInc(unsigned* p, unsigned most) {
  const unsigned old = *p;
  *p = old >= most ? 0 : old + 1;
  return old;
}
}  // namespace

namespace ffai {
namespace {

// The barriers: consumers always have freed a stage, copies land when they are waited for.
struct Fills {
  uint32_t sent = 0;
  long long awaited = -1;  // the parity of the last wait
};
std::map<uint64_t*, Fills> fills;
bool mbar_wait(uint64_t* bar, uint32_t parity, volatile int*, unsigned*, unsigned code) {
  if (code == kErrTimeoutDrain && threadIdx.x == 0) fills[bar].awaited = parity;
  return true;
}
void mbar_arrive_expect_tx_w(uint64_t* bar, uint32_t) {
  if (threadIdx.x == 0) ++fills[bar].sent;
}
void tma_load_3d_w(void*, const CUtensorMap*, uint64_t*, int, int, int) {}

#include "parts.inc"

alignas(1024) uint8_t ct_smem[kCtSmem];

template <typename F>
void as_warp(F f) {
  std::vector<std::thread> all;
  for (unsigned t = 0; t < 32; ++t)
    all.emplace_back([=] {
      threadIdx.x = t;
      f();
    });
  for (auto& t : all) t.join();
}

// As the kernel makes it of a stretch.
Walk start_of(const ChunkParams& p, const Stretch& x) {
  Walk w{};
  w.left = x.left;
  if (x.left > 0) {
    bool bad = false;
    w.s = chunk_seq(p, x.b, bad);
    w.b = x.b, w.h = x.h, w.m = x.m, w.step = x.step, w.unit0 = x.unit0;
    walk_unit(w, p);
  }
  return w;
}

struct Problem {
  std::vector<int> cu{0}, lens, table;
  std::vector<unsigned> tickets;
  unsigned err = 0;
  ChunkParams p{};
};
void make(Problem& a, std::mt19937& g, int ctas) {
  const auto below = [&](int n) { return static_cast<int>(g() % n); };
  const int B = 1 + below(40), heads = 1 + below(3), group = 1 + below(4);
  const int kind = below(3);
  for (int b = 0; b < B; ++b) {
    const int n = kind == 0 ? below(4) : kind == 1 ? below(700) : below(8) ? 1 : below(1500);
    a.cu.push_back(a.cu.back() + n);
    a.lens.push_back(max(0, n + (below(2) ? below(5000) : below(64)) - below(3) / 2 * 40));
  }
  a.p.max_pages = (1500 + 5000 + 63) / 64;
  a.table.assign(static_cast<size_t>(B) * a.p.max_pages, 0);
  a.tickets.assign(2 * ctas, 0);
  a.p.cu_q = a.cu.data(), a.p.seq_lens = a.lens.data(), a.p.block_table = a.table.data();
  a.p.tickets = a.tickets.data();
  a.p.batch = B, a.p.tokens = a.cu.back(), a.p.num_pages = 1;
  a.p.kv_heads = heads, a.p.heads = heads * group;
  a.p.causal = below(2), a.p.min_share = 2, a.p.err = &a.err;
}

// Every CTA leaves at some point of its stretch, or ends it: the tickets of all units
// are taken once, so the words are zero behind the call.  rest: as the kernel does; else
// what is left in them is counted.
int tickets(std::mt19937& g, bool rest) {
  int left = 0, shared = 0;
  for (int round = 0; round < 40; ++round) {
    Problem a;
    gridDim.x = 1 + g() % 40;
    make(a, g, gridDim.x);
    if (a.p.tokens == 0) continue;
    for (blockIdx.x = 0; blockIdx.x < gridDim.x; ++blockIdx.x) {
      Stretch x{};
      int2 s_warp[2];
      as_warp([&] { find_stretch<kPxRows, kChKeys, 32, 1>(a.p, &x, s_warp); });
      for (int t = 0; t < 2; ++t) {
        Walk w = start_of(a.p, x);
        const int stop = g() % 3 ? static_cast<int>(g() % 6) : INT_MAX;  // units, and the next one's ticket or not
        bool taken = false;
        for (int i = 0; w.left > 0; ++i, walk_next(w, a.p)) {
          if (i == stop && g() % 2) break;
          if (!walk_whole(w) && (walk_pair(w) || t == 0)) {
            ++shared;
            take_ticket(a.p, w, walk_teams(w, x.share), t);
          }
          if (i == stop) {
            taken = true;
            break;
          }
        }
        if (rest) take_the_rest(a.p, w, x.share, t, taken);
      }
    }
    for (unsigned n : a.tickets) left += n != 0;
  }
  if (shared < 400) printf("few units are shared: %d\n", shared);
  return left;
}

// The producer of every CTA, where nothing has gone wrong yet when it has sent its last
// copies: it has waited for the last one into each place all the same.
int copies_in_flight(std::mt19937& g) {
  int flying = 0;
  for (int round = 0; round < 5; ++round) {
    Problem a;
    gridDim.x = 1 + g() % 20;
    make(a, g, gridDim.x);
    for (blockIdx.x = 0; blockIdx.x < gridDim.x; ++blockIdx.x) {
      Stretch x{};
      int2 s_warp[2];
      fills.clear();
      as_warp([&] {
        find_stretch<kPxRows, kChKeys, 32, 1>(a.p, &x, s_warp);
        if (threadIdx.x == 0) CT_BARS->start = start_of(a.p, x);
        __syncthreads();
        ct_producer(nullptr, nullptr, a.p);
      });
      for (const auto& [bar, f] : fills) flying += f.sent > 0 && f.awaited != (f.sent - 1) % 2;
    }
  }
  return flying;
}

}  // namespace
}  // namespace ffai

int main() {
  std::mt19937 g(1);
  if (const int n = ffai::tickets(g, true)) printf("%d words are above zero\n", n);
  if (!ffai::tickets(g, false)) printf("nothing is left in the words by CTAs that take no tickets on their way out\n");
  if (const int n = ffai::copies_in_flight(g)) printf("%d copies may be in flight when their CTA exits\n", n);
}

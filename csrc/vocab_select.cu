// Top-k log-probabilities and sampling over rows of logits [N, V].
//
// topk_logprobs: the k largest logits of a row (ties: lower token first) with log p = z/tau - lse(z/tau).
// sample_tokens: one token per row, drawn from softmax(z/tau) restricted by top-k, top-p and min-p: with e_i the
//   row's given Exp(1) numbers, argmax over the kept tokens of w_i / e_i, w_i = exp((z_i - max z)/tau), is a sample
//   (the smallest of independent exponential times with rates w_i). All three filters keep a prefix of the rank
//   order (greater logit first, then lower token), which is what the kernels use.
//
// Both are bound by reading the logits once. A thread copies its own vectors through a private ring in shared memory
// (cp.async, no barriers), so that many loads are in flight without registers. Selection needs no buffer along the
// way: the pass keeps the largest logit of each group (a thread's elements over a few steps, 4096 groups in a slice).
// Where k of 256 threads, or of the groups, reach some logit, at least k elements do; only groups whose maximum
// reaches it can hold such elements. So about k groups are read again (k times 48 elements at V = 151,936: 11% more
// bytes for k = 64), and of the elements that reach the threshold, hardly more than k, the k best are taken by 64-bit
// words of logit order and token (no ties). Before, a buffer of candidates with a rising threshold took 327 us for the
// top 64 of 2048 x 151,936 fp32 logits, most of it in barriers and in pushing; this takes 237 (5.3 TB/s; k = 1 190).
//
// Sampling from a row with a top-k of 256 and less reads the logits, and the random numbers of the listed tokens: 70 us
// for 512 fp32 rows (top 20), 18 for 64 bf16 ones. Every other row reads both in one pass, in which all tokens race:
// 124 us for the 512 (5.0 TB/s of 622 MB), 405 for 2048. Without a top-p, min-p or top-k that is all. Else the winner
// is the sample if it is kept, which a pass over the logits tells (nothing but a comparison for a min-p); 512 rows at
// top-p 0.9 take 240 us. A list of the 256 best for these rows too was no help: it holds the kept tokens of peaked
// rows only, and costs more than it saves.
#include "common.cuh"
#include "vocab.cuh"
#include "vocab.h"

namespace ts {
namespace {

namespace cg = cooperative_groups;
using namespace vocab;

constexpr int kMaxTop = 256;
constexpr int kMaxParts = 8;
constexpr int kGroups = 4096;                // groups of a slice whose maxima are kept
constexpr int kMaxList = 512;                // groups that are read again, at most
constexpr int kMaxRounds = 40;               // winners of a race that are tried before the kept tokens are looked for
constexpr float kColdest = 1e-6f;            // colder rows are greedy

template <typename T, int NT>
struct Shared {
  uint64_t win[kMaxTop];
  uint64_t wbest[NT / 32];
  uint64_t pbest[2];  // this CTA's partial results, read by its cluster (two sets, used in turn)
  float wm[NT / 32], ws[NT / 32];
  int wc[NT / 32];
  uint32_t hist[2][256], sel_min, sel_max;
  float pm[2], ps[2], jm, js;
  float ybest;        // of the race so far: some thread's, not always the latest
  uint64_t jbest;
  int jcount, jflag;
  int pcount[2], pflag[2];
  int count;          // candidates (may pass the room for them: then they were not stored)
  int nwin;           // entries in win
  int sel_need, sel_bin, sel_done, sel_have;
  int nlist;          // groups on the list (may pass its room: then they were not noted)
  uint16_t list[kMaxList];
  uint32_t top[kMaxTop];
  __align__(16) uint32_t keys[kGroups];          // order of the groups' maxima
  __align__(16) uint4 ring[kRing * NT];          // the rings; afterwards the candidates

  static constexpr int kCand = kRing * NT * 2;
  static constexpr int kWork = sizeof(uint32_t) * kGroups + sizeof(uint4) * kRing * NT;
  static_assert(kCand >= kMaxParts * kMaxTop && kCand >= kMaxTop + NT * Slice<T>::kVec + 16, "room for the candidates");
  __device__ uint64_t* cand() { return reinterpret_cast<uint64_t*>(ring); }
  __device__ uint4* work() { return reinterpret_cast<uint4*>(keys); }  // all of it, for the race's ring
};

// A lower bound of the k-th largest of x[0, n) above or at which exactly `reach` >= k of them are: k, or more where
// the k-th is one of several equal ones, and then it is the bound itself. Values up to `none` do not count; `reach` is
// 0 where fewer than k others are. All threads call it, after a barrier that follows the last write to x. Digits of
// eight bits from the first bit in which the upper 32 differ.
template <typename X, typename T, int NT>
__device__ __noinline__ X kth_largest(Shared<T, NT>& sh, const X* x, int n, int k, X none, int& reach) {
  constexpr int kBits = 8 * sizeof(X);
  const int tid = threadIdx.x;
  if (tid < 256) {
    sh.hist[0][tid] = 0;
    sh.hist[1][tid] = 0;
  }
  if (tid == 0) {
    sh.sel_min = 0xffffffffu;
    sh.sel_max = 0;
    sh.sel_have = 0;
  }
  __syncthreads();
  uint32_t mn = 0xffffffffu, mx = 0;
  int have = 0;
  for (int i = tid; i < n; i += NT) {
    const X full = x[i];
    if (full <= none) continue;
    const uint32_t v = (uint32_t)(full >> (kBits - 32));
    ++have;
    mn = min(mn, v);
    mx = max(mx, v);
  }
  mn = __reduce_min_sync(0xffffffffu, mn);
  mx = __reduce_max_sync(0xffffffffu, mx);
  have = __reduce_add_sync(0xffffffffu, have);
  if ((tid & 31) == 0 && have > 0) {
    atomicMin(&sh.sel_min, mn);
    atomicMax(&sh.sel_max, mx);
    atomicAdd(&sh.sel_have, have);
  }
  __syncthreads();
  if (sh.sel_have < k) {
    reach = 0;
    return none;
  }
  mn = sh.sel_min;
  mx = sh.sel_max;
  int prev = mn == mx ? kBits - 32 : kBits - __clz(mn ^ mx);  // the bits from here on are decided
  X prefix = prev == kBits ? X(0) : (X)((X)mx << (kBits - 32)) >> prev << prev;
  int need = k;
  if (prev == 0) {  // (32-bit values that are all equal)
    reach = sh.sel_have;
    return prefix;
  }
  for (int turn = 0;; turn ^= 1) {
    const int width = min(8, prev), shift = prev - width;
    const uint32_t mask = (1u << width) - 1;
    for (int i = tid; i < n; i += NT) {
      const X v = x[i];
      if (v > none && (prev == kBits || (v >> prev) == (prefix >> prev))) atomicAdd(&sh.hist[turn][(uint32_t)(v >> shift) & mask], 1u);
    }
    __syncthreads();
    if (tid < 32) {
      // lane l sums the 8 bins from 255 - 8l downwards
      uint32_t h[8], sum = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += h[j] = sh.hist[turn][255 - 8 * tid - j];
      uint32_t incl = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, incl, o);
        if (tid >= o) incl += up;
      }
      uint32_t above = incl - sum;
      if ((int)above < need && (int)incl >= need) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          if ((int)above < need && (int)(above + h[j]) >= need) {
            sh.sel_bin = 255 - 8 * tid - j;
            sh.sel_need = need - (int)above;
            sh.sel_done = (int)h[j];
            break;
          }
          above += h[j];
        }
      }
      __syncwarp();
#pragma unroll
      for (int j = 0; j < 8; ++j) sh.hist[turn][255 - 8 * tid - j] = 0;
    }
    __syncthreads();
    prefix |= (X)sh.sel_bin << shift;
    need = sh.sel_need;
    prev = shift;
    if (sh.sel_done == need || shift == 0) break;  // the whole bin belongs to the k, or its entries are equal
  }
  reach = k - need + sh.sel_done;
  return prefix;
}

// The k largest of the candidates, all different, to sh.win (in no order); n >= k. `least`: a lower bound of them
// above which no other candidate is.
template <typename T, int NT>
__device__ void select_k(Shared<T, NT>& sh, int n, int k, uint64_t& least) {
  int reach;
  least = kth_largest<uint64_t>(sh, sh.cand(), n, k, 0, reach);
  if (threadIdx.x == 0) sh.nwin = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += NT) {
    const uint64_t x = sh.cand()[i];
    if (x >= least) {
      const int at = atomicAdd(&sh.nwin, 1);
      if (at < kMaxTop) sh.win[at] = x;
    }
  }
  __syncthreads();
}

// A threshold that at least k of 256 groups' values (`mine`, the greatest of a group's threads) reach, the same in all
// threads, or 0: exact but for the last 12 bits. Each warp looks for itself, bit by bit, with 8 values in a lane.
template <typename T, int NT>
__device__ __noinline__ uint32_t group_threshold(Shared<T, NT>& sh, uint32_t mine, int k) {
  constexpr int kWidth = NT / kMaxTop;  // threads of a group
  const int tid = threadIdx.x, lane = tid & 31;
#pragma unroll
  for (int o = 1; o < kWidth; o <<= 1) mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, o));
  if (tid % kWidth == 0) sh.top[tid / kWidth] = mine;
  __syncthreads();
  uint32_t v[8], mx = 0, mn = 0xffffffffu;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    v[j] = sh.top[lane + 32 * j];
    mx = max(mx, v[j]);
    mn = min(mn, v[j]);
  }
  mx = __reduce_max_sync(0xffffffffu, mx);
  mn = __reduce_min_sync(0xffffffffu, mn);
  if (mn == mx) return mx;
  const int first = 31 - __clz(mn ^ mx);
  uint32_t lo = first >= 31 ? 0u : (mx >> (first + 1)) << (first + 1);  // the digits that all have
  for (int bit = first; bit >= 12; --bit) {
    const uint32_t cand = lo | (1u << bit);
    int n = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) n += v[j] >= cand;
    n = __reduce_add_sync(0xffffffffu, n);
    if (n >= k) lo = cand;
    if (n == k) break;
  }
  return lo;
}

// Leaves the slice's k largest (all of it where it is shorter) in sh.win, sh.nwin entries of which some may be
// smaller, in no order; and this thread's part of the statistics.
template <typename T, int NT>
__device__ __noinline__ Stat scan_slice(Shared<T, NT>& sh, const Slice<T> sl, int k, float c) {
  using S = Steps<T, NT>;
  constexpr int VEC = S::VEC, Q = S::kVecs, kSegs = kGroups / NT;
  constexpr uint32_t kMinusInf = 0x007fffffu;  // order of -inf
  const int tid = threadIdx.x;
  Stat st;
  S steps(sl, sh.ring);
  const int edges = sl.head + sl.tail;
  float zedge = -INFINITY;  // an element of the unaligned ends
  const int iedge = tid < sl.head ? tid : sl.nvec * VEC + tid;
  if (tid < edges) {
    zedge = to_f(sl.p[iedge]);
    stat_raise(st.m, st.s, fmaxf(zedge, -INFINITY), c);
    st.s += sum_exp<1>(&zedge, st.m, c);
  }
  const int span = max(1, (steps.count + kSegs - 1) / kSegs);  // steps of a group
  const int groups = (steps.count + span - 1) / span * NT;
  {
    float gmax = -INFINITY;
    uint32_t* key = sh.keys + tid;
    for (int t = 0, in = 0; t < steps.count; ++t) {
      float z[Q][VEC];
      steps.read(t, z);
      const float zmax = vec_max<16>(&z[0][0]);
      stat_raise(st.m, st.s, zmax, c);
      st.s += sum_exp<16>(&z[0][0], st.m, c);
      gmax = fmaxf(gmax, zmax);
      if (++in == span || t + 1 == steps.count) {
        *key = gmax > -INFINITY ? order_key(gmax) : 0u;
        key += NT;
        gmax = -INFINITY;
        in = 0;
      }
    }
  }
  copy_wait<0>();
  if (tid == 0) {
    sh.count = 0;
    sh.nlist = 0;
  }
  // Elements whose order is at least `least` are candidates. The k-th largest of 256 threads' maxima is a little lower
  // than that of the 4096 groups (73 groups reach it instead of 64 where k is 64, 173 instead of 128) and costs one
  // barrier instead of about ten; from half of the threads on it says too little.
  uint32_t least = 0, even = 0;
  bool many = false;
  auto note_groups = [&]() {
    for (int i = tid; i < groups; i += NT) {
      if (sh.keys[i] >= least) {
        const int at = atomicAdd(&sh.nlist, 1);
        if (at < kMaxList) sh.list[at] = (uint16_t)i;
      }
    }
    __syncthreads();
  };
  bool found = false;
  if (k <= kMaxTop / 2) {
    least = group_threshold<T, NT>(sh, st.m > -INFINITY ? order_key(st.m) : 0u, k);
    if (least > kMinusInf) {
      note_groups();
      found = sh.nlist <= kMaxList;
    }
  }
  __syncthreads();
  if (!found) {  // the same in all threads
    int reach;
    least = kth_largest<uint32_t>(sh, sh.keys, groups, k, kMinusInf, reach);
    if (reach == 0) ++least;  // fewer than k groups with a logit above -inf: all such logits
    even = least;             // where very many logits are equal, of these only the first tokens
    many = reach > kMaxList;
    if (many) ++least;
    if (tid == 0) sh.nlist = 0;
    __syncthreads();
    note_groups();
  }
  uint64_t* cand = sh.cand();
  auto push = [&](uint64_t x) {
    const int at = atomicAdd(&sh.count, 1);
    if (at < Shared<T, NT>::kCand) cand[at] = x;
  };
  if (tid < edges && order_key(zedge) >= least) push(rank_key(zedge, sl.lo + iedge));
  __syncthreads();
  const int width = span * Q;  // vectors of a group
  const int tasks = sh.nlist * width;
  auto vec_of = [&](int i) {
    const int g = sh.list[i / width];
    return (g / NT * width + i % width) * NT + g % NT;
  };
  constexpr int U = 4;
  for (int i0 = tid; i0 < tasks; i0 += U * NT) {
    uint4 raw[U];
    int v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      v[u] = i0 + u * NT < tasks ? vec_of(i0 + u * NT) : sl.nvec;
      if (v[u] < sl.nvec) raw[u] = *reinterpret_cast<const uint4*>(sl.body() + (long long)v[u] * VEC);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (v[u] >= sl.nvec) continue;
      float z[VEC];
      unpack<T>(raw[u], z);
      if (order_key(vec_max<VEC>(z)) < least) continue;
#pragma unroll
      for (int e = 0; e < VEC; ++e)
        if (order_key(z[e]) >= least) push(rank_key(z[e], sl.lo + sl.head + v[u] * VEC + e));
    }
  }
  __syncthreads();
  int n = sh.count;
  __syncthreads();
  if (n > Shared<T, NT>::kCand) {
    // groups that hold many such elements: again, a vector of each thread at a time, and only the k best are kept
    if (tid == 0) sh.count = 0;
    __syncthreads();
    if (tid < edges && order_key(zedge) >= least) push(rank_key(zedge, sl.lo + iedge));
    uint64_t floor = (uint64_t)least << 32;
    for (int i0 = 0; i0 < tasks; i0 += NT) {
      const int v = i0 + tid < tasks ? vec_of(i0 + tid) : sl.nvec;
      if (v < sl.nvec) {
        for (int e = 0; e < VEC; ++e) {
          const int i = sl.head + v * VEC + e;
          const uint64_t x = rank_key(to_f(sl.p[i]), sl.lo + i);
          if (x >= floor) push(x);
        }
      }
      __syncthreads();
      n = sh.count;
      __syncthreads();
      if (n > Shared<T, NT>::kCand - NT * VEC) {
        select_k<T, NT>(sh, n, k, floor);
        for (int i = tid; i < k; i += NT) cand[i] = sh.win[i];
        if (tid == 0) sh.count = k;
        __syncthreads();
        n = k;
      }
    }
  }
  // Too few: the first tokens of the next order (the equal ones, or -inf), and after -inf NaN.
  for (int next = many ? 2 : 0; n < k && next < 3; next = next == 0 ? 1 : 3) {
    const uint32_t order = next == 2 ? even : next == 0 ? kMinusInf : 0u;
    for (int i0 = 0; i0 < sl.n && n < k; i0 += NT) {
      const int i = i0 + tid;
      if (i < sl.n) {
        const float z = to_f(sl.p[i]);
        if (order_key(z) == order) push(rank_key(z, sl.lo + i));
      }
      __syncthreads();
      n = sh.count;
      __syncthreads();
    }
  }
  if (n > kMaxTop) {
    uint64_t floor;
    select_k<T, NT>(sh, n, k, floor);
  } else {
    for (int i = tid; i < n; i += NT) sh.win[i] = cand[i];
    if (tid == 0) sh.nwin = n;
    __syncthreads();
  }
  return st;
}

// The lanes' (m, s) joined; all lanes get lane 0's. An exchange by xor leaves each lane its own rounding of s: the
// multiply-add of a merge rounds one of its two products, and the two sides of an exchange differ in which.
TS_DEVICE void warp_stat(Stat& st, float c) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, st.m, o), s2 = __shfl_xor_sync(0xffffffffu, st.s, o);
    stat_merge(st.m, st.s, m2, s2, c);
  }
  st.m = __shfl_sync(0xffffffffu, st.m, 0);
  st.s = __shfl_sync(0xffffffffu, st.s, 0);
}

// Block-wide (m, s); all threads get the same bits, which they compare with sums to decide about loops with barriers.
template <typename T, int NT>
__device__ void block_stat(Shared<T, NT>& sh, Stat& st, float c) {
  warp_stat(st, c);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) {
    sh.wm[threadIdx.x >> 5] = st.m;
    sh.ws[threadIdx.x >> 5] = st.s;
  }
  __syncthreads();
  // one warp joins the warps' pairs, and its result is everyone's
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    st.m = lane < NT / 32 ? sh.wm[lane] : -INFINITY;
    st.s = lane < NT / 32 ? sh.ws[lane] : 0.f;
    warp_stat(st, c);
    if (lane == 0) {
      sh.jm = st.m;
      sh.js = st.s;
    }
  }
  __syncthreads();
  st.m = sh.jm;
  st.s = sh.js;
}

// The row's statistics from the parts': one warp of each part reads them. All threads get them.
template <typename T, int NT>
__device__ Stat join_stat(Shared<T, NT>& sh, Stat st, float c) {
  cg::cluster_group cl = cg::this_cluster();
  const int parts = (int)cl.num_blocks();
  if (parts == 1) return st;
  if (threadIdx.x == 0) {
    sh.pm[0] = st.m;
    sh.ps[0] = st.s;
  }
  cl.sync();
  if (threadIdx.x < 32) {
    const int r = threadIdx.x;
    st.m = -INFINITY;
    st.s = 0.f;
    if (r < parts) {
      const Shared<T, NT>* o = cl.map_shared_rank(&sh, r);
      st.m = o->pm[0];
      st.s = o->ps[0];
    }
#pragma unroll
    for (int o = kMaxParts / 2; o > 0; o >>= 1) {
      const float m2 = __shfl_xor_sync(0xffffffffu, st.m, o), s2 = __shfl_xor_sync(0xffffffffu, st.s, o);
      stat_merge(st.m, st.s, m2, s2, c);
    }
    if (r == 0) {
      sh.jm = st.m;
      sh.js = st.s;
    }
  }
  __syncthreads();
  return {sh.jm, sh.js};
}

// The row's k largest from the parts' lists: part 0 gets them in sh.win in rank order (sh.nwin of them); every part
// gets the row's statistics.
template <typename T, int NT>
__device__ void join_parts(Shared<T, NT>& sh, int k, float c, Stat& st) {
  const int tid = threadIdx.x;
  cg::cluster_group cl = cg::this_cluster();
  const int parts = (int)cl.num_blocks();
  if (parts > 1) {
    const bool first = cl.block_rank() == 0;
    st = join_stat(sh, st, c);
    int n = 0;
    if (first) {
      // list r goes behind those before it
      const int lane = tid & 31, warp = tid >> 5;
      const int cnt = lane < parts ? cl.map_shared_rank(&sh, lane)->nwin : 0;
      int incl = cnt;
#pragma unroll
      for (int o = 1; o < kMaxParts; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += up;
      }
      n = __shfl_sync(0xffffffffu, incl, kMaxParts - 1);
      for (int r = warp; r < parts; r += NT / 32) {
        const int at = __shfl_sync(0xffffffffu, incl - cnt, r), len = __shfl_sync(0xffffffffu, cnt, r);
        const Shared<T, NT>* o = cl.map_shared_rank(&sh, r);
        for (int i = lane; i < len; i += 32) sh.cand()[at + i] = o->win[i];
      }
    }
    cl.sync();
    if (first) {
      if (n > kMaxTop) {
        uint64_t least;
        select_k<T, NT>(sh, n, k, least);
      } else {
        if (tid < n) sh.win[tid] = sh.cand()[tid];
        if (tid == 0) sh.nwin = n;
        __syncthreads();
      }
    }
  }
  if (cl.block_rank() == 0) {
    // rank order: an entry's place is the number of greater ones
    const int n = sh.nwin;
    uint64_t mine = 0;
    int at = 0;
    if (tid < n) {
      mine = sh.win[tid];
      for (int j = 0; j < n; ++j) at += sh.win[j] > mine;
    }
    __syncthreads();
    if (tid < n && at < k) sh.win[at] = mine;
    if (tid == 0) sh.nwin = min(n, k);
    __syncthreads();
  }
}

template <typename T, int NT>
__global__ void __launch_bounds__(NT) topk_kernel(const T* __restrict__ logits, long long stride, int v, int k,
                                                  float temperature, int64_t* __restrict__ ids,
                                                  float* __restrict__ logprobs) {
  extern __shared__ __align__(16) uint8_t raw[];
  Shared<T, NT>& sh = *reinterpret_cast<Shared<T, NT>*>(raw);
  cg::cluster_group cl = cg::this_cluster();
  const int parts = (int)cl.num_blocks();
  const int row = blockIdx.x / parts;
  const float c = kLog2e / temperature;
  Slice<T> sl(logits + row * stride, v, (int)cl.block_rank(), parts);
  Stat st = scan_slice<T, NT>(sh, sl, k, c);
  block_stat(sh, st, c);
  join_parts(sh, k, c, st);
  if (cl.block_rank() == 0) {
    const float m = st.m == -INFINITY ? 0.f : st.m;
    const float ls = st.s == 0.f ? 0.f : logf(st.s);  // a row of -inf alone: its log-probs are -inf
    for (int i = threadIdx.x; i < k; i += NT) {
      const uint64_t x = sh.win[i];
      ids[(long long)row * k + i] = rank_id(x);
      logprobs[(long long)row * k + i] = (rank_value(x) - m) / temperature - ls;
    }
  }
}

// ------------------------------------------------------------------ sampling
TS_DEVICE float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The race's winner so far among this thread's tokens, by y = z·c - log2 e (log2 of the key, up to the row's
// constant). y is off by less than margin(y), so what counts in the end is the exact key w / e of the few tokens
// within the margin of the best. A thread keeps one token: `tie` says that another one came as near, and then the
// tokens are gone over again with exact keys. Threads look only at tokens within the margin of the best that any of
// the block has seen (sh.ybest, read and written without order: whatever it holds is some token's y).
struct Race {
  float y = -INFINITY, z = 0.f, e = 1.f;
  int id = -1;
  bool tie = false;

  // c's and the difference's roundings, 2^-24 each of values up to |y| and log2 e; lg2.approx; the key's own
  static TS_DEVICE float margin(float y) { return 1e-4f + 1e-6f * fabsf(y); }
  TS_DEVICE void take(float y2, float z2, float e2, int id2) {
    if (!(y2 > y - margin(y)) && y != -INFINITY) return;
    if (!(y2 > -INFINITY)) return;
    const bool near = y != -INFINITY && !(y2 > y + margin(y));
    tie = near || y2 == INFINITY;
    if (y2 > y) {
      y = y2;
      z = z2;
      e = e2;
      id = id2;
    }
  }
};

TS_DEVICE float weight(float z, float m, float temperature) { return expf((z - m) / temperature); }
// (key, token) in one word: the greater key first, then the lower token; 0 is nothing
TS_DEVICE uint64_t race_key(float w, float e, int id) {
  const float key = w / e;
  return key >= 0.f ? ((uint64_t)__float_as_uint(key) << 32) | (uint32_t)~(uint32_t)id : 0;
}

// One pass over logits and random numbers together: statistics and the race among all tokens. A step is 8 elements of
// each thread (two vectors of fp32 logits or one of 16-bit ones, and two of random numbers) through its ring. The 32
// bytes of random numbers beside one 16-bit vector are copied by the warp, 512 bytes at a time: each thread for itself
// would fetch every 32-byte sector twice.
template <typename T, int NT>
__device__ __noinline__ void scan_free(Shared<T, NT>& sh, const Slice<T> sl, const float* __restrict__ noise, float c,
                                       Stat& st_out, Race& race_out) {
  constexpr int VEC = Slice<T>::kVec, Q = 8 / VEC;
  constexpr int kPieces = Q + 2;  // 16-byte pieces of a step
  constexpr int kFit = Shared<T, NT>::kWork / (NT * 16 * kPieces);
  constexpr int R = kFit < 4 ? kFit : 4;  // steps in flight
  static_assert(R >= 2, "a ring of two");
  const int tid = threadIdx.x;
  Stat st;
  Race race;
  uint4* const ring = sh.work() + tid;
  const T* src = sl.body() + tid * VEC;
  const float* nsrc = noise + sl.head;
  const bool wide = (reinterpret_cast<uintptr_t>(nsrc) & 15) == 0;
  const int steps = (sl.nvec + Q * NT - 1) / (Q * NT), whole = sl.nvec / (Q * NT);
  const int lane = tid & 31, warp0 = tid - lane;
  auto has = [&](int t, int q) { return (t * Q + q) * NT + tid < sl.nvec; };
  auto copy_noise = [&](uint4* to, const float* from) {
    if (wide) {
      copy16(to, from);
    } else {
#pragma unroll
      for (int w = 0; w < 4; ++w) copy4(reinterpret_cast<float*>(to) + w, from + w);
    }
  };
  // `slot` is the step's place in the ring, at this thread
  auto fetch = [&](int t, uint4* slot) {
    if (VEC == 4) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        if (t < whole || (t < steps && has(t, q))) {
          const long long i = (long long)(t * 2 + q) * (NT * VEC);
          copy16(slot + q * NT, src + i);
          copy_noise(slot + (2 + q) * NT, nsrc + i + tid * VEC);
        }
      }
    } else {
      if (t < whole || (t < steps && has(t, 0))) copy16(slot, src + (long long)t * (NT * VEC));
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int v = t * NT + warp0 + q * 16 + lane / 2;  // the vector whose random numbers these are
        if (t < whole || (t < steps && v < sl.nvec))
          copy_noise(slot + NT - tid + warp0 * 2 + q * 32 + lane, nsrc + (long long)v * VEC + (lane & 1) * 4);
      }
    }
    copy_commit();
  };
#pragma unroll
  for (int t = 0; t < R; ++t) fetch(t, ring + t * kPieces * NT);
  if (tid == 0) sh.ybest = -INFINITY;
  __syncthreads();
  if (tid < sl.head + sl.tail) {
    const int i = tid < sl.head ? tid : sl.nvec * VEC + tid;
    const float z = to_f(sl.p[i]), e = noise[i];
    stat_raise(st.m, st.s, fmaxf(z, -INFINITY), c);
    st.s += sum_exp<1>(&z, st.m, c);
    race.take(fmaf(z, c, -lg2(e)), z, e, sl.lo + i);
  }
  volatile float* shared_y = &sh.ybest;
  int place = 0;
  for (int t = 0; t < steps; ++t) {
    copy_wait<R - 1>();
    if (VEC == 8) __syncwarp();
    uint4* const slot = ring + place * kPieces * NT;
    float z[8], e[8], y[8];
#pragma unroll
    for (int q = 0; q < Q; ++q) unpack<T>(slot[q * NT], z + q * VEC);
#pragma unroll
    for (int q = 0; q < 2; ++q)
      unpack<float>(VEC == 4 ? slot[(2 + q) * NT] : slot[NT + tid + q], e + 4 * q);
    if (VEC == 8) __syncwarp();
    if (t >= whole) {
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        if (!has(t, q)) {
#pragma unroll
          for (int x = 0; x < VEC; ++x) {
            z[q * VEC + x] = -INFINITY;  // (y is then -inf too, which never wins)
            e[q * VEC + x] = 1.f;
          }
        }
      }
    }
    fetch(t + R, slot);
    place = place + 1 == R ? 0 : place + 1;
    stat_raise(st.m, st.s, vec_max<8>(z), c);
    st.s += sum_exp<8>(z, st.m, c);
#pragma unroll
    for (int x = 0; x < 8; ++x) y[x] = fmaf(z[x], c, -lg2(e[x]));
    const float known = *shared_y, least = known - Race::margin(known);
    if (vec_max<8>(y) > least) {
#pragma unroll
      for (int x = 0; x < 8; ++x)
        if (y[x] > least)
          race.take(y[x], z[x], e[x], sl.lo + sl.head + ((t * Q + x / VEC) * NT + tid) * VEC + x % VEC);
      if (race.y > known) *shared_y = race.y;
    }
  }
  copy_wait<0>();
  st_out = st;
  race_out = race;
}

struct Bound {  // tokens ranked before (z, id); `none`: all tokens
  bool none = true;
  float z = 0.f;
  int id = 0;
  TS_DEVICE bool before(float x, int i) const { return none || x > z || (x == z && i < id); }
};

// How many tokens rank before `bound`, and their mass.
template <typename T, int NT>
__device__ __noinline__ void count_before(Shared<T, NT>& sh, const Slice<T> sl, float m, float c, const Bound& bound,
                                          int& count, float& mass) {
  constexpr int VEC = Slice<T>::kVec, Q = 16 / VEC;
  const int tid = threadIdx.x;
  Steps<T, NT> steps(sl, sh.ring);
  const float bz = bound.z;
  const int bi = bound.id;
  // as in sum_exp: the mass is compared with a total that is made so
  const float r = m * c;
  const bool fused = fabsf(r) <= kFusedMost;
  auto power = [&](float a) { return fused ? ex2(fmaf(a, c, -r)) : rel_exp(a, m, c); };
  int n = 0;
  float s0 = 0.f, s1 = 0.f;
  if (tid < sl.head + sl.tail) {
    const int i = tid < sl.head ? tid : sl.nvec * VEC + tid;
    const float a = to_f(sl.p[i]);
    if (bound.before(a, sl.lo + i)) {
      ++n;
      s0 += power(a);
    }
  }
  for (int t = 0; t < steps.count; ++t) {
    float z[Q][VEC];
    steps.read(t, z);
    bool even = false;
#pragma unroll
    for (int q = 0; q < Q; ++q) {
#pragma unroll
      for (int e = 0; e < VEC; e += 2) {
        const float a = z[q][e], b = z[q][e + 1];
        const float ea = power(a), eb = power(b);
        n += (a > bz) + (b > bz);
        s0 += a > bz ? ea : 0.f;
        s1 += b > bz ? eb : 0.f;
        even |= a == bz || b == bz;
      }
    }
    if (even) {
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const int id = sl.lo + sl.head + ((t * Q + q) * NT + tid) * VEC;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          if (z[q][e] == bz && id + e < bi && steps.has(t, q)) {
            ++n;
            s0 += power(bz);
          }
        }
      }
    }
  }
  copy_wait<0>();
  count = n;
  s0 += s1;
  mass = fused ? fmaf(s0, -kLn2 * fmaf(m, c, -r), s0) : s0;
}

// The race among the tokens before `bound` with weight min_p at least (none is below zmin). Random numbers are read
// where a vector holds such a token.
template <typename T, int NT>
__device__ __noinline__ void race_before(Shared<T, NT>& sh, const Slice<T> sl, const float* __restrict__ noise, float m,
                                         float temperature, float c, float min_p, float zmin, const Bound& bound,
                                         Race& race) {
  constexpr int VEC = Slice<T>::kVec;
  constexpr int U = VEC == 4 ? 4 : 2;
  const int tid = threadIdx.x;
  const float bz = bound.z;
  const int bi = bound.id;
  const float floor = fmaxf(bz, zmin);
  const bool all = !(min_p > 0.f);
  Race r;
  volatile float* shared_y = &sh.ybest;
  if (tid == 0) sh.ybest = -INFINITY;
  __syncthreads();
  auto one = [&](float z, float e, int id) {
    const float y = fmaf(z, c, -lg2(e)), known = *shared_y;
    if (y > known - Race::margin(known) && (z > bz || (z == bz && id < bi)) && z >= zmin &&
        (all || weight(z, m, temperature) >= min_p || z == m)) {
      r.take(y, z, e, id);
      if (r.y > known) *shared_y = r.y;
    }
  };
  if (tid < sl.head + sl.tail) {
    const int i = tid < sl.head ? tid : sl.nvec * VEC + tid;
    one(to_f(sl.p[i]), noise[i], sl.lo + i);
  }
  const T* body = sl.body();
  const float* nb = noise + sl.head;
  const bool wide = (reinterpret_cast<uintptr_t>(nb) & 15) == 0;
  for (int i0 = tid; i0 < sl.nvec; i0 += U * NT) {
    uint4 raw[U];
    float e[U][VEC];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (i0 + u * NT < sl.nvec) raw[u] = load_stream(body + (long long)(i0 + u * NT) * VEC);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long i = (long long)(i0 + u * NT) * VEC;
      float z[VEC];
      unpack<T>(raw[u], z);
      if (i0 + u * NT < sl.nvec && vec_max<VEC>(z) >= floor) {
        if (wide) {
#pragma unroll
          for (int q = 0; q < VEC; q += 4) unpack<float>(load_stream(nb + i + q), e[u] + q);
        } else {
#pragma unroll
          for (int q = 0; q < VEC; ++q) e[u][q] = nb[i + q];
        }
      } else {
#pragma unroll
        for (int q = 0; q < VEC; ++q) e[u][q] = INFINITY;  // (never wins)
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = sl.head + (i0 + u * NT) * VEC;
      float z[VEC];
      unpack<T>(raw[u], z);
#pragma unroll
      for (int q = 0; q < VEC; ++q) one(z[q], e[u][q], sl.lo + i + q);
    }
  }
  race = r;
}

// The best exact key of those tokens (of all tokens, where there is no bound).
template <typename T, int NT>
__device__ __noinline__ uint64_t scan_exact(const Slice<T> sl, const float* __restrict__ noise, float m,
                                            float temperature, float min_p, float zmin, const Bound& bound) {
  uint64_t best = 0;
  for (int i = threadIdx.x; i < sl.n; i += NT) {
    const float z = to_f(sl.p[i]);
    const int id = sl.lo + i;
    if (bound.none || (bound.before(z, id) && z >= zmin)) {
      const float w = weight(z, m, temperature);
      if (w >= min_p || z == m) {
        const uint64_t key = race_key(w, noise[i], id);
        best = key > best ? key : best;
      }
    }
  }
  return best;
}

// Cluster-wide sums and bests; all threads of all parts get them. `turn` alternates between calls.
template <typename T, int NT>
__device__ void join_keys(Shared<T, NT>& sh, int& turn, int& count, float& mass, uint64_t& best, int& flag) {
  cg::cluster_group cl = cg::this_cluster();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto fold = [&]() {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      count += __shfl_xor_sync(0xffffffffu, count, o);
      mass += __shfl_xor_sync(0xffffffffu, mass, o);
      const uint64_t b = __shfl_xor_sync(0xffffffffu, best, o);
      best = b > best ? b : best;
    }
  };
  flag = __syncthreads_or(flag);
  fold();
  if (lane == 0) {
    sh.wm[warp] = mass;
    sh.wc[warp] = count;
    sh.wbest[warp] = best;
  }
  __syncthreads();
  if (warp == 0) {
    mass = lane < NT / 32 ? sh.wm[lane] : 0.f;
    count = lane < NT / 32 ? sh.wc[lane] : 0;
    best = lane < NT / 32 ? sh.wbest[lane] : 0;
    fold();
    if (lane == 0) {
      sh.ps[turn] = mass;
      sh.pcount[turn] = count;
      sh.pbest[turn] = best;
      sh.pflag[turn] = flag;
    }
  }
  cl.sync();
  const int parts = (int)cl.num_blocks();
  if (warp == 0) {
    count = 0;
    mass = 0.f;
    best = 0;
    flag = 0;
    if (lane < parts) {
      const Shared<T, NT>* o = cl.map_shared_rank(&sh, lane);
      mass = o->ps[turn];
      count = o->pcount[turn];
      best = o->pbest[turn];
      flag = o->pflag[turn];
    }
    fold();
    flag = __reduce_or_sync(0xffffffffu, flag);
    if (lane == 0) {
      sh.js = mass;
      sh.jcount = count;
      sh.jbest = best;
      sh.jflag = flag;
    }
  }
  __syncthreads();
  mass = sh.js;
  count = sh.jcount;
  best = sh.jbest;
  flag = sh.jflag;
  turn ^= 1;
}

// The bound before which tokens are kept by top-k and top-p (`p` of the total mass), by bisection of the 64-bit ranks;
// the token of rank `out` is not kept.
template <typename T, int NT>
__device__ __noinline__ Bound kept_bound(Shared<T, NT>& sh, const Slice<T> sl, float m, float c, float total,
                                         long long top_k, float p, uint64_t out, int& turn) {
  uint64_t lo = out, hi = ((uint64_t)order_key(m) << 32) | 0xffffffffu;  // nothing ranks before hi
  Bound b;
  b.none = false;
  auto set = [&](uint64_t x) {
    const uint32_t order = (uint32_t)(x >> 32), id = ~(uint32_t)x;
    b.z = key_value(order);
    b.id = id > 0x7fffffffu || order == 0x7fffffffu ? 0x7fffffff : (int)id;  // (no logit has -0's own order)
  };
  while (hi - lo > 1) {
    const uint64_t mid = lo + (hi - lo) / 2;
    set(mid);
    int count = 0, flag = 0;
    float mass = 0.f;
    uint64_t best = 0;
    count_before<T, NT>(sh, sl, m, c, b, count, mass);
    join_keys(sh, turn, count, mass, best, flag);
    if (count == 0 || (count < top_k && mass < p * total)) hi = mid;
    else lo = mid;
  }
  set(lo);  // a token of rank hi and those before it are kept: what ranks before lo
  return b;
}

// The first-ranked token.
template <typename T, int NT>
__device__ __noinline__ int first_rank(Shared<T, NT>& sh, const Slice<T>& sl, int& turn) {
  uint64_t best = 0;
  for (int i = threadIdx.x; i < sl.n; i += NT) {
    const uint64_t x = rank_key(to_f(sl.p[i]), sl.lo + i);
    best = x > best ? x : best;
  }
  int count = 0, flag = 0;
  float mass = 0.f;
  join_keys(sh, turn, count, mass, best, flag);
  return rank_id(best);
}

template <typename T, int NT>
__global__ void __launch_bounds__(NT, NT == 256 ? 4 : 1) sample_kernel(const T* __restrict__ logits, long long stride,
                                                    const float* __restrict__ noise, long long nstride, int v,
                                                    SampleArgs a, int64_t* __restrict__ tokens,
                                                    float* __restrict__ logprobs) {
  extern __shared__ __align__(16) uint8_t raw[];
  Shared<T, NT>& sh = *reinterpret_cast<Shared<T, NT>*>(raw);
  cg::cluster_group cl = cg::this_cluster();
  const int parts = (int)cl.num_blocks(), part = (int)cl.block_rank();
  const int row = blockIdx.x / parts;
  const int tid = threadIdx.x;
  float temperature = a.temperature ? a.temperature[row] : a.temperature_s;
  const float top_p = a.top_p ? a.top_p[row] : a.top_p_s;
  const float min_p = fminf(a.min_p ? a.min_p[row] : a.min_p_s, 1.f);
  const long long top_k = a.top_k ? a.top_k[row] : a.top_k_s;
  const bool greedy = !(temperature >= kColdest);
  if (greedy) temperature = 1.f;
  const float c = kLog2e / temperature;
  const bool by_k = top_k > 0 && top_k < v, by_p = top_p < 1.f, by_m = min_p > 0.f;
  const bool race_first = !greedy && !(by_k && top_k <= kMaxTop);
  const int k = greedy ? 1 : (int)top_k;  // of the list
  const T* lrow = logits + row * stride;
  const float* nrow = noise ? noise + row * nstride : nullptr;
  Slice<T> sl(lrow, v, part, parts);
  const float* ns = nrow ? nrow + sl.lo : nullptr;
  Stat st;
  Race race;
  int turn = 0;
  if (race_first) {
    scan_free<T, NT>(sh, sl, ns, c, st, race);
    block_stat(sh, st, c);
    st = join_stat(sh, st, c);
    turn = 1;
  } else {
    st = scan_slice<T, NT>(sh, sl, k, c);
    block_stat(sh, st, c);
    join_parts(sh, k, c, st);
  }
  const float m = st.m, total = st.s;
  auto result = [&](int id) {
    tokens[row] = id;
    logprobs[row] = id < 0 ? __int_as_float(0x7fc00000) : (to_f(lrow[id]) - m) / temperature - logf(total);
  };
  if (!(total > 0.f && total < INFINITY)) {  // the same in every part: no distribution
    if (part == 0 && tid == 0) result(-1);
    cl.sync();
    return;
  }
  if (part == 0 && !race_first) {
    if (greedy) {
      if (tid == 0) result(rank_id(sh.win[0]));
    } else {
      // the list in rank order: weights, the mass before each, and the race among the kept
      const int n = sh.nwin;
      const uint64_t x = tid < n ? sh.win[tid] : 0;
      const float w = tid < n ? weight(rank_value(x), m, temperature) : 0.f;
      float incl = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const float up = __shfl_up_sync(0xffffffffu, incl, o);
        if ((tid & 31) >= o) incl += up;
      }
      if ((tid & 31) == 31) sh.wm[tid >> 5] = incl;
      __syncthreads();
      float before = incl - w;
      if (tid < n)
        for (int q = 0; q < (tid >> 5); ++q) before += sh.wm[q];
      const bool kept = tid < n && (tid == 0 || ((!by_p || before < top_p * total) && w >= min_p));
      uint64_t best = kept ? race_key(w, nrow[rank_id(x)], rank_id(x)) : 0;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const uint64_t b = __shfl_xor_sync(0xffffffffu, best, o);
        best = b > best ? b : best;
      }
      if ((tid & 31) == 0) sh.wbest[tid >> 5] = best;
      __syncthreads();
      if (tid == 0) {
        for (int q = 0; q < kMaxTop / 32; ++q) best = sh.wbest[q] > best ? sh.wbest[q] : best;
        result(rank_id(best ? best : sh.win[0]));
      }
    }
  }
  if (!race_first) {
    cl.sync();  // no part leaves while another may still read its shared memory
    return;
  }
  // The best key of all tokens is the sample if it is kept: two passes over the logits alone where there is a top-k
  // or top-p (the race, and what ranks before the winner), else one. If it is not kept, no token ranked after it is
  // (the filters keep a prefix of the rank order), and the best key of those before it is next.
  // No token below zmin has weight min_p (the weight itself decides about those above).
  const float zmin = by_m ? m + temperature * (logf(min_p) - 1e-4f) - 1e-5f * fabsf(m) : -INFINITY;
  Bound bound;
  int id = -1, rounds = 0;
  bool settled = false;  // all tokens before `bound` are kept by top-k and top-p
  for (;;) {
    // the best of y, and then of the exact keys of the tokens within its margin
    int c0 = 0, f0 = 0, tie = 0;
    float m0 = 0.f;
    uint64_t best = race.id >= 0 ? (uint64_t)order_key(race.y) << 32 : 0;
    join_keys(sh, turn, c0, m0, best, f0);
    const float ybest = key_value((uint32_t)(best >> 32));
    best = 0;
    if (race.id >= 0 && race.y >= ybest - Race::margin(ybest)) {
      best = race_key(weight(race.z, m, temperature), race.e, race.id);
      tie = race.tie;
    }
    join_keys(sh, turn, c0, m0, best, tie);
    if (tie || (best >> 32) == 0) {  // no single winner by y (or a key that vanished): by exact keys
      best = scan_exact<T, NT>(sl, ns, m, temperature, bound.none ? 0.f : min_p, zmin, bound);
      join_keys(sh, turn, c0, m0, best, f0);
    }
    if (best == 0) {  // random numbers that are none: the first of the ranks
      id = first_rank<T, NT>(sh, sl, turn);
      break;
    }
    id = rank_id(best);
    if (settled) break;
    const float z = to_f(lrow[id]);
    bound.none = false;
    bound.id = id;
    bound.z = z;
    if (weight(z, m, temperature) >= min_p || z == m) {
      if (!by_k && !by_p) break;
      int count = 0;
      float mass = 0.f;
      count_before<T, NT>(sh, sl, m, c, bound, count, mass);
      best = 0;
      join_keys(sh, turn, count, mass, best, f0);
      if (count == 0 || ((!by_k || count < top_k) && (!by_p || mass < top_p * total))) break;
    }
    // A winner that is not kept takes about half of what ranks before the last one away, so with random numbers this
    // goes on for 1 + log(1 / kept share) rounds. Numbers that are not random can make it a round for each token.
    if (++rounds == kMaxRounds) {
      bound = kept_bound<T, NT>(sh, sl, m, c, total, by_k ? top_k : (long long)v, by_p ? top_p : INFINITY,
                                rank_key(z, id), turn);
      settled = true;
    }
    race = Race();
    race_before<T, NT>(sh, sl, ns, m, temperature, c, min_p, zmin, bound, race);
  }
  if (part == 0 && tid == 0) result(id);
  cl.sync();  // no part leaves while another may still read its shared memory
}

// Parts (CTAs, a cluster) of a row, in doublings up to eight while they are at most `most` CTAs an SM in all and a part
// has `least` logits. Joining the parts of a row costs more than it brings where the rows alone fill the SMs. Measured
// in us, with 1 / 2 / 4 / 8 parts, V = 151,936: top 20 of 64 bf16 rows 24 / 19 / 19 / 23, of 200 31 / 29 / 43 / 62;
// top 64 of 300 fp32 rows 45 / 58 / 64 / 82.
int row_parts(int64_t rows, int v, int sms, int most, int least) {
  int parts = 1;
  while (parts < kMaxParts && 2 * rows * parts <= (int64_t)most * sms && v / (2 * parts) >= least) parts *= 2;
  return parts;
}
// A part takes all the threads of an SM where there are fewer parts than SMs.
bool few_rows(int64_t rows, int parts, int sms) { return rows * parts <= sms; }

template <typename T, int NT, typename... KArgs, typename... Args>
cudaError_t launch_rows(const VocabLaunch& l, void (*kernel)(KArgs...), int64_t rows, int parts, Args&&... args) {
  const int bytes = (int)sizeof(Shared<T, NT>);
  const cudaError_t e = l.set_smem((const void*)kernel, bytes);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * parts));
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = l.stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = parts;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

template <typename T>
cudaError_t topk_of(const VocabLaunch& l, const VocabRows& x, int k, float temperature, int64_t* ids, float* lp) {
  const int parts = row_parts(x.n, x.v, l.sms, 3, 32768);
  if (few_rows(x.n, parts, l.sms))
    return launch_rows<T, 1024>(l, topk_kernel<T, 1024>, x.n, parts, (const T*)x.logits, x.stride, x.v, k, temperature,
                                ids, lp);
  return launch_rows<T, 256>(l, topk_kernel<T, 256>, x.n, parts, (const T*)x.logits, x.stride, x.v, k, temperature, ids,
                             lp);
}
template <typename T>
cudaError_t sample_of(const VocabLaunch& l, const VocabRows& x, const float* noise, long long nstride,
                      const SampleArgs& a, int64_t* tokens, float* lp) {
  // The settings decide how often a row is read: once for a small top-k, once with the random numbers without a filter,
  // and again for each winner of the race that has to be looked at under a top-p or min-p, which wants more parts (512
  // fp32 rows, top-p 0.9, 1 / 2 / 4 / 8 parts: 450 / 331 / 280 / 334 us). Settings of each row may be any of these.
  const bool mixed = a.temperature || a.top_k || a.top_p || a.min_p;
  const bool list = a.temperature_s < kColdest || (a.top_k_s > 0 && a.top_k_s <= kMaxTop);
  const bool filter = a.top_p_s < 1.f || a.min_p_s > 0.f || a.top_k_s > 0;
  const int parts = mixed    ? row_parts(x.n, x.v, l.sms, 8, 16384)
                    : list   ? row_parts(x.n, x.v, l.sms, 3, 32768)
                    : filter ? row_parts(x.n, x.v, l.sms, 16, 16384)
                             : row_parts(x.n, x.v, l.sms, 3, 16384);
  if (few_rows(x.n, parts, l.sms))
    return launch_rows<T, 1024>(l, sample_kernel<T, 1024>, x.n, parts, (const T*)x.logits, x.stride, noise, nstride,
                                x.v, a, tokens, lp);
  return launch_rows<T, 256>(l, sample_kernel<T, 256>, x.n, parts, (const T*)x.logits, x.stride, noise, nstride, x.v, a,
                             tokens, lp);
}

}  // namespace

cudaError_t vocab_topk(const VocabLaunch& l, const VocabRows& x, int k, float temperature, int64_t* ids, float* lp) {
  switch (x.type) {
    case kRowsF32: return topk_of<float>(l, x, k, temperature, ids, lp);
    case kRowsBf16: return topk_of<__nv_bfloat16>(l, x, k, temperature, ids, lp);
    default: return topk_of<__half>(l, x, k, temperature, ids, lp);
  }
}

cudaError_t vocab_sample(const VocabLaunch& l, const VocabRows& x, const float* noise, long long nstride,
                         const SampleArgs& a, int64_t* tokens, float* lp) {
  switch (x.type) {
    case kRowsF32: return sample_of<float>(l, x, noise, nstride, a, tokens, lp);
    case kRowsBf16: return sample_of<__nv_bfloat16>(l, x, noise, nstride, a, tokens, lp);
    default: return sample_of<__half>(l, x, noise, nstride, a, tokens, lp);
  }
}

int vocab_max_top() { return kMaxTop; }

}  // namespace ts

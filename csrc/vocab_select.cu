// Top-k log-probabilities and sampling over rows of logits [N, V].
//
// topk_logprobs: the k largest logits of a row (ties: lower token first) with log p = z/tau - lse(z/tau).
// sample_tokens: one token per row, drawn from softmax(z/tau) restricted by top-k, top-p and min-p: with e_i the
//   row's given Exp(1) numbers, argmax over the kept tokens of w_i / e_i, w_i = exp((z_i - max z)/tau), is a sample
//   (the smallest of independent exponential times with rates w_i). All three filters keep a prefix of the rank
//   order (greater logit first, then lower token), which is what the kernels use.
//
// One pass over the row. A slice keeps a threshold under which no element can be among its k largest, appends the
// elements above it to a buffer in shared memory and, when that runs full, cuts it back to the k best (radix select
// on 64-bit words of logit order and token, so that there are no ties) and raises the threshold. The first tile's
// threshold is the k-th largest of the threads' own maxima.
#include "common.cuh"
#include "vocab.cuh"
#include "vocab.h"

namespace ts {
namespace {

namespace cg = cooperative_groups;
using namespace vocab;

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxTop = 256;
constexpr int kPer = 16;                     // elements of a thread in a tile
constexpr int kTile = kThreads * kPer;       // 4096
constexpr int kLimit = 1024;                 // entries that are kept before the buffer is cut back
constexpr int kCap = kLimit + kTile + 32;
constexpr int kMaxParts = 8;
static_assert(kMaxParts * kMaxTop <= kCap, "the parts' lists meet in one buffer");

struct Shared {
  uint64_t buf[kCap];
  uint64_t win[kMaxTop];
  uint32_t hist[256];
  float wm[kWarps], ws[kWarps];
  uint64_t wbest[kWarps];
  // this CTA's partial results, read by its cluster (two sets, used in turn)
  float pm[2], ps[2];
  uint64_t pbest[2];
  int pcount[2];
  int count;      // entries in buf
  int nwin;       // entries in win
  int sel_need, sel_bin, sel_done;
  int verdict;    // of part 0: 0 done, 1 the general search follows
};

struct Stat {
  float m = -INFINITY, s = 0.f;
};

// Leaves the `k` largest of sh.buf[0, n) in sh.win (unordered) and a lower bound of the smallest in `least`;
// n >= k. All threads call it after a barrier that follows the last write to buf.
__device__ void select_k(Shared& sh, int n, int k, uint64_t& least) {
  uint64_t prefix = 0;  // decided digits of the k-th largest
  int need = k;
  int shift = 56;
  const int tid = threadIdx.x;
  for (;; shift -= 8) {
    sh.hist[tid] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kThreads) {
      const uint64_t x = sh.buf[i];
      if (shift == 56 || (x >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&sh.hist[(x >> shift) & 255], 1u);
    }
    __syncthreads();
    if (tid < 32) {
      // lane l sums the 8 bins from 255 - 8l downwards
      uint32_t h[8], sum = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) sum += h[j] = sh.hist[255 - 8 * tid - j];
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
            sh.sel_done = (int)h[j] == need - (int)above;
            break;
          }
          above += h[j];
        }
      }
    }
    __syncthreads();
    prefix |= (uint64_t)sh.sel_bin << shift;
    need = sh.sel_need;
    if (sh.sel_done || shift == 0) break;  // every entry of the bin belongs to the k
  }
  least = prefix;
  if (tid == 0) sh.nwin = 0;
  __syncthreads();
  for (int i = tid; i < n; i += kThreads) {
    const uint64_t x = sh.buf[i];
    if (x >= prefix) {
      const int at = atomicAdd(&sh.nwin, 1);
      if (at < kMaxTop) sh.win[at] = x;
    }
  }
  __syncthreads();
}

// The slice's k largest (all of it where it is shorter) in sh.win / sh.nwin, and its statistics per thread.
template <typename T>
__device__ void scan_slice(Shared& sh, const Slice<T>& sl, int k, float c, Stat& st) {
  constexpr int VEC = Slice<T>::kVec;
  constexpr int U = kPer / VEC;
  const int tid = threadIdx.x, lane = tid & 31;
  const T* body = sl.body();
  if (tid == 0) sh.count = 0;
  __syncthreads();

  bool open = true;        // no threshold yet: every element is appended
  uint32_t tkey = 0;       // else: elements whose order is above it (strictly: at equal logits the lower token is in)

  // appends this thread's elements whose bit is set in `take`; returns the entries used so far (of this warp's view)
  auto append = [&](uint32_t take, auto&& entry) -> int {
    const int mine = __popc(take);
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    const int total = __shfl_sync(0xffffffffu, incl, 31);
    if (total == 0) return 0;
    int base = 0;
    if (lane == 31) base = atomicAdd(&sh.count, total);
    base = __shfl_sync(0xffffffffu, base, 31);
    int at = base + incl - mine;
    while (take) {
      const int e = __ffs(take) - 1;
      take &= take - 1;
      if (at < kCap) sh.buf[at] = entry(e);
      ++at;
    }
    return base + total;
  };
  auto cut = [&]() {  // all threads; buf complete
    const int n = sh.count;
    __syncthreads();  // all have read it before anyone appends again
    if (n < k) return;
    uint64_t least;
    select_k(sh, n, k, least);
    for (int i = tid; i < k; i += kThreads) sh.buf[i] = sh.win[i];
    if (tid == 0) sh.count = k;
    open = false;
    tkey = (uint32_t)(least >> 32);
    __syncthreads();
  };
  // the unaligned ends (fewer elements than a vector): one element of each of the first threads
  auto edge = [&](int first, int cnt) {
    uint32_t take = 0;
    float v = -INFINITY;
    const int i = first + tid;
    if (tid < cnt) {
      v = to_f(sl.p[i]);
      stat_raise(st.m, st.s, fmaxf(v, -INFINITY), c);
      st.s += sum_exp<1>(&v, st.m, c);
      take = open || order_key(v) > tkey;
    }
    if (tid < 32) append(take, [&](int) { return rank_key(v, sl.lo + i); });
  };

  if (sl.head > 0) edge(0, sl.head);

  const int tiles = (sl.nvec + U * kThreads - 1) / (U * kThreads);
  uint4 next[U];
  auto load = [&](int t) {
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int i = (t * U + j) * kThreads + tid;
      if (i < sl.nvec) next[j] = load_stream(body + (long long)i * VEC);
    }
  };
  if (tiles > 0) load(0);
  for (int t = 0; t < tiles; ++t) {
    float v[kPer];
    uint32_t valid = 0;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int i = (t * U + j) * kThreads + tid;
      if (i < sl.nvec) {
        unpack<T>(next[j], v + j * VEC);
        valid |= ((1u << VEC) - 1u) << (j * VEC);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[j * VEC + e] = -INFINITY;
      }
    }
    if (t + 1 < tiles) load(t + 1);
    float tmax = -INFINITY;
#pragma unroll
    for (int e = 0; e < kPer; ++e) tmax = fmaxf(tmax, v[e]);
    stat_raise(st.m, st.s, tmax, c);
    st.s += sum_exp<kPer>(v, st.m, c);
    if (t == 0 && open) {
      // a threshold that at least k of the threads' maxima reach: bitwise from the top, exact to 2^-11 of a logit
      uint32_t mine = 0;
      if (tmax > -INFINITY) {
        mine = order_key(tmax);
      } else {  // nothing but -inf, NaN (which tmax leaves out) and places past the end
#pragma unroll
        for (int e = 0; e < kPer; ++e)
          if ((valid >> e) & 1) mine = max(mine, order_key(v[e]));
      }
      uint32_t lo = 0;
      for (int bit = 31; bit >= 12; --bit) {
        const uint32_t cand = lo | (1u << bit);
        const int cnt = __syncthreads_count(mine >= cand);
        if (cnt >= k) lo = cand;
        if (cnt == k) break;
      }
      if (lo > 0) {
        tkey = lo - 1;
            open = false;
      }
    }
    int used = 0;
    if (__any_sync(0xffffffffu, open || order_key(tmax) > tkey)) {
      uint32_t take = 0;
#pragma unroll
      for (int e = 0; e < kPer; ++e)
        if (open || order_key(v[e]) > tkey) take |= 1u << e;
      used = append(take & valid, [&](int e) {
        float x = 0.f;
#pragma unroll
        for (int q = 0; q < kPer; ++q)
          if (q == e) x = v[q];
        const int i = (t * U + e / VEC) * kThreads + tid;
        return rank_key(x, sl.lo + sl.head + i * VEC + e % VEC);
      });
    }
    if (__syncthreads_or(t == 0 || used > kLimit)) cut();
  }
  if (sl.tail > 0) edge(sl.head + sl.nvec * VEC, sl.tail);
  __syncthreads();
  const int n = sh.count;
  if (n > k) {
    uint64_t least;
    select_k(sh, n, k, least);
  } else {
    for (int i = tid; i < n; i += kThreads) sh.win[i] = sh.buf[i];
    if (tid == 0) sh.nwin = n;
    __syncthreads();
  }
}

// Block-wide (m, s); all threads get it.
__device__ void block_stat(Shared& sh, Stat& st, float c) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, st.m, o), s2 = __shfl_xor_sync(0xffffffffu, st.s, o);
    stat_merge(st.m, st.s, m2, s2, c);
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) {
    sh.wm[threadIdx.x >> 5] = st.m;
    sh.ws[threadIdx.x >> 5] = st.s;
  }
  __syncthreads();
  Stat all;
  for (int w = 0; w < kWarps; ++w) stat_merge(all.m, all.s, sh.wm[w], sh.ws[w], c);
  st = all;
}

// The row's k largest from the parts' lists: part 0 gets them in sh.win in rank order (sh.nwin of them); every part
// gets the row's statistics.
__device__ void join_parts(Shared& sh, int k, float c, Stat& st) {
  const int tid = threadIdx.x;
  cg::cluster_group cl = cg::this_cluster();
  const int parts = (int)cl.num_blocks();
  if (parts > 1) {
    if (tid == 0) {
      sh.pm[0] = st.m;
      sh.ps[0] = st.s;
    }
    cl.sync();
    Stat row;
    for (int r = 0; r < parts; ++r) {
      Shared* o = cl.map_shared_rank(&sh, r);
      stat_merge(row.m, row.s, o->pm[0], o->ps[0], c);
    }
    st = row;
    int n = 0;
    if (cl.block_rank() == 0) {
      for (int r = 0; r < parts; ++r) {
        Shared* o = cl.map_shared_rank(&sh, r);
        const int cnt = o->nwin;
        for (int i = tid; i < cnt; i += kThreads) sh.buf[n + i] = o->win[i];
        n += cnt;
      }
    }
    cl.sync();
    if (cl.block_rank() == 0) {
      uint64_t least;
      if (n > k) {
        select_k(sh, n, k, least);
      } else {
        for (int i = tid; i < n; i += kThreads) sh.win[i] = sh.buf[i];
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
    if (tid < n) sh.win[at] = mine;
    __syncthreads();
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) topk_kernel(const T* __restrict__ logits, long long stride, int v, int k,
                                                        float temperature, int64_t* __restrict__ ids,
                                                        float* __restrict__ logprobs) {
  extern __shared__ __align__(16) uint8_t raw[];
  Shared& sh = *reinterpret_cast<Shared*>(raw);
  cg::cluster_group cl = cg::this_cluster();
  const int parts = (int)cl.num_blocks();
  const int row = blockIdx.x / parts;
  const float c = kLog2e / temperature;
  Slice<T> sl(logits + row * stride, v, (int)cl.block_rank(), parts);
  Stat st;
  scan_slice<T>(sh, sl, k, c, st);
  block_stat(sh, st, c);
  join_parts(sh, k, c, st);
  if (cl.block_rank() == 0) {
    const float m = st.m == -INFINITY ? 0.f : st.m;
    const float ls = st.s == 0.f ? 0.f : logf(st.s);  // a row of -inf alone: its log-probs are -inf
    for (int i = threadIdx.x; i < k; i += kThreads) {
      const uint64_t x = sh.win[i];
      ids[(long long)row * k + i] = rank_id(x);
      logprobs[(long long)row * k + i] = (rank_value(x) - m) / temperature - ls;
    }
  }
}

constexpr float kColdest = 1e-6f;  // colder rows are greedy

// One pass over the slice for the token search of rows whose kept set is not known: of the tokens ranked before
// `bound` (all, where it is ~0) the number and mass before `bound`, and the best key w/e among those with w >= min_p.
template <typename T>
__device__ void scan_keys(const Slice<T>& sl, const float* __restrict__ noise, float m, float temperature,
                          float min_p, uint64_t bound, int& count, float& mass, uint64_t& best) {
  constexpr int VEC = Slice<T>::kVec;
  const int tid = threadIdx.x;
  auto one = [&](float z, float e, int id) {
    if (bound != 0 && rank_key(z, id) <= bound) return;
    const float w = expf((z - m) / temperature);
    ++count;
    mass += w;
    if (w >= min_p) {
      const float key = w / e;
      if (key >= 0.f) {
        const uint64_t x = ((uint64_t)__float_as_uint(key) << 32) | (uint32_t)~(uint32_t)id;
        if (x > best) best = x;
      }
    }
  };
  for (int i = tid; i < sl.head; i += kThreads) one(to_f(sl.p[i]), noise[i], sl.lo + i);
  const T* body = sl.body();
  const float* nb = noise + sl.head;
  const bool wide = (reinterpret_cast<uintptr_t>(nb) & 15) == 0;
  for (int i = tid; i < sl.nvec; i += kThreads) {
    float z[VEC], e[VEC];
    unpack<T>(load_stream(body + (long long)i * VEC), z);
    if (wide) {
#pragma unroll
      for (int q = 0; q < VEC; q += 4) unpack<float>(load_stream(nb + (long long)i * VEC + q), e + q);
    } else {
#pragma unroll
      for (int q = 0; q < VEC; ++q) e[q] = nb[(long long)i * VEC + q];
    }
#pragma unroll
    for (int q = 0; q < VEC; ++q) one(z[q], e[q], sl.lo + sl.head + i * VEC + q);
  }
  const int t0 = sl.head + sl.nvec * VEC;
  for (int i = tid; i < sl.tail; i += kThreads) one(to_f(sl.p[t0 + i]), noise[t0 + i], sl.lo + t0 + i);
}

// Row-wide (cluster-wide) sums and best of scan_keys; all threads of all parts get them. `turn` alternates.
__device__ void join_keys(Shared& sh, int turn, int& count, float& mass, uint64_t& best) {
  cg::cluster_group cl = cg::this_cluster();
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    count += __shfl_xor_sync(0xffffffffu, count, o);
    mass += __shfl_xor_sync(0xffffffffu, mass, o);
    const uint64_t b = __shfl_xor_sync(0xffffffffu, best, o);
    best = b > best ? b : best;
  }
  __syncthreads();
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) == 0) {
    sh.wm[warp] = mass;
    sh.hist[warp] = count;
    sh.wbest[warp] = best;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    count = 0;
    mass = 0.f;
    best = 0;
    for (int w = 0; w < kWarps; ++w) {
      mass += sh.wm[w];
      count += (int)sh.hist[w];
      best = sh.wbest[w] > best ? sh.wbest[w] : best;
    }
    sh.ps[turn] = mass;
    sh.pcount[turn] = count;
    sh.pbest[turn] = best;
  }
  cl.sync();
  count = 0;
  mass = 0.f;
  best = 0;
  for (int r = 0; r < (int)cl.num_blocks(); ++r) {
    Shared* o = cl.map_shared_rank(&sh, r);
    mass += o->ps[turn];
    count += o->pcount[turn];
    best = o->pbest[turn] > best ? o->pbest[turn] : best;
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const T* __restrict__ logits, long long stride,
                                                          const float* __restrict__ noise, long long nstride, int v,
                                                          SampleArgs a, int64_t* __restrict__ tokens,
                                                          float* __restrict__ logprobs) {
  extern __shared__ __align__(16) uint8_t raw[];
  Shared& sh = *reinterpret_cast<Shared*>(raw);
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
  const bool by_k = top_k > 0 && top_k < v, by_p = top_p < 1.f;
  const bool free_row = !greedy && !by_k && !by_p && !(min_p > 0.f);
  const int k = greedy || free_row ? 1 : by_k && top_k < kMaxTop ? (int)top_k : min(v, kMaxTop);
  const T* lrow = logits + row * stride;
  const float* nrow = noise ? noise + row * nstride : nullptr;
  Slice<T> sl(lrow, v, part, parts);
  Stat st;
  scan_slice<T>(sh, sl, k, c, st);
  block_stat(sh, st, c);
  join_parts(sh, k, c, st);
  const float m = st.m, total = st.s;
  auto result = [&](int id) {
    tokens[row] = id;
    logprobs[row] = id < 0 ? __int_as_float(0x7fc00000) : (to_f(lrow[id]) - m) / temperature - logf(total);
  };
  if (!(total > 0.f && total < INFINITY)) {  // the same in every part: no distribution
    if (part == 0 && tid == 0) result(-1);
    return;
  }
  if (part == 0) {
    if (greedy) {
      if (tid == 0) {
        result(rank_id(sh.win[0]));
        sh.verdict = 0;
      }
    } else if (free_row) {
      if (tid == 0) sh.verdict = 1;
    } else {
      // the list in rank order: weights, the mass before each, and whether the list holds all that is kept
      const int n = sh.nwin;
      const uint64_t x = tid < n ? sh.win[tid] : 0;
      const float w = tid < n ? expf((rank_value(x) - m) / temperature) : 0.f;
      float incl = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const float up = __shfl_up_sync(0xffffffffu, incl, o);
        if ((tid & 31) >= o) incl += up;
      }
      if ((tid & 31) == 31) sh.wm[tid >> 5] = incl;
      __syncthreads();
      float before = incl - w;
      for (int q = 0; q < (tid >> 5); ++q) before += sh.wm[q];
      const bool kept = tid < n && (tid == 0 || ((!by_p || before < top_p * total) && w >= min_p));
      const bool open = kept && tid == n - 1 && n < v && !(by_k && top_k <= n);
      const int more = __syncthreads_or(open);
      if (!more) {
        uint64_t best = 0;
        if (kept) {
          const float key = w / nrow[rank_id(x)];
          if (key >= 0.f) best = ((uint64_t)__float_as_uint(key) << 32) | (uint32_t)x;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const uint64_t b = __shfl_xor_sync(0xffffffffu, best, o);
          best = b > best ? b : best;
        }
        if ((tid & 31) == 0) sh.wbest[tid >> 5] = best;
        __syncthreads();
        if (tid == 0) {
          for (int q = 0; q < kWarps; ++q) best = sh.wbest[q] > best ? sh.wbest[q] : best;
          result(rank_id(best ? best : sh.win[0]));
        }
      }
      if (tid == 0) sh.verdict = more ? 1 : 0;
    }
  }
  cl.sync();
  const int verdict = cl.map_shared_rank(&sh, 0)->verdict;
  if (verdict) {
    // General search. The best key over all tokens is the sample if it is kept. If it is not, no token ranked after
    // it is kept either (the filters keep a prefix of the rank order), and the best key of those before it is next.
    const float* ns = nrow + sl.lo;
    uint64_t bound = 0;  // 0: all tokens
    int id = -1;
    for (int turn = 0;; turn ^= 1) {
      int count = 0;
      float mass = 0.f;
      uint64_t best = 0;
      scan_keys<T>(sl, ns, m, temperature, min_p, bound, count, mass, best);
      join_keys(sh, turn, count, mass, best);
      if (bound != 0) {
        const bool kept = count == 0 || ((!by_k || count < top_k) && (!by_p || mass < top_p * total));
        if (kept || best == 0) break;
      }
      if (best == 0) break;
      id = rank_id(best);
      if (free_row) break;
      bound = rank_key(to_f(lrow[id]), id);
    }
    if (part == 0 && tid == 0) result(id >= 0 ? id : rank_id(sh.win[0]));
  }
  cl.sync();  // no part leaves while another may still read its shared memory
}

// Parts (CTAs) of a row: one where the rows alone fill the SMs, up to a cluster of eight where there are few.
int row_parts(int64_t rows, int v, int sms) {
  int parts = 1;
  while (parts < kMaxParts && rows * parts < 2 * sms && v / (2 * parts) >= kTile) parts *= 2;
  return parts;
}

template <typename... KArgs, typename... Args>
cudaError_t launch_rows(const VocabLaunch& l, void (*kernel)(KArgs...), int64_t rows, int parts, Args&&... args) {
  const cudaError_t e = l.set_smem((const void*)kernel, (int)sizeof(Shared));
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * parts));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = sizeof(Shared);
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
  return launch_rows(l, topk_kernel<T>, x.n, row_parts(x.n, x.v, l.sms), (const T*)x.logits, x.stride, x.v, k,
                     temperature, ids, lp);
}
template <typename T>
cudaError_t sample_of(const VocabLaunch& l, const VocabRows& x, const float* noise, long long nstride,
                      const SampleArgs& a, int64_t* tokens, float* lp) {
  return launch_rows(l, sample_kernel<T>, x.n, row_parts(x.n, x.v, l.sms), (const T*)x.logits, x.stride, noise, nstride,
                     x.v, a, tokens, lp);
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

// Distillation from a teacher's top entries: loss rows over student logits [N, V] and the logits' gradient.
//
// Per row, with a = z/tau, log p = a - lse(a), S the teacher's entries (token id, log-prob t), q = exp(t):
//   forward  KL(q || p):  L = sum_S q (t - log p)     [+ Q (log Q - log P)]
//   reverse  KL(p || q):  L = sum_S p (log p - t)     [+ P (log P - log Q)]
// P and Q are what p and q give to the tokens outside S, one class together ("tail"). The gradient goes through the
// log-probs of S alone (dP = -sum dp): with g_k = dL/dlog p_k and G = sum g_k,
//   dL/dz_j = (g_j [j in S] - G p_j) / tau,
// in closed form (mass = sum_S q + Q; u = log p - t, u_T = log P - log Q):
//   forward  entries p mass - q,                    G = Q/P - mass       (without the tail: G = -sum_S q, mass likewise)
//   reverse  entries p (u - L),                     G = L - u_T
//            without the tail: p (u + 1 - L - sum_S p),  G = L + sum_S p
// P is summed over the tokens outside S directly: as 1 - sum_S p it would have no digits left where S holds nearly
// all of the mass, and the gradient divides by it. The K entries' arithmetic is done in 64 bits for the same reason
// (Q = 1 - sum q); K numbers against a row of V.
//
// Both kernels move each logit once: the forward reads the row (a bitmap of S in shared memory takes its tokens out of
// the sum), the backward reads it and writes the gradient, then overwrites the entries of S with values that the
// forward has left per entry. Memory bounds them: 1000 x 151,936 bf16 logits with 64 entries take 82 us forward (3.7
// TB/s; at 11 logits a clock and SM for full rate the forward's 11 instructions a logit, issued 63% of the time, come
// close) and 102 us backward (6.0 TB/s). For a few rows the launches and the caller's autograd take more than
// the kernels (33 fp32 rows: 21 + 9 of 70 us).
#include "bounds.cuh"
#include "common.cuh"
#include "vocab.cuh"
#include "vocab.h"

#include <algorithm>

namespace ts {
namespace {

namespace cg = cooperative_groups;
using namespace vocab;

constexpr int kSiteTeacherId = 4;  // bounds site: a teacher token id outside the vocabulary
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxTop = 256;  // teacher entries of a row: one per thread
constexpr int kMaxParts = 8;
constexpr double kLeastTail = 1e-7;  // of the teacher: about the resolution of its fp32 log-probs

struct Block2 {
  double x[kWarps], y[kWarps];
};
// Sums of x and of y over the block, to all threads.
__device__ void block_sum2(Block2& b, double& x, double& y) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    x += __shfl_xor_sync(0xffffffffu, x, o);
    y += __shfl_xor_sync(0xffffffffu, y, o);
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) {
    b.x[threadIdx.x >> 5] = x;
    b.y[threadIdx.x >> 5] = y;
  }
  __syncthreads();
  x = y = 0.0;
  for (int w = 0; w < kWarps; ++w) {
    x += b.x[w];
    y += b.y[w];
  }
}

// The block's largest m; then sums relative to it meet without a chain of rescalings, each of which would round.
__device__ float block_max(float* red, float m) {
  m = warp_max(m);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
  m = red[0];
  for (int w = 1; w < kWarps; ++w) m = fmaxf(m, red[w]);
  return m;
}
TS_DEVICE double rescaled(float m, float s, float to, float c) {
  return m == -INFINITY || m == to ? (double)s : (double)s * exp2(((double)m - (double)to) * c);
}

// The row's loss and gradient coefficients, by one block: thread k holds entry k (logit z, log-prob t; `have` where it
// counts), the tokens outside S come as (m, s_tail) with s_tail = sum 2^((z - m)·c), m = -inf if there are none.
__device__ void finish_row(Block2& b, float* red, long long row, int k, float z, float t, bool have, float m,
                           double s_tail, float c, float tau, bool reverse, bool tail, const DistillOut& out) {
  const int tid = threadIdx.x;
  const float m_tail = m;
  m = fmaxf(m_tail, block_max(red, have ? z : -INFINITY));
  if (m == -INFINITY) m = 0.f;
  // 2^-1074 is the least number of 64 bits: where the tokens outside S have less of the mass they count as having none
  const double a_tail = m_tail == -INFINITY ? 0.0 : ((double)m_tail - (double)m) * c;
  const double f_tail = exp2(a_tail);
  const double st = s_tail * f_tail;
  const double a2 = ((double)z - (double)m) * c;
  const double e = have ? exp2(a2) : 0.0;
  const double q = have ? exp((double)t) : 0.0;
  double se = e, sq = q;
  block_sum2(b, se, sq);
  const double s = st + se;
  const double ls = log(s);
  const double logp = a2 * 0.693147180559945309417 - ls;
  const double p = e / s;
  const double tp = st / s;
  const bool with_tail = tail && !(tp == 0.0);
  double lt = 0.0, tq = 0.0, ltq = 0.0;
  if (with_tail) {
    lt = a_tail * 0.693147180559945309417 + log(s_tail) - ls;
    tq = fmax(1.0 - sq, kLeastTail);
    ltq = log(tq);
  }
  double l = 0.0;
  if (have) {
    if (!reverse) l = q * ((double)t - logp);
    else if (!(p == 0.0)) l = p * (logp - (double)t);
  }
  double sl = l, sp = have ? p : 0.0;
  block_sum2(b, sl, sp);
  // The sums over g_k in closed form: g_k - G p_k and G themselves would cancel where P is small. For the tokens outside
  // S the backward multiplies by G p_j; G may be about Q/P and p_j no more than P, each of them past fp32 where P is
  // small, so what it gets is relative to the largest logit outside S: p_j = 2^((z_j - m_tail) c) f_tail / s, and
  // G f_tail / s is about Q / s_tail.
  double g, gs;  // of this entry, and G f_tail / s
  if (!reverse) {
    if (with_tail) sl += tq * (ltq - lt);
    const double mass = sq + tq;
    g = p * mass - q;
    gs = (with_tail ? tq / s_tail : 0.0) - mass * f_tail / s;
  } else {
    if (with_tail) sl += tp * (lt - ltq);
    const double off = with_tail ? sl : sl + sp - 1.0;
    g = p == 0.0 ? 0.0 : p * (logp - (double)t - off);
    gs = (with_tail ? off - (lt - ltq) : sl + sp) * f_tail / s;
  }
  if (tid < k) out.entry[row * k + tid] = have ? (float)(g / (double)tau) : 0.f;
  if (tid == 0) {
    out.loss[row] = (float)sl;
    out.ref[row] = m_tail == -INFINITY ? 0.f : m_tail;
    out.gs[row] = s_tail == 0.0 && s > 0.0 ? 0.f : (float)(gs / (double)tau);  // 0: no token outside S
  }
}

// Entry k of the row: its token, or -1 where there is none (an id outside [0, V), a log-prob of -inf, or an id that
// an earlier entry has).
__device__ int entry_slot(int* ids_s, const int64_t* ids, const float* lp, long long row, int k, int v, float& t) {
  const int tid = threadIdx.x;
  int slot = -1;
  t = 0.f;
  if (tid < k) {
    const int64_t id = ids[row * k + tid];
    t = lp[row * k + tid];
    if (id >= v || id < -1) TS_BOUND_RECORD(kSiteTeacherId, id);
    if (id >= 0 && id < v && !(t == -INFINITY)) slot = (int)id;
    ids_s[tid] = slot;
  }
  __syncthreads();
  if (slot >= 0) {
    for (int j = 0; j < tid; ++j) {
      if (ids_s[j] == slot) {
        slot = -1;
        break;
      }
    }
  }
  __syncthreads();
  if (tid < k) ids_s[tid] = slot;
  return slot;
}

struct RowShared {
  Block2 b;
  float red[kWarps];
  float pm;
  double ps;
  int ids[kMaxTop];
};

template <typename T>
__global__ void __launch_bounds__(kThreads) distill_rows_fwd_kernel(const T* __restrict__ logits, long long stride,
                                                                    int v, const int64_t* __restrict__ ids,
                                                                    const float* __restrict__ lp, int k, float tau,
                                                                    bool reverse, bool tail, DistillOut out,
                                                                    int words) {
  constexpr int VEC = Slice<T>::kVec;
  __shared__ RowShared sh;
  extern __shared__ __align__(16) uint4 room[];  // the threads' rings, then
  uint32_t* bitmap = reinterpret_cast<uint32_t*>(room + kRing * kThreads);
  // ... a bit for each token: id - lo - head + VEC, so that a vector's bits share a byte
  cg::cluster_group cl = cg::this_cluster();
  const int parts = (int)cl.num_blocks(), part = (int)cl.block_rank();
  const long long row = blockIdx.x / parts;
  const int tid = threadIdx.x;
  const float c = kLog2e / tau;
  const T* lrow = logits + row * stride;
  for (int i = tid; i < words; i += kThreads) bitmap[i] = 0;
  float t;
  const int slot = entry_slot(sh.ids, ids, lp, row, k, v, t);
  if (part == 0 && tid < k) out.slots[row * k + tid] = slot;
  if (!__syncthreads_or(slot >= 0)) {  // the same in every part: a row without entries has no loss
    if (part == 0) {
      if (tid < k) out.entry[row * k + tid] = 0.f;
      if (tid == 0) out.loss[row] = out.ref[row] = out.gs[row] = 0.f;
    }
    return;
  }
  Slice<T> sl(lrow, v, part, parts);
  Steps<T, kThreads> steps(sl, room);
  const float zk = part == 0 && slot >= 0 ? to_f(lrow[slot]) : 0.f;
  if (slot >= sl.lo && slot < sl.lo + sl.n) {
    const int bit = slot - sl.lo - sl.head + VEC;
    atomicOr(&bitmap[bit >> 5], 1u << (bit & 31));
  }
  __syncthreads();
  float m = -INFINITY, s = 0.f;
  if (tid < sl.head + sl.tail) {
    const int i = tid < sl.head ? tid : sl.nvec * VEC + tid;
    const int bit = i - sl.head + VEC;
    if (!((bitmap[bit >> 5] >> (bit & 31)) & 1)) {
      const float z = to_f(sl.p[i]);
      stat_raise(m, s, fmaxf(z, -INFINITY), c);
      s += sum_exp<1>(&z, m, c);
    }
  }
  const uint8_t* bytes = reinterpret_cast<const uint8_t*>(bitmap);
  for (int step = 0; step < steps.count; ++step) {
    constexpr int Q = Steps<T, kThreads>::kVecs;
    float z[Q][VEC];
    steps.read(step, z);
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int i = (step * Q + q) * kThreads + tid;  // (past the end: no bits, and -inf)
      const uint32_t in = i >= sl.nvec ? 0u
                          : VEC == 8   ? (uint32_t)bytes[i + 1]
                                       : (bytes[(i + 1) >> 1] >> (((i + 1) & 1) * 4)) & 15u;
      if (in) {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if ((in >> e) & 1) z[q][e] = -INFINITY;
      }
    }
    stat_raise(m, s, vec_max<16>(&z[0][0]), c);
    s += sum_exp<16>(&z[0][0], m, c);
  }
  copy_wait<0>();
  const float top = block_max(sh.red, m);
  double total = rescaled(m, s, top, c), none = 0.0;
  block_sum2(sh.b, total, none);
  m = top;
  if (parts > 1) {
    if (tid == 0) {
      sh.pm = m;
      sh.ps = total;
    }
    cl.sync();
    if (part == 0) {
      for (int r = 1; r < parts; ++r) m = fmaxf(m, cl.map_shared_rank(&sh, r)->pm);
      total = 0.0;
      for (int r = 0; r < parts; ++r) {
        RowShared* o = cl.map_shared_rank(&sh, r);
        total += o->pm == -INFINITY || o->pm == m ? o->ps : o->ps * exp2(((double)o->pm - (double)m) * c);
      }
    }
    cl.sync();  // no part leaves before its sums are read
    if (part != 0) return;
  }
  finish_row(sh.b, sh.red, row, k, zk, t, slot >= 0, m, total, c, tau, reverse, tail, out);
}

// d[n, j] = -g gs 2^((z - ref)·c) (past fp32, perhaps, at the entries of S), and then g · entry at these; rows without a
// gradient are zeros and are not read. TWO: `out` gets d rounded to bf16 and `lo` what the rounding leaves, rounded to
// bf16, which together hold 16 bits of it.
template <typename T, typename O, bool TWO>
__global__ void __launch_bounds__(kThreads) distill_rows_bwd_kernel(const T* __restrict__ logits, long long stride,
                                                                    int v, const int* __restrict__ slots,
                                                                    const float* __restrict__ ref,
                                                                    const float* __restrict__ gs,
                                                                    const float* __restrict__ entry,
                                                                    const float* __restrict__ grad, int k, float tau,
                                                                    int parts, O* __restrict__ out, O* __restrict__ lo,
                                                                    long long ostride) {
  constexpr int VEC = Slice<T>::kVec;
  const long long row = blockIdx.x / parts;
  const int part = blockIdx.x % parts;
  const int tid = threadIdx.x;
  const float c = kLog2e / tau;
  const float g = grad[row];
  const float coef = g == 0.f ? 0.f : -g * gs[row];
  const float m = ref[row];
  Slice<T> sl(logits + row * stride, v, part, parts);
  O* o = out + row * ostride + sl.lo;
  O* o2 = TWO ? lo + row * ostride + sl.lo : nullptr;
  auto d = [&](float z) { return coef * ex2((z - m) * c); };
  auto put = [&](int i, float x) {
    o[i] = from_f<O>(x);
    if constexpr (TWO) o2[i] = from_f<O>(x - to_f(from_f<O>(x)));
  };
  if (tid < sl.head + sl.tail) {
    const int i = tid < sl.head ? tid : sl.nvec * VEC + tid;
    put(i, coef == 0.f ? 0.f : d(to_f(sl.p[i])));
  }
  const T* body = sl.body();
  constexpr int OB = VEC * sizeof(O);  // output bytes of a vector: 8, 16 or 32
  const uintptr_t at = reinterpret_cast<uintptr_t>(o + sl.head) | (TWO ? reinterpret_cast<uintptr_t>(o2 + sl.head) : 0);
  const bool wide = at % (OB < 16 ? OB : 16) == 0;
  auto put_vec = [&](O* w, const float* x) {
    union {
      O e[VEC];
      uint4 q[OB >= 16 ? OB / 16 : 1];
      uint2 h;
    } u;
#pragma unroll
    for (int e = 0; e < VEC; ++e) u.e[e] = from_f<O>(x[e]);
    if constexpr (OB == 8) {
      *reinterpret_cast<uint2*>(w) = u.h;
    } else {
#pragma unroll
      for (int q = 0; q < OB / 16; ++q) reinterpret_cast<uint4*>(w)[q] = u.q[q];
    }
  };
  constexpr int U = 16 / VEC;
  for (int i0 = tid; i0 < sl.nvec; i0 += U * kThreads) {
    uint4 raw[U];
#pragma unroll
    for (int j = 0; j < U; ++j)
      if (coef != 0.f && i0 + j * kThreads < sl.nvec) raw[j] = load_stream(body + (long long)(i0 + j * kThreads) * VEC);
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int i = i0 + j * kThreads;
      if (i >= sl.nvec) break;
      float z[VEC];
      if (coef == 0.f) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) z[e] = 0.f;
      } else {
        unpack<T>(raw[j], z);
#pragma unroll
        for (int e = 0; e < VEC; ++e) z[e] = d(z[e]);
      }
      const int w = sl.head + i * VEC;
      if (wide) {
        put_vec(o + w, z);
        if constexpr (TWO) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) z[e] -= to_f(from_f<O>(z[e]));
          put_vec(o2 + w, z);
        }
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) put(w + e, z[e]);
      }
    }
  }
  __syncthreads();
  if (tid < k) {
    const int slot = slots[row * k + tid];
    if (slot >= sl.lo && slot < sl.lo + sl.n) put(slot - sl.lo, g == 0.f ? 0.f : g * entry[row * k + tid]);
  }
}

// ---- the head's forward: its epilogue wants the entries in order, and leaves sums over pieces of the vocabulary
__global__ void __launch_bounds__(kThreads) sort_entries_kernel(const int64_t* __restrict__ ids,
                                                                const float* __restrict__ lp, int k, int v,
                                                                int* __restrict__ ids_out, float* __restrict__ lp_out) {
  __shared__ int slots[kMaxTop];
  const long long row = blockIdx.x;
  const int tid = threadIdx.x;
  float t;
  const int slot = entry_slot(slots, ids, lp, row, k, v, t);
  __syncthreads();
  if (tid >= k) return;
  int at = 0;
  for (int j = 0; j < k; ++j) {
    const int o = slots[j];
    at += slot >= 0 ? (o >= 0 && o < slot) : (o >= 0 || j < tid);
  }
  ids_out[row * k + at] = slot >= 0 ? slot : 0x7fffffff;
  lp_out[row * k + at] = t;
}

__global__ void __launch_bounds__(kThreads) head_finish_kernel(HeadStats st, const float* __restrict__ lp, float tau,
                                                               bool reverse, bool tail, DistillOut out) {
  __shared__ Block2 b;
  __shared__ float red[kWarps];
  const long long row = blockIdx.x;
  const int tid = threadIdx.x;
  const int id = tid < st.k ? st.ids[row * st.k + tid] : 0x7fffffff;
  const bool have = id != 0x7fffffff;
  if (tid < st.k) out.slots[row * st.k + tid] = have ? id : -1;
  if (!__syncthreads_or(have)) {  // a row without entries has no loss
    if (tid < st.k) out.entry[row * st.k + tid] = 0.f;
    if (tid == 0) out.loss[row] = out.ref[row] = out.gs[row] = 0.f;
    return;
  }
  const float* pm = st.pm + row * st.parts;
  const float* ps = st.ps + row * st.parts;
  float m = -INFINITY;
  for (int i = tid; i < st.parts; i += kThreads) m = fmaxf(m, pm[i]);
  m = block_max(red, m);
  double total = 0.0, none = 0.0;
  for (int i = tid; i < st.parts; i += kThreads) total += rescaled(pm[i], ps[i], m, st.c);
  block_sum2(b, total, none);
  const float z = have ? st.zk[row * st.k + tid] : 0.f;
  const float t = have ? lp[row * st.k + tid] : 0.f;
  finish_row(b, red, row, st.k, z, t, have, m, total, st.c, tau, reverse, tail, out);
}

// Parts of a row, in doublings up to eight while they are at most `most` CTAs an SM in all and a part has `least`
// logits. The forward's parts are a cluster that joins its sums (in us, with 1 / 2 / 4 / 8 parts, V = 151,936: 64 bf16
// rows 25 / 19 / 17 / 21, 1000 79 / 92 / 123 / 194); the backward's know nothing of each other, and shorter ones even
// out the last round (1000 bf16 rows 132 / 117 / 107 / 107).
int row_parts(int64_t rows, int v, int sms, int most, int least) {
  int parts = 1;
  while (parts < kMaxParts && 2 * rows * parts <= (int64_t)most * sms && v / (2 * parts) >= least) parts *= 2;
  return parts;
}

template <typename T>
cudaError_t fwd_of(const VocabLaunch& l, const VocabRows& x, const DistillArgs& a, const DistillOut& out) {
  int parts = row_parts(x.n, x.v, l.sms, 3, 32768);
  while (parts < kMaxParts && x.v / parts > 1000000) parts *= 2;  // the bitmap has to fit
  const int len = ((x.v + parts - 1) / parts + 63) / 64 * 64;
  const int words = (len + 16 + 31) / 32 + 1;
  const int bytes = kRing * kThreads * 16 + words * 4;
  const cudaError_t e = l.set_smem((const void*)distill_rows_fwd_kernel<T>, bytes);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(x.n * parts));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = l.stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = parts;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, distill_rows_fwd_kernel<T>, (const T*)x.logits, x.stride, x.v, a.ids, a.lp, a.k, a.tau,
                            a.reverse, a.tail, out, words);
}

template <typename T, typename O, bool TWO = false>
cudaError_t bwd_of(const VocabLaunch& l, const VocabRows& x, const DistillArgs& a, const DistillOut& f,
                   const float* grad, void* out, void* lo, long long ostride) {
  const int parts = std::max(row_parts(x.n, x.v, l.sms, 1 << 20, 16384), row_parts(x.n, x.v, l.sms, 6, 4096));
  distill_rows_bwd_kernel<T, O, TWO><<<(unsigned)(x.n * parts), kThreads, 0, l.stream>>>(
      (const T*)x.logits, x.stride, x.v, f.slots, f.ref, f.gs, f.entry, grad, a.k, a.tau, parts, (O*)out, (O*)lo, ostride);
  return cudaGetLastError();
}

}  // namespace

cudaError_t distill_rows_forward(const VocabLaunch& l, const VocabRows& x, const DistillArgs& a, const DistillOut& out) {
  switch (x.type) {
    case kRowsF32: return fwd_of<float>(l, x, a, out);
    case kRowsBf16: return fwd_of<__nv_bfloat16>(l, x, a, out);
    default: return fwd_of<__half>(l, x, a, out);
  }
}

cudaError_t distill_rows_backward(const VocabLaunch& l, const VocabRows& x, const DistillArgs& a, const DistillOut& f,
                                  const float* grad, RowType otype, void* out, void* lo, long long ostride) {
  if (lo != nullptr) {
    if (x.type != kRowsF32 || otype != kRowsBf16) return cudaErrorInvalidValue;
    return bwd_of<float, __nv_bfloat16, true>(l, x, a, f, grad, out, lo, ostride);
  }
  if (x.type == kRowsF32) {
    if (otype == kRowsF32) return bwd_of<float, float>(l, x, a, f, grad, out, lo, ostride);
    if (otype == kRowsBf16) return bwd_of<float, __nv_bfloat16>(l, x, a, f, grad, out, lo, ostride);
    return bwd_of<float, __half>(l, x, a, f, grad, out, lo, ostride);
  }
  if (otype != x.type) return cudaErrorInvalidValue;
  if (x.type == kRowsBf16) return bwd_of<__nv_bfloat16, __nv_bfloat16>(l, x, a, f, grad, out, lo, ostride);
  return bwd_of<__half, __half>(l, x, a, f, grad, out, lo, ostride);
}

cudaError_t distill_sort_entries(const VocabLaunch& l, const DistillArgs& a, int64_t n, int v, int* ids, float* lp) {
  sort_entries_kernel<<<(unsigned)n, kThreads, 0, l.stream>>>(a.ids, a.lp, a.k, v, ids, lp);
  return cudaGetLastError();
}

cudaError_t distill_head_finish(const VocabLaunch& l, const HeadStats& st, const float* lp, int64_t n, float tau,
                                bool reverse, bool tail, const DistillOut& out) {
  head_finish_kernel<<<(unsigned)n, kThreads, 0, l.stream>>>(st, lp, tau, reverse, tail, out);
  return cudaGetLastError();
}

cudaError_t distill_bounds(unsigned long long* word, bool reset) {
  cudaError_t e = cudaMemcpyFromSymbol(word, g_bounds_word, sizeof(*word));
  if (e == cudaSuccess && reset && *word != 0) {
    const unsigned long long zero = 0;
    e = cudaMemcpyToSymbol(g_bounds_word, &zero, sizeof(zero));
  }
  return e;
}

}  // namespace ts

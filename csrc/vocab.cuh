// Pieces shared by the kernels that walk rows of a vocabulary (csrc/vocab_select.cu, csrc/distill.cu).
//
// A row of V logits (fp32, bf16 or fp16; any row stride, any alignment of the type) is cut into `parts` slices, one
// per CTA of a cluster; a slice is an unaligned head, a body of 16-byte vectors and a tail. Log-sum-exp statistics
// are kept online as (m, s): the largest logit and s = sum of 2^((z - m)·c), c = log2(e)/temperature.
#pragma once

#include "common.cuh"

#include <cooperative_groups.h>

namespace ts {
namespace vocab {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

TS_DEVICE float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 2^((z - m)·c) for z <= m; an m of -inf (nothing but -inf so far) stands for 0
TS_DEVICE float rel_exp(float z, float m, float c) { return ex2((z - (m == -INFINITY ? 0.f : m)) * c); }

// |m c| up to which an exponent is one multiply-add, z·c - r with r = m·c rounded, and the sum is multiplied by
// 1 - ln2 (m c - r) afterwards: r is off by 2^-11 at most there, so what the first order leaves out is 6e-8. Above, as
// for masks of finite values (a thread may have seen nothing else yet), for logits with a large offset and for cold
// rows, the difference is taken first.
constexpr float kFusedMost = 16384.f;

// Sum of rel_exp over N values. In z·c - r the product is exact inside the multiply-add, so what is rounded is r, the
// same for all values, and the difference.
template <int N>
TS_DEVICE float sum_exp(const float* z, float m, float c) {
  float s0 = 0.f, s1 = 0.f;
  const float r = m * c;
  if (fabsf(r) <= kFusedMost) {
#pragma unroll
    for (int e = 0; e + 1 < N; e += 2) {
      s0 += ex2(fmaf(z[e], c, -r));
      s1 += ex2(fmaf(z[e + 1], c, -r));
    }
    if (N & 1) s0 += ex2(fmaf(z[N - 1], c, -r));
    s0 += s1;
    return fmaf(s0, -kLn2 * fmaf(m, c, -r), s0);
  }
#pragma unroll
  for (int e = 0; e < N; ++e) s0 += rel_exp(z[e], m, c);
  return s0;
}

// (m, s): raise the reference to `to`, or merge another pair. An empty side has m = -inf and s = 0 (or NaN: it stays).
TS_DEVICE void stat_raise(float& m, float& s, float to, float c) {
  if (to > m) {
    if (m != -INFINITY) s *= rel_exp(m, to, c);
    m = to;
  }
}
TS_DEVICE void stat_merge(float& m, float& s, float m2, float s2, float c) {
  const float mx = fmaxf(m, m2);
  s = s * (m == -INFINITY ? 1.f : rel_exp(m, mx, c)) + s2 * (m2 == -INFINITY ? 1.f : rel_exp(m2, mx, c));
  m = mx;
}

template <typename T>
struct Slice {
  static constexpr int kVec = 16 / sizeof(T);
  const T* p;  // first element
  int lo;      // its token id
  int n, head, nvec, tail;

  TS_DEVICE Slice(const T* row, int v, int part, int parts) {
    const int len = ((v + parts - 1) / parts + 63) / 64 * 64;
    lo = (int)min((long long)v, (long long)part * len);
    n = min(len, v - lo);
    p = row + lo;
    const int off = (int)((reinterpret_cast<uintptr_t>(p) & 15) / sizeof(T));
    head = min(n, off ? kVec - off : 0);
    nvec = (n - head) / kVec;
    tail = n - head - nvec * kVec;
  }
  TS_DEVICE const T* body() const { return p + head; }
};

TS_DEVICE uint4 load_stream(const void* p) {
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}

template <typename T>
TS_DEVICE void unpack(const uint4& raw, float* v) {
  Vec<T> x;
  x.raw = raw;
#pragma unroll
  for (int e = 0; e < Vec<T>::N; ++e) v[e] = to_f(x.e[e]);
}

// Order of the logits as unsigned integers: larger is greater, equal values (also -0 and +0) are equal, NaN is least.
TS_DEVICE uint32_t order_key(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);
  if (v != v) return 0u;
  return u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
TS_DEVICE float key_value(uint32_t k) { return __uint_as_float((k >> 31) ? k ^ 0x80000000u : ~k); }
// Rank of (logit, token) in one word: greater logits first, then lower tokens.
TS_DEVICE uint64_t rank_key(float v, int id) { return ((uint64_t)order_key(v) << 32) | (uint32_t)~(uint32_t)id; }
TS_DEVICE int rank_id(uint64_t k) { return (int)~(uint32_t)k; }
TS_DEVICE float rank_value(uint64_t k) { return key_value((uint32_t)(k >> 32)); }

TS_DEVICE void copy16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src)
               : "memory");
}
TS_DEVICE void copy4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src)
               : "memory");
}
TS_DEVICE void copy_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N> TS_DEVICE void copy_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory"); }

// Largest of a vector's values; NaN is left out (-inf if there is nothing else).
template <int N>
TS_DEVICE float vec_max(const float* z) {
  float x = -INFINITY;
#pragma unroll
  for (int e = 0; e < N; ++e) x = fmaxf(x, z[e]);
  return x;
}

constexpr int kRing = 8;  // vectors of a thread in its ring

// This thread's vectors of a slice through its private ring, a step of 16 elements (four vectors, or two of 16-bit
// types) at a time: vectors t·kVecs + q, q < kVecs, of every thread. Places past the end read as -inf.
template <typename T, int NT>
struct Steps {
  static constexpr int VEC = Slice<T>::kVec;
  static constexpr int kVecs = 16 / VEC;
  static constexpr int kAhead = kRing / kVecs;  // steps in flight
  const T* src;
  uint4* ring;
  int nvec, count;

  __device__ Steps(const Slice<T>& sl, uint4* rings)
      : src(sl.body() + threadIdx.x * VEC), ring(rings + threadIdx.x), nvec(sl.nvec),
        count((sl.nvec + kVecs * NT - 1) / (kVecs * NT)) {
#pragma unroll
    for (int t = 0; t < kAhead; ++t) fetch(t);
  }
  TS_DEVICE bool has(int t, int q) const { return (t * kVecs + q) * NT + (int)threadIdx.x < nvec; }
  TS_DEVICE void fetch(int t) {
    uint4* to = ring + (t % kAhead) * (kVecs * NT);
    const T* from = src + (long long)t * (kVecs * NT * VEC);
    if ((t + 1) * kVecs * NT <= nvec) {
#pragma unroll
      for (int q = 0; q < kVecs; ++q) copy16(to + q * NT, from + q * NT * VEC);
    } else {
#pragma unroll
      for (int q = 0; q < kVecs; ++q)
        if (has(t, q)) copy16(to + q * NT, from + q * NT * VEC);
    }
    copy_commit();
  }
  // step t (in order), and the fetch of the one that takes its place
  TS_DEVICE void read(int t, float (&z)[kVecs][VEC]) {
    copy_wait<kAhead - 1>();
    const uint4* at = ring + (t % kAhead) * (kVecs * NT);
#pragma unroll
    for (int q = 0; q < kVecs; ++q) unpack<T>(at[q * NT], z[q]);
    if ((t + 1) * kVecs * NT > nvec) {
#pragma unroll
      for (int q = 0; q < kVecs; ++q) {
        if (!has(t, q)) {
#pragma unroll
          for (int e = 0; e < VEC; ++e) z[q][e] = -INFINITY;
        }
      }
    }
    fetch(t + kAhead);
  }
};

struct Stat {
  float m = -INFINITY, s = 0.f;
};

}  // namespace vocab
}  // namespace ts

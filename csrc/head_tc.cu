// tcgen05 products of the distillation head: logits = h Wᵀ with the loss's statistics in the epilogue, dH = d W over
// slices of the vocabulary, dW = dᵀ h.
//
// CTA pairs (cta_group::2): a cluster of two CTAs computes a 256 x 256 tile, each staging 128 rows of A and 128 of B
// per 64-deep K block through a six-stage TMA ring. Where too many of such tiles' rows would be past the last one,
// single CTAs compute 128 x 256 tiles, each staging 128 rows of A and 256 of B through four stages. d may come as two
// bf16 halves, d = hi + lo (16 bits): a stage then holds both (four and three stages), and B is read once for the two
// products that add into one accumulator.
//   warp 0  TMA producer, warp 1 MMA issuer (one lane each; the even CTA issues for the pair), warps 2-3 idle
//   warps 4-11  epilogue: two warps for each 32-row slab of tensor memory, half of the tile's columns each
// The contraction is accumulated in chunks: tensor memory holds one chunk's sum (two buffers, used in turn), and the
// epilogue warps add the chunks in registers with rounded fp32 additions, because the tensor core's own accumulation
// truncates. At D = 2048 the logits are 2.1e-6 (of their norm) from 64 bits in one chunk, 4.7e-7 in chunks of 512 and
// 2.4e-7 in chunks of 256 (an fp32 library product 3.9e-7), and the loss 2e-5, 2e-6 and 1e-6. A chunk's reading costs
// the MMAs about 1000 clocks, so 2048 x 151,936 logits take 0.98 ms in chunks of 512 and 1.17 in chunks of 256. The
// logits go by 256, the gradients, which are rounded to bf16, by 2048.
//
// Measured at 2048 rows x 2048 x 151,936: logits with statistics 1.17 ms (1088 TFLOP/s), kept in fp32 as well 1.24; with
// d in halves dH 1.57 ms and dW 1.56 (1630 TFLOP/s of the four products), which the tensor cores bound; with d rounded
// 0.94 and 0.93 (1360), bound by 14 TB/s from L2 (62 of 64 bytes a clock and SM at full rate). The library's bf16 products
// take 0.87 each. What the halves are for: rounded, a row's dlogits do not sum to 0 any more, and dH is 1.1e-2 off where
// the entries' weight rows are nearly the same, and 1.9e-3 to 3.3e-3 on random ones; in halves 1.7e-3, which is its own
// rounding. At 97 rows x 2560 the weight's 778 MB bound all three (0.17, 0.17 and 0.31 ms, the last a write: clearing
// that much memory takes 0.20; d rounded 0.15 and 0.28).
//
// Every wait is bounded (tc::mbar_wait); tensor memory is always freed. Loads have no multicast.
#include "common.cuh"
#include "tc.cuh"
#include "vocab.cuh"
#include "vocab.h"

#include <algorithm>

namespace ts {
namespace {

using namespace vocab;

constexpr int kBM = 128, kBN = 256, kBK = 64;
constexpr int kChunkLogits = 4, kChunkGrad = 32;  // K blocks of a chunk
constexpr uint32_t kABytes = kBM * kBK * 2;  // 16 KB
template <bool PAIR, bool TWO>  // TWO: a stage holds both halves of A
struct Ring {
  static constexpr int kStages = (PAIR ? 6 : 4) - (TWO ? (PAIR ? 2 : 1) : 0);
  static constexpr int kBRows = PAIR ? 128 : 256;  // of B in each CTA
  static constexpr uint32_t kAll = (TWO ? 2 : 1) * kABytes;
  static constexpr uint32_t kStageBytes = kAll + kBRows * kBK * 2;
  static_assert(kStages * kStageBytes == 6 * 32768, "the rings take the same room");
};
constexpr int kEpiWarps = 8;
constexpr int kThreads = 128 + 32 * kEpiWarps;
// Registers of a thread after the split of the block's (384 threads x 168 at launch): the first warpgroup gives, the
// epilogue's two take. 128 x 56 + 256 x 224 is the launch's 64,512.
constexpr int kRegsLaunch = 168, kRegsGive = 56, kRegsTake = 224;
static_assert(128 * kRegsGive + 32 * kEpiWarps * kRegsTake <= kThreads * kRegsLaunch, "no more registers than launched");
constexpr uint32_t kEpiOff = 6 * 32768;  // 4 KB of staging for each epilogue warp
constexpr uint32_t kBarOff = kEpiOff + kEpiWarps * 4096;
constexpr uint32_t kSmem = kBarOff + 256 + 1024;
static_assert(kSmem <= 232448, "shared memory");

enum Out { kNone = 0, kF32 = 1, kBf16 = 2 };

struct Bars {
  uint64_t full[6], empty[6], acc_full[2], acc_empty[2];
  uint32_t tmem_slot;
  int abort;
};

struct Shape {
  int m, n, k;      // C [m, n] = A [m, k] B [k, n]
  int tile;         // rows of a unit's tile: 256 (pairs) or 128
  int splits;       // slices of the contraction, one unit of work each
  int split_rows;   // rows of C between two slices' outputs
};

struct Work {
  int mb, nb, kb0, kb1, row_off;
};

// Unit u: slices outermost, so that what runs at one time reads the same part of both operands; then groups of eight
// row blocks, which share B's columns.
TS_DEVICE Work work_of(const Shape& s, int u) {
  const int mt = (s.m + s.tile - 1) / s.tile, nt = (s.n + kBN - 1) / kBN, kt = (s.k + kBK - 1) / kBK;
  const int z = u / (mt * nt), t = u % (mt * nt);
  const int group = t / (8 * nt), r = t % (8 * nt), first = group * 8, gm = min(8, mt - first);
  Work w;
  w.mb = first + r % gm;
  w.nb = r / gm;
  const int per = (kt + s.splits - 1) / s.splits;
  w.kb0 = min(kt, z * per);
  w.kb1 = min(kt, w.kb0 + per);
  w.row_off = z * s.split_rows;
  return w;
}

TS_DEVICE void store_tile(const CUtensorMap* map, uint32_t src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];\n" ::"l"(map), "r"(src),
               "r"(x), "r"(y)
               : "memory");
  asm volatile("cp.async.bulk.commit_group;\n" ::: "memory");
}
TS_DEVICE void store_read_wait() { asm volatile("cp.async.bulk.wait_group.read 0;\n" ::: "memory"); }
TS_DEVICE void store_wait() { asm volatile("cp.async.bulk.wait_group 0;\n" ::: "memory"); }

TS_DEVICE uint32_t pack2(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

// This lane's values (row `lane`) of a chunk of 32 rows of 128 bytes (32 fp32 or 64 bf16) at (col, row0), through the
// warp's 4 KB of staging in the output map's 128-byte swizzle, which keeps the writes of 32 rows apart in the banks.
// bf16 chunks of 64-byte rows took the output of a short contraction (97 rows' dW) 0.24 ms.
template <int OUT>
TS_DEVICE void store_chunk(uint32_t buf, bool& busy, const CUtensorMap* map, const float* o, int col, int row0) {
  const int lane = threadIdx.x & 31;
  if (busy) {  // the store before has read the buffer
    if (lane == 0) store_read_wait();
    __syncwarp();
  }
  busy = true;
  const uint32_t rowb = buf + (uint32_t)lane * 128;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t at = rowb + (uint32_t)((j ^ (lane & 7)) << 4);
    if constexpr (OUT == kF32) {
      asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};\n" ::"r"(at), "f"(o[4 * j]), "f"(o[4 * j + 1]),
                   "f"(o[4 * j + 2]), "f"(o[4 * j + 3])
                   : "memory");
    } else {
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};\n" ::"r"(at), "r"(pack2(o[8 * j], o[8 * j + 1])),
                   "r"(pack2(o[8 * j + 2], o[8 * j + 3])), "r"(pack2(o[8 * j + 4], o[8 * j + 5])),
                   "r"(pack2(o[8 * j + 6], o[8 * j + 7]))
                   : "memory");
    }
  }
  tc::fence_async_smem();
  __syncwarp();
  if (lane == 0) store_tile(map, buf, col, row0);
}

// The search for a row's first entry at or after a column: the entries are sorted by token, and those that do not count
// are last with a token past any column. A step's load is begun well before its outcome is used.
struct EntrySearch {
  const int* ids;
  int col, lo, hi, seen;
  TS_DEVICE void look() {
    if (lo < hi) seen = __ldg(ids + ((lo + hi) >> 1));
  }
  TS_DEVICE void narrow() {
    if (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (seen < col) lo = mid + 1;
      else hi = mid;
    }
  }
};

template <bool A_MN, bool B_MN, int OUT, bool STATS, int kChunk, bool PAIR, bool TWO>
__global__ void __launch_bounds__(kThreads, 1)
    head_gemm_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_a2,
                     const __grid_constant__ CUtensorMap tm_b, const __grid_constant__ CUtensorMap tm_c, Shape shape,
                     HeadStats st, int* __restrict__ err) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  Bars* bars = reinterpret_cast<Bars*>(smem + kBarOff);
  const uint32_t sbase = tc::smem_addr(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kStages = Ring<PAIR, TWO>::kStages;
  constexpr uint32_t kStageBytes = Ring<PAIR, TWO>::kStageBytes, kAll = Ring<PAIR, TWO>::kAll;
  constexpr int kTileM = PAIR ? 2 * kBM : kBM;
  const uint32_t rank = PAIR ? tc::cluster_rank() : 0;
  const int units = ((shape.m + kTileM - 1) / kTileM) * ((shape.n + kBN - 1) / kBN) * shape.splits;
  const int cid = PAIR ? blockIdx.x >> 1 : blockIdx.x, ncl = PAIR ? gridDim.x >> 1 : gridDim.x;
  volatile int* abort = &bars->abort;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      tc::mbar_init(&bars->full[s], 1);
      tc::mbar_init(&bars->empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      tc::mbar_init(&bars->acc_full[b], 1);
      tc::mbar_init(&bars->acc_empty[b], (PAIR ? 2 : 1) * kEpiWarps);  // the epilogue warps (of both CTAs)
    }
    bars->abort = 0;
    tc::fence_barrier_init();
  }
  if (warp == 1) {
    if constexpr (PAIR) tc::tmem_alloc_pair(&bars->tmem_slot, 512);
    else tc::tmem_alloc(&bars->tmem_slot, 512);
  }
  tc::tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) tc::cluster_sync();  // both CTAs' barriers exist before any remote arrive or byte count
  tc::tc_fence_after();
  const uint32_t tmem = bars->tmem_slot;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kRegsGive));
    if (warp == 0) {
      if (lane == 0) {
        tc::prefetch_tmap(&tm_a);
        if constexpr (TWO) tc::prefetch_tmap(&tm_a2);
        tc::prefetch_tmap(&tm_b);
        int it = 0;
        for (int u = cid; u < units; u += ncl) {
          const Work w = work_of(shape, u);
          const int arow = w.mb * kTileM + (int)rank * kBM, bcol = w.nb * kBN + (int)rank * (kBN / 2);
          for (int kb = w.kb0; kb < w.kb1; ++kb, ++it) {
            const int s = it % kStages;
            if (it >= kStages && !tc::mbar_wait(&bars->empty[s], ((it - kStages) / kStages) & 1, abort, err, 301))
              goto producer_done;
            uint64_t* full = &bars->full[s];
            if (rank == 0) tc::mbar_expect_tx(full, (PAIR ? 2 : 1) * kStageBytes);
            const uint32_t full0 = PAIR ? tc::map_cluster(tc::smem_addr(full), 0) : 0;
            auto load = [&](uint8_t* to, const CUtensorMap* map, int x, int y) {
              if constexpr (PAIR) tc::tma_load_2d_pair(to, map, x, y, full0);
              else tc::tma_load_2d(to, map, x, y, full);
            };
            uint8_t* a = smem + s * kStageBytes;
            uint8_t* b = a + kAll;
            const int kx = kb * kBK;
            auto load_a = [&](uint8_t* to, const CUtensorMap* map) {
              if constexpr (!A_MN) {
                load(to, map, kx, arow);  // box 64 (k) x 128 (m)
              } else {
#pragma unroll
                for (int j = 0; j < kBM / 64; ++j) load(to + j * 64 * 128, map, arow + j * 64, kx);  // [K][M]: 64 m x 64 k
              }
            };
            load_a(a, &tm_a);
            if constexpr (TWO) load_a(a + kABytes, &tm_a2);
            if constexpr (!B_MN) {
#pragma unroll
              for (int j = 0; j < Ring<PAIR, TWO>::kBRows / 128; ++j)
                load(b + j * 128 * 128, &tm_b, kx, bcol + j * 128);  // box 64 (k) x 128 (n)
            } else {
#pragma unroll
              for (int j = 0; j < Ring<PAIR, TWO>::kBRows / 64; ++j)
                load(b + j * 64 * 128, &tm_b, bcol + j * 64, kx);  // [K][N]: 64 n x 64 k
            }
          }
        }
      producer_done:;
      }
    } else if (warp == 1) {
      if (lane == 0 && rank == 0) {
        const uint32_t idesc = tc::idesc_bf16(kTileM, kBN, A_MN, B_MN);
        int it = 0, chunk = 0;
        bool ok = true;
        for (int u = cid; ok && u < units; u += ncl) {
          const Work w = work_of(shape, u);
          for (int kc = w.kb0; ok && kc < w.kb1; kc += kChunk, ++chunk) {
            const int buf = chunk & 1;
            if (chunk >= 2 && !tc::mbar_wait(&bars->acc_empty[buf], ((chunk - 2) >> 1) & 1, abort, err, 311)) {
              ok = false;
              break;
            }
            tc::tc_fence_after();
            const uint32_t acc = tmem + buf * kBN;
            const int kend = min(kc + kChunk, w.kb1);
            for (int kb = kc; kb < kend; ++kb, ++it) {
              const int s = it % kStages;
              if (!tc::mbar_wait(&bars->full[s], (it / kStages) & 1, abort, err, 312)) {
                ok = false;
                break;
              }
              tc::tc_fence_after();
              const uint32_t a = sbase + s * kStageBytes, b = a + kAll;
#pragma unroll
              for (int kk = 0; kk < kBK / 16; ++kk) {
                const uint64_t bd = B_MN ? tc::sdesc_sw128(b + kk * 16 * 128, 64 * 128, 1024)
                                         : tc::sdesc_sw128(b + kk * 32, 16, 1024);
                auto product = [&](uint32_t from, bool add) {
                  const uint64_t ad = A_MN ? tc::sdesc_sw128(from + kk * 16 * 128, 64 * 128, 1024)
                                           : tc::sdesc_sw128(from + kk * 32, 16, 1024);
                  if constexpr (PAIR) tc::mma_bf16_pair(acc, ad, bd, idesc, add);
                  else tc::mma_bf16(acc, ad, bd, idesc, add);
                };
                product(a, kb > kc || kk > 0);
                if constexpr (TWO) product(a + kABytes, true);
              }
              if constexpr (PAIR) tc::mma_commit_pair(&bars->empty[s]);
              else tc::mma_commit(&bars->empty[s]);
            }
            if (ok) {
              if constexpr (PAIR) tc::mma_commit_pair(&bars->acc_full[buf]);
              else tc::mma_commit(&bars->acc_full[buf]);
            }
          }
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(kRegsTake));
    const int sub = warp & 3;            // the 32-row slab of tensor memory that this warp can read
    const int ew = warp - 4, half = ew >> 2;  // and its half of the tile's columns
    const uint32_t lane_base = tmem + ((uint32_t)(sub * 32) << 16) + half * (kBN / 2);
    const uint32_t acc_empty0 = PAIR ? tc::map_cluster(tc::smem_addr(&bars->acc_empty[0]), 0) : 0;
    const uint32_t acc_empty1 = PAIR ? tc::map_cluster(tc::smem_addr(&bars->acc_empty[1]), 0) : 0;
    const uint32_t stage = sbase + kEpiOff + (uint32_t)ew * 4096;
    bool ok = true;
    int chunk = 0;
    bool busy = false;
    for (int u = cid; ok && u < units; u += ncl) {
      const Work w = work_of(shape, u);
      const int row0 = w.mb * kTileM + (int)rank * kBM + sub * 32, row = row0 + lane;
      const int col0 = w.nb * kBN + half * (kBN / 2);
      EntrySearch find{nullptr, col0, 0, 0, 0};
      if constexpr (STATS) {
        if (row < shape.m) {
          find.ids = st.ids + (long long)row * st.k;
          find.hi = st.k;
        }
      }
      float acc[kBN / 2];
#pragma unroll
      for (int x = 0; x < kBN / 2; ++x) acc[x] = 0.f;
#pragma unroll 1
      for (int kc = w.kb0; kc < w.kb1; kc += kChunk, ++chunk) {
        const int buf = chunk & 1;
        if constexpr (STATS) find.look();
        if (lane == 0) ok = tc::mbar_wait(&bars->acc_full[buf], (chunk >> 1) & 1, abort, err, 321);
        ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
        if (!ok) break;
        tc::tc_fence_after();
        if constexpr (STATS) {
          find.narrow();
          find.look();
        }
        const uint32_t from = lane_base + buf * kBN;
#pragma unroll
        for (int g = 0; g < 4; g += 2) {
          float va[32], vb[32];
          tc::tmem_ld32(from + g * 32, va);
          tc::tmem_ld32(from + g * 32 + 32, vb);
          tc::tmem_ld_wait();
#pragma unroll
          for (int x = 0; x < 32; ++x) {
            acc[g * 32 + x] += va[x];
            acc[g * 32 + 32 + x] += vb[x];
          }
        }
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if constexpr (PAIR) tc::mbar_arrive_cluster(buf ? acc_empty1 : acc_empty0);
          else tc::mbar_arrive(&bars->acc_empty[buf]);
        }
        if constexpr (STATS) find.narrow();
      }
      if (!ok) break;
      if (row0 >= shape.m) continue;  // the same in the whole warp
      float m = -INFINITY, s = 0.f;
      int at = 0, next = 0x7fffffff, after = 0x7fffffff;  // the row's next entry and the one behind it
      if constexpr (STATS) {
        while (find.lo < find.hi) {
          find.look();
          find.narrow();
        }
        at = find.lo;
        if (at < (find.ids ? st.k : 0)) next = __ldg(find.ids + at);
        if (at + 1 < (find.ids ? st.k : 0)) after = __ldg(find.ids + at + 1);
      }
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int col = col0 + g * 32;
        float* v = acc + g * 32;
        if (col < shape.n) {
          if constexpr (OUT == kF32) store_chunk<OUT>(stage, busy, &tm_c, v, col, w.row_off + row0);
          if constexpr (OUT == kBf16) {
            if (g % 2 == 0) store_chunk<OUT>(stage, busy, &tm_c, v, col, w.row_off + row0);
          }
          if constexpr (STATS) {
            // the entries' logits go to their places and out of the sums
            uint32_t hit = 0;
            while (next < col + 32) {
              const int x = next - col;
              hit |= 1u << x;
              float z = v[0];
#pragma unroll
              for (int q = 1; q < 32; ++q)
                if (q == x) z = v[q];
              st.zk[(long long)row * st.k + at] = z;
              ++at;
              next = after;
              after = at + 1 < st.k ? __ldg(find.ids + at + 1) : 0x7fffffff;
            }
            if (col + 32 > shape.n) hit |= 0xffffffffu << (shape.n - col);
            if (__any_sync(0xffffffffu, hit != 0)) {
#pragma unroll
              for (int q = 0; q < 32; ++q)
                if ((hit >> q) & 1) v[q] = -INFINITY;
            }
            stat_raise(m, s, [&] {
              float x = -INFINITY;
#pragma unroll
              for (int q = 0; q < 32; ++q) x = fmaxf(x, v[q]);
              return x;
            }(), st.c);
            s += sum_exp<32>(v, m, st.c);
          }
        }
      }
      if constexpr (STATS) {
        if (row < shape.m) {
          const long long o = (long long)row * st.parts + 2 * w.nb + half;
          st.pm[o] = m;
          st.ps[o] = s;
        }
      }
    }
    if (OUT != kNone && lane == 0) store_wait();  // staged stores are done before shared memory goes away
    __syncwarp();
  }
  tc::tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) tc::cluster_sync();  // no CTA leaves while its pair may still read its shared memory or arrive on it
  if (warp == 1) {
    tc::tc_fence_after();
    if constexpr (PAIR) tc::tmem_dealloc_pair(tmem, 512);
    else tc::tmem_dealloc(tmem, 512);
  }
}

// out bf16 [rows, cols] = the sum of the slices' fp32 products, in order
__global__ void __launch_bounds__(256) sum_slices_kernel(const float* __restrict__ x, long long slice, int splits,
                                                         __nv_bfloat16* __restrict__ out, long long n4) {
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n4; i += gridDim.x * 256ll) {
    float4 a = reinterpret_cast<const float4*>(x)[i];
    for (int z = 1; z < splits; ++z) {
      const float4 b = reinterpret_cast<const float4*>(x + z * slice)[i];
      a.x += b.x;
      a.y += b.y;
      a.z += b.z;
      a.w += b.w;
    }
    reinterpret_cast<uint2*>(out)[i] = make_uint2(pack2(a.x, a.y), pack2(a.z, a.w));
  }
}

template <bool PAIR>
void fill_config(cudaLaunchConfig_t& cfg, cudaLaunchAttribute& attr, int ctas, cudaStream_t stream) {
  cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = stream;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = PAIR ? 2 : 1;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
}

// Pairs of CTAs (or CTAs) that the device holds at one time: the persistent grid.
template <bool A_MN, bool B_MN, int OUT, bool STATS, int kChunk, bool PAIR, bool TWO>
cudaError_t resident(const VocabLaunch& l, int& held) {
  static int have[16] = {0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  int& n = have[dev & 15];
  if (n == 0) {
    const auto kernel = head_gemm_kernel<A_MN, B_MN, OUT, STATS, kChunk, PAIR, TWO>;
    e = l.set_smem((const void*)kernel, (int)kSmem);
    if (e != cudaSuccess) return e;
    if (PAIR) {
      cudaLaunchConfig_t cfg;
      cudaLaunchAttribute attr;
      fill_config<PAIR>(cfg, attr, 2 * l.sms, 0);
      int most = 0;
      e = cudaOccupancyMaxActiveClusters(&most, kernel, &cfg);
      if (e != cudaSuccess) return e;
      n = std::max(1, std::min(most, l.sms / 2));
    } else {
      n = l.sms;  // one CTA an SM
    }
  }
  held = n;
  return cudaSuccess;
}

template <bool A_MN, bool B_MN, int OUT, bool STATS, int kChunk, bool PAIR, bool TWO>
cudaError_t launch_as(const VocabLaunch& l, const CUtensorMap& a, const CUtensorMap& a2, const CUtensorMap& b,
                      const CUtensorMap& c, Shape shape, const HeadStats& st, int* err) {
  shape.tile = PAIR ? 2 * kBM : kBM;
  int held = 0;
  const cudaError_t e = resident<A_MN, B_MN, OUT, STATS, kChunk, PAIR, TWO>(l, held);
  if (e != cudaSuccess) return e;
  const int units = ((shape.m + shape.tile - 1) / shape.tile) * ((shape.n + kBN - 1) / kBN) * shape.splits;
  cudaLaunchConfig_t cfg;
  cudaLaunchAttribute attr;
  fill_config<PAIR>(cfg, attr, (PAIR ? 2 : 1) * std::min(units, held), l.stream);
  return cudaLaunchKernelEx(&cfg, head_gemm_kernel<A_MN, B_MN, OUT, STATS, kChunk, PAIR, TWO>, a, a2, b, c, shape, st,
                            err);
}

// Pairs or single CTAs: a pair's tile takes 7% less time a row (logits of 2048 rows 1.25 ms, of single CTAs 1.35) but
// rounds the rows up to 256 instead of 128 (97 rows 0.225 / 0.176 ms, 300 0.32 / 0.27, 600 0.47 / 0.43).
bool in_pairs(int rows) {
  const int pairs = (rows + 255) / 256 * 256, single = (rows + 127) / 128 * 128;
  return 100ll * single >= 93ll * pairs;
}

template <bool A_MN, bool B_MN, int OUT, bool STATS, int kChunk, bool TWO>
cudaError_t launch(const VocabLaunch& l, const CUtensorMap& a, const CUtensorMap& a2, const CUtensorMap& b,
                   const CUtensorMap& c, const Shape& shape, const HeadStats& st, int* err) {
  if (in_pairs(shape.m)) return launch_as<A_MN, B_MN, OUT, STATS, kChunk, true, TWO>(l, a, a2, b, c, shape, st, err);
  return launch_as<A_MN, B_MN, OUT, STATS, kChunk, false, TWO>(l, a, a2, b, c, shape, st, err);
}

}  // namespace

int head_parts(int v) { return 2 * ((v + kBN - 1) / kBN); }

// Slices of dH's contraction over the vocabulary: the fewest that fill the pairs' rounds to 95%, or the fullest.
int head_splits(const VocabLaunch& l, int rows, int d, int v) {
  const bool two = in_pairs(rows);
  int pairs = 0;
  const cudaError_t e = two ? resident<false, true, kF32, false, kChunkGrad, true, false>(l, pairs)
                            : resident<false, true, kF32, false, kChunkGrad, false, false>(l, pairs);
  if (e != cudaSuccess) return 1;
  const int tile = two ? 2 * kBM : kBM;
  const int tiles = ((rows + tile - 1) / tile) * ((d + kBN - 1) / kBN);
  const int kt = (v + kBK - 1) / kBK;
  int best = 1;
  double full = 0.0;
  for (int s = 1; s <= 32 && kt / s >= 32; ++s) {
    const int units = tiles * s, rounds = (units + pairs - 1) / pairs;
    const double f = (double)units / ((double)rounds * pairs);
    if (f > full + 1e-9) {
      full = f;
      best = s;
    }
    if (full >= 0.95) break;
  }
  return best;
}

cudaError_t head_logits(const VocabLaunch& l, const CUtensorMap& h, const CUtensorMap& w, const CUtensorMap* out,
                        int rows, int d, int v, const HeadStats& st, int* err) {
  const Shape s{rows, v, d, 0, 1, 0};
  if (out != nullptr) return launch<false, false, kF32, true, kChunkLogits, false>(l, h, h, w, *out, s, st, err);
  return launch<false, false, kNone, true, kChunkLogits, false>(l, h, h, w, h, s, st, err);
}

cudaError_t head_logits_again(const VocabLaunch& l, const CUtensorMap& h, const CUtensorMap& w, const CUtensorMap& out,
                              int rows, int d, int v, int* err) {
  return launch<false, false, kF32, false, kChunkLogits, false>(l, h, h, w, out, Shape{rows, v, d, 0, 1, 0}, HeadStats{},
                                                                err);
}

cudaError_t head_dh(const VocabLaunch& l, const CUtensorMap& dl, const CUtensorMap* lo, const CUtensorMap& w,
                    const CUtensorMap& out, int rows, int d, int v, int splits, int split_rows, const float* parts,
                    void* dh, int* err) {
  const Shape s{rows, d, v, 0, splits, split_rows};
  const HeadStats none{};
  if (splits == 1)
    return lo ? launch<false, true, kBf16, false, kChunkGrad, true>(l, dl, *lo, w, out, s, none, err)
              : launch<false, true, kBf16, false, kChunkGrad, false>(l, dl, dl, w, out, s, none, err);
  const cudaError_t e = lo ? launch<false, true, kF32, false, kChunkGrad, true>(l, dl, *lo, w, out, s, none, err)
                           : launch<false, true, kF32, false, kChunkGrad, false>(l, dl, dl, w, out, s, none, err);
  if (e != cudaSuccess) return e;
  const long long n4 = (long long)rows * d / 4;
  const int blocks = (int)std::min<long long>((n4 + 255) / 256, 8ll * l.sms);
  sum_slices_kernel<<<blocks, 256, 0, l.stream>>>(parts, (long long)split_rows * d, splits, (__nv_bfloat16*)dh, n4);
  return cudaGetLastError();
}

cudaError_t head_dw(const VocabLaunch& l, const CUtensorMap& dl, const CUtensorMap* lo, const CUtensorMap& h,
                    const CUtensorMap& out, int rows, int d, int v, int* err) {
  const Shape s{v, d, rows, 0, 1, 0};
  return lo ? launch_as<true, true, kBf16, false, kChunkGrad, true, true>(l, dl, *lo, h, out, s, HeadStats{}, err)
            : launch_as<true, true, kBf16, false, kChunkGrad, true, false>(l, dl, dl, h, out, s, HeadStats{}, err);
}

}  // namespace ts

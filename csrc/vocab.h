// Launchers of the vocabulary-row kernels (csrc/vocab_select.cu, csrc/distill.cu), for csrc/vocab_bind.cpp: plain
// pointers, so that the kernel sources compile without torch's headers. Each returns the launch's error.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace ts {

enum RowType { kRowsF32 = 0, kRowsBf16 = 1, kRowsF16 = 2 };

struct VocabLaunch {
  cudaStream_t stream;
  int sms;
  cudaError_t (*set_smem)(const void* kernel, int bytes);  // raises a kernel's dynamic shared memory limit
};

struct VocabRows {  // logits [n, v], rows contiguous, `stride` elements apart
  const void* logits;
  RowType type;
  int64_t n;
  int v;
  long long stride;
};

struct SampleArgs {  // each setting: per row, or (null) the scalar
  const float* temperature;
  const int64_t* top_k;
  const float* top_p;
  const float* min_p;
  float temperature_s, top_p_s, min_p_s;
  long long top_k_s;
};

struct DistillArgs {
  const int64_t* ids;  // [n, k] teacher tokens
  const float* lp;     // [n, k] their log-probs
  int k;
  float tau;
  bool reverse, tail;
};

struct DistillOut {
  float* loss;   // [n]
  int* slots;    // [n, k] the entries that count (token, or -1)
  float* ref;    // [n] the largest logit outside the entries: p_j is in proportion to 2^((z_j - ref) c), c = log2(e) / tau
  float* gs;     // [n] the row's gradient outside the entries is -gs 2^((z_j - ref) c)
  float* entry;  // [n, k] the gradient at the entries
};

struct HeadStats {      // what the logits' epilogue leaves per row
  const int* ids = nullptr;  // [rows, k] the entries' tokens in ascending order; 0x7fffffff: none
  int k = 0;
  float c = 0.f;        // log2(e) / tau
  float* pm = nullptr;  // [rows, parts] of the tokens that are no entry: the largest logit of each 128 columns ...
  float* ps = nullptr;  // ... and their sum of 2^((z - m) c)
  float* zk = nullptr;  // [rows, k] the entries' logits
  int parts = 0;
};

int vocab_max_top();
cudaError_t vocab_topk(const VocabLaunch& l, const VocabRows& x, int k, float temperature, int64_t* ids, float* lp);
cudaError_t vocab_sample(const VocabLaunch& l, const VocabRows& x, const float* noise, long long nstride,
                         const SampleArgs& a, int64_t* tokens, float* lp);
cudaError_t distill_rows_forward(const VocabLaunch& l, const VocabRows& x, const DistillArgs& a, const DistillOut& out);
cudaError_t distill_rows_backward(const VocabLaunch& l, const VocabRows& x, const DistillArgs& a, const DistillOut& f,
                                  const float* grad, RowType otype, void* out, void* lo, long long ostride);
// entries in ascending order of their tokens, those that do not count last (token 0x7fffffff)
cudaError_t distill_sort_entries(const VocabLaunch& l, const DistillArgs& a, int64_t n, int v, int* ids, float* lp);
// loss and gradient coefficients from the head's statistics; `lp` sorted as st.ids
cudaError_t distill_head_finish(const VocabLaunch& l, const HeadStats& st, const float* lp, int64_t n, float tau,
                                bool reverse, bool tail, const DistillOut& out);

// Products of the head (csrc/head_tc.cu). Operand maps: bf16, boxes of 64 along the contiguous dimension and 128 rows
// (64 where the contraction is not the contiguous dimension); output maps: boxes of 32 rows of 128 bytes.
int head_parts(int v);
int head_splits(const VocabLaunch& l, int rows, int d, int v);
cudaError_t head_logits(const VocabLaunch& l, const CUtensorMap& h, const CUtensorMap& w, const CUtensorMap* out,
                        int rows, int d, int v, const HeadStats& st, int* err);
cudaError_t head_logits_again(const VocabLaunch& l, const CUtensorMap& h, const CUtensorMap& w, const CUtensorMap& out,
                              int rows, int d, int v, int* err);
// dlogits in two bf16 halves, or (`lo` null) rounded to bf16
cudaError_t head_dh(const VocabLaunch& l, const CUtensorMap& dl, const CUtensorMap* lo, const CUtensorMap& w,
                    const CUtensorMap& out, int rows, int d, int v, int splits, int split_rows, const float* parts,
                    void* dh, int* err);
cudaError_t head_dw(const VocabLaunch& l, const CUtensorMap& dl, const CUtensorMap* lo, const CUtensorMap& h,
                    const CUtensorMap& out, int rows, int d, int v, int* err);

cudaError_t distill_bounds(unsigned long long* word, bool reset);

}  // namespace ts

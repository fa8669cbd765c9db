// Launchers of the vocabulary-row kernels (csrc/vocab_select.cu, csrc/distill.cu), for csrc/vocab_bind.cpp: plain
// pointers, so that the kernel sources compile without torch's headers. Each returns the launch's error.
#pragma once

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
  float* ref;    // [n] m, the largest logit: p_j = 2^((z_j - m) c) / s, c = log2(e) / tau
  float* gs;     // [n] G / (s tau): the row's gradient outside the entries is -gs 2^((z_j - m) c)
  float* entry;  // [n, k] the gradient at the entries
};

int vocab_max_top();
cudaError_t vocab_topk(const VocabLaunch& l, const VocabRows& x, int k, float temperature, int64_t* ids, float* lp);
cudaError_t vocab_sample(const VocabLaunch& l, const VocabRows& x, const float* noise, long long nstride,
                         const SampleArgs& a, int64_t* tokens, float* lp);
cudaError_t distill_rows_forward(const VocabLaunch& l, const VocabRows& x, const DistillArgs& a, const DistillOut& out);
cudaError_t distill_rows_backward(const VocabLaunch& l, const VocabRows& x, const DistillArgs& a, const DistillOut& f,
                                  const float* grad, RowType otype, void* out, long long ostride);
cudaError_t distill_bounds(unsigned long long* word, bool reset);

}  // namespace ts

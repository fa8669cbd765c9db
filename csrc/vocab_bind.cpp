// Tensor entry points of the vocabulary-row kernels: argument checks, outputs and the current stream.
#include "common.h"
#include "vocab.h"

namespace ts {
namespace {

void check_rows(const at::Tensor& t, const char* name) {
  TS_CHECK(t.is_cuda() && t.dim() == 2, name, " must be a CUDA matrix");
  TS_CHECK(t.size(1) <= 1 || t.stride(1) == 1, name, " must have contiguous rows");
  TS_CHECK(t.size(1) >= 1 && t.size(1) <= 8000000 && t.size(0) < (int64_t(1) << 27), name, ": sizes out of range");
}

RowType row_type(const at::Tensor& t, const char* name) {
  const auto ty = t.scalar_type();
  TS_CHECK(ty == at::kFloat || ty == at::kBFloat16 || ty == at::kHalf, name, " must be fp32, bf16 or fp16");
  return ty == at::kFloat ? kRowsF32 : ty == at::kBFloat16 ? kRowsBf16 : kRowsF16;
}

cudaError_t set_smem(const void* kernel, int bytes) {
  ensure_smem(kernel, bytes);
  return cudaSuccess;
}

VocabLaunch launch_on(const at::Tensor& t) { return {stream(), sm_count(t.get_device()), set_smem}; }

VocabRows rows_of(const at::Tensor& t, const char* name) {
  check_rows(t, name);
  return {t.data_ptr(), row_type(t, name), t.size(0), (int)t.size(1), (long long)t.stride(0)};
}

}  // namespace

// logits [N, V] (fp32, bf16 or fp16, rows contiguous) -> ids int64 [N, k], log-probs fp32 [N, k], greatest first.
std::vector<at::Tensor> topk_logprobs(const at::Tensor& logits, int64_t k, double temperature) {
  const VocabRows x = rows_of(logits, "logits");
  TS_CHECK(k >= 1 && k <= vocab_max_top() && k <= x.v, "topk_logprobs: k must be in [1, min(256, V)]");
  TS_CHECK(temperature > 0, "topk_logprobs: temperature must be positive");
  const c10::cuda::CUDAGuard guard(logits.device());
  auto ids = at::empty({x.n, k}, logits.options().dtype(at::kLong));
  auto lp = at::empty({x.n, k}, logits.options().dtype(at::kFloat));
  if (x.n == 0) return {ids, lp};
  TS_CUDA_CHECK(vocab_topk(launch_on(logits), x, (int)k, (float)temperature, ids.data_ptr<int64_t>(),
                           lp.data_ptr<float>()));
  return {ids, lp};
}

// One token per row of logits [N, V]; noise fp32 [N, V] (may be absent when every row is greedy); each setting is a
// number or a tensor [N] (temperature, top_p, min_p fp32; top_k int64). Returns tokens int64 [N], log-probs fp32 [N].
std::vector<at::Tensor> sample_tokens(const at::Tensor& logits, const c10::optional<at::Tensor>& noise,
                                      const c10::optional<at::Tensor>& temperature_t, double temperature,
                                      const c10::optional<at::Tensor>& top_k_t, int64_t top_k,
                                      const c10::optional<at::Tensor>& top_p_t, double top_p,
                                      const c10::optional<at::Tensor>& min_p_t, double min_p) {
  const VocabRows x = rows_of(logits, "logits");
  if (noise) {
    check_rows(*noise, "noise");
    TS_CHECK(noise->scalar_type() == at::kFloat && noise->sizes() == logits.sizes() &&
                 noise->device() == logits.device(),
             "sample_tokens: noise must be fp32 with the logits' shape and device");
  } else {
    TS_CHECK(!temperature_t && temperature == 0, "sample_tokens: noise may be left out at temperature 0 only");
  }
  auto per_row = [&](const c10::optional<at::Tensor>& t, at::ScalarType ty, const char* name) -> const void* {
    if (!t) return nullptr;
    check_cuda(*t, name);
    TS_CHECK(t->dim() == 1 && t->size(0) == x.n && t->scalar_type() == ty && t->device() == logits.device(), name,
             " must be a number or have one entry per row");
    return t->data_ptr();
  };
  SampleArgs a;
  a.temperature = (const float*)per_row(temperature_t, at::kFloat, "temperature");
  a.top_k = (const int64_t*)per_row(top_k_t, at::kLong, "top_k");
  a.top_p = (const float*)per_row(top_p_t, at::kFloat, "top_p");
  a.min_p = (const float*)per_row(min_p_t, at::kFloat, "min_p");
  a.temperature_s = (float)temperature;
  a.top_k_s = top_k;
  a.top_p_s = (float)top_p;
  a.min_p_s = (float)min_p;
  const c10::cuda::CUDAGuard guard(logits.device());
  auto tok = at::empty({x.n}, logits.options().dtype(at::kLong));
  auto lp = at::empty({x.n}, logits.options().dtype(at::kFloat));
  if (x.n == 0) return {tok, lp};
  TS_CUDA_CHECK(vocab_sample(launch_on(logits), x, noise ? noise->data_ptr<float>() : nullptr,
                             noise ? (long long)noise->stride(0) : 0, a, tok.data_ptr<int64_t>(),
                             lp.data_ptr<float>()));
  return {tok, lp};
}

// logits [N, V]; teacher ids int64 [N, K] and log-probs fp32 [N, K] (id -1 or log-prob -inf: no entry).
// Returns loss [N], and what the backward reads: slots int32 [N, K], ref [N], gs [N], entry [N, K].
std::vector<at::Tensor> distill_rows_fwd(const at::Tensor& logits, const at::Tensor& ids, const at::Tensor& lp,
                                         double tau, bool reverse, bool tail) {
  const VocabRows x = rows_of(logits, "logits");
  check_cuda(ids, "teacher_ids");
  check_cuda(lp, "teacher_logprobs");
  TS_CHECK(ids.dim() == 2 && ids.size(0) == x.n && ids.scalar_type() == at::kLong && lp.sizes() == ids.sizes() &&
               lp.scalar_type() == at::kFloat,
           "teacher_ids must be int64 [N, K] and teacher_logprobs fp32 [N, K]");
  const int64_t k = ids.size(1);
  TS_CHECK(k >= 1 && k <= vocab_max_top(), "teacher entries per row must be in [1, 256]");
  TS_CHECK(tau > 0, "temperature must be positive");
  TS_CHECK(ids.device() == logits.device() && lp.device() == logits.device(), "operands on different devices");
  const c10::cuda::CUDAGuard guard(logits.device());
  const auto f32 = logits.options().dtype(at::kFloat);
  auto loss = at::empty({x.n}, f32), ref = at::empty({x.n}, f32), gs = at::empty({x.n}, f32);
  auto entry = at::empty({x.n, k}, f32);
  auto slots = at::empty({x.n, k}, logits.options().dtype(at::kInt));
  if (x.n == 0) return {loss, slots, ref, gs, entry};
  const DistillArgs a{ids.data_ptr<int64_t>(), lp.data_ptr<float>(), (int)k, (float)tau, reverse, tail};
  const DistillOut out{loss.data_ptr<float>(), slots.data_ptr<int>(), ref.data_ptr<float>(), gs.data_ptr<float>(),
                       entry.data_ptr<float>()};
  TS_CUDA_CHECK(distill_rows_forward(launch_on(logits), x, a, out));
  return {loss, slots, ref, gs, entry};
}

// The gradient of the logits for upstream gradients grad [N] fp32, in `out` [N, V] (its rows may be strided): the
// logits' type, or bf16 / fp16 for fp32 logits.
void distill_rows_bwd(const at::Tensor& logits, const at::Tensor& slots, const at::Tensor& ref, const at::Tensor& gs,
                      const at::Tensor& entry, const at::Tensor& grad, double tau, at::Tensor& out) {
  const VocabRows x = rows_of(logits, "logits");
  check_rows(out, "gradient");
  check_cuda(grad, "grad");
  TS_CHECK(out.sizes() == logits.sizes() && out.device() == logits.device(), "the gradient must have the logits' shape");
  TS_CHECK(grad.scalar_type() == at::kFloat && grad.dim() == 1 && grad.size(0) == x.n, "grad must be fp32 [N]");
  const c10::cuda::CUDAGuard guard(logits.device());
  if (x.n == 0) return;
  const DistillArgs a{nullptr, nullptr, (int)slots.size(1), (float)tau, false, false};
  const DistillOut f{nullptr, slots.data_ptr<int>(), ref.data_ptr<float>(), gs.data_ptr<float>(),
                     entry.data_ptr<float>()};
  TS_CUDA_CHECK(distill_rows_backward(launch_on(logits), x, a, f, grad.data_ptr<float>(), row_type(out, "gradient"),
                                      out.data_ptr(), (long long)out.stride(0)));
}

uint64_t bounds_word_distill(bool reset) {
  unsigned long long w = 0;
  TS_CUDA_CHECK(distill_bounds(&w, reset));
  return (uint64_t)w;
}

}  // namespace ts

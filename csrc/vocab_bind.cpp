// Tensor entry points of the vocabulary-row kernels: argument checks, outputs and the current stream.
#include "common.h"
#include "vocab.h"

#include <atomic>

namespace ts {

CUtensorMap make_bf16_map(const void* base, uint64_t inner, uint64_t outer, uint64_t row_stride_elems,
                          uint32_t box_rows);
CUtensorMap make_out_map(void* base, bool f32, uint64_t cols, uint64_t rows, uint64_t ld);
at::Tensor& tc_error_flag(const at::Device& dev);

namespace {

std::atomic<int64_t> g_more_launches{0};

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
// logits' type, or bf16 / fp16 for fp32 logits. With `lo` (fp32 logits, both bf16) the two add up to the gradient.
void distill_rows_bwd(const at::Tensor& logits, const at::Tensor& slots, const at::Tensor& ref, const at::Tensor& gs,
                      const at::Tensor& entry, const at::Tensor& grad, double tau, at::Tensor& out,
                      const c10::optional<at::Tensor>& lo) {
  const VocabRows x = rows_of(logits, "logits");
  check_rows(out, "gradient");
  check_cuda(grad, "grad");
  TS_CHECK(out.sizes() == logits.sizes() && out.device() == logits.device(), "the gradient must have the logits' shape");
  if (lo) {
    check_rows(*lo, "gradient");
    TS_CHECK(lo->sizes() == out.sizes() && lo->device() == out.device() && lo->strides() == out.strides() &&
                 lo->scalar_type() == at::kBFloat16 && out.scalar_type() == at::kBFloat16 &&
                 logits.scalar_type() == at::kFloat,
             "the gradient's halves must be two bf16 tensors of one layout, of fp32 logits");
  }
  TS_CHECK(grad.scalar_type() == at::kFloat && grad.dim() == 1 && grad.size(0) == x.n, "grad must be fp32 [N]");
  const c10::cuda::CUDAGuard guard(logits.device());
  if (x.n == 0) return;
  const DistillArgs a{nullptr, nullptr, (int)slots.size(1), (float)tau, false, false};
  const DistillOut f{nullptr, slots.data_ptr<int>(), ref.data_ptr<float>(), gs.data_ptr<float>(),
                     entry.data_ptr<float>()};
  TS_CUDA_CHECK(distill_rows_backward(launch_on(logits), x, a, f, grad.data_ptr<float>(), row_type(out, "gradient"),
                                      out.data_ptr(), lo ? lo->data_ptr() : nullptr, (long long)out.stride(0)));
}

namespace {

// The gradient as the end of what can be differentiated: it depends on the logits and the upstream gradient, but asking
// for that dependence is an error.
struct DifferentiatedOnce : torch::autograd::Function<DifferentiatedOnce> {
  static at::Tensor forward(torch::autograd::AutogradContext*, const at::Tensor& d, const at::Tensor&, const at::Tensor&) {
    return d;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext*, torch::autograd::variable_list) {
    TS_CHECK(false, "topk_distill_loss is differentiable once: its gradient on CUDA has no gradient of its own");
    return {};
  }
};

// The loss on logits as a native autograd node: its backward needs no interpreter, which for a few rows was most of
// the call's time.
struct DistillRows : torch::autograd::Function<DistillRows> {
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& ids,
                            const at::Tensor& lp, double tau, bool reverse, bool tail) {
    auto r = distill_rows_fwd(logits, ids, lp, tau, reverse, tail);
    ctx->save_for_backward({logits, r[1], r[2], r[3], r[4]});
    ctx->saved_data["tau"] = tau;
    return r[0];
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    at::Tensor d;
    if (grads[0].defined()) {
      const auto s = ctx->get_saved_variables();
      {
        const at::AutoGradMode off(false);
        d = at::empty(s[0].sizes(), s[0].options());
        distill_rows_bwd(s[0], s[1], s[2], s[3], s[4], grads[0].to(at::kFloat).contiguous(),
                         ctx->saved_data["tau"].toDouble(), d, c10::nullopt);
        if (d.size(0) > 0) ++g_more_launches;
      }
      if (at::GradMode::is_enabled()) d = DifferentiatedOnce::apply(d, s[0], grads[0]);  // (create_graph)
    }
    return {d, {}, {}, {}, {}, {}};
  }
};

void check_bf16(const at::Tensor& t, const char* name) {
  check_cuda(t, name);
  TS_CHECK(t.dim() == 2 && t.scalar_type() == at::kBFloat16 && t.size(1) % 8 == 0 && t.size(0) < (int64_t(1) << 30) &&
               t.size(1) < (int64_t(1) << 30),
           name, " must be a bf16 matrix whose rows are a multiple of 8 long");
}
void check_head(const at::Tensor& h, const at::Tensor& w) {
  check_bf16(h, "hidden");
  check_bf16(w, "weight");
  TS_CHECK(h.size(1) == w.size(1) && w.size(0) % 8 == 0 && w.size(0) >= 8 && w.size(0) <= 8000000 && h.size(1) >= 8 &&
               h.device() == w.device(),
           "hidden [N, D] and weight [V, D] with V a multiple of 8");
}
int* error_word(const at::Tensor& t) { return tc_error_flag(t.device()).data_ptr<int>(); }
CUtensorMap k_rows(const at::Tensor& t) {  // [rows, k], the contraction along the rows
  return make_bf16_map(t.data_ptr(), t.size(1), t.size(0), t.size(1), 128);
}
CUtensorMap k_cols(const at::Tensor& t) {  // [k, cols], the contraction down the columns
  return make_bf16_map(t.data_ptr(), t.size(1), t.size(0), t.size(1), 64);
}
CUtensorMap out_map(const at::Tensor& t) {  // boxes of 32 rows of 128 bytes
  if (t.scalar_type() == at::kFloat) return make_out_map(t.data_ptr(), true, t.size(1), t.size(0), t.size(1));
  return make_bf16_map(t.data_ptr(), t.size(1), t.size(0), t.size(1), 32);
}

}  // namespace

// distill_rows_fwd's loss, differentiable in the logits
at::Tensor distill_rows(const at::Tensor& logits, const at::Tensor& ids, const at::Tensor& lp, double tau, bool reverse,
                        bool tail) {
  return DistillRows::apply(logits, ids, lp, tau, reverse, tail);
}

// hidden [N, D] and weight [V, D] bf16, teacher entries [N, K]: loss and what the backward reads, as distill_rows_fwd;
// with `keep` the fp32 logits [N, V] too (else None).
std::vector<c10::optional<at::Tensor>> distill_head_fwd(const at::Tensor& h, const at::Tensor& w, const at::Tensor& ids,
                                                        const at::Tensor& lp, double tau, bool reverse, bool tail,
                                                        bool keep) {
  check_head(h, w);
  check_cuda(ids, "teacher_ids");
  check_cuda(lp, "teacher_logprobs");
  const int64_t n = h.size(0), d = h.size(1), v = w.size(0);
  TS_CHECK(ids.dim() == 2 && ids.size(0) == n && ids.scalar_type() == at::kLong && lp.sizes() == ids.sizes() &&
               lp.scalar_type() == at::kFloat && ids.device() == h.device() && lp.device() == h.device(),
           "teacher_ids must be int64 [N, K] and teacher_logprobs fp32 [N, K]");
  const int64_t k = ids.size(1);
  TS_CHECK(k >= 1 && k <= vocab_max_top(), "teacher entries per row must be in [1, 256]");
  TS_CHECK(tau > 0, "temperature must be positive");
  const c10::cuda::CUDAGuard guard(h.device());
  const auto f32 = h.options().dtype(at::kFloat), i32 = h.options().dtype(at::kInt);
  auto loss = at::empty({n}, f32), ref = at::empty({n}, f32), gs = at::empty({n}, f32), entry = at::empty({n, k}, f32);
  auto slots = at::empty({n, k}, i32);
  c10::optional<at::Tensor> logits;
  if (keep) logits = at::empty({n, v}, f32);
  if (n == 0) return {loss, slots, ref, gs, entry, logits};
  const int parts = head_parts((int)v);
  auto sorted_ids = at::empty({n, k}, i32);
  auto sorted_lp = at::empty({n, k}, f32), zk = at::empty({n, k}, f32), sums = at::empty({2, n, parts}, f32);
  const VocabLaunch l = launch_on(h);
  const DistillArgs a{ids.data_ptr<int64_t>(), lp.data_ptr<float>(), (int)k, (float)tau, reverse, tail};
  TS_CUDA_CHECK(distill_sort_entries(l, a, n, (int)v, sorted_ids.data_ptr<int>(), sorted_lp.data_ptr<float>()));
  HeadStats st;
  st.ids = sorted_ids.data_ptr<int>();
  st.k = (int)k;
  st.c = 1.4426950408889634f / (float)tau;
  st.pm = sums.data_ptr<float>();
  st.ps = st.pm + n * parts;
  st.zk = zk.data_ptr<float>();
  st.parts = parts;
  CUtensorMap out{};
  if (keep) out = out_map(*logits);
  TS_CUDA_CHECK(head_logits(l, k_rows(h), k_rows(w), keep ? &out : nullptr, (int)n, (int)d, (int)v, st, error_word(h)));
  const DistillOut o{loss.data_ptr<float>(), slots.data_ptr<int>(), ref.data_ptr<float>(), gs.data_ptr<float>(),
                     entry.data_ptr<float>()};
  TS_CUDA_CHECK(distill_head_finish(l, st, sorted_lp.data_ptr<float>(), n, (float)tau, reverse, tail, o));
  return {loss, slots, ref, gs, entry, logits};
}

// fp32 logits [N, V] as distill_head_fwd computes them
at::Tensor distill_head_logits(const at::Tensor& h, const at::Tensor& w) {
  check_head(h, w);
  const c10::cuda::CUDAGuard guard(h.device());
  auto out = at::empty({h.size(0), w.size(0)}, h.options().dtype(at::kFloat));
  if (h.size(0) == 0) return out;
  TS_CUDA_CHECK(head_logits_again(launch_on(h), k_rows(h), k_rows(w), out_map(out), (int)h.size(0), (int)h.size(1),
                                  (int)w.size(0), error_word(h)));
  return out;
}

namespace {
void check_halves(const at::Tensor& dl, const c10::optional<at::Tensor>& lo) {
  check_bf16(dl, "dlogits");
  if (!lo) return;
  check_bf16(*lo, "dlogits");
  TS_CHECK(lo->sizes() == dl.sizes() && lo->device() == dl.device(), "the halves of the dlogits differ in shape");
}
}  // namespace

// dH [N, D] = (d + lo) [N, V] · weight [V, D], bf16
void distill_head_dh(const at::Tensor& dl, const c10::optional<at::Tensor>& lo, const at::Tensor& w, at::Tensor& dh) {
  check_halves(dl, lo);
  check_bf16(w, "weight");
  check_bf16(dh, "dhidden");
  const int64_t n = dl.size(0), v = dl.size(1), d = w.size(1);
  TS_CHECK(w.size(0) == v && dh.size(0) == n && dh.size(1) == d && dl.device() == w.device() &&
               dh.device() == w.device(),
           "distill_head_dh shapes");
  const c10::cuda::CUDAGuard guard(dl.device());
  if (n == 0) return;
  const VocabLaunch l = launch_on(dl);
  const int splits = head_splits(l, (int)n, (int)d, (int)v);
  const int split_rows = (int)((n + 255) / 256 * 256);  // whole tiles: a slice's last one writes no row of the next
  at::Tensor parts;
  if (splits > 1) parts = at::empty({(int64_t)splits * split_rows, d}, dl.options().dtype(at::kFloat));
  CUtensorMap low{};
  if (lo) low = k_rows(*lo);
  TS_CUDA_CHECK(head_dh(l, k_rows(dl), lo ? &low : nullptr, k_cols(w), out_map(splits > 1 ? parts : dh), (int)n, (int)d,
                        (int)v, splits, split_rows, splits > 1 ? parts.data_ptr<float>() : nullptr, dh.data_ptr(),
                        error_word(dl)));
  if (splits > 1) ++g_more_launches;  // the sum of the slices
}

// dW [V, D] = (d + lo)ᵀ [V, N] · hidden [N, D], bf16
at::Tensor distill_head_dw(const at::Tensor& dl, const c10::optional<at::Tensor>& lo, const at::Tensor& h) {
  check_halves(dl, lo);
  check_bf16(h, "hidden");
  TS_CHECK(dl.size(0) == h.size(0) && dl.device() == h.device(), "distill_head_dw shapes");
  const c10::cuda::CUDAGuard guard(dl.device());
  auto dw = at::empty({dl.size(1), h.size(1)}, dl.options());
  if (h.size(0) == 0) return dw.zero_();
  CUtensorMap low{};
  if (lo) low = k_cols(*lo);
  TS_CUDA_CHECK(head_dw(launch_on(dl), k_cols(dl), lo ? &low : nullptr, k_cols(h), out_map(dw), (int)h.size(0),
                        (int)h.size(1), (int)dl.size(1), error_word(dl)));
  return dw;
}

// Kernels since the last reset that no call of an entry point stands for: the loss rows' gradient, which autograd calls,
// and those that only some calls launch.
int64_t more_launches(bool reset) { return reset ? g_more_launches.exchange(0) : g_more_launches.load(); }

uint64_t bounds_word_distill(bool reset) {
  unsigned long long w = 0;
  TS_CUDA_CHECK(distill_bounds(&w, reset));
  return (uint64_t)w;
}

}  // namespace ts

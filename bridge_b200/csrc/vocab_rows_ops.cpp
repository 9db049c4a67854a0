// Torch entry points of the kernels over rows of logits (vocab_rows.cu): argument checks, allocation, launch.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <cmath>

#include "vocab_rows.h"

namespace {

using OptTensor = c10::optional<torch::Tensor>;

void check(cudaError_t e) { TORCH_CHECK(e == cudaSuccess, "CUDA error ", cudaGetErrorString(e)); }

bb::RowType row_type(const torch::Tensor& x) {
  switch (x.scalar_type()) {
    case at::kFloat: return bb::RowType::f32;
    case at::kHalf: return bb::RowType::f16;
    case at::kBFloat16: return bb::RowType::bf16;
    default: TORCH_CHECK(false, "logits must be float32, float16 or bfloat16");
  }
}
void check_rows(const torch::Tensor& x) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2 && (x.size(1) == 1 || x.stride(1) == 1),
              "logits must be a CUDA matrix with unit column stride");
  TORCH_CHECK(x.size(1) >= 1 && x.size(1) <= bb::kMaxVocab && x.size(0) < (1l << 28),
              "logits: at most 2^22 columns and 2^28 rows");
}
void check_vec(const OptTensor& t, int64_t n, at::ScalarType dt, const torch::Tensor& x, const char* what) {
  if (!t.has_value()) return;
  TORCH_CHECK(t->device() == x.device() && t->scalar_type() == dt && t->is_contiguous() && t->numel() == n, what);
}
// The forms that the kernels take as they are; anything else is checked and brought into them by the caller.
bool plain_rows(const torch::Tensor& x) {
  return x.is_cuda() && x.dim() == 2 && x.size(1) >= 1 && x.size(1) <= bb::kMaxVocab && x.size(0) < (1l << 28) &&
         (x.size(1) == 1 || x.stride(1) == 1) &&
         (x.scalar_type() == at::kBFloat16 || x.scalar_type() == at::kHalf || x.scalar_type() == at::kFloat);
}
bool plain_floats(const OptTensor& t, const torch::Tensor& x) {
  return !t.has_value() || (t->dim() == 1 && t->size(0) == x.size(0) && t->scalar_type() == at::kFloat &&
                            t->is_contiguous() && t->device() == x.device() && !t->requires_grad());
}
bool positive(double v) { return v > 0.0 && std::isfinite(v); }

template <typename V>
V* ptr(const OptTensor& t) {
  return t.has_value() ? t->data_ptr<V>() : nullptr;
}

bb::DistillArgs distill_args(const torch::Tensor& logits_like, const torch::Tensor& ids, const torch::Tensor& logq,
                             const OptTensor& weights, const OptTensor& temp, double temp1, double scale, bool tail,
                             int64_t vocab_start, int64_t vocab_total) {
  const int64_t U = logits_like.size(0), K = ids.size(1);
  TORCH_CHECK(K >= 1 && K <= bb::kMaxTop, "teacher entries per row out of range");
  TORCH_CHECK(U < (1l << 31) && vocab_total < (1l << 31), "size out of range");
  check_vec(ids, U * K, at::kLong, logits_like, "teacher ids must be int64 [U, K]");
  check_vec(logq, U * K, at::kFloat, logits_like, "teacher log-probs must be float32 [U, K]");
  check_vec(weights, U, at::kFloat, logits_like, "weights must be float32 [U]");
  check_vec(temp, U, at::kFloat, logits_like, "temperature must be float32 [U]");
  bb::DistillArgs a{};
  a.ids = ids.data_ptr<int64_t>();
  a.logq = logq.data_ptr<float>();
  a.weights = ptr<float>(weights);
  a.temp = ptr<float>(temp);
  a.inv_temp1 = 1.0 / temp1, a.scale = scale;
  a.U = (int)U, a.K = (int)K;
  a.vocab_start = vocab_start, a.vocab_total = vocab_total;
  a.tail = tail;
  return a;
}

// ---------------------------------------------------------------------------------------- token log-probs
struct Scores {
  torch::Tensor logp, entropy, stats, ids, top;      // undefined where not asked for
};

Scores score_rows(const torch::Tensor& logits, const OptTensor& tokens, const OptTensor& temp, double temp1, int64_t k,
                  bool entropy, bool stats, int64_t vocab_start, bool open) {
  const c10::cuda::CUDAGuard guard(logits.device());
  const int64_t U = logits.size(0), V = logits.size(1);
  const auto f32 = logits.options().dtype(at::kFloat).requires_grad(false);
  Scores o;
  if (tokens.has_value()) o.logp = at::empty(tokens->sizes(), f32);
  if (entropy) o.entropy = at::empty({U}, f32);
  if (stats) o.stats = at::empty({U, 3}, f32);
  if (k) {
    o.ids = at::empty({U, k}, f32.dtype(at::kLong));
    o.top = at::empty({U, k}, f32);
  }
  if (U == 0) return o;
  bb::TokenArgs a{};
  a.tokens = ptr<int64_t>(tokens);
  a.temp = ptr<float>(temp);
  a.inv_temp1 = 1.0 / temp1;
  a.U = (int)U, a.V = (int)V, a.n = tokens.has_value() ? (int)(tokens->numel() / U) : 0, a.k = (int)k;
  a.stride = logits.stride(0), a.vocab_start = vocab_start;
  a.logp = tokens.has_value() ? o.logp.data_ptr<float>() : nullptr;
  a.entropy = entropy ? o.entropy.data_ptr<float>() : nullptr;
  a.stats = stats ? o.stats.data_ptr<float>() : nullptr;
  a.top_ids = k ? o.ids.data_ptr<int64_t>() : nullptr;
  a.top_logp = k ? o.top.data_ptr<float>() : nullptr;
  a.open = open;
  check(bb::launch_token_logprob(row_type(logits), logits.data_ptr(), a, at::cuda::getCurrentCUDAStream()));
  return o;
}

void check_scoring(const torch::Tensor& logits, const OptTensor& tokens, const OptTensor& temp, int64_t k) {
  check_rows(logits);
  const int64_t U = logits.size(0);
  if (tokens.has_value()) {
    TORCH_CHECK(tokens->dim() >= 1 && tokens->dim() <= 2 && tokens->size(0) == U, "tokens must be [U] or [U, n]");
    check_vec(tokens, tokens->numel(), at::kLong, logits, "tokens must be contiguous int64 on the logits' device");
  }
  check_vec(temp, U, at::kFloat, logits, "temperature must be float32 [U]");
  TORCH_CHECK(k >= 0 && k <= bb::kMaxTop && k <= logits.size(1), "top_k out of range");
}

torch::Tensor score_rows_bwd(const torch::Tensor& logits, const OptTensor& tokens, const OptTensor& temp, double temp1,
                             const torch::Tensor& stats, const OptTensor& d_logp, const OptTensor& d_entropy,
                             int64_t vocab_start, int64_t vocab_total) {
  const c10::cuda::CUDAGuard guard(logits.device());
  const int64_t U = logits.size(0), V = logits.size(1);
  auto grad = at::empty({U, V}, logits.options().requires_grad(false));
  if (U == 0) return grad;
  const bool given = tokens.has_value() && d_logp.has_value();
  bb::TokenArgs a{};
  a.tokens = given ? ptr<int64_t>(tokens) : nullptr;
  a.d_logp = given ? ptr<float>(d_logp) : nullptr;
  a.d_entropy = ptr<float>(d_entropy);
  a.temp = ptr<float>(temp);
  a.inv_temp1 = 1.0 / temp1;
  a.U = (int)U, a.V = (int)V, a.n = given ? (int)(tokens->numel() / U) : 0;
  a.stride = logits.stride(0), a.vocab_start = vocab_start, a.vocab_total = vocab_total;
  a.stats = stats.data_ptr<float>();
  check(bb::launch_token_logprob_bwd(row_type(logits), logits.data_ptr(), grad.data_ptr(), a,
                                     at::cuda::getCurrentCUDAStream()));
  return grad;
}

// Both nodes' gradients are made from sums that their forward kept: constants to a second differentiation, and nothing
// here carries a tangent.
void first_order(const char* name) {
  TORCH_CHECK(!at::GradMode::is_enabled(), name, " has no second derivative (backward was called with create_graph=True)");
}
void no_tangent(const torch::Tensor& x, const char* name) {
  TORCH_CHECK_NOT_IMPLEMENTED(!x._fw_grad(0).defined(), name, " has no forward-mode derivative");
}

OptTensor optional(const torch::Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }
OptTensor upstream(const torch::Tensor& g) {
  return g.defined() ? OptTensor(g.to(at::kFloat).contiguous()) : OptTensor();
}

// Differentiable in `logits` through the log-probs and the entropy.
class ScoreRows : public torch::autograd::Function<ScoreRows> {
 public:
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const torch::Tensor& logits,
                                                const OptTensor& tokens, const OptTensor& temp, double temp1, int64_t k,
                                                bool entropy) {
    const Scores o = score_rows(logits, tokens, temp, temp1, k, entropy, true, 0, false);
    const torch::Tensor none;
    ctx->save_for_backward({logits, tokens.value_or(none), temp.value_or(none), o.stats});
    ctx->saved_data["temp1"] = temp1;
    ctx->saved_data["logp"] = tokens.has_value();
    ctx->set_materialize_grads(false);
    torch::autograd::variable_list out;
    for (const auto& t : {o.logp, o.entropy, o.ids, o.top})
      if (t.defined()) out.push_back(t);
    if (k) ctx->mark_non_differentiable({o.ids, o.top});
    return out;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    first_order("token_logprobs");
    const auto saved = ctx->get_saved_variables();
    const bool has_logp = ctx->saved_data["logp"].toBool();
    size_t at = 0;
    OptTensor d_logp, d_entropy;
    if (has_logp) d_logp = upstream(grads[at++]);
    if (at < grads.size()) d_entropy = upstream(grads[at]);      // (the alternatives' are never defined)
    torch::Tensor g;
    if (d_logp.has_value() || d_entropy.has_value())
      g = score_rows_bwd(saved[0], optional(saved[1]), optional(saved[2]), ctx->saved_data["temp1"].toDouble(),
                         saved[3], d_logp, d_entropy, 0, saved[0].size(1));
    return {g, torch::Tensor(), torch::Tensor(), torch::Tensor(), torch::Tensor(), torch::Tensor()};
  }
};

// ------------------------------------------------------------------------------------------- distillation
// Rows of a whole vocabulary: KL [U] and, unless `grad` is null, their gradient into it.
void distill_into(const torch::Tensor& logits, bb::DistillArgs a, const torch::Tensor* rows, const torch::Tensor* grad) {
  if (a.U == 0) return;
  a.V = (int)logits.size(1), a.stride = logits.stride(0);
  a.rows = rows ? rows->data_ptr<float>() : nullptr;
  check(bb::launch_distill(row_type(logits), logits.data_ptr(), grad ? grad->data_ptr() : nullptr, a,
                           at::cuda::getCurrentCUDAStream()));
}

torch::Tensor sum_rows(const torch::Tensor& rows, const OptTensor& weights, double denom) {
  auto out = at::empty({}, rows.options());
  check(bb::launch_weighted_sum(rows.data_ptr<float>(), ptr<float>(weights), (int)rows.numel(), 1.0 / denom,
                                out.data_ptr<float>(), at::cuda::getCurrentCUDAStream()));
  return out;
}

void scale_grad(const torch::Tensor& x, const torch::Tensor& num, double den) {
  if (x.numel() == 0) return;
  check(bb::launch_scale_unless_one(row_type(x), x.data_ptr(), x.numel(), num.data_ptr<float>(), (float)den,
                                    at::cuda::getCurrentCUDAStream()));
}

// The loss (differentiable in `logits`; the gradient is written by the forward) and the rows.
class DistillLoss : public torch::autograd::Function<DistillLoss> {
 public:
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const torch::Tensor& logits,
                                                const torch::Tensor& ids, const torch::Tensor& logq,
                                                const OptTensor& weights, const OptTensor& temp, double temp1,
                                                bool tail, double denom, double grad_scale) {
    const c10::cuda::CUDAGuard guard(logits.device());
    const auto plain = logits.options().requires_grad(false);
    auto rows = at::empty({logits.size(0)}, plain.dtype(at::kFloat));
    auto grad = at::empty(logits.sizes(), plain);
    const auto a = distill_args(logits, ids, logq, weights, temp, temp1, grad_scale / denom, tail, 0,
                                logits.size(1));
    distill_into(logits, a, &rows, &grad);
    ctx->saved_data["grad"] = grad;
    ctx->saved_data["grad_scale"] = grad_scale;
    if (logits.scalar_type() == at::kHalf) {      // what the gradient takes once more if the loss is scaled otherwise
      const torch::Tensor none;
      ctx->save_for_backward({logits, ids, logq, weights.value_or(none), temp.value_or(none)});
      ctx->saved_data["temp1"] = temp1;
      ctx->saved_data["tail"] = tail;
      ctx->saved_data["denom"] = denom;
    }
    ctx->mark_non_differentiable({rows});
    return {sum_rows(rows, weights, denom), rows};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    first_order("topk_distill_loss");
    const auto held = ctx->saved_data.find("grad");
    TORCH_CHECK(held != ctx->saved_data.end(),
                "topk_distill_loss: the gradient was already taken by an earlier backward");
    auto grad = held->second.toTensor();      // handed on without a copy, so there is one backward
    ctx->saved_data.erase(held);
    const c10::cuda::CUDAGuard guard(grad.device());
    const auto dloss = grads[0].to(at::kFloat);
    const double grad_scale = ctx->saved_data["grad_scale"].toDouble();
    const torch::Tensor none;
    if (grad.scalar_type() == at::kHalf) {
      // FP16 has no room for a scale after the rounding (what a loss scaler is there to save is 0 by then): the gradient
      // is written again from the logits, unless the factor is the announced one
      const auto saved = ctx->get_saved_variables();
      auto a = distill_args(saved[0], saved[1], saved[2], optional(saved[3]), optional(saved[4]),
                            ctx->saved_data["temp1"].toDouble(), grad_scale / ctx->saved_data["denom"].toDouble(),
                            ctx->saved_data["tail"].toBool(), 0, saved[0].size(1));
      a.num = dloss.data_ptr<float>(), a.den = (float)grad_scale;
      distill_into(saved[0], a, nullptr, &grad);
    } else {
      scale_grad(grad, dloss, grad_scale);
    }
    return {grad, none, none, none, none, none, none, none, none};
  }
};

}  // namespace

// (log-probs, entropy, ids, their log-probs), None where not asked for; empty where the arguments are not in the form
// that the kernels take.
std::vector<torch::Tensor> token_logprobs(torch::Tensor logits, OptTensor tokens, OptTensor temp, double temp1,
                                          int64_t k, bool entropy) {
  const bool fits = plain_rows(logits) && plain_floats(temp, logits) && positive(temp1) && k >= 0 && k <= bb::kMaxTop &&
                    k <= logits.size(1) &&
                    (!tokens.has_value() ||
                     (tokens->dim() >= 1 && tokens->dim() <= 2 && tokens->size(0) == logits.size(0) &&
                      tokens->scalar_type() == at::kLong && tokens->is_contiguous() &&
                      tokens->device() == logits.device()));
  if (!fits) return {};
  no_tangent(logits, "token_logprobs");
  const bool differentiable = logits.requires_grad() && at::GradMode::is_enabled() && (tokens.has_value() || entropy);
  if (!differentiable) {
    const Scores o = score_rows(logits, tokens, temp, temp1, k, entropy, false, 0, false);
    return {o.logp, o.entropy, o.ids, o.top};
  }
  const auto out = ScoreRows::apply(logits, tokens, temp, temp1, k, entropy);
  std::vector<torch::Tensor> r(4);
  size_t at = 0;
  if (tokens.has_value()) r[0] = out[at++];
  if (entropy) r[1] = out[at++];
  if (k) r[2] = out[at], r[3] = out[at + 1];
  return r;
}

// A shard of the vocabulary: open sums [U, 3], the tokens' x c, and the shard's best (ids, logits).
std::vector<torch::Tensor> token_logprob_open(torch::Tensor logits, OptTensor tokens, OptTensor temp, double temp1,
                                              int64_t k, bool entropy, int64_t vocab_start) {
  check_scoring(logits, tokens, temp, k);
  const Scores o = score_rows(logits, tokens, temp, temp1, k, entropy, true, vocab_start, true);
  return {o.logp, o.stats, o.ids, o.top};
}

torch::Tensor token_logprob_bwd(torch::Tensor logits, OptTensor tokens, OptTensor temp, double temp1,
                                torch::Tensor stats, OptTensor d_logp, OptTensor d_entropy, int64_t vocab_start,
                                int64_t vocab_total) {
  check_scoring(logits, tokens, temp, 0);
  const int64_t U = logits.size(0);
  if (tokens.has_value()) check_vec(d_logp, tokens->numel(), at::kFloat, logits, "d_logp must be float32 like tokens");
  check_vec(stats, 3 * U, at::kFloat, logits, "stats must be float32 [U, 3]");
  check_vec(d_entropy, U, at::kFloat, logits, "d_entropy must be float32 [U]");
  return score_rows_bwd(logits, tokens, temp, temp1, stats, d_logp, d_entropy, vocab_start, vocab_total);
}

// (loss, KL [U]) of a whole vocabulary; empty where the arguments are not in the form that the kernels take.
std::vector<torch::Tensor> topk_distill(torch::Tensor logits, torch::Tensor ids, torch::Tensor logq, OptTensor weights,
                                        OptTensor temp, double temp1, bool tail, double denom, double grad_scale) {
  const auto entries = [&](const torch::Tensor& t, at::ScalarType dt) {
    return t.dim() == 2 && t.size(0) == logits.size(0) && t.size(1) >= 1 && t.size(1) <= bb::kMaxTop &&
           t.scalar_type() == dt && t.is_contiguous() && t.device() == logits.device() && !t.requires_grad();
  };
  const bool fits = plain_rows(logits) && plain_floats(temp, logits) && plain_floats(weights, logits) &&
                    positive(temp1) && positive(denom) && positive(grad_scale) && entries(ids, at::kLong) &&
                    entries(logq, at::kFloat) && logq.size(1) == ids.size(1);
  if (!fits) return {};
  no_tangent(logits, "topk_distill_loss");
  if (logits.requires_grad() && at::GradMode::is_enabled()) {
    const auto o = DistillLoss::apply(logits, ids, logq, weights, temp, temp1, tail, denom, grad_scale);
    return {o[0], o[1]};
  }
  const c10::cuda::CUDAGuard guard(logits.device());
  auto rows = at::empty({logits.size(0)}, logits.options().dtype(at::kFloat).requires_grad(false));
  const auto a = distill_args(logits, ids, logq, weights, temp, temp1, 1.0, tail, 0, logits.size(1));
  distill_into(logits, a, &rows, nullptr);
  return {sum_rows(rows, weights, denom), rows};
}

// KL [U] of a whole vocabulary; with `want_grad` the contiguous logits become their own gradient.
torch::Tensor distill_rows_inplace(torch::Tensor logits, torch::Tensor ids, torch::Tensor logq, OptTensor weights,
                                   OptTensor temp, double temp1, double scale, bool tail, bool want_grad) {
  check_rows(logits);
  TORCH_CHECK(!want_grad || logits.is_contiguous(), "in-place gradients need contiguous logits");
  const c10::cuda::CUDAGuard guard(logits.device());
  auto rows = at::empty({logits.size(0)}, logits.options().dtype(at::kFloat));
  const auto a = distill_args(logits, ids, logq, weights, temp, temp1, scale, tail, 0, logits.size(1));
  distill_into(logits, a, &rows, want_grad ? &logits : nullptr);
  return rows;
}

// A shard of the vocabulary, in three steps: open sums (joined over the shards by the caller), finish, gradient.
std::vector<torch::Tensor> distill_open(torch::Tensor logits, torch::Tensor ids, torch::Tensor logq, OptTensor weights,
                                        OptTensor temp, double temp1, int64_t vocab_start, int64_t vocab_total) {
  check_rows(logits);
  const c10::cuda::CUDAGuard guard(logits.device());
  const int64_t U = logits.size(0), V = logits.size(1);
  auto a = distill_args(logits, ids, logq, weights, temp, temp1, 1.0, true, vocab_start, vocab_total);
  const auto f32 = logits.options().dtype(at::kFloat);
  auto stats = torch::empty({U, 2}, f32), xc = torch::empty({U, ids.size(1)}, f32);
  if (U) {
    a.V = (int)V, a.stride = logits.stride(0);
    a.stats = stats.data_ptr<float>();
    a.xc = xc.data_ptr<float>();
    a.open = true;
    check(bb::launch_distill(row_type(logits), logits.data_ptr(), nullptr, a, at::cuda::getCurrentCUDAStream()));
  }
  return {stats, xc};
}

std::vector<torch::Tensor> distill_finish(torch::Tensor stats, torch::Tensor xc, torch::Tensor ids, torch::Tensor logq,
                                          OptTensor weights, OptTensor temp, double temp1, double scale, bool tail,
                                          int64_t vocab_total) {
  TORCH_CHECK(stats.is_cuda() && stats.dim() == 2, "stats must be a CUDA matrix");
  const c10::cuda::CUDAGuard guard(stats.device());
  const int64_t U = stats.size(0), K = ids.size(1);
  auto a = distill_args(stats, ids, logq, weights, temp, temp1, scale, tail, 0, vocab_total);
  check_vec(stats, 2 * U, at::kFloat, stats, "stats must be float32 [U, 2]");
  check_vec(xc, U * K, at::kFloat, stats, "entries must be float32 [U, K]");
  auto rows = torch::empty({U}, stats.options()), coef = torch::empty({U, 2}, stats.options());
  auto fix = torch::empty({U, K}, stats.options());
  if (U) {
    a.stats = stats.data_ptr<float>();
    a.xc = xc.data_ptr<float>();
    a.rows = rows.data_ptr<float>();
    a.coef = coef.data_ptr<float>();
    a.fix = fix.data_ptr<float>();
    check(bb::launch_distill_finish(a, at::cuda::getCurrentCUDAStream()));
  }
  return {rows, coef, fix};
}

torch::Tensor distill_grad(torch::Tensor logits, torch::Tensor ids, torch::Tensor coef, torch::Tensor fix,
                           OptTensor temp, double temp1, int64_t vocab_start, int64_t vocab_total, bool inplace) {
  check_rows(logits);
  const c10::cuda::CUDAGuard guard(logits.device());
  const int64_t U = logits.size(0), V = logits.size(1), K = ids.size(1);
  auto a = distill_args(logits, ids, fix, {}, temp, temp1, 1.0, true, vocab_start, vocab_total);
  check_vec(coef, 2 * U, at::kFloat, logits, "coef must be float32 [U, 2]");
  check_vec(fix, U * K, at::kFloat, logits, "fix must be float32 [U, K]");
  TORCH_CHECK(!inplace || logits.is_contiguous(), "in-place gradients need contiguous logits");
  auto grad = inplace ? logits : torch::empty({U, V}, logits.options());
  if (U) {
    a.V = (int)V, a.stride = logits.stride(0);
    a.coef = coef.data_ptr<float>();
    a.fix = fix.data_ptr<float>();
    check(bb::launch_distill_grad(row_type(logits), logits.data_ptr(), grad.data_ptr(), a,
                                  at::cuda::getCurrentCUDAStream()));
  }
  return grad;
}

torch::Tensor weighted_rows_sum(torch::Tensor rows, OptTensor weights, double denom) {
  TORCH_CHECK(rows.is_cuda() && rows.scalar_type() == at::kFloat && rows.is_contiguous(), "rows must be float32");
  const c10::cuda::CUDAGuard guard(rows.device());
  check_vec(weights, rows.numel(), at::kFloat, rows, "weights must be float32 [U]");
  return sum_rows(rows, weights, denom);
}

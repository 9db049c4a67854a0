// Torch entry points of the kernels over rows of logits (vocab_rows.cu): argument checks, allocation, launch.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

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
  TORCH_CHECK(x.size(1) >= 1 && x.size(1) < (1l << 30) && x.size(0) < (1l << 31), "logits: size out of range");
}
void check_vec(const OptTensor& t, int64_t n, at::ScalarType dt, const torch::Tensor& x, const char* what) {
  if (!t.has_value()) return;
  TORCH_CHECK(t->device() == x.device() && t->scalar_type() == dt && t->is_contiguous() && t->numel() == n, what);
}
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
  a.temp1 = temp1, a.scale = scale;
  a.U = (int)U, a.K = (int)K;
  a.vocab_start = vocab_start, a.vocab_total = vocab_total;
  a.tail = tail;
  return a;
}

}  // namespace

std::vector<torch::Tensor> token_logprob_fwd(torch::Tensor logits, OptTensor tokens, OptTensor temp, double temp1,
                                             int64_t k, bool entropy, int64_t vocab_start, bool open) {
  check_rows(logits);
  const c10::cuda::CUDAGuard guard(logits.device());
  const int64_t U = logits.size(0), V = logits.size(1), n = tokens.has_value() ? tokens->size(1) : 0;
  check_vec(tokens, U * n, at::kLong, logits, "tokens must be int64 [U, n]");
  check_vec(temp, U, at::kFloat, logits, "temperature must be float32 [U]");
  TORCH_CHECK(k >= 0 && k <= bb::kMaxTop && k <= V, "top_k out of range");
  const auto f32 = logits.options().dtype(at::kFloat);
  auto logp = torch::empty({U, n}, f32), ent = torch::empty({entropy ? U : 0}, f32), stats = torch::empty({U, 3}, f32);
  auto ids = torch::empty({U, k}, f32.dtype(at::kLong)), top = torch::empty({U, k}, f32);
  if (U) {
    bb::TokenArgs a{};
    a.tokens = ptr<int64_t>(tokens);
    a.temp = ptr<float>(temp);
    a.temp1 = temp1;
    a.U = (int)U, a.V = (int)V, a.n = (int)n, a.k = (int)k;
    a.stride = logits.stride(0), a.vocab_start = vocab_start;
    a.logp = logp.data_ptr<float>();
    a.entropy = entropy ? ent.data_ptr<float>() : nullptr;
    a.stats = stats.data_ptr<float>();
    a.top_ids = ids.data_ptr<int64_t>();
    a.top_logp = top.data_ptr<float>();
    a.open = open;
    check(bb::launch_token_logprob(row_type(logits), logits.data_ptr(), a, at::cuda::getCurrentCUDAStream()));
  }
  return {logp, ent, stats, ids, top};
}

torch::Tensor token_logprob_bwd(torch::Tensor logits, OptTensor tokens, OptTensor temp, double temp1,
                                torch::Tensor stats, OptTensor d_logp, OptTensor d_entropy, int64_t vocab_start,
                                int64_t vocab_total) {
  check_rows(logits);
  const c10::cuda::CUDAGuard guard(logits.device());
  const int64_t U = logits.size(0), V = logits.size(1);
  const bool given = tokens.has_value() && d_logp.has_value();
  const int64_t n = given ? tokens->size(1) : 0;
  if (given) {
    check_vec(tokens, U * n, at::kLong, logits, "tokens must be int64 [U, n]");
    check_vec(d_logp, U * n, at::kFloat, logits, "d_logp must be float32 [U, n]");
  }
  check_vec(temp, U, at::kFloat, logits, "temperature must be float32 [U]");
  check_vec(stats, 3 * U, at::kFloat, logits, "stats must be float32 [U, 3]");
  check_vec(d_entropy, U, at::kFloat, logits, "d_entropy must be float32 [U]");
  auto grad = torch::empty({U, V}, logits.options());
  if (U) {
    bb::TokenArgs a{};
    a.tokens = given ? ptr<int64_t>(tokens) : nullptr;
    a.d_logp = given ? ptr<float>(d_logp) : nullptr;
    a.d_entropy = ptr<float>(d_entropy);
    a.temp = ptr<float>(temp);
    a.temp1 = temp1;
    a.U = (int)U, a.V = (int)V, a.n = (int)n;
    a.stride = logits.stride(0), a.vocab_start = vocab_start, a.vocab_total = vocab_total;
    a.stats = stats.data_ptr<float>();
    check(bb::launch_token_logprob_bwd(row_type(logits), logits.data_ptr(), grad.data_ptr(), a,
                                       at::cuda::getCurrentCUDAStream()));
  }
  return grad;
}

// Rows of a whole vocabulary: (KL [U], gradient or empty).  `inplace` writes the gradient over the logits.
std::vector<torch::Tensor> distill_rows(torch::Tensor logits, torch::Tensor ids, torch::Tensor logq, OptTensor weights,
                                        OptTensor temp, double temp1, double scale, bool tail, bool want_grad,
                                        bool inplace) {
  check_rows(logits);
  const c10::cuda::CUDAGuard guard(logits.device());
  const int64_t U = logits.size(0), V = logits.size(1);
  auto a = distill_args(logits, ids, logq, weights, temp, temp1, scale, tail, 0, V);
  TORCH_CHECK(bb::distill_smem(V) <= 200 * 1024, "distillation kernel: vocabulary above ", 200 * 1024 * 8, " tokens");
  TORCH_CHECK(!inplace || logits.is_contiguous(), "in-place gradients need contiguous logits");
  auto rows = torch::empty({U}, logits.options().dtype(at::kFloat));
  auto grad = !want_grad ? torch::empty({0, V}, logits.options())
                         : (inplace ? logits : torch::empty({U, V}, logits.options()));
  if (U) {
    a.V = (int)V, a.stride = logits.stride(0);
    a.rows = rows.data_ptr<float>();
    check(bb::launch_distill(row_type(logits), want_grad ? bb::Distill::loss_and_grad : bb::Distill::loss,
                             logits.data_ptr(), want_grad ? grad.data_ptr() : nullptr, a,
                             at::cuda::getCurrentCUDAStream()));
  }
  return {rows, grad};
}

// A shard of the vocabulary, in three steps: open sums (joined over the shards by the caller), finish, gradient.
std::vector<torch::Tensor> distill_open(torch::Tensor logits, torch::Tensor ids, torch::Tensor logq, OptTensor weights,
                                        OptTensor temp, double temp1, int64_t vocab_start, int64_t vocab_total) {
  check_rows(logits);
  const c10::cuda::CUDAGuard guard(logits.device());
  const int64_t U = logits.size(0), V = logits.size(1);
  auto a = distill_args(logits, ids, logq, weights, temp, temp1, 1.0, true, vocab_start, vocab_total);
  TORCH_CHECK(bb::distill_smem(V) <= 200 * 1024, "distillation kernel: vocabulary above ", 200 * 1024 * 8, " tokens");
  const auto f32 = logits.options().dtype(at::kFloat);
  auto stats = torch::empty({U, 2}, f32), xc = torch::empty({U, ids.size(1)}, f32);
  if (U) {
    a.V = (int)V, a.stride = logits.stride(0);
    a.stats = stats.data_ptr<float>();
    a.xc = xc.data_ptr<float>();
    check(bb::launch_distill(row_type(logits), bb::Distill::open, logits.data_ptr(), nullptr, a,
                             at::cuda::getCurrentCUDAStream()));
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
  auto out = torch::empty({}, rows.options());
  check(bb::launch_weighted_sum(rows.data_ptr<float>(), ptr<float>(weights), (int)rows.numel(), 1.0 / denom,
                                out.data_ptr<float>(), at::cuda::getCurrentCUDAStream()));
  return out;
}

void scale_unless_one(torch::Tensor x, torch::Tensor num, double den) {
  TORCH_CHECK(x.is_cuda() && x.is_contiguous() && num.device() == x.device() && num.scalar_type() == at::kFloat &&
                  num.numel() == 1,
              "scale: contiguous CUDA tensor and one float32 factor");
  if (x.numel() == 0) return;
  const c10::cuda::CUDAGuard guard(x.device());
  check(bb::launch_scale_unless_one(row_type(x), x.data_ptr(), x.numel(), num.data_ptr<float>(), (float)den,
                                    at::cuda::getCurrentCUDAStream()));
}

// Torch entry points of the adapter kernels (adapter_linear.cu): argument checks, allocation, autograd.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <algorithm>
#include <tuple>

#include "adapter_linear.h"

torch::Tensor gemm(torch::Tensor a, torch::Tensor b, bool a_mn, bool b_mn, c10::optional<torch::Tensor> out,
                   bool accumulate);

namespace {

using OptTensor = c10::optional<torch::Tensor>;
using Meta = std::vector<int64_t>;   // rows, slots, units, blocks, then where the plan's parts begin in its buffer

void check(cudaError_t e) { TORCH_CHECK(e == cudaSuccess, "CUDA error ", cudaGetErrorString(e)); }

bool aligned(const torch::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
// Rows that a tensor map can describe: unit columns, rows 16 bytes apart or a multiple of it, not on top of each other.
bool plain_rows(const torch::Tensor& t) {
  return t.dim() == 2 && t.stride(1) == 1 && aligned(t) &&
         (t.size(0) <= 1 || (t.stride(0) % 8 == 0 && t.stride(0) >= t.size(1)));
}
long row_stride(const torch::Tensor& t) { return t.size(0) <= 1 ? t.size(1) : t.stride(0); }
torch::Tensor as_rows(const torch::Tensor& t) {
  return plain_rows(t) ? t : t.clone(at::MemoryFormat::Contiguous);
}

bb::AdapterPlan plan_of(const torch::Tensor& buf, const Meta& meta) {
  const int* p = buf.data_ptr<int>();
  return {p + meta[4], p + meta[5], p + meta[6], p + meta[7], p + meta[8], p + meta[9], p + meta[10],
          (int)meta[2], (int)meta[3], (int)meta[1]};
}

struct Sizes {
  int T, K, N, S, R;
  bool half;
  explicit Sizes(const torch::Tensor& x, const torch::Tensor& a, const torch::Tensor& b)
      : T((int)x.size(0)), K((int)a.size(2)), N((int)b.size(1)), S((int)a.size(0)), R((int)a.size(1)),
        half(a.scalar_type() == at::kHalf) {}
};

struct Products {
  torch::Tensor u, y;      // undefined where not asked for
};

// u = scale A x and y = W x + B u from (x, W, A, B); with `mn` du = scale B^T dy and dx = W^T dy + A^T du from
// (dy, W, B, A).  u is for the gradients, in two parts.
Products products(const torch::Tensor& x, const torch::Tensor& w, const torch::Tensor& op, const torch::Tensor& low, bool mn,
                  bool want_u, bool want_y, const torch::Tensor& buf, const Meta& meta, double scale,
                  const OptTensor& scales) {
  bb::AdapterProduct a{};
  a.mn = mn, a.keep_u = want_u;
  a.T = (int)x.size(0), a.K = (int)x.size(1), a.N = (int)w.size(mn ? 1 : 0);
  a.S = (int)op.size(0), a.R = (int)op.size(mn ? 2 : 1);
  a.half = op.scalar_type() == at::kHalf;
  a.x = x.data_ptr(), a.op = op.data_ptr(), a.w = w.data_ptr(), a.low = low.data_ptr();
  a.ldx = row_stride(x), a.ldw = row_stride(w);
  a.scale = (float)scale;
  a.scales = scales.has_value() ? scales->data_ptr<float>() : nullptr;
  a.plan = plan_of(buf, meta);
  const auto opts = op.options().requires_grad(false);
  const auto stream = at::cuda::getCurrentCUDAStream();
  const bb::AdapterNeeds needs = want_y ? bb::adapter_product_needs(a) : bb::AdapterNeeds{true, 0};
  Products out;
  if (needs.u) {
    out.u = at::empty({want_u ? 2 : 1, a.T, a.R}, opts);
    a.u = out.u.data_ptr();
  }
  if (!want_y) {
    check(bb::launch_adapter_shrink(a, stream));
    return out;
  }
  out.y = at::empty({a.T, a.N}, opts);
  a.y = out.y.data_ptr();
  torch::Tensor sums;      // the call's own: two of them may run at once
  if (needs.workspace) {
    sums = at::empty({(int64_t)needs.workspace}, opts.dtype(at::kByte));
    a.workspace = sums.data_ptr();
  }
  check(bb::launch_adapter_product(a, stream));
  return out;
}

void first_order() {
  TORCH_CHECK(!at::GradMode::is_enabled(),
              "adapter_linear has no second derivative (backward was called with create_graph=True)");
}

class AdapterLinear : public torch::autograd::Function<AdapterLinear> {
 public:
  static torch::Tensor forward(torch::autograd::AutogradContext* ctx, const torch::Tensor& x, const torch::Tensor& w,
                               const torch::Tensor& a, const torch::Tensor& b, const torch::Tensor& buf,
                               const Meta& meta, double scale, const OptTensor& scales, const OptTensor& a_main,
                               const OptTensor& b_main, const OptTensor& w_main) {
    const c10::cuda::CUDAGuard guard(x.device());
    torch::Tensor u, y;
    if (x.size(0)) {
      const Products out = products(x, w, a, b, false, true, true, buf, meta, scale, scales);
      u = out.u, y = out.y;
    } else {
      u = at::empty({0, a.size(1)}, a.options().requires_grad(false));
      y = at::empty({0, w.size(0)}, a.options().requires_grad(false));
    }
    const torch::Tensor none;
    ctx->save_for_backward({x, w, a, b, u, buf, scales.value_or(none)});
    ctx->saved_data["meta"] = meta;
    ctx->saved_data["scale"] = scale;
    if (a_main.has_value()) ctx->saved_data["a_main"] = *a_main;
    if (b_main.has_value()) ctx->saved_data["b_main"] = *b_main;
    if (w_main.has_value()) ctx->saved_data["w_main"] = *w_main;
    return y;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    first_order();
    const auto saved = ctx->get_saved_variables();
    const torch::Tensor &x = saved[0], &w = saved[1], &a = saved[2], &b = saved[3], &u = saved[4], &buf = saved[5];
    const OptTensor scales = saved[6].defined() ? OptTensor(saved[6]) : OptTensor();
    const Meta meta = ctx->saved_data["meta"].toIntVector();
    const double scale = ctx->saved_data["scale"].toDouble();
    const auto main = [&](const char* name) {
      const auto at = ctx->saved_data.find(name);
      return at == ctx->saved_data.end() ? OptTensor() : OptTensor(at->second.toTensor());
    };
    const OptTensor a_main = main("a_main"), b_main = main("b_main"), w_main = main("w_main");
    const c10::cuda::CUDAGuard guard(x.device());
    const bool want_x = ctx->needs_input_grad(0), want_w = ctx->needs_input_grad(1), want_a = ctx->needs_input_grad(2),
               want_b = ctx->needs_input_grad(3);
    const torch::Tensor none;
    torch::Tensor dx, dw, da, db;
    if (x.size(0) == 0) {
      if (want_x) dx = at::empty(x.sizes(), a.options().requires_grad(false));
      if (want_w && !w_main.has_value()) dw = at::zeros(w.sizes(), a.options().requires_grad(false));
      if (want_a && !a_main.has_value()) da = at::zeros(a.sizes(), a.options().requires_grad(false));
      if (want_b && !b_main.has_value()) db = at::zeros(b.sizes(), a.options().requires_grad(false));
      return {dx, dw, da, db, none, none, none, none, none, none, none};
    }
    const auto dy = as_rows(grads[0]);
    torch::Tensor du;
    if (want_x || want_a) {
      const Products out = products(dy, w, b, a, true, want_a, want_x, buf, meta, scale, scales);
      du = out.u, dx = out.y;
    }
    if (want_w) {
      const auto rows = [](const torch::Tensor& t) { return t.as_strided(t.sizes(), {row_stride(t), 1}); };
      if (w_main.has_value()) gemm(rows(dy), rows(x), true, true, w_main, true);
      else dw = gemm(rows(dy), rows(x), true, true, c10::nullopt, false);
    }
    if (want_a || want_b) {
      const Sizes n(x, a, b);
      bb::AdapterGrads g{};
      if (want_a) {
        if (!a_main.has_value()) da = at::empty(a.sizes(), a.options().requires_grad(false));
        g.da = a_main.has_value() ? a_main->data_ptr() : da.data_ptr();
        g.add_a = a_main.has_value();
        g.du = du.data_ptr();
      }
      if (want_b) {
        if (!b_main.has_value()) db = at::empty(b.sizes(), b.options().requires_grad(false));
        g.db = b_main.has_value() ? b_main->data_ptr() : db.data_ptr();
        g.add_b = b_main.has_value();
        g.u = u.data_ptr();
      }
      g.x = x.data_ptr(), g.dy = dy.data_ptr();
      g.ldx = row_stride(x), g.lddy = row_stride(dy);
      g.T = n.T, g.K = n.K, g.N = n.N, g.S = n.S, g.R = n.R, g.half = n.half;
      g.plan = plan_of(buf, meta);
      check(bb::launch_adapter_grads(g, at::cuda::getCurrentCUDAStream()));
    }
    return {dx, dw, da, db, none, none, none, none, none, none, none};
  }
};

// A plan lies inside an object that its owner may let go while kernels of another stream than the one it was made on still
// read it: its memory is not handed out again before they are done.  (One that a graph is captured with has to be kept.)
void read_by(const torch::Tensor& buf, const at::cuda::CUDAStream& stream) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  check(cudaStreamIsCapturing(stream, &status));
  if (status == cudaStreamCaptureStatusNone)
    c10::cuda::CUDACachingAllocator::recordStream(buf.storage().data_ptr(), stream);
}

bool main_fits(const OptTensor& m, const torch::Tensor& p) {
  return !m.has_value() || (m->scalar_type() == at::kFloat && m->is_contiguous() && m->numel() == p.numel() &&
                            m->device() == p.device() && aligned(*m));
}

}  // namespace

// y [T, N]; undefined where the arguments are not in the form that the kernels take.
torch::Tensor adapter_linear(torch::Tensor x, torch::Tensor w, torch::Tensor a, torch::Tensor b, torch::Tensor buf,
                             Meta meta, double scale, OptTensor scales, OptTensor a_main, OptTensor b_main,
                             OptTensor w_main) {
  const auto type = x.scalar_type();
  const auto like_x = [&](const torch::Tensor& t) { return t.scalar_type() == type && t.device() == x.device(); };
  const bool fits =
      x.is_cuda() && (type == at::kBFloat16 || type == at::kHalf) && x.dim() == 2 && w.dim() == 2 && a.dim() == 3 &&
      b.dim() == 3 && like_x(w) && like_x(a) && like_x(b) && x.size(1) == w.size(1) && a.size(2) == x.size(1) &&
      b.size(1) == w.size(0) && a.size(0) == b.size(0) && a.size(1) == b.size(2) && a.size(0) >= 1 && x.size(1) >= 8 &&
      w.size(0) >= 8 && a.size(1) >= 8 && x.size(1) % 8 == 0 && w.size(0) % 8 == 0 && a.size(1) % 8 == 0 &&
      a.size(1) <= bb::kMaxAdapterRank && x.size(0) < (1l << 30) && x.size(1) < (1l << 30) && w.size(0) < (1l << 30) &&
      a.size(0) < (1l << 16) && plain_rows(x) && plain_rows(w) && a.is_contiguous() && aligned(a) &&
      b.is_contiguous() && aligned(b) && meta.size() == 11 && meta[0] == x.size(0) && meta[1] <= a.size(0) &&
      buf.device() == x.device() && buf.scalar_type() == at::kInt && buf.is_contiguous() &&
      (!scales.has_value() || (scales->dim() == 1 && scales->size(0) == a.size(0) && scales->is_contiguous() &&
                               scales->scalar_type() == at::kFloat && scales->device() == x.device() &&
                               !scales->requires_grad())) &&
      !(w.requires_grad() && type == at::kHalf) && main_fits(a_main, a) && main_fits(b_main, b) && main_fits(w_main, w);
  if (!fits) return {};
  for (const auto& t : {x, w, a, b})
    TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), "adapter_linear has no forward-mode derivative");
  const c10::cuda::CUDAGuard guard(x.device());
  if (x.size(0)) read_by(buf, at::cuda::getCurrentCUDAStream());
  if (at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad() || a.requires_grad() || b.requires_grad()))
    return AdapterLinear::apply(x, w, a, b, buf, meta, scale, scales, a_main, b_main, w_main);
  if (x.size(0) == 0) return at::empty({0, w.size(0)}, x.options().requires_grad(false));
  return products(x, w, a, b, false, false, true, buf, meta, scale, scales).y;
}

// The plan of a batch on `device`, laid out as ops/adapter.py's _lay_out says (which makes the same without CUDA), and
// its meta.  The copy is complete when this returns: kernels read a plan before they wait for the stream.
std::tuple<torch::Tensor, Meta> adapter_plan(const std::vector<int64_t>& cu, const std::vector<int64_t>& slots,
                                             const torch::Device& device) {
  const int64_t rows = cu.back(), tiles = (rows + 255) / 256;
  const int64_t top = slots.empty() ? 0 : *std::max_element(slots.begin(), slots.end()) + 1;
  struct Pair {
    int32_t slot;
    uint32_t off[8];
  };
  struct Block {
    int32_t row, n;
  };
  std::vector<int32_t> row_slot(rows), tile_start{0}, unit_start{0}, units;
  std::vector<Pair> pairs;
  std::vector<int64_t> seen(top, -1);              // tile in which a slot was met last
  std::vector<std::vector<Block>> blocks(top);
  int64_t open = -1, begin = 0;                    // the run of rows of one slot that is under way
  const auto close = [&](int64_t end) {
    for (int64_t r = begin; open >= 0 && r < end; r += 64)
      blocks[open].push_back({(int32_t)r, (int32_t)std::min<int64_t>(64, end - r)});
  };
  for (size_t i = 0; i < slots.size(); ++i) {
    if (cu[i] == cu[i + 1]) continue;
    std::fill(row_slot.begin() + cu[i], row_slot.begin() + cu[i + 1], (int32_t)slots[i]);
    if (slots[i] != open) close(cu[i]), open = slots[i], begin = cu[i];
  }
  close(rows);
  for (int64_t t = 0; t < tiles; ++t) {
    const int64_t lo = t * 256, hi = std::min(rows, lo + 256);
    std::vector<int32_t> here;
    for (int64_t r = lo; r < hi; ++r)
      if (const int32_t s = row_slot[r]; s >= 0 && seen[s] != t) seen[s] = t, here.push_back(s);
    std::sort(here.begin(), here.end());
    const size_t first = pairs.size();
    for (const int32_t s : here) {
      Pair p{s, {}};
      std::fill(p.off, p.off + 8, 0xffffffffu);
      pairs.push_back(p);
    }
    for (int64_t r = lo; r < hi; ++r)
      if (const int32_t s = row_slot[r]; s >= 0) {
        const size_t at = first + (std::lower_bound(here.begin(), here.end(), s) - here.begin());
        pairs[at].off[(r - lo) / 32] &= ~(1u << ((r - lo) % 32));
      }
    tile_start.push_back((int32_t)pairs.size());
    for (int half = 0; half < 2; ++half) {
      for (size_t k = first; k < pairs.size(); ++k) {
        const uint32_t* off = pairs[k].off + 4 * half;
        if ((off[0] & off[1] & off[2] & off[3]) == 0xffffffffu) continue;
        units.insert(units.end(), {(int32_t)(2 * t + half), pairs[k].slot, 0, 0});
        for (int w = 0; w < 4; ++w) units.push_back((int32_t)off[w]);
      }
      unit_start.push_back((int32_t)(units.size() / 8));
    }
  }
  std::vector<int32_t> flat;
  Meta meta{rows, top, (int64_t)units.size() / 8, 0};
  const auto begin_part = [&] {
    flat.resize((flat.size() + 3) / 4 * 4);        // each part begins at 16 bytes
    meta.push_back((int64_t)flat.size());
  };
  const auto part = [&](const std::vector<int32_t>& v) {
    begin_part();
    flat.insert(flat.end(), v.begin(), v.end());
  };
  part(row_slot);
  part(tile_start);
  begin_part();
  for (const Pair& p : pairs) {
    flat.insert(flat.end(), {p.slot, 0, 0, 0});
    for (const uint32_t w : p.off) flat.push_back((int32_t)w);
  }
  part(unit_start);
  part(units);
  std::vector<int32_t> block_start{0}, list;
  for (int64_t s = 0; s < top; ++s) {
    for (const Block& b : blocks[s]) list.insert(list.end(), {b.row, b.n, (int32_t)s, 0});
    block_start.push_back((int32_t)(list.size() / 4));
  }
  meta[3] = (int64_t)list.size() / 4;
  part(block_start);
  part(list);
  flat.resize((flat.size() + 3) / 4 * 4);
  const auto host = torch::from_blob(flat.data(), {(int64_t)flat.size()}, at::kInt);
  return {host.to(device, /*non_blocking=*/false, /*copy=*/true), meta};
}

int64_t adapter_error_code() { return bb::adapter_error_code(); }

// torch bindings of the embedding, block-norm and gradient-norm kernels.  Every entry checks
// what the kernel assumes, makes the tensors' device current and launches on its current stream.
#include "training_ops.h"

#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <algorithm>
#include <vector>

#include "kernels.h"

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef c10::optional<at::Tensor> Opt;

int dt_code(const at::Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat:
      return smpk::F32;
    case at::kHalf:
      return smpk::F16;
    case at::kBFloat16:
      return smpk::BF16;
    default:
      TORCH_CHECK(false, name, ": unsupported dtype ", t.scalar_type());
  }
  return -1;
}

hipStream_t stream() { return at::hip::getCurrentHIPStream().stream(); }

void check(int rc, const char* what) { TORCH_CHECK(rc == 0, what, " launch failed with code ", rc); }

// A tensor that is its memory and nothing else, as the kernels take it.  Not so: dual numbers, the
// tensors of function transforms (vmap, torch.func) and of classes that dispatch operations themselves
// (fake or distributed ones), lazily negated and zero tensors.
bool plain(const at::Tensor& t, bool duals) {
  using Key = c10::DispatchKey;
  static const c10::DispatchKeySet other({Key::Python, Key::Batched, Key::FuncTorchBatched, Key::FuncTorchGradWrapper,
                                          Key::BatchedNestedTensor, Key::Functionalize, Key::Conjugate, Key::Negative,
                                          Key::ZeroTensor});
  return !t.key_set().has_any(other) && !t.is_nested() && !(duals && t._fw_grad(/*level=*/0).defined());
}

// There may be dual numbers: asked once a call, a tensor's own tangent takes a lock.
bool duals_live() { return torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr; }

// No trace, mode or function transform is active, which would have to know of the launch.
bool unobserved() {
  return !torch::jit::tracer::isTracing() && !c10::impl::TorchDispatchModeTLS::any_modes_set() &&
         !c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::FuncTorchDynamicLayerFrontMode);
}

// ------------------------------------------------------------------- embedding
smpk::IndexList index_list(const c10::optional<at::Tensor>& ids, int64_t n, int64_t start, int64_t rows,
                           int64_t period, const at::Tensor& like) {
  smpk::IndexList l;
  l.start = start;
  l.rows = rows;
  l.period = period < 1 ? 1 : period;
  if (ids.has_value()) {
    TORCH_CHECK(ids->device() == like.device() && ids->is_contiguous() && ids->numel() == n, "embedding: bad ids");
    TORCH_CHECK(ids->scalar_type() == at::kLong || ids->scalar_type() == at::kInt, "embedding: ids int32 or int64");
    l.ids = ids->data_ptr();
    l.wide = ids->scalar_type() == at::kLong;
  }
  return l;
}

void check_table_dims(const at::Tensor& w) {
  TORCH_CHECK(w.is_cuda() && w.dim() == 2, "embedding: a table must be a GPU matrix");
}

// Elements of a row one after the other (of one element: whatever its stride says).
bool rows_dense(const at::Tensor& w) { return w.stride(1) == 1 || w.size(1) == 1; }

void check_table(const at::Tensor& w) {
  TORCH_CHECK(w.is_cuda() && w.dim() == 2 && rows_dense(w) && w.size(1) < (1ll << 31), "embedding: bad table");
}

// n tokens: ids (or, for the positions, none: t % period) into w [rows, d], rows dense along d
at::Tensor embedding_fwd(at::Tensor ids, at::Tensor weight, double scale, int64_t start, bool foreign_zero,
                         c10::optional<at::Tensor> pos, c10::optional<at::Tensor> pos_weight, int64_t period) {
  check_table(weight);
  const c10::DeviceGuard guard(weight.device());
  const int64_t n = ids.numel(), d = weight.size(1);
  if (pos_weight.has_value()) {
    check_table(*pos_weight);
    TORCH_CHECK(pos_weight->size(1) == d && pos_weight->scalar_type() == weight.scalar_type() &&
                    pos_weight->device() == weight.device(),
                "embedding: the position table differs from the token table");
  }
  const auto li = index_list(ids, n, start, weight.size(0), 1, weight);
  smpk::IndexList lp;
  if (pos_weight.has_value()) lp = index_list(pos, n, 0, pos_weight->size(0), period, weight);
  auto y = at::empty({n, d}, weight.options());
  check(smpk::embedding_fwd(dt_code(weight, "weight"), li, weight.data_ptr(), weight.stride(0),
                            static_cast<float>(scale), foreign_zero ? 1 : 0, lp,
                            pos_weight.has_value() ? pos_weight->data_ptr() : nullptr,
                            pos_weight.has_value() ? pos_weight->stride(0) : 0, y.data_ptr(), n, d, stream()),
        "embedding_fwd");
  return y;
}

// Gradients of the token table (ids, scale, start, skip) and of the position table (pos or, without
// them, t % period): rows x d tensors of dy's type.  dw / dp: written, or added to (accumulate);
// null: not wanted.
void embedding_bwd(at::Tensor dy, at::Tensor ids, c10::optional<at::Tensor> pos, int64_t period, double scale,
                   int64_t start, int64_t skip, c10::optional<at::Tensor> dw, bool dw_accumulate,
                   c10::optional<at::Tensor> dp, bool dp_accumulate) {
  const c10::DeviceGuard guard(dy.device());
  TORCH_CHECK(dy.is_cuda() && dy.dim() == 2 && dy.is_contiguous(), "embedding: bad dy");
  const int64_t n = dy.size(0), d = dy.size(1);
  TORCH_CHECK(n <= (1ll << 27), "embedding: more than 2^27 tokens");
  smpk::EmbeddingGrad t[2];
  int count = 0;
  int64_t bytes = 0;
  int64_t at[2][5];  // keys, tokens, counts, part, marks in the workspace
  bool brief = true;
  for (int i = 0; i < 2; ++i) {
    const auto& g = i == 0 ? dw : dp;
    if (!g.has_value()) continue;
    brief = brief && smpk::embedding_bwd_short(n, d, g->size(0), (i == 0 ? dw_accumulate : dp_accumulate) ? 0 : g->nbytes());
  }
  for (int i = 0; i < 2; ++i) {
    const auto& g = i == 0 ? dw : dp;
    if (!g.has_value()) continue;
    TORCH_CHECK(g->dim() == 2 && g->is_contiguous() && g->size(1) == d && g->scalar_type() == dy.scalar_type() &&
                    g->device() == dy.device() && g->size(0) < (1ll << 31) - 1,
                "embedding: bad gradient");
    smpk::EmbeddingGrad& e = t[count];
    const int64_t rows = g->size(0);
    const bool sequence = i == 1 && !pos.has_value();
    if (sequence)
      TORCH_CHECK(period >= 1 && n % period == 0 && period <= rows, "embedding: no whole sequences of positions");
    e.ids = i == 0 ? index_list(ids, n, start, rows, 1, dy) : index_list(pos, n, 0, rows, period, dy);
    e.scale = i == 0 ? static_cast<float>(scale) : 1.f;
    e.skip = i == 0 ? skip : -1;
    e.dw = g->data_ptr();
    e.accumulate = i == 0 ? dw_accumulate : dp_accumulate;
    if (brief) {
      ++count;
      continue;
    }
    e.plan = smpk::embedding_bwd_plan(n, d, rows, sequence ? std::max<int64_t>(n / period, 1) : 0);
    const bool sort = !sequence && n > 0;
    const int64_t lists = e.plan.one_launch ? 4 * n : 8 * n;
    const int64_t size[5] = {sort ? lists : 0, sort ? lists : 0, sort && !e.plan.one_launch ? e.plan.sort_blocks << (e.plan.bits + 2) : 0,
                             e.plan.join ? e.plan.chunks * 8 * d : 0, sort && !e.accumulate ? rows : 0};
    for (int k = 0; k < 5; ++k) {
      at[count][k] = bytes;
      bytes += (size[k] + 15) / 16 * 16;
    }
    ++count;
  }
  if (count == 0) return;
  if (brief) {
    check(smpk::embedding_bwd_of_short(dt_code(dy, "embedding"), dy.data_ptr(), n, d, t, count, stream()), "embedding_bwd");
    return;
  }
  auto ws = at::empty({bytes}, dy.options().dtype(at::kByte));
  uint8_t* const base = ws.data_ptr<uint8_t>();
  for (int i = 0; i < count; ++i) {
    t[i].keys = reinterpret_cast<uint32_t*>(base + at[i][0]);
    t[i].tokens = reinterpret_cast<int32_t*>(base + at[i][1]);
    t[i].counts = reinterpret_cast<int32_t*>(base + at[i][2]);
    t[i].part = reinterpret_cast<float*>(base + at[i][3]);
    t[i].marks = base + at[i][4];
  }
  check(smpk::embedding_bwd(dt_code(dy, "embedding"), dy.data_ptr(), n, d, t, count, stream()), "embedding_bwd");
}

// backward() will add the gradient of the leaf `t` to t.grad.  Not so torch.autograd.grad, which returns
// it, nor a pass that builds a graph, whose sum has to be part of that graph.
bool accumulates(const at::Tensor& t) {
  if (at::GradMode::is_enabled()) return false;
  const auto* info = torch::autograd::get_current_graph_task_exec_info();
  if (info == nullptr || info->empty()) return true;
  const auto it = info->find(torch::autograd::impl::try_get_grad_accumulator(t).get());
  return it != info->end() && it->second.needed_ && !it->second.captures_;
}

// Something other than the sum into t.grad wants the gradient of the leaf `t`: a hook of the tensor
// or of its accumulator, which may change it before it is added.
bool hooked(const at::Tensor& t) {
  if (!torch::autograd::impl::hooks(t).empty()) return true;
  const auto accumulator = torch::autograd::impl::try_get_grad_accumulator(t);
  return accumulator && !(accumulator->pre_hooks().empty() && accumulator->post_hooks().empty());
}

// The sum into t.grad belongs on the stream that was current when the accumulator of the leaf `t` was made,
// and autograd makes the caller wait for that stream alone.  A node of another stream returns its gradient,
// which autograd brings there.
bool here(const at::Tensor& t) {
  const auto accumulator = torch::autograd::impl::try_get_grad_accumulator(t);
  const auto of_leaf = accumulator ? accumulator->stream() : std::nullopt;
  return !of_leaf.has_value() || of_leaf->id() == at::hip::getCurrentHIPStream(t.device().index()).id();
}

// The gradient of `t` goes straight into its bound slot of the flat buffer: the caller saw the
// parameter's mark, the slot has to be there still.
bool bound(const at::Tensor& t, bool marked) {
  if (!marked || !t.defined() || !t.is_leaf() || hooked(t) || !here(t)) return false;
  const at::Tensor& g = t.grad();
  return g.defined() && g.scalar_type() == t.scalar_type() && g.sizes() == t.sizes() && g.is_contiguous() &&
         accumulates(t);
}

// Autograd takes a leaf's gradient on the stream that was current when the leaf's accumulator was made.
// If that is the default stream, as where an eager graph of the leaf is alive, no capture can include it:
// an error here, before autograd tries, which would end the process.
void check_capture(at::ArrayRef<at::Tensor> inputs, const char* name) {
  if (stream() == nullptr) return;  // the default stream: never captured
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  TORCH_CHECK(hipStreamIsCapturing(stream(), &status) == hipSuccess, name, ": the stream's capture is invalid");
  if (status == hipStreamCaptureStatusNone) return;
  for (const at::Tensor& t : inputs) {
    if (!t.defined() || !t.is_leaf() || !t.requires_grad()) continue;
    const auto accumulator = torch::autograd::impl::try_get_grad_accumulator(t);
    const auto at = accumulator ? accumulator->stream() : std::nullopt;
    TORCH_CHECK(!at.has_value() || at->id() != 0, name,
                ": this backward pass is captured while a graph of the same parameters, made on the default stream, is "
                "alive: drop that graph first (its outputs and losses), or make it on another stream");
  }
}

at::Tensor embedding(at::Tensor weight, Opt pos_weight, at::Tensor ids, Opt pos, double scale, int64_t start,
                     bool foreign_zero, int64_t skip, bool mark_w, bool mark_p);

// The gradients of both tables as functions of dy, for passes that build a graph: linear in dy, so the
// derivative is a lookup in the tables' second gradients, and that can be differentiated again.
class EmbeddingGradFunction : public torch::autograd::Function<EmbeddingGradFunction> {
 public:
  // {dw, dp}, those of w_shape / p_shape that are not empty
  static variable_list forward(AutogradContext* ctx, const at::Tensor& dy, const at::Tensor& ids, const Opt& pos,
                               int64_t period, double scale, int64_t start, int64_t skip,
                               std::vector<int64_t> w_shape, std::vector<int64_t> p_shape) {
    ctx->save_for_backward({ids, pos.has_value() ? *pos : at::Tensor()});
    ctx->saved_data["args"] = std::vector<int64_t>{period, start, skip, !w_shape.empty(), !p_shape.empty()};
    ctx->saved_data["scale"] = scale;
    Opt dw, dp;
    variable_list out;
    if (!w_shape.empty()) out.push_back(*(dw = at::empty(w_shape, dy.options())));
    if (!p_shape.empty()) out.push_back(*(dp = at::empty(p_shape, dy.options())));
    embedding_bwd(dy, ids, pos, period, scale, start, skip, dw, false, dp, false);
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto args = ctx->saved_data["args"].toIntVector();
    const bool has_w = args[3], has_p = args[4];
    Opt gp, pos;
    if (has_p) gp = grads.back();
    at::Tensor gw = has_w ? grads[0] : at::zeros({1, gp->size(1)}, gp->options());
    const int64_t d = gw.size(1), skip = args[2];
    if (has_w && skip >= 0 && skip < gw.size(0))  // the row that takes no gradient passes none on
      gw = at::cat({gw.narrow(0, 0, skip), at::zeros({1, d}, gw.options()),
                    gw.narrow(0, skip + 1, gw.size(0) - skip - 1)});
    const at::Tensor ids = has_p ? saved[0].view({-1, args[0]}) : saved[0];
    if (has_p && saved[1].defined()) pos = saved[1].view(ids.sizes());
    variable_list out(9);
    out[0] = embedding(gw, gp, ids, pos, ctx->saved_data["scale"].toDouble(), args[1], true, has_w ? skip : -1, false,
                       false).view({-1, d});
    return out;
  }
};

// Both gradients by torch's operations, which see to duals, batches and graphs of a dy that is not plain:
// added up in fp32 and rounded once.
at::Tensor table_gradient(const at::Tensor& dy, const at::Tensor& ids, at::IntArrayRef shape, double scale, int64_t start,
                          int64_t skip) {
  const at::Tensor row = ids.to(at::kLong) - start;
  const at::Tensor other = (row < 0).logical_or(row >= shape[0]).logical_or(row == (skip < 0 ? shape[0] : skip));
  const at::Tensor sum = at::zeros(shape, ids.options().dtype(at::kFloat))
                             .index_add(0, row.masked_fill(other, 0), dy.to(at::kFloat).masked_fill(other.unsqueeze(1), 0));
  return (sum * scale).to(dy.scalar_type());
}

// Autograd's nodes are C++: a short call's time is the host's, and the backward needs no interpreter.
class EmbeddingFunction : public torch::autograd::Function<EmbeddingFunction> {
 public:
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& weight, const Opt& pos_weight,
                            const at::Tensor& ids, const Opt& pos, int64_t period, double scale, int64_t start,
                            bool foreign_zero, int64_t skip, bool mark_w, bool mark_p) {
    // the tables' values are not needed again: they may change before the backward
    ctx->saved_data["weight"] = weight;
    if (pos_weight.has_value()) ctx->saved_data["pos_weight"] = *pos_weight;
    ctx->save_for_backward({ids, pos.has_value() ? *pos : at::Tensor()});
    ctx->saved_data["args"] = std::vector<int64_t>{period, start, skip, mark_w, mark_p};
    ctx->saved_data["scale"] = scale;
    return embedding_fwd(ids, weight, scale, start, foreign_zero, pos, pos_weight, period);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto args = ctx->saved_data["args"].toIntVector();
    const double scale = ctx->saved_data["scale"].toDouble();
    const at::Tensor w = ctx->saved_data["weight"].toTensor();
    const bool two = ctx->saved_data.count("pos_weight") != 0;
    const at::Tensor p = two ? ctx->saved_data["pos_weight"].toTensor() : at::Tensor();
    check_capture({w, p}, "embedding");
    variable_list out(11);
    if (!plain(grads[0], duals_live())) {
      const at::Tensor dy = grads[0].reshape({-1, w.size(1)});
      const at::Tensor place =
          saved[1].defined() ? saved[1] : at::arange(dy.size(0), saved[0].options()).remainder(args[0]);
      if (ctx->needs_input_grad(0)) out[0] = table_gradient(dy, saved[0], w.sizes(), scale, args[1], args[2]);
      if (two && ctx->needs_input_grad(1)) out[1] = table_gradient(dy, place, p.sizes(), 1.0, 0, -1);
      return out;
    }
    const at::Tensor dy = grads[0].reshape({-1, w.size(1)}).contiguous();
    Opt dw, dp, pos;
    if (saved[1].defined()) pos = saved[1];
    if (at::GradMode::is_enabled() && dy.requires_grad()) {
      std::vector<int64_t> w_shape, p_shape;
      if (ctx->needs_input_grad(0)) w_shape = w.sizes().vec();
      if (two && ctx->needs_input_grad(1)) p_shape = p.sizes().vec();
      size_t k = 0;
      const auto g = EmbeddingGradFunction::apply(dy, saved[0], pos, args[0], scale, args[1], args[2], w_shape, p_shape);
      if (!w_shape.empty()) out[0] = g[k++];
      if (!p_shape.empty()) out[1] = g[k++];
      return out;
    }
    bool add_w = false, add_p = false;
    auto target = [&](const at::Tensor& t, bool marked, Opt& g, bool& add, at::Tensor& result) {
      add = bound(t, marked);
      g = add ? t.grad() : at::empty(t.sizes(), t.options());
      if (add) {
        torch::autograd::impl::bump_version(*g);
      } else {
        result = *g;
      }
    };
    if (ctx->needs_input_grad(0)) target(w, args[3], dw, add_w, out[0]);
    if (two && ctx->needs_input_grad(1)) target(p, args[4], dp, add_p, out[1]);
    if (add_w && add_p && dw->data_ptr() == dp->data_ptr()) {  // one parameter as both tables: one after the other
      embedding_bwd(dy, saved[0], pos, args[0], scale, args[1], args[2], dw, true, c10::nullopt, false);
      embedding_bwd(dy, saved[0], pos, args[0], scale, args[1], args[2], c10::nullopt, false, dp, true);
    } else {
      embedding_bwd(dy, saved[0], pos, args[0], scale, args[1], args[2], dw, add_w, dp, add_p);
    }
    return out;
  }
};

// scale * weight[ids - start] (+ pos_weight[pos]) -> [*ids.shape, dim], differentiable in both tables
at::Tensor embedding(at::Tensor weight, Opt pos_weight, at::Tensor ids, Opt pos, double scale, int64_t start,
                     bool foreign_zero, int64_t skip, bool mark_w, bool mark_p) {
  check_table_dims(weight);
  auto dense = [](const at::Tensor& t) { return rows_dense(t) ? t : t.contiguous(); };
  auto shape = ids.sizes().vec();
  shape.push_back(weight.size(1));
  const int64_t period = pos_weight.has_value() && !pos.has_value() ? std::max<int64_t>(ids.size(-1), 1) : 1;
  const at::Tensor flat = ids.reshape({-1}).contiguous();
  if (pos.has_value()) pos = pos->reshape({-1}).contiguous();
  weight = dense(weight);
  if (pos_weight.has_value()) {
    check_table_dims(*pos_weight);
    pos_weight = dense(*pos_weight);
  }
  const bool grad = at::GradMode::is_enabled() &&
                    (weight.requires_grad() || (pos_weight.has_value() && pos_weight->requires_grad()));
  if (!grad) return embedding_fwd(flat, weight, scale, start, foreign_zero, pos, pos_weight, period).view(shape);
  return EmbeddingFunction::apply(weight, pos_weight, flat, pos, period, scale, start, foreign_zero, skip, mark_w, mark_p)
      .view(shape);
}

// None where the kernels do not take the call: the caller has the same in torch's operations
Opt embedding_call(at::Tensor weight, Opt pos_weight, at::Tensor ids, Opt pos, double scale, int64_t start,
                   bool foreign_zero, int64_t skip, bool mark_w, bool mark_p) {
  const bool duals = duals_live();
  bool take = unobserved() && plain(weight, duals) && plain(ids, duals);
  for (const Opt* t : {&pos_weight, &pos}) take = take && (!t->has_value() || plain(**t, duals));
  if (!take) return c10::nullopt;
  return embedding(weight, pos_weight, ids, pos, scale, start, foreign_zero, skip, mark_w, mark_p);
}

// ------------------------------------------------------------------ block norm

const void* ptr(const Opt& t) { return t.has_value() ? t->data_ptr() : nullptr; }

// Arguments that the forward and the backward share, checked.
smpk::BlockNormArgs block_args(const Opt& x, const at::Tensor& res, const at::Tensor& w, const Opt& b, const Opt& pw,
                               const Opt& pb, const Opt& gate, int64_t gate_rows, double alpha, double eps, bool rms) {
  TORCH_CHECK(res.is_cuda() && res.dim() >= 1 && res.is_contiguous(), "block_norm: rows must be dense");
  const int64_t d = res.size(-1);
  TORCH_CHECK(d >= 1 && d <= 16384, "block_norm: width ", d, " is not within 1 .. 16384");
  const int64_t rows = res.numel() / d;
  dt_code(res, "block_norm");
  auto like = [&](const Opt& t) {
    return !t.has_value() || (t->device() == res.device() && t->is_contiguous() && t->sizes() == res.sizes() &&
                              t->scalar_type() == res.scalar_type());
  };
  TORCH_CHECK(like(x), "block_norm: x differs from the residual");
  auto vec = [&](const Opt& t) {
    return !t.has_value() || (t->device() == res.device() && t->is_contiguous() && t->numel() == d &&
                              t->scalar_type() == w.scalar_type());
  };
  TORCH_CHECK(w.scalar_type() == res.scalar_type() || w.scalar_type() == at::kFloat, "block_norm: weight dtype");
  TORCH_CHECK(vec(w) && vec(b) && vec(pw) && vec(pb), "block_norm: weights and biases must be alike");
  if (gate.has_value()) {
    TORCH_CHECK(gate->device() == res.device() && gate->is_contiguous() && gate_rows >= 1 &&
                    (rows == 0 || (gate->numel() == rows / gate_rows * d && rows % gate_rows == 0)) &&
                    (gate->scalar_type() == res.scalar_type() || gate->scalar_type() == at::kFloat),
                "block_norm: bad gate");
  }
  smpk::BlockNormArgs a;
  a.x = ptr(x);
  a.res = res.data_ptr();
  a.w = w.data_ptr();
  a.b = ptr(b);
  a.pw = ptr(pw);
  a.pb = ptr(pb);
  a.gate = ptr(gate);
  a.w_f32 = w.scalar_type() == at::kFloat;
  a.gate_f32 = gate.has_value() && gate->scalar_type() == at::kFloat;
  a.rms = rms;
  a.rows = rows;
  a.gate_rows = gate.has_value() ? gate_rows : (a.rows < 1 ? 1 : a.rows);
  a.groups = a.rows / a.gate_rows;
  a.d = static_cast<int>(d);
  a.alpha = static_cast<float>(alpha);
  a.eps = static_cast<float>(eps);
  return a;
}

// {y, s, stats}; s is empty without x, stats without need_stats
std::vector<at::Tensor> block_norm_fwd(Opt x, at::Tensor res, at::Tensor w, Opt b, Opt pw, Opt pb, Opt gate,
                                       int64_t gate_rows, double alpha, double eps, bool rms, bool need_stats) {
  const c10::DeviceGuard guard(res.device());
  auto a = block_args(x, res, w, b, pw, pb, gate, gate_rows, alpha, eps, rms);
  auto y = at::empty_like(res);
  auto s = x.has_value() ? at::empty_like(res) : at::empty({0}, res.options());
  auto stats = at::empty({need_stats ? a.rows : 0, 4}, res.options().dtype(at::kFloat));
  a.y = y.data_ptr();
  a.s = x.has_value() ? s.data_ptr() : nullptr;
  a.stats = need_stats ? stats.data_ptr<float>() : nullptr;
  check(smpk::block_norm_fwd(dt_code(res, "block_norm"), a, stream()), "block_norm_fwd");
  return {y, s, stats};
}

// Gradients of x, residual, w, b, pw, pb, gate: those of `need` (undefined otherwise).  into[i]: the
// bound gradient of w, b, pw, pb, gate, added to in place (and returned undefined).
std::vector<Opt> block_norm_bwd(Opt dy, Opt ds, Opt x, at::Tensor res, at::Tensor w, Opt b, Opt pw, Opt pb, Opt gate,
                                int64_t gate_rows, double alpha, double eps, bool rms, at::Tensor stats,
                                std::vector<bool> need, std::vector<Opt> into) {
  const c10::DeviceGuard guard(res.device());
  auto a = block_args(x, res, w, b, pw, pb, gate, gate_rows, alpha, eps, rms);
  TORCH_CHECK(need.size() == 7 && into.size() == 5, "block_norm: bad lists");
  TORCH_CHECK(stats.is_contiguous() && stats.scalar_type() == at::kFloat && stats.numel() == 4 * a.rows,
              "block_norm: bad statistics");
  for (const Opt* t : {&dy, &ds})
    TORCH_CHECK(!t->has_value() || ((*t)->is_contiguous() && (*t)->sizes() == res.sizes() &&
                                    (*t)->scalar_type() == res.scalar_type() && (*t)->device() == res.device()),
                "block_norm: bad gradient");
  const Opt vectors[5] = {Opt(w), b, pw, pb, gate};
  std::vector<Opt> out(7);
  at::Tensor target[5];
  for (int i = 0; i < 5; ++i) {
    if (!need[2 + i]) continue;
    TORCH_CHECK(vectors[i].has_value(), "block_norm: gradient of an absent vector");
    if (into[i].has_value()) {
      TORCH_CHECK(into[i]->is_contiguous() && into[i]->numel() == vectors[i]->numel() &&
                      into[i]->scalar_type() == vectors[i]->scalar_type() && into[i]->device() == res.device(),
                  "block_norm: bad bound gradient");
      target[i] = *into[i];
    } else {
      target[i] = a.rows > 0 ? at::empty_like(*vectors[i]) : at::zeros_like(*vectors[i]);
      out[2 + i] = target[i];
    }
  }
  at::Tensor dx, dres;
  if (need[0]) {
    TORCH_CHECK(x.has_value(), "block_norm: gradient of an absent x");
    out[0] = dx = at::empty_like(res);
    a.dx = dx.data_ptr();
  }
  if (need[1]) {
    out[1] = dres = at::empty_like(res);
    a.dres = dres.data_ptr();
  }
  if (a.rows == 0) return out;  // (bound gradients stay as they are)
  a.dy = ptr(dy);
  a.ds = ptr(ds);
  a.stats = stats.data_ptr<float>();
  smpk::BlockNormPlan p;
  check(smpk::block_norm_bwd_plan(a.rows, a.d, a.gate_rows, p), "block_norm_bwd_plan");
  a.split = p.split;
  const auto f32 = res.options().dtype(at::kFloat);
  const int64_t groups = a.rows / a.gate_rows;
  const bool gate_rows_own = need[6] && groups > 1;  // one sum for each gate row, not one for all rows
  at::Tensor parts, gate_part, pq;
  if (p.two_pass) {
    pq = at::empty({a.rows, 2}, f32);
    a.pq = pq.data_ptr<float>();
  }
  int sums = 0;
  for (int i = 0; i < 5; ++i) sums += target[i].defined() && !(i == 4 && gate_rows_own);
  if (sums) parts = at::empty({sums, p.blocks, a.d}, f32);
  smpk::BlockNormJoin join;
  int used = 0;
  for (int i = 0; i < 5; ++i) {
    if (!target[i].defined()) continue;
    auto& it = join.item[join.count];
    it.dt = dt_code(target[i], "block_norm");
    it.out = target[i].data_ptr();
    it.accumulate = into[i].has_value();
    if (i == 4 && gate_rows_own) {
      if (p.split == 1 && !it.accumulate) {  // written by the units
        a.gate_direct = 1;
        a.dgate = it.out;
        continue;
      }
      TORCH_CHECK(p.split > 1, "block_norm: a bound gradient of a gate with many rows");
      gate_part = at::empty({p.units, a.d}, f32);
      a.gate_part = gate_part.data_ptr<float>();
      it.part = a.gate_part;
      it.split = p.split;
      it.groups = groups;
    } else {
      a.part[i] = parts.data_ptr<float>() + used++ * p.blocks * a.d;
      it.part = a.part[i];
      it.split = p.blocks;
      it.groups = 1;
    }
    ++join.count;
  }
  check(smpk::block_norm_bwd(dt_code(res, "block_norm"), a, p, stream()), "block_norm_bwd");
  check(smpk::block_norm_join(join, a.d, stream()), "block_norm_join");
  return out;
}

// The backward launches kernels that autograd does not see: a second derivative is an error.
variable_list once(variable_list grads, const char* name) {
  if (!at::GradMode::is_enabled()) return grads;
  for (auto& g : grads)
    if (g.defined()) g = g.detach().set_requires_grad(true);  // whatever is built on it reaches the error
  const auto error = std::make_shared<torch::autograd::DelayedError>(
      std::string(name) + " cannot be differentiated twice", static_cast<int64_t>(grads.size()));
  return (*error)(std::move(grads));
}

class BlockNormFunction : public torch::autograd::Function<BlockNormFunction> {
 public:
  static variable_list forward(AutogradContext* ctx, const Opt& x, const at::Tensor& res, const at::Tensor& w,
                               const Opt& b, const Opt& pw, const Opt& pb, const Opt& gate, int64_t gate_rows,
                               double alpha, double eps, bool rms, std::vector<int64_t> marks) {
    auto out = block_norm_fwd(x, res, w, b, pw, pb, gate, gate_rows, alpha, eps, rms, true);
    auto opt = [](const Opt& t) { return t.has_value() ? *t : at::Tensor(); };
    // s is not kept: the backward forms it again from x and the residual (block_norm.hip)
    ctx->save_for_backward({opt(x), res, w, opt(b), opt(pw), opt(pb), opt(gate), out[2]});
    ctx->saved_data["marks"] = marks;
    ctx->saved_data["gate_rows"] = gate_rows;
    ctx->saved_data["alpha"] = alpha;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["rms"] = rms;
    ctx->set_materialize_grads(false);
    out.resize(x.has_value() ? 2 : 1);
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list result(12);
    auto opt = [](const at::Tensor& t) { return t.defined() ? Opt(t) : Opt(); };
    const Opt dy = opt(grads[0].defined() ? grads[0].contiguous() : grads[0]);
    const Opt ds = grads.size() > 1 ? opt(grads[1].defined() ? grads[1].contiguous() : grads[1]) : Opt();
    if (!dy.has_value() && !ds.has_value()) return result;
    const bool duals = duals_live();
    TORCH_CHECK((!dy.has_value() || plain(*dy, duals)) && (!ds.has_value() || plain(*ds, duals)),
                "block_norm: the gradient of an output must be a plain tensor, not a dual, batched or otherwise wrapped "
                "one (calls made inside a function transform or on dual numbers take such gradients)");
    const auto v = ctx->get_saved_variables();
    check_capture(v, "block_norm");
    const auto marks = ctx->saved_data["marks"].toIntVector();
    std::vector<bool> need(7, false);
    for (size_t i = 0, edge = 0; i < 7; ++i)  // (autograd counts the tensors that are there)
      if (v[i].defined()) need[i] = ctx->needs_input_grad(edge++);
    std::vector<Opt> into(5);
    for (size_t i = 0; i < 5; ++i) {
      const at::Tensor& t = v[2 + i];
      if (!need[2 + i] || !bound(t, marks[i] != 0)) continue;
      if (i == 4 && t.numel() != t.size(-1)) continue;  // a gate with many rows may be written without a partial sum
      bool again = false;  // a parameter used twice is added to in place only once
      for (size_t k = 0; k < i; ++k) again = again || (into[k].has_value() && into[k]->is_same(t.grad()));
      if (again) continue;
      into[i] = t.grad();
      torch::autograd::impl::bump_version(*into[i]);
    }
    const auto out = block_norm_bwd(dy, ds, opt(v[0]), v[1], v[2], opt(v[3]), opt(v[4]), opt(v[5]), opt(v[6]),
                                    ctx->saved_data["gate_rows"].toInt(), ctx->saved_data["alpha"].toDouble(),
                                    ctx->saved_data["eps"].toDouble(), ctx->saved_data["rms"].toBool(), v[7], need,
                                    into);
    for (size_t i = 0; i < 7; ++i)
      if (out[i].has_value()) result[i] = *out[i];
    return once(std::move(result), "block_norm");
  }
};

// {y, s} (y alone without x), differentiable in all tensors; marks: which of w, b, pw, pb, gate are
// parameters bound to the flat gradient buffer.  None where the kernels do not take the call, as above.
c10::optional<variable_list> block_norm(Opt x, at::Tensor res, at::Tensor w, Opt b, Opt pw, Opt pb, Opt gate, int64_t gate_rows,
                         double alpha, double eps, bool rms, std::vector<int64_t> marks) {
  TORCH_CHECK(marks.size() == 5, "block_norm: bad lists");
  const bool duals = duals_live();
  bool take = unobserved() && plain(res, duals) && plain(w, duals);
  for (const Opt* t : {&x, &b, &pw, &pb, &gate}) take = take && (!t->has_value() || plain(**t, duals));
  if (!take) return c10::nullopt;
  auto dense = [](Opt& t) {
    if (t.has_value()) t = t->contiguous();
  };
  dense(x);
  dense(b);
  dense(pw);
  dense(pb);
  dense(gate);
  res = res.contiguous();
  w = w.contiguous();
  bool grad = res.requires_grad() || w.requires_grad();
  for (const Opt* t : {&x, &b, &pw, &pb, &gate}) grad = grad || (t->has_value() && (*t)->requires_grad());
  if (grad && at::GradMode::is_enabled())
    return BlockNormFunction::apply(x, res, w, b, pw, pb, gate, gate_rows, alpha, eps, rms, marks);
  auto out = block_norm_fwd(x, res, w, b, pw, pb, gate, gate_rows, alpha, eps, rms, false);
  out.resize(x.has_value() ? 2 : 1);
  return out;
}

// --------------------------------------------------------------- gradient norm
// [start, end) of the memory of a dense tensor
std::pair<uintptr_t, uintptr_t> extent(const at::Tensor& t) {
  const auto p = reinterpret_cast<uintptr_t>(t.data_ptr());
  return {p, p + static_cast<uintptr_t>(t.nbytes())};
}

// No element may be written twice, or written while another tensor's turn reads it.
void check_disjoint(const std::vector<at::Tensor>& in, const std::vector<at::Tensor>& out) {
  struct Range {
    uintptr_t s, e;
    bool write;
  };
  std::vector<Range> r;
  r.reserve(in.size() * 2);
  for (size_t i = 0; i < in.size(); ++i) {
    if (in[i].numel() == 0) continue;
    const auto a = extent(in[i]), b = extent(out[i]);
    r.push_back({b.first, b.second, true});
    if (a != b || in[i].scalar_type() != out[i].scalar_type()) r.push_back({a.first, a.second, false});
  }
  std::sort(r.begin(), r.end(), [](const Range& x, const Range& y) { return x.s < y.s; });
  uintptr_t end = 0, write_end = 0;
  for (const Range& x : r) {
    TORCH_CHECK_VALUE(x.s >= write_end && (!x.write || x.s >= end),
                      "clip_grad_norm_: two tensors of the list share memory");
    end = std::max(end, x.e);
    if (x.write) write_end = std::max(write_end, x.e);
  }
}

bool is_float(const at::Tensor& t) {
  return t.scalar_type() == at::kFloat || t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16;
}

// {power fp64 [1], norm fp32 []}; with `out`, also out[i] = grads[i] * scale * min(1, max_norm / (norm + 1e-6)).
// Tensors with gaps (slices, expanded views) go through dense copies.
std::vector<at::Tensor> grad_norm(std::vector<at::Tensor> grads, bool inf, double scale,
                                  c10::optional<std::vector<at::Tensor>> out, double max_norm) {
  TORCH_CHECK_VALUE(!grads.empty() && grads[0].defined() && grads[0].is_cuda(), "no GPU tensors");
  const at::Device device = grads[0].device();
  const c10::DeviceGuard guard(device);
  const bool duals = duals_live();
  int64_t total = 0;
  std::vector<at::Tensor> dest;
  if (out.has_value()) {
    TORCH_CHECK_VALUE(out->size() == grads.size(), grads.size(), " gradients, ", out->size(), " outputs");
    dest = *out;
  }
  for (size_t i = 0; i < grads.size(); ++i) {
    at::Tensor& t = grads[i];
    TORCH_CHECK_VALUE(t.defined() && t.layout() == at::kStrided && is_float(t) && plain(t, duals), "tensor ", i,
                      " is none of them (or no plain tensor)");
    TORCH_CHECK_VALUE(t.device() == device, "tensor ", i, " is on ", t.device(), ", not on ", device);
    total += t.numel();
    if (out.has_value()) {
      at::Tensor& o = dest[i];
      TORCH_CHECK_VALUE(o.is_same(t) || (o.defined() && o.layout() == at::kStrided && is_float(o) && plain(o, duals) &&
                                         o.device() == device && o.sizes() == t.sizes()),
                        "output ", i, " differs from its gradient in shape or device, or is none of them");
      for (int64_t k = 0; k < o.dim(); ++k)
        TORCH_CHECK_VALUE(o.stride(k) != 0 || o.size(k) <= 1, "output ", i, " is expanded: it cannot be written");
    }
    if (!t.is_non_overlapping_and_dense()) t = t.contiguous();
    if (out.has_value()) {
      at::Tensor& o = dest[i];
      if (!o.is_non_overlapping_and_dense() || (o.numel() != 0 && o.strides() != t.strides()))
        o = at::empty_like(t, t.options().dtype(o.scalar_type()));  // copied to the output at the end
    }
  }
  if (out.has_value()) check_disjoint(grads, dest);
  const int64_t size = smpk::grad_chunk_size(total);
  std::vector<smpk::GradList> lists(1);
  lists[0].count = 0;
  lists[0].first[0] = 0;
  lists[0].first_chunk = 0;
  for (size_t i = 0; i < grads.size(); ++i) {
    const int64_t n = grads[i].numel();
    if (n == 0) continue;
    if (lists.back().count == smpk::kGradList) {
      const int64_t next = lists.back().first_chunk + lists.back().first[lists.back().count];
      lists.emplace_back();
      lists.back().count = 0;
      lists.back().first[0] = 0;
      lists.back().first_chunk = next;
    }
    smpk::GradList& l = lists.back();
    const int k = l.count++;
    l.p[k] = grads[i].data_ptr();
    l.o[k] = out.has_value() ? dest[i].data_ptr() : nullptr;
    l.n[k] = n;
    l.dt[k] = static_cast<uint8_t>(dt_code(grads[i], "grad_norm"));
    l.odt[k] = out.has_value() ? static_cast<uint8_t>(dt_code(dest[i], "grad_norm")) : 0;
    l.first[k + 1] = l.first[k] + static_cast<uint32_t>((n + size - 1) / size);
  }
  const int64_t chunks = lists.back().first_chunk + lists.back().first[lists.back().count];
  const auto opts = grads[0].options();
  auto part = at::empty({chunks + 1}, opts.dtype(at::kDouble));  // (the last holds the factor)
  auto power = at::empty({1}, opts.dtype(at::kDouble));
  auto norm = at::empty({}, opts.dtype(at::kFloat));
  float* const factor = reinterpret_cast<float*>(part.data_ptr<double>() + chunks);
  for (const auto& l : lists)
    check(smpk::grad_partials(l, size, inf ? 1 : 0, part.data_ptr<double>(), stream()), "grad_partials");
  const bool each = out.has_value() && chunks > 0 && chunks <= smpk::kGradJoinEach;
  if (each) {
    for (const auto& l : lists)
      check(smpk::grad_join_scale(l, size, part.data_ptr<double>(), chunks, inf ? 1 : 0, scale, max_norm,
                                  power.data_ptr<double>(), norm.data_ptr<float>(), stream()),
            "grad_join_scale");
  } else {
    check(smpk::grad_join(part.data_ptr<double>(), chunks, inf ? 1 : 0, scale, max_norm, power.data_ptr<double>(),
                          norm.data_ptr<float>(), out.has_value() ? factor : nullptr, stream()),
          "grad_join");
  }
  if (out.has_value()) {
    if (!each)
      for (auto l = lists.rbegin(); l != lists.rend(); ++l)
        check(smpk::grad_scale(*l, size, factor, stream()), "grad_scale");
    for (size_t i = 0; i < dest.size(); ++i) {
      if (dest[i].is_same((*out)[i])) {  // a graph that holds it may not use it any more
        if (!dest[i].is_inference()) torch::autograd::impl::bump_version(dest[i]);
      } else {
        (*out)[i].copy_(dest[i]);
      }
    }
  }
  return {power, norm};
}

}  // namespace

void register_training_ops(py::module_& m) {
  m.def("block_norm", &block_norm, py::arg("x"), py::arg("res"), py::arg("w"), py::arg("b"), py::arg("pw"),
        py::arg("pb"), py::arg("gate"), py::arg("gate_rows"), py::arg("alpha"), py::arg("eps"), py::arg("rms"),
        py::arg("marks"));
  m.def("grad_norm", &grad_norm, py::arg("grads"), py::arg("inf"), py::arg("scale"), py::arg("out") = py::none(),
        py::arg("max_norm") = 0.0);
  m.def("embedding", &embedding_call, py::arg("weight"), py::arg("pos_weight"), py::arg("ids"), py::arg("pos"),
        py::arg("scale"), py::arg("start"), py::arg("foreign_zero"), py::arg("skip"), py::arg("mark_w"),
        py::arg("mark_p"));
}

// torch bindings of the embedding, block-norm and gradient-norm kernels.  Every entry checks
// what the kernel assumes, makes the tensors' device current and launches on its current stream.
#include "training_ops.h"

#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>

#include <algorithm>
#include <vector>

#include "kernels.h"

namespace {

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

void check_table(const at::Tensor& w) {
  TORCH_CHECK(w.is_cuda() && w.dim() == 2 && w.stride(1) == 1 && w.size(1) < (1ll << 31), "embedding: bad table");
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

// dw [rows, d] = (or += accumulate) the gradient of the table whose rows `ids` (or t % period) chose
void embedding_bwd(at::Tensor dy, c10::optional<at::Tensor> ids, int64_t period, double scale, int64_t start,
                   int64_t skip, at::Tensor dw, bool accumulate) {
  const c10::DeviceGuard guard(dw.device());
  TORCH_CHECK(dy.is_cuda() && dy.dim() == 2 && dy.is_contiguous() && dy.device() == dw.device(), "embedding: bad dy");
  const int64_t n = dy.size(0), d = dy.size(1);
  TORCH_CHECK(dw.dim() == 2 && dw.is_contiguous() && dw.size(1) == d && dw.scalar_type() == dy.scalar_type(),
              "embedding: bad dw");
  TORCH_CHECK(n < (1ll << 31) && dw.size(0) < (1ll << 31) - 1, "embedding: too many tokens or rows");
  const auto li = index_list(ids, n, start, dw.size(0), period, dw);
  check(smpk::embedding_bwd(dt_code(dw, "weight"), li, dy.data_ptr(), n, d, static_cast<float>(scale), skip,
                            dw.data_ptr(), accumulate ? 1 : 0, stream()),
        "embedding_bwd");
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
    if (a != b) r.push_back({a.first, a.second, false});
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

// {power fp64 [1], norm fp32 []}; with `out`, also out[i] = grads[i] * scale * min(1, max_norm / (norm + 1e-6))
std::vector<at::Tensor> grad_norm(std::vector<at::Tensor> grads, bool inf, double scale,
                                  c10::optional<std::vector<at::Tensor>> out, double max_norm) {
  TORCH_CHECK(!grads.empty(), "grad_norm: no tensors");
  const c10::DeviceGuard guard(grads[0].device());
  int64_t total = 0;
  for (size_t i = 0; i < grads.size(); ++i) {
    const at::Tensor& t = grads[i];
    TORCH_CHECK(t.is_cuda() && t.device() == grads[0].device() && t.is_non_overlapping_and_dense(),
                "grad_norm: dense tensors of one GPU expected");
    dt_code(t, "grad_norm");
    total += t.numel();
  }
  if (out.has_value()) {
    TORCH_CHECK(out->size() == grads.size(), "grad_norm: lists of different lengths");
    for (size_t i = 0; i < grads.size(); ++i) {
      const at::Tensor& o = (*out)[i];
      TORCH_CHECK(o.device() == grads[0].device() && o.sizes() == grads[i].sizes() &&
                      (o.numel() == 0 || o.strides() == grads[i].strides()),
                  "grad_norm: out differs from its gradient");
      dt_code(o, "grad_norm");
    }
    check_disjoint(grads, *out);
  }
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
    l.o[k] = out.has_value() ? (*out)[i].data_ptr() : nullptr;
    l.n[k] = n;
    l.dt[k] = static_cast<uint8_t>(dt_code(grads[i], "grad_norm"));
    l.odt[k] = out.has_value() ? static_cast<uint8_t>(dt_code((*out)[i], "grad_norm")) : 0;
    l.first[k + 1] = l.first[k] + static_cast<uint32_t>((n + size - 1) / size);
  }
  const int64_t chunks = lists.back().first_chunk + lists.back().first[lists.back().count];
  const auto opts = grads[0].options();
  auto part = at::empty({chunks < 1 ? 1 : chunks}, opts.dtype(at::kDouble));
  auto power = at::empty({1}, opts.dtype(at::kDouble));
  auto norm = at::empty({}, opts.dtype(at::kFloat));
  auto factor = at::empty({1}, opts.dtype(at::kFloat));
  for (const auto& l : lists)
    check(smpk::grad_partials(l, size, inf ? 1 : 0, part.data_ptr<double>(), stream()), "grad_partials");
  check(smpk::grad_join(part.data_ptr<double>(), chunks, inf ? 1 : 0, scale, max_norm, power.data_ptr<double>(),
                        norm.data_ptr<float>(), out.has_value() ? factor.data_ptr<float>() : nullptr, stream()),
        "grad_join");
  if (out.has_value())
    for (const auto& l : lists) check(smpk::grad_scale(l, size, factor.data_ptr<float>(), stream()), "grad_scale");
  return {power, norm};
}

}  // namespace

void register_training_ops(py::module_& m) {
  m.def("grad_norm", &grad_norm, py::arg("grads"), py::arg("inf"), py::arg("scale"), py::arg("out") = py::none(),
        py::arg("max_norm") = 0.0);
  m.def("embedding_fwd", &embedding_fwd, py::arg("ids"), py::arg("weight"), py::arg("scale"), py::arg("start"),
        py::arg("foreign_zero"), py::arg("pos"), py::arg("pos_weight"), py::arg("period"));
  m.def("embedding_bwd", &embedding_bwd, py::arg("dy"), py::arg("ids"), py::arg("period"), py::arg("scale"),
        py::arg("start"), py::arg("skip"), py::arg("dw"), py::arg("accumulate"));
}

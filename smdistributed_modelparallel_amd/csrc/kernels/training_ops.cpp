// torch bindings of the embedding, block-norm and gradient-norm kernels.  Every entry checks
// what the kernel assumes, makes the tensors' device current and launches on its current stream.
#include "training_ops.h"

#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>

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

}  // namespace

void register_training_ops(py::module_& m) {
  m.def("embedding_fwd", &embedding_fwd, py::arg("ids"), py::arg("weight"), py::arg("scale"), py::arg("start"),
        py::arg("foreign_zero"), py::arg("pos"), py::arg("pos_weight"), py::arg("period"));
  m.def("embedding_bwd", &embedding_bwd, py::arg("dy"), py::arg("ids"), py::arg("period"), py::arg("scale"),
        py::arg("start"), py::arg("skip"), py::arg("dw"), py::arg("accumulate"));
}

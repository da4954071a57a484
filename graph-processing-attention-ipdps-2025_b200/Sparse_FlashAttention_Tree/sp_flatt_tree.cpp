// Torch-extension binding `spfa_tree` (additive; the reference has no cache and one head): attention of drafted token trees over
// a paged key / value cache, with the (m, l, O) state of the other operators.
#include "cache_common.h"

using namespace spfa_binding;

// Row i of Q [n, query heads, d] sees the committed positions [0, lens[b]) of its sequence b and the drafted positions
// lens[b] + j with tree_mask[i, j]. m, l [n, query heads] float32 and O [n, query heads, d] are updated in place; first = True
// takes the incoming state as empty without reading it.
torch::Tensor spfa_tree_rows(torch::Tensor Q, torch::Tensor K_pages, torch::Tensor V_pages, torch::Tensor page_table,
                             torch::Tensor lens, torch::Tensor cu_rows, torch::Tensor tree_mask, torch::Tensor m, torch::Tensor l,
                             torch::Tensor O, OptTensor K_scale, OptTensor V_scale, bool first) {
  CacheArgs a(K_pages, V_pages, page_table, lens, K_scale, V_scale);
  a.check_cu(cu_rows);
  const int dtype = rows_dtype(Q, "Q", a);
  TORCH_CHECK(Q.dim() == 3 && Q.size(1) >= 1 && Q.size(1) % a.c.n_heads == 0,
              "Q must be [rows, query heads, d] with a multiple of the cache's heads");
  const int64_t n = Q.size(0), heads = Q.size(1);
  const Rows q(Q, "Q", n, heads, a, Q.scalar_type()), o(O, "O", n, heads, a, Q.scalar_type());
  TORCH_CHECK(tree_mask.device() == a.dev && (tree_mask.scalar_type() == torch::kBool || tree_mask.scalar_type() == torch::kUInt8) &&
                  tree_mask.dim() == 2 && tree_mask.size(0) == n && tree_mask.is_contiguous(),
              "tree_mask must be a contiguous torch.bool / torch.uint8 tensor [rows, drafted positions] on the cache's device");
  for (const torch::Tensor* t : {&m, &l})
    TORCH_CHECK(t->device() == a.dev && t->scalar_type() == torch::kFloat32 && t->dim() == 2 && t->size(0) == n &&
                    t->size(1) == heads && t->is_contiguous(),
                "m and l must be contiguous float32 [rows, query heads] on the cache's device");
  if (n == 0 || a.c.n_seq == 0) return O;
  c10::cuda::CUDAGuard guard(a.dev);
  Workspace ws(spfa_tree_workspace_bytes(&a.c, dtype, n, heads), a.dev);
  raise_for_status(spfa_tree_forward(&a.c, dtype, Q.data_ptr(), q.stride, cu_rows.data_ptr<int32_t>(), n, heads,
                                     static_cast<const uint8_t*>(tree_mask.data_ptr()), tree_mask.size(1), m.data_ptr<float>(),
                                     l.data_ptr<float>(), O.data_ptr(), o.stride, first ? 1 : 0, ws.ptr, ws.bytes,
                                     at::cuda::getCurrentCUDAStream().stream()));
  return O;
}

PYBIND11_MODULE(TORCH_EXTENSION_NAME, mod) {
  namespace py = pybind11;
  mod.def("forward", &spfa_tree_rows, "Attention of drafted token trees over a paged cache (CUDA)", py::arg("Q"), py::arg("K_pages"),
          py::arg("V_pages"), py::arg("page_table"), py::arg("lens"), py::arg("cu_rows"), py::arg("tree_mask"), py::arg("m"),
          py::arg("l"), py::arg("O"), py::arg("K_scale") = py::none(), py::arg("V_scale") = py::none(), py::arg("first") = false);
}

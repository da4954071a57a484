// Torch-extension binding `spfa_cache` (additive; the reference has no cache): paged key / value caches that hold their rows as
// they are or in 8 bits. Rows of a call are packed: row i belongs to the sequence b with cu_rows[b] <= i < cu_rows[b + 1] and
// stands for position lens[b] + i - cu_rows[b].
#include "cache_common.h"

using namespace spfa_binding;

// Writes the rows K, V [n, heads, d] to their positions, quantised where the cache is.
void spfa_cache_append_rows(torch::Tensor K, torch::Tensor V, torch::Tensor K_pages, torch::Tensor V_pages, torch::Tensor page_table,
                            torch::Tensor lens, torch::Tensor cu_rows, OptTensor K_scale, OptTensor V_scale) {
  CacheArgs a(K_pages, V_pages, page_table, lens, K_scale, V_scale);
  a.check_cu(cu_rows);
  const int dtype = rows_dtype(K, "K", a);
  const Rows k(K, "K", K.size(0), a.c.n_heads, a, K.scalar_type()), v(V, "V", K.size(0), a.c.n_heads, a, K.scalar_type());
  if (K.size(0) == 0 || a.c.n_seq == 0) return;
  c10::cuda::CUDAGuard guard(a.dev);
  raise_for_status(spfa_cache_append(&a.c, dtype, K.data_ptr(), k.stride, V.data_ptr(), v.stride, cu_rows.data_ptr<int32_t>(),
                                     K.size(0), at::cuda::getCurrentCUDAStream().stream()));
}

// Fills the rows K, V [n, heads, d] from their positions. Rows of no position are left as they are.
std::tuple<torch::Tensor, torch::Tensor> spfa_cache_read_rows(torch::Tensor K_pages, torch::Tensor V_pages, torch::Tensor page_table,
                                                              torch::Tensor lens, torch::Tensor cu_rows, torch::Tensor K,
                                                              torch::Tensor V, OptTensor K_scale, OptTensor V_scale) {
  CacheArgs a(K_pages, V_pages, page_table, lens, K_scale, V_scale);
  a.check_cu(cu_rows);
  const int dtype = rows_dtype(K, "K", a);
  const Rows k(K, "K", K.size(0), a.c.n_heads, a, K.scalar_type()), v(V, "V", K.size(0), a.c.n_heads, a, K.scalar_type());
  if (K.size(0) == 0 || a.c.n_seq == 0) return {K, V};
  c10::cuda::CUDAGuard guard(a.dev);
  raise_for_status(spfa_cache_read(&a.c, dtype, K.data_ptr(), k.stride, V.data_ptr(), v.stride, cu_rows.data_ptr<int32_t>(),
                                   K.size(0), at::cuda::getCurrentCUDAStream().stream()));
  return {K, V};
}

// Moves position lens[b] + kept[b, i] to lens[b] + i for i < n_kept[b]: what is left of a drafted tree once its path is accepted.
void spfa_cache_keep_rows(torch::Tensor K_pages, torch::Tensor V_pages, torch::Tensor page_table, torch::Tensor lens,
                          torch::Tensor kept, torch::Tensor n_kept, OptTensor K_scale, OptTensor V_scale) {
  CacheArgs a(K_pages, V_pages, page_table, lens, K_scale, V_scale);
  check_index(kept, "kept", 2, a.dev);
  check_index(n_kept, "n_kept", 1, a.dev);
  TORCH_CHECK(kept.size(0) == a.c.n_seq && n_kept.size(0) == a.c.n_seq, "kept and n_kept must have one row per sequence");
  if (kept.numel() == 0) return;
  c10::cuda::CUDAGuard guard(a.dev);
  raise_for_status(spfa_cache_keep(&a.c, kept.data_ptr<int32_t>(), kept.size(1), n_kept.data_ptr<int32_t>(),
                                   at::cuda::getCurrentCUDAStream().stream()));
}

PYBIND11_MODULE(TORCH_EXTENSION_NAME, mod) {
  namespace py = pybind11;
  mod.def("append", &spfa_cache_append_rows, "Write rows of K and V into a paged cache (CUDA)", py::arg("K"), py::arg("V"),
          py::arg("K_pages"), py::arg("V_pages"), py::arg("page_table"), py::arg("lens"), py::arg("cu_rows"),
          py::arg("K_scale") = py::none(), py::arg("V_scale") = py::none());
  mod.def("read", &spfa_cache_read_rows, "Read rows of K and V back from a paged cache (CUDA)", py::arg("K_pages"), py::arg("V_pages"),
          py::arg("page_table"), py::arg("lens"), py::arg("cu_rows"), py::arg("K"), py::arg("V"), py::arg("K_scale") = py::none(),
          py::arg("V_scale") = py::none());
  mod.def("keep", &spfa_cache_keep_rows, "Move the kept drafted rows of a paged cache to the front (CUDA)", py::arg("K_pages"),
          py::arg("V_pages"), py::arg("page_table"), py::arg("lens"), py::arg("kept"), py::arg("n_kept"),
          py::arg("K_scale") = py::none(), py::arg("V_scale") = py::none());
}

// Shared by the bindings of the paged caches: the description of a cache from its tensors, and the checks of its arguments.
//
// K_pages, V_pages [n_pages, page_size, heads, d] in any memory order whose last dimension is contiguous; K_scale, V_scale
// [n_pages, page_size, heads] float32 in any order, of the 8-bit types (torch.float8_e4m3fn, torch.int8) only; page_table
// [sequences, pages], lens [sequences] and cu_rows [sequences + 1] int32, contiguous. All on the pages' device. Contents of the
// index tensors are not looked at here: what they may hold is the library's business (include/spfa_b200.h).
#pragma once
#include "binding_common.h"

namespace spfa_binding {

using OptTensor = c10::optional<torch::Tensor>;

inline int cache_dtype_code(torch::ScalarType t, const char* name) {
  switch (t) {
    case torch::kFloat32: return SPFA_DTYPE_F32;
    case torch::kFloat16: return SPFA_DTYPE_F16;
    case torch::kBFloat16: return SPFA_DTYPE_BF16;
    case torch::kFloat8_e4m3fn: return SPFA_DTYPE_E4M3;
    case torch::kInt8: return SPFA_DTYPE_INT8;
    default: TORCH_CHECK(false, name, " must be float32, float16, bfloat16, float8_e4m3fn or int8; got ", t);
  }
}

inline void check_index(const torch::Tensor& t, const char* name, int64_t dim, const torch::Device& dev) {
  TORCH_CHECK(t.device() == dev, name, " must be on the cache's device");
  TORCH_CHECK(t.scalar_type() == torch::kInt32, name, " must be torch.int32");
  TORCH_CHECK(t.dim() == dim, name, " must have ", dim, " dimension(s)");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}

struct CacheArgs {
  spfa_kv_cache c{};
  torch::Device dev{torch::kCPU};

  CacheArgs(const torch::Tensor& K, const torch::Tensor& V, const torch::Tensor& table, const torch::Tensor& lens,
            const OptTensor& K_scale, const OptTensor& V_scale)
      : dev(K.device()) {
    TORCH_CHECK(K.is_cuda(), "K_pages must be a CUDA tensor");
    TORCH_CHECK(V.device() == dev, "V_pages must be on the device of K_pages");
    TORCH_CHECK(K.dim() == 4 && V.dim() == 4, "K_pages and V_pages must be 4-D [n_pages, page_size, heads, d]");
    TORCH_CHECK(K.sizes() == V.sizes() && K.scalar_type() == V.scalar_type(), "K_pages and V_pages must have one shape and dtype");
    TORCH_CHECK(K.size(1) >= 1 && K.size(2) >= 1 && K.size(3) >= 1, "pages must hold at least one position, head and element");
    TORCH_CHECK((K.stride(3) == 1 && V.stride(3) == 1) || K.size(3) == 1, "the last dimension of the pages must be contiguous");
    c.dtype = cache_dtype_code(K.scalar_type(), "K_pages");
    c.K = K.data_ptr();
    c.V = V.data_ptr();
    for (int i = 0; i < 3; ++i) {
      c.K_stride[i] = K.stride(i);
      c.V_stride[i] = V.stride(i);
    }
    c.n_pages = K.size(0);
    c.page_size = K.size(1);
    c.n_heads = K.size(2);
    TORCH_CHECK(K.size(3) <= 1024, spfa_status_string(SPFA_ERR_EMBED_DIM));
    c.d = (int32_t)K.size(3);
    const bool quantised = c.dtype == SPFA_DTYPE_E4M3 || c.dtype == SPFA_DTYPE_INT8;
    TORCH_CHECK(K_scale.has_value() == quantised && V_scale.has_value() == quantised,
                quantised ? "an 8-bit cache needs K_scale and V_scale" : "K_scale and V_scale belong to 8-bit caches only");
    if (quantised) {
      const torch::Tensor* s[2] = {&*K_scale, &*V_scale};
      for (int x = 0; x < 2; ++x) {
        TORCH_CHECK(s[x]->device() == dev && s[x]->scalar_type() == torch::kFloat32 && s[x]->dim() == 3 &&
                        s[x]->size(0) == c.n_pages && s[x]->size(1) == c.page_size && s[x]->size(2) == c.n_heads,
                    "K_scale and V_scale must be float32 [n_pages, page_size, heads] on the cache's device");
        for (int i = 0; i < 3; ++i) (x ? c.V_scale_stride : c.K_scale_stride)[i] = s[x]->stride(i);
      }
      c.K_scale = K_scale->data_ptr<float>();
      c.V_scale = V_scale->data_ptr<float>();
    }
    check_index(table, "page_table", 2, dev);
    check_index(lens, "lens", 1, dev);
    TORCH_CHECK(table.size(0) == lens.size(0), "page_table and lens must have one row per sequence");
    c.page_table = table.data_ptr<int32_t>();
    c.lens = lens.data_ptr<int32_t>();
    c.n_seq = lens.size(0);
    c.table_width = table.size(1);
    // an empty tensor has no address, and nothing is read through this one
    static const int64_t nowhere[2] = {0, 0};
    auto some = [&](auto*& p) {
      if (!p) p = reinterpret_cast<std::remove_reference_t<decltype(p)>>(const_cast<int64_t*>(nowhere));
    };
    some(c.K);
    some(c.V);
    some(c.page_table);
    some(c.lens);
    if (quantised) {
      some(c.K_scale);
      some(c.V_scale);
    }
  }

  void check_cu(const torch::Tensor& cu) const {
    check_index(cu, "cu_rows", 1, dev);
    TORCH_CHECK(cu.size(0) == c.n_seq + 1, "cu_rows must have one entry more than there are sequences");
  }
};

// Rows [n, heads, d] of one call, d contiguous; the two strides.
struct Rows {
  int64_t stride[2];
  Rows(const torch::Tensor& t, const char* name, int64_t n, int64_t heads, const CacheArgs& a, torch::ScalarType dtype) {
    TORCH_CHECK(t.device() == a.dev, name, " must be on the cache's device");
    TORCH_CHECK(t.scalar_type() == dtype, name, " must be ", dtype, ", got ", t.scalar_type());
    TORCH_CHECK(t.dim() == 3 && t.size(0) == n && t.size(1) == heads && t.size(2) == a.c.d, name, " must be [", n, ", ", heads, ", ",
                a.c.d, "], got ", t.sizes());
    TORCH_CHECK(t.stride(2) == 1 || t.size(2) == 1, "the last dimension of ", name, " must be contiguous");
    stride[0] = t.stride(0);
    stride[1] = t.stride(1);
  }
};

inline int rows_dtype(const torch::Tensor& t, const char* name, const CacheArgs& a) {
  const int code = cache_dtype_code(t.scalar_type(), name);
  TORCH_CHECK(code <= SPFA_DTYPE_BF16, name, " must be float32, float16 or bfloat16");
  TORCH_CHECK(a.c.dtype == code || a.c.dtype == SPFA_DTYPE_E4M3 || a.c.dtype == SPFA_DTYPE_INT8, name,
              " must have the cache's dtype (8-bit caches take float32, float16 and bfloat16)");
  return code;
}

}  // namespace spfa_binding

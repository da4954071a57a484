// Host side of the paged caches: checks of a spfa_kv_cache and the view that the kernels take.
#pragma once
#include "cache_common.cuh"
#include "capi_common.cuh"

namespace spfa {

inline int dtype_bytes(int dtype) {
  switch (dtype) {
    case SPFA_DTYPE_F32: return 4;
    case SPFA_DTYPE_F16:
    case SPFA_DTYPE_BF16: return 2;
    case SPFA_DTYPE_E4M3:
    case SPFA_DTYPE_INT8: return 1;
    default: return 0;
  }
}
inline bool aligned_to(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

constexpr int64_t kMost32 = (1LL << 31) - 1;

// Status of a cache description on its own and with rows of type `dtype` (-1: a call without rows).
inline int check_cache(const spfa_kv_cache* c, int dtype) {
  if (!c || !c->K || !c->V || !c->page_table || !c->lens) return SPFA_ERR_BAD_ARG;
  const int size = dtype_bytes(c->dtype);
  if (size == 0 || (dtype != -1 && (dtype < SPFA_DTYPE_F32 || dtype > SPFA_DTYPE_BF16))) return SPFA_ERR_BAD_ARG;
  if (size > 1 && dtype != -1 && dtype != c->dtype) return SPFA_ERR_BAD_ARG;
  if (size == 1 && (!c->K_scale || !c->V_scale || !aligned4(c->K_scale) || !aligned4(c->V_scale))) return SPFA_ERR_BAD_ARG;
  if (!aligned_to(c->K, size) || !aligned_to(c->V, size) || !aligned4(c->page_table) || !aligned4(c->lens)) return SPFA_ERR_BAD_ARG;
  if (c->d < 1 || c->d > 1024) return SPFA_ERR_EMBED_DIM;
  if (c->n_pages < 0 || c->page_size < 1 || c->n_heads < 1 || c->n_seq < 0 || c->table_width < 0) return SPFA_ERR_BAD_ARG;
  if (c->n_pages > kMost32 || c->page_size > kMost32 || c->n_heads > 65535 || c->n_seq >= kMost32 || c->table_width > kMost32)
    return SPFA_ERR_TOO_LARGE;
  for (int i = 0; i < 3; ++i)
    if (c->K_stride[i] < 0 || c->V_stride[i] < 0 || (size == 1 && (c->K_scale_stride[i] < 0 || c->V_scale_stride[i] < 0)))
      return SPFA_ERR_BAD_ARG;
  return SPFA_OK;
}

// Whether every element of something that a call writes has a place of its own, as far as strides of 0 tell.
inline bool apart(const int64_t* count, const int64_t* stride, int n) {
  for (int i = 0; i < n; ++i)
    if (count[i] > 1 && stride[i] == 0) return false;
  return true;
}
// check_cache of a call that writes into the cache.
inline int check_written_cache(const spfa_kv_cache* c, int dtype) {
  const int rc = check_cache(c, dtype);
  if (rc != SPFA_OK) return rc;
  const int64_t count[3] = {c->n_pages, c->page_size, c->n_heads};
  if (!apart(count, c->K_stride, 3) || !apart(count, c->V_stride, 3)) return SPFA_ERR_BAD_ARG;
  if (dtype_bytes(c->dtype) == 1 && (!apart(count, c->K_scale_stride, 3) || !apart(count, c->V_scale_stride, 3))) return SPFA_ERR_BAD_ARG;
  return SPFA_OK;
}

inline CacheView cache_view(const spfa_kv_cache* c) {
  CacheView v{};
  v.K.data = static_cast<char*>(c->K);
  v.V.data = static_cast<char*>(c->V);
  const bool quantised = dtype_bytes(c->dtype) == 1;
  v.K.scale = quantised ? c->K_scale : nullptr;
  v.V.scale = quantised ? c->V_scale : nullptr;
  for (int i = 0; i < 3; ++i) {
    v.K.stride[i] = c->K_stride[i];
    v.V.stride[i] = c->V_stride[i];
    v.K.s_stride[i] = c->K_scale_stride[i];
    v.V.s_stride[i] = c->V_scale_stride[i];
  }
  v.table = c->page_table;
  v.lens = c->lens;
  v.n_pages = c->n_pages;
  v.page_size = (int32_t)c->page_size;
  v.n_heads = (int32_t)c->n_heads;
  v.d = c->d;
  v.n_seq = (int32_t)c->n_seq;
  v.table_width = c->table_width;
  v.capacity = c->table_width > kMost32 / c->page_size ? kMost32 : c->table_width * c->page_size;
  return v;
}

// Whether rows of the cache can be taken as pieces of n elements (n * bytes a power of two, at most 16 bytes).
inline bool cache_rows_align(const spfa_kv_cache* c, int n) {
  const size_t bytes = (size_t)n * dtype_bytes(c->dtype);
  if (c->d % n || !aligned_to(c->K, bytes) || !aligned_to(c->V, bytes)) return false;
  for (int i = 0; i < 3; ++i)
    if (c->K_stride[i] % n || c->V_stride[i] % n) return false;
  return true;
}
inline bool rows_align(const void* p, const int64_t* stride, int elem_bytes, int n) {
  return aligned_to(p, (size_t)n * elem_bytes) && stride[0] % n == 0 && stride[1] % n == 0;
}

// f(tag of the rows' type, tag of the cache's type) with the types as null pointers.
template <class F>
int with_cache_types(int dtype, int cache_dtype, F&& f) {
  auto held = [&](auto* t) {
    using T = typename std::remove_pointer<decltype(t)>::type;
    if (cache_dtype == SPFA_DTYPE_E4M3) return f(t, static_cast<e4m3*>(nullptr));
    if (cache_dtype == SPFA_DTYPE_INT8) return f(t, static_cast<int8_t*>(nullptr));
    return f(t, static_cast<T*>(nullptr));
  };
  if (dtype == SPFA_DTYPE_F32) return held(static_cast<float*>(nullptr));
  if (dtype == SPFA_DTYPE_F16) return held(static_cast<__half*>(nullptr));
  if (dtype == SPFA_DTYPE_BF16) return held(static_cast<__nv_bfloat16*>(nullptr));
  return (int)SPFA_ERR_BAD_ARG;
}

}  // namespace spfa

// C ABI of the paged key / value caches: append, read, keep. Declared in include/spfa_b200.h.
#include "cache_kernels.cuh"
#include "cache_view.cuh"

namespace spfa {
namespace {

int check_rows_arg(const void* K, const int64_t* ks, const void* V, const int64_t* vs, const int32_t* cu, int64_t n_rows, int dtype) {
  if (!K || !V || !ks || !vs || !cu || !aligned4(cu) || n_rows < 0) return SPFA_ERR_BAD_ARG;
  if (n_rows > kMost32) return SPFA_ERR_TOO_LARGE;
  const int size = dtype_bytes(dtype);
  if (!aligned_to(K, size) || !aligned_to(V, size) || ks[0] < 0 || ks[1] < 0 || vs[0] < 0 || vs[1] < 0) return SPFA_ERR_BAD_ARG;
  return SPFA_OK;
}

// launch(rows, blocks) for the rows of the call, `lanes` threads for each of a row's `parts`; thread numbers stay below 2^31.
template <class F>
int launch_over_rows(cache::RowsView rows, int64_t parts, int lanes, F&& launch) {
  const int64_t most = (kMost32 - cache::kThreads) / (parts * lanes);
  for (rows.first = 0; rows.first < rows.n_rows; rows.first += most) {
    const int64_t n = rows.n_rows - rows.first < most ? rows.n_rows - rows.first : most;
    launch(rows, (unsigned)((n * parts * lanes + cache::kThreads - 1) / cache::kThreads));
    g_launches.fetch_add(1);
  }
  return launch_status();
}

// Threads that fill the machine (148 SMs of 2048): from there on a group of lanes takes four heads of its row. Four against one, in us, of
// an append and a read that are repeated: 64 rows of 8 e4m3 heads 8.2 : 6.0 (in a graph), 131072 rows of 8 int8 heads 334 : 414, of
// which append 189 (4.3 TB/s) and read 145 (5.6 TB/s).
constexpr int64_t kManyThreads = 148 * 2048;

template <bool kAppend, class T, class TC>
int launch_rows(const spfa_kv_cache* c, const cache::RowsView& rows, cudaStream_t st) {
  constexpr int VE = 16 / (int)sizeof(T);
  const CacheView view = cache_view(c);
  // Pieces of 16 bytes of the rows' type: a row of up to 32 of them stays in its lanes' registers. Others go element by element.
  if (c->d <= VE * 32 && cache_rows_align(c, VE) && rows_align(rows.K, rows.k_stride, sizeof(T), VE) &&
      rows_align(rows.V, rows.v_stride, sizeof(T), VE)) {
    auto run = [&](auto lanes, auto heads) {
      constexpr int LPR = decltype(lanes)::value, HC = decltype(heads)::value;
      return launch_over_rows(rows, (c->n_heads + HC - 1) / HC, LPR, [&](const cache::RowsView& r, unsigned blocks) {
        if constexpr (kAppend) cache::append_kernel<T, TC, VE, LPR, HC><<<blocks, cache::kThreads, 0, st>>>(r, view);
        else cache::read_kernel<T, TC, VE, LPR, HC><<<blocks, cache::kThreads, 0, st>>>(r, view);
      });
    };
    auto by_heads = [&](auto lanes) {
      return (c->n_heads > 1 && rows.n_rows * c->n_heads * decltype(lanes)::value > kManyThreads)
                 ? run(lanes, std::integral_constant<int, 4>())
                 : run(lanes, std::integral_constant<int, 1>());
    };
    const int need = c->d / VE;
    if (need <= 4) return by_heads(std::integral_constant<int, 4>());
    if (need <= 8) return by_heads(std::integral_constant<int, 8>());
    if (need <= 16) return by_heads(std::integral_constant<int, 16>());
    return by_heads(std::integral_constant<int, 32>());
  }
  return launch_over_rows(rows, c->n_heads, 32, [&](const cache::RowsView& r, unsigned blocks) {
    if constexpr (kAppend) cache::append_any_kernel<T, TC><<<blocks, cache::kThreads, 0, st>>>(r, view);
    else cache::read_any_kernel<T, TC><<<blocks, cache::kThreads, 0, st>>>(r, view);
  });
}

template <bool kAppend>
int rows_call(const spfa_kv_cache* c, int dtype, void* K, const int64_t* ks, void* V, const int64_t* vs, const int32_t* cu,
              int64_t n_rows, void* stream) {
  int rc = kAppend ? check_written_cache(c, dtype) : check_cache(c, dtype);
  if (rc == SPFA_OK) rc = check_rows_arg(K, ks, V, vs, cu, n_rows, dtype);
  if (rc != SPFA_OK) return rc;
  const int64_t count[2] = {n_rows, c->n_heads};
  if (!kAppend && (!apart(count, ks, 2) || !apart(count, vs, 2))) return SPFA_ERR_BAD_ARG;
  if (n_rows == 0 || c->n_seq == 0 || c->n_pages == 0 || c->table_width == 0) return SPFA_OK;
  cache::RowsView rows{static_cast<char*>(K), static_cast<char*>(V), {ks[0], ks[1]}, {vs[0], vs[1]}, cu, n_rows, 0};
  return with_cache_types(dtype, c->dtype, [&](auto* t, auto* tc) {
    using T = typename std::remove_pointer<decltype(t)>::type;
    using TC = typename std::remove_pointer<decltype(tc)>::type;
    return launch_rows<kAppend, T, TC>(c, rows, (cudaStream_t)stream);
  });
}

}  // namespace
}  // namespace spfa

using namespace spfa;

extern "C" {

int spfa_cache_append(const spfa_kv_cache* c, int dtype, const void* K, const int64_t* K_stride, const void* V,
                      const int64_t* V_stride, const int32_t* cu_rows, int64_t n_rows, void* stream) {
  return rows_call<true>(c, dtype, const_cast<void*>(K), K_stride, const_cast<void*>(V), V_stride, cu_rows, n_rows, stream);
}

int spfa_cache_read(const spfa_kv_cache* c, int dtype, void* K, const int64_t* K_stride, void* V, const int64_t* V_stride,
                    const int32_t* cu_rows, int64_t n_rows, void* stream) {
  return rows_call<false>(c, dtype, K, K_stride, V, V_stride, cu_rows, n_rows, stream);
}

int spfa_cache_keep(const spfa_kv_cache* c, const int32_t* kept, int64_t width, const int32_t* n_kept, void* stream) {
  const int rc = check_written_cache(c, -1);
  if (rc != SPFA_OK) return rc;
  if (width < 0 || (width > 0 && !kept) || !n_kept || !aligned4(kept) || !aligned4(n_kept)) return SPFA_ERR_BAD_ARG;
  if (width > kMost32 || c->n_seq * c->n_heads > kMost32) return SPFA_ERR_TOO_LARGE;
  if (width == 0 || c->n_seq == 0 || c->n_pages == 0 || c->table_width == 0) return SPFA_OK;
  const CacheView view = cache_view(c);
  const int size = dtype_bytes(c->dtype);
  const unsigned blocks = (unsigned)(c->n_seq * c->n_heads);
  cudaStream_t st = (cudaStream_t)stream;
  if (cache_rows_align(c, 16 / size)) cache::keep_kernel<uint4><<<blocks, 128, 0, st>>>(view, kept, width, n_kept, size);
  else if (cache_rows_align(c, 4 / size)) cache::keep_kernel<uint32_t><<<blocks, 128, 0, st>>>(view, kept, width, n_kept, size);
  else if (size == 2) cache::keep_kernel<uint16_t><<<blocks, 128, 0, st>>>(view, kept, width, n_kept, size);
  else cache::keep_kernel<uint8_t><<<blocks, 128, 0, st>>>(view, kept, width, n_kept, size);
  g_launches.fetch_add(1);
  return launch_status();
}

}  // extern "C"

// Host side of the tree attention, one translation unit per type of Q: the kernels are compiled in parallel.
#pragma once
#include "cache_view.cuh"
#include "tensor_map.cuh"
#include "tree_direct.cuh"
#include "tree_kernels.cuh"
#include "tree_tiled.cuh"

namespace spfa {
namespace tree {

// Launches the context and merge kernels of one call. `vec`: rows of Q, O and the cache are whole 4-element pieces; `tiled`: on the
// tensor cores (16-bit only; the caller has checked tiled_shape). The *_usable functions: whether this build's kernels can run.
int launch_f32(const spfa_kv_cache* c, const Call& a, const MergeArgs& g, bool vec, cudaStream_t st);
int launch_f16(const spfa_kv_cache* c, const Call& a, const MergeArgs& g, bool vec, bool tiled, cudaStream_t st);
int launch_bf16(const spfa_kv_cache* c, const Call& a, const MergeArgs& g, bool vec, bool tiled, cudaStream_t st);
bool usable_f16(const spfa_kv_cache* c, int subs);
bool usable_bf16(const spfa_kv_cache* c, int subs);

constexpr int kTiledKeys = 64;  // a tile of context_tiled_kernel

// Units and grid of context_any_kernel for rows of d elements: 32 rows where a sequence has more than 16 on average and a CTA's shared
// memory holds them. 32 against 16, in us (float32, d = 64, 4 sequences of 4096 keys, 2 heads a key head): 16 tokens 35 : 42, 8 tokens
// 39 : 27.
inline int any_padded(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : d <= 256 ? 256 : d <= 512 ? 512 : 1024; }
inline int any_rows(const Call& a) { return a.c.d <= 128 && a.n_rows * a.group > 16LL * a.c.n_seq ? 32 : 16; }
inline int any_ctas(int d) { return 148 * (d <= 256 ? 2 : 1); }

// Opts a kernel into its dynamic shared memory, once per device and kernel.
template <auto kernel>
bool opt_in(int bytes) {
  static std::atomic<int> done[64];  // per device: 0 unknown, 1 done
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
  if (done[dev].load(std::memory_order_relaxed)) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
  done[dev].store(1, std::memory_order_relaxed);
  return true;
}

template <int DP, int R, class TQ, class TC>
int launch_context_any(const Call& a, bool vec, cudaStream_t st) {
  using P = PlanAny<DP, R>;
  if (!opt_in<context_any_kernel<DP, R, TQ, TC>>(P::kBytes)) return SPFA_ERR_LAUNCH;
  context_any_kernel<DP, R, TQ, TC><<<(unsigned)a.n_cta, P::kThreads, P::kBytes, st>>>(a, vec ? 1 : 0);
  g_launches.fetch_add(1);
  return launch_status();
}

// The merge kernel may start while the context kernel drains (programmatic dependent launch).
template <class TQ, class TC, int VE, int NC, int GR>
int launch_merge(const Call& a, const MergeArgs& g, cudaStream_t st) {
  const int64_t blocks = (a.n_rows * a.c.n_heads * ((a.group + GR - 1) / GR) + 3) / 4;
  if (blocks * 4 > kMost32) return SPFA_ERR_TOO_LARGE;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(128);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, merge_kernel<TQ, TC, VE, NC, GR>, a, g) != cudaSuccess) return SPFA_ERR_LAUNCH;
  g_launches.fetch_add(1);
  return launch_status();
}

// From this many rows on (as many warps as 148 SMs hold) a warp merges four rows of a token: calls of 53,248 rows over 512 keys take 181 us,
// one by one 242. Below, one warp's latency counts, and one row is quicker: 256 rows over 4096 keys 21.1 us, by fours 28.6.
constexpr int64_t kMergeRows = 148 * 16;
template <class TQ, class TC>
int launch_merge_any(const Call& a, const MergeArgs& g, bool vec, cudaStream_t st) {
  const int d = a.c.d;
  if (vec) {
    const bool four = a.group > 1 && (a.unit_rows % a.group == 0 || a.group % 4 == 0) && a.n_rows * a.n_q_heads > kMergeRows;
    if (d <= 128) return four ? launch_merge<TQ, TC, 4, 1, 4>(a, g, st) : launch_merge<TQ, TC, 4, 1, 1>(a, g, st);
    if (d <= 256) return launch_merge<TQ, TC, 4, 2, 1>(a, g, st);
    return launch_merge<TQ, TC, 4, 8, 1>(a, g, st);
  }
  if (d <= 128) return launch_merge<TQ, TC, 1, 4, 1>(a, g, st);
  return launch_merge<TQ, TC, 1, 32, 1>(a, g, st);
}

template <class TQ, class TC, int R>
int launch_direct_rows(const Call& a, const MergeArgs& g, cudaStream_t st) {
  const DirectPlan plan(a.c.d * (int)sizeof(TC));
  if (!opt_in<direct_kernel<TQ, TC, R>>(227 * 1024)) return SPFA_ERR_LAUNCH;
  const int64_t blocks = a.n_rows * a.c.n_heads * ((a.group + R - 1) / R);
  direct_kernel<TQ, TC, R><<<(unsigned)blocks, plan.warps * 32, plan.bytes, st>>>(a, g);
  g_launches.fetch_add(1);
  return launch_status();
}
template <class TQ, class TC>
int launch_direct(const Call& a, const MergeArgs& g, cudaStream_t st) {
  if (a.group == 1) return launch_direct_rows<TQ, TC, 1>(a, g, st);
  if (a.group == 2) return launch_direct_rows<TQ, TC, 2>(a, g, st);
  if (a.group <= 4) return launch_direct_rows<TQ, TC, 4>(a, g, st);
  return launch_direct_rows<TQ, TC, kDirectRows>(a, g, st);
}

template <class TQ, class TC>
int launch_any(const Call& a, const MergeArgs& g, bool vec, cudaStream_t st) {
  const int d = a.c.d;
  if (a.direct) return launch_direct<TQ, TC>(a, g, st);
  int rc = SPFA_OK;
  const bool wide = a.row_tile == 32;
  if (d <= 64) rc = wide ? launch_context_any<64, 32, TQ, TC>(a, vec, st) : launch_context_any<64, 16, TQ, TC>(a, vec, st);
  else if (d <= 128) rc = wide ? launch_context_any<128, 32, TQ, TC>(a, vec, st) : launch_context_any<128, 16, TQ, TC>(a, vec, st);
  else if (d <= 256) rc = launch_context_any<256, 16, TQ, TC>(a, vec, st);
  else if (d <= 512) rc = launch_context_any<512, 16, TQ, TC>(a, vec, st);
  else rc = launch_context_any<1024, 16, TQ, TC>(a, vec, st);
  return rc != SPFA_OK ? rc : launch_merge_any<TQ, TC>(a, g, vec, st);
}

// What the copy engine can address: 16-byte rows and strides below 2^40 bytes, boxes that do not cut a page into unaligned pieces. A
// dimension whose elements share their memory (a tensor expanded over heads: stride 0) is left to the kernels that compute addresses.
inline bool tiled_shape(const spfa_kv_cache* c) {
  const int size = dtype_bytes(c->dtype);
  if (c->d > 128 || c->n_pages < 1 || !cache_rows_align(c, 16 / size) || (c->page_size % 8 && c->page_size < kTiledKeys)) return false;
  const int64_t count[3] = {c->n_pages, c->page_size, c->n_heads};
  for (int i = 0; i < 3; ++i) {
    if (c->K_stride[i] * size >= (1LL << 40) || c->V_stride[i] * size >= (1LL << 40)) return false;
    if (count[i] > 1 && (c->K_stride[i] == 0 || c->V_stride[i] == 0)) return false;
  }
  return true;
}

// Pages as (element, slot, head, page), fetched as boxes of a page's slots (at most kTiledKeys) x 128 bytes of 16-bit elements in the
// swizzle of the tensor cores, or x `bytes` codes of an 8-bit cache, as they lie or in that swizzle. Elements behind d and slots behind a page are zeros.
template <class T>
bool make_page_map(CUtensorMap* tm, const spfa_kv_cache* c, void* base, const int64_t* stride, int bytes, bool swizzle) {
  TensorMapEncodeTiledFn enc = tensor_map_encoder();
  if (!enc) return false;
  constexpr bool kByte = sizeof(T) == 1;
  const cuuint64_t dims[4] = {(cuuint64_t)c->d, (cuuint64_t)c->page_size, (cuuint64_t)c->n_heads, (cuuint64_t)c->n_pages};
  cuuint64_t strides[3] = {(cuuint64_t)stride[1] * sizeof(T), (cuuint64_t)stride[2] * sizeof(T), (cuuint64_t)stride[0] * sizeof(T)};
  for (int i = 0; i < 3; ++i)
    if (strides[i] == 0) strides[i] = 16;  // of a dimension of one element: tiled_shape lets no other pass
  const cuuint32_t box[4] = {kByte ? (cuuint32_t)bytes : 64u, (cuuint32_t)(c->page_size < kTiledKeys ? c->page_size : kTiledKeys), 1u, 1u};
  const cuuint32_t estr[4] = {1u, 1u, 1u, 1u};
  const CUtensorMapDataType type = kByte ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                         : (std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16);
  return enc(tm, type, 4, base, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
             swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// As band16_usable: setmaxnreg.inc must be covered by what the launch allocates.
template <int DP, class T, class TC, int NSUB>
bool tiled_usable() {
  using P = PlanTree<DP, T, TC, NSUB>;
  static std::atomic<int> cached[64];  // per device: 0 unknown, 1 usable, 2 not
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
  int v = cached[dev].load(std::memory_order_relaxed);
  if (v == 0) {
    cudaFuncAttributes attr;
    auto kern = context_tiled_kernel<DP, T, TC, NSUB>;
    const bool ok = cudaFuncGetAttributes(&attr, kern) == cudaSuccess &&
                    attr.numRegs * P::kThreads >= P::kRegsNeeded &&
                    cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, P::kDynSmem) == cudaSuccess;
    v = ok ? 1 : 2;
    cached[dev].store(v, std::memory_order_relaxed);
  }
  return v == 1;
}

// f(tag of the cache's type, padded d, row tiles of a CTA)
template <class TQ, class F>
auto with_tiled(const spfa_kv_cache* c, int subs, F&& f) {
  auto by_subs = [&](auto* t, auto dp) {
    return subs == 1 ? f(t, dp, std::integral_constant<int, 1>()) : f(t, dp, std::integral_constant<int, 2>());
  };
  auto by_d = [&](auto* t) {
    return c->d <= 64 ? by_subs(t, std::integral_constant<int, 64>()) : by_subs(t, std::integral_constant<int, 128>());
  };
  if (c->dtype == SPFA_DTYPE_E4M3) return by_d(static_cast<e4m3*>(nullptr));
  if (c->dtype == SPFA_DTYPE_INT8) return by_d(static_cast<int8_t*>(nullptr));
  return by_d(static_cast<TQ*>(nullptr));
}

template <class TQ>
bool usable_by_cache(const spfa_kv_cache* c, int subs) {
  return with_tiled<TQ>(c, subs, [](auto* t, auto dp, auto n) {
    return tiled_usable<decltype(dp)::value, TQ, typename std::remove_pointer<decltype(t)>::type, decltype(n)::value>();
  });
}

template <class TQ>
int launch_tiled(const spfa_kv_cache* c, const Call& a, const MergeArgs& g, bool vec, cudaStream_t st) {
  return with_tiled<TQ>(c, a.row_tile / 128, [&](auto* t, auto dp, auto n) -> int {
    using TC = typename std::remove_pointer<decltype(t)>::type;
    constexpr int DP = decltype(dp)::value, NSUB = decltype(n)::value;
    using P = PlanTree<DP, TQ, TC, NSUB>;
    int* err = tile_error_word();
    CUtensorMap tmK, tmV;
    if (!err || !make_page_map<TC>(&tmK, c, c->K, c->K_stride, P::kRawK ? 128 : DP, !P::kConvertK) ||
        !make_page_map<TC>(&tmV, c, c->V, c->V_stride, DP, !P::kQuant))
      return SPFA_ERR_LAUNCH;
    context_tiled_kernel<DP, TQ, TC, NSUB><<<(unsigned)a.n_cta, P::kThreads, P::kDynSmem, st>>>(tmK, tmV, a, err);
    g_launches.fetch_add(1);
    const int rc = launch_status();
    return rc != SPFA_OK ? rc : launch_merge_any<TQ, TC>(a, g, vec, st);
  });
}

template <class TQ>
int launch_by_cache(const spfa_kv_cache* c, const Call& a, const MergeArgs& g, bool vec, cudaStream_t st) {
  if (c->dtype == SPFA_DTYPE_E4M3) return launch_any<TQ, e4m3>(a, g, vec, st);
  if (c->dtype == SPFA_DTYPE_INT8) return launch_any<TQ, int8_t>(a, g, vec, st);
  return launch_any<TQ, TQ>(a, g, vec, st);
}

}  // namespace tree
}  // namespace spfa

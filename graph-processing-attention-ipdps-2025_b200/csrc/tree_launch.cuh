// Host side of the tree attention, one translation unit per type of Q: the kernels are compiled in parallel.
#pragma once
#include "cache_view.cuh"
#include "tree_kernels.cuh"

namespace spfa {
namespace tree {

// Launches the context and merge kernels of one call; `vec`: rows of Q, O and the cache are whole 4-element pieces.
int launch_f32(const spfa_kv_cache* c, const Call& a, const MergeArgs& g, bool vec, cudaStream_t st);
int launch_f16(const spfa_kv_cache* c, const Call& a, const MergeArgs& g, bool vec, cudaStream_t st);
int launch_bf16(const spfa_kv_cache* c, const Call& a, const MergeArgs& g, bool vec, cudaStream_t st);

constexpr int kAnyRows = 16;  // row tile of context_any_kernel
inline int any_tile_keys(int d) { return d <= 128 ? 64 : (d <= 256 ? 32 : 16); }

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

template <int DP, class TQ, class TC>
int launch_context_any(const Call& a, bool vec, cudaStream_t st) {
  using P = PlanAny<DP>;
  if (!opt_in<context_any_kernel<DP, TQ, TC>>(P::kBytes)) return SPFA_ERR_LAUNCH;
  context_any_kernel<DP, TQ, TC><<<(unsigned)a.n_cta, P::kThreads, P::kBytes, st>>>(a, vec ? 1 : 0);
  g_launches.fetch_add(1);
  return launch_status();
}

// The merge kernel may start while the context kernel drains (programmatic dependent launch).
template <class TQ, class TC, int VE, int NC>
int launch_merge(const Call& a, const MergeArgs& g, cudaStream_t st) {
  const int64_t blocks = (a.n_rows * a.n_q_heads + 3) / 4;
  if (blocks > kMost32) return SPFA_ERR_TOO_LARGE;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(128);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, merge_kernel<TQ, TC, VE, NC>, a, g) != cudaSuccess) return SPFA_ERR_LAUNCH;
  g_launches.fetch_add(1);
  return launch_status();
}

template <class TQ, class TC>
int launch_merge_any(const Call& a, const MergeArgs& g, bool vec, cudaStream_t st) {
  const int d = a.c.d;
  if (vec) {
    if (d <= 128) return launch_merge<TQ, TC, 4, 1>(a, g, st);
    if (d <= 256) return launch_merge<TQ, TC, 4, 2>(a, g, st);
    return launch_merge<TQ, TC, 4, 8>(a, g, st);
  }
  if (d <= 128) return launch_merge<TQ, TC, 1, 4>(a, g, st);
  return launch_merge<TQ, TC, 1, 32>(a, g, st);
}

template <class TQ, class TC>
int launch_any(const Call& a, const MergeArgs& g, bool vec, cudaStream_t st) {
  const int d = a.c.d;
  int rc = SPFA_OK;
  if (d <= 64) rc = launch_context_any<64, TQ, TC>(a, vec, st);
  else if (d <= 128) rc = launch_context_any<128, TQ, TC>(a, vec, st);
  else if (d <= 256) rc = launch_context_any<256, TQ, TC>(a, vec, st);
  else if (d <= 512) rc = launch_context_any<512, TQ, TC>(a, vec, st);
  else rc = launch_context_any<1024, TQ, TC>(a, vec, st);
  return rc != SPFA_OK ? rc : launch_merge_any<TQ, TC>(a, g, vec, st);
}

template <class TQ>
int launch_by_cache(const spfa_kv_cache* c, const Call& a, const MergeArgs& g, bool vec, cudaStream_t st) {
  if (c->dtype == SPFA_DTYPE_E4M3) return launch_any<TQ, e4m3>(a, g, vec, st);
  if (c->dtype == SPFA_DTYPE_INT8) return launch_any<TQ, int8_t>(a, g, vec, st);
  return launch_any<TQ, TQ>(a, g, vec, st);
}

}  // namespace tree
}  // namespace spfa

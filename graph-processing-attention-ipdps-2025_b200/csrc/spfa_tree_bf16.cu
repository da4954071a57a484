// Tree attention with Q and O of type __nv_bfloat16.
#include "tree_launch.cuh"

namespace spfa {
namespace tree {

int launch_bf16(const spfa_kv_cache* c, const Call& a, const MergeArgs& g, bool vec, bool tiled, cudaStream_t st) {
  return tiled ? launch_tiled<__nv_bfloat16>(c, a, g, vec, st) : launch_by_cache<__nv_bfloat16>(c, a, g, vec, st);
}

bool usable_bf16(const spfa_kv_cache* c, int subs) { return usable_by_cache<__nv_bfloat16>(c, subs); }

}  // namespace tree
}  // namespace spfa

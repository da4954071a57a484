// Tree attention with Q and O of type __half.
#include "tree_launch.cuh"

namespace spfa {
namespace tree {

int launch_f16(const spfa_kv_cache* c, const Call& a, const MergeArgs& g, bool vec, bool tiled, cudaStream_t st) {
  return tiled ? launch_tiled<__half>(c, a, g, vec, st) : launch_by_cache<__half>(c, a, g, vec, st);
}

bool usable_f16(const spfa_kv_cache* c, int subs) { return usable_by_cache<__half>(c, subs); }

}  // namespace tree
}  // namespace spfa

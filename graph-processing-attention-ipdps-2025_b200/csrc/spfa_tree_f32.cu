// Tree attention with Q and O of type float.
#include "tree_launch.cuh"

namespace spfa {
namespace tree {

int launch_f32(const spfa_kv_cache* c, const Call& a, const MergeArgs& g, bool vec, cudaStream_t st) {
  return launch_by_cache<float>(c, a, g, vec, st);
}

}  // namespace tree
}  // namespace spfa

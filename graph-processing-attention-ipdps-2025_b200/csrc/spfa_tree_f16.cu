// Tree attention with Q and O of type __half.
#include "tree_launch.cuh"

namespace spfa {
namespace tree {

int launch_f16(const spfa_kv_cache* c, const Call& a, const MergeArgs& g, bool vec, cudaStream_t st) {
  return launch_by_cache<__half>(c, a, g, vec, st);
}

}  // namespace tree
}  // namespace spfa

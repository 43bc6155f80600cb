// The drafted-tree attention kernel over LK_KV_E4M3 caches.
#include "paged_tree.cuh"

namespace lk {

int tree_launch_e4m3(const TreeParams& p, int dtype, int D, int NT, unsigned grid, cudaStream_t s) {
  return tree::by_type<LK_KV_E4M3>(p, dtype, D, NT, grid, s);
}

}  // namespace lk

// The drafted-tree attention kernels over LK_KV_INT8 caches.
#include "paged_tree.cuh"
#include "paged_tree_tc.cuh"

namespace lk {

int tree_launch_i8(const TreeParams& p, int dtype, int D, int NT, unsigned grid, cudaStream_t s) {
  return NT == 0 ? treetc::by_type<LK_KV_INT8>(p, dtype, D, grid, s)
                 : tree::by_type<LK_KV_INT8>(p, dtype, D, NT, grid, s);
}

}  // namespace lk

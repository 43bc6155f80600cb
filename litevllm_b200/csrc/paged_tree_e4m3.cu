// The drafted-tree attention kernels over LK_KV_E4M3 caches.
#include "paged_tree.cuh"
#include "paged_tree_tc.cuh"

namespace lk {

int tree_launch_e4m3(const TreeParams& p, int dtype, int D, int NT, unsigned grid, cudaStream_t s) {
  return NT == 0 ? treetc::by_type<LK_KV_E4M3>(p, dtype, D, grid, s)
                 : tree::by_type<LK_KV_E4M3>(p, dtype, D, NT, grid, s);
}

}  // namespace lk

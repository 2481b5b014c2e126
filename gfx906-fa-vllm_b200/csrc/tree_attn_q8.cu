// tree_attn_q8.cu -- tree-attention kernels for V format 2 (Q8_0 token rows).
#include "tree_attn_tc.cuh"

namespace g9 {
cudaError_t launch_tree_tc_v2(const TreeTcParams& pp, int nq, cudaStream_t stream) {
  return nq == 1 ? launch_tree_tc_t<1, 2>(pp, stream) : launch_tree_tc_t<2, 2>(pp, stream);
}
}  // namespace g9

G9_ERROR_ACCESSORS(tree_v2)

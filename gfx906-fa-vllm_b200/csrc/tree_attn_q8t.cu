// tree_attn_q8t.cu -- tree-attention kernels for V format 3 (page-transposed Q8_0 records).
#include "tree_attn_tc.cuh"

namespace g9 {
cudaError_t launch_tree_tc_v3(const TreeTcParams& pp, int nq, cudaStream_t stream) {
  return nq == 1 ? launch_tree_tc_t<1, 3>(pp, stream) : launch_tree_tc_t<2, 3>(pp, stream);
}
}  // namespace g9

G9_ERROR_ACCESSORS(tree_v3)

// tree_attn_bf16.cu -- tree-attention kernels for V format 1 (bf16 rows).
#include "tree_attn_tc.cuh"

namespace g9 {
cudaError_t launch_tree_tc_v1(const TreeTcParams& pp, int nq, cudaStream_t stream) {
  return nq == 1 ? launch_tree_tc_t<1, 1>(pp, stream) : launch_tree_tc_t<2, 1>(pp, stream);
}
}  // namespace g9

G9_ERROR_ACCESSORS(tree_v1)

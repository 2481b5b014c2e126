// tree_attn_f16.cu -- tree-attention kernels for V format 0 (fp16 rows).
#include "tree_attn_tc.cuh"

namespace g9 {
cudaError_t launch_tree_tc_v0(const TreeTcParams& pp, int nq, cudaStream_t stream) {
  return nq == 1 ? launch_tree_tc_t<1, 0>(pp, stream) : launch_tree_tc_t<2, 0>(pp, stream);
}
}  // namespace g9

G9_ERROR_ACCESSORS(tree_v0)

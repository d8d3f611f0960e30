// Gradient of the residual branch, bf16 stream (branch_bwd.cuh).
#include "branch_bwd.cuh"

namespace fwn {

cudaError_t launch_branch_bwd_bf16(const BranchBwdParams& p, cudaStream_t st) {
  return p.y_bf16 ? branch_bwd_by<bf16, bf16>(p, st) : branch_bwd_by<bf16, float>(p, st);
}

}  // namespace fwn

// balance on __nv_bfloat16 scores.
#include "score_balance.cuh"

namespace trnopt {

cudaError_t balance_launch_bf16(int device, const BalanceProblem& p, const BalanceWork& wk, cudaStream_t stream) {
  return launch<__nv_bfloat16>(device, p, wk, stream);
}

}  // namespace trnopt

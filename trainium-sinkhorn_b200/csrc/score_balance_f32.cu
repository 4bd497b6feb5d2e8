// balance on float scores.
#include "score_balance.cuh"

namespace trnopt {

cudaError_t balance_launch_f32(int device, const BalanceProblem& p, const BalanceWork& wk, cudaStream_t stream) {
  return launch<float>(device, p, wk, stream);
}

}  // namespace trnopt

// balance on __half scores.
#include "score_balance.cuh"

namespace trnopt {

cudaError_t balance_launch_f16(int device, const BalanceProblem& p, const BalanceWork& wk, cudaStream_t stream) {
  return launch<__half>(device, p, wk, stream);
}

}  // namespace trnopt

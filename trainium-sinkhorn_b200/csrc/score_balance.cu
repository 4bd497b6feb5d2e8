// Launch shape and workspace of balance (the kernel is in score_balance.cuh, compiled per type of score).
#include <math.h>

#include <atomic>

#include "kernels.h"
#include "scores.h"

namespace trnopt {

namespace {

int sm_count(int device) {
  static std::atomic<int> sms[kMaxDevices];
  if (device < 0 || device >= kMaxDevices) device = 0;
  int n = sms[device].load(std::memory_order_relaxed);
  if (n == 0) {
    cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device);
    sms[device].store(n, std::memory_order_relaxed);
  }
  return n;
}

// the counter and the fixed-point sums
size_t zeroed_bytes(int cols) { return 256 + (size_t)2 * ((cols + 3) & ~3) * sizeof(unsigned long long); }

}  // namespace

// CTAs: one for problems that it takes in two steps, else up to one per SM with a step's rows each. Two steps in one CTA
// against two CTAs: 2 iterations of 1000 x 8 8.2 / 12.3 us, of 512 x 64 16.4 / 17.8 us; 12 iterations 25 / 29 us and
// 51 / 48 us. (Four steps in one CTA, 2000 x 24: 5.5 us an iteration; four CTAs' steps cost 3 us.)
int balance_grid(int device, int rows, int cols) {
  const long long steps = ((long long)rows * lanes_per_row(cols) + kBalanceThreads - 1) / kBalanceThreads;
  if (steps <= 2) return 1;
  const int most = sm_count(device) < 255 ? sm_count(device) : 255;    // (counted in a byte)
  return steps < most ? (int)steps : most;
}

size_t balance_workspace_bytes(int device, int rows, int cols) {
  return zeroed_bytes(cols) + (size_t)2 * balance_grid(device, rows, cols) * ((cols + 3) & ~3) * sizeof(float);
}

cudaError_t balance_launch(int device, int type, const BalanceProblem& p, void* ws, cudaStream_t stream) {
  char* const at = static_cast<char*>(ws);
  const BalanceWork wk{reinterpret_cast<unsigned*>(at), reinterpret_cast<unsigned long long*>(at + 256),
                       reinterpret_cast<float*>(at + zeroed_bytes(p.cols)), device_error_word(), p.b ? 0.0 : log2((double)p.cols),
                       (p.b ? 1.0 : (double)p.cols) / (p.a ? 1.0 : (double)p.rows)};
  if (balance_grid(device, p.rows, p.cols) > 1) {
    const cudaError_t e = cudaMemsetAsync(ws, 0, zeroed_bytes(p.cols), stream);
    if (e != cudaSuccess) return e;
  }
  switch (type) {
    case TRNOPT_F32: return balance_launch_f32(device, p, wk, stream);
    case TRNOPT_F16: return balance_launch_f16(device, p, wk, stream);
    default: return balance_launch_bf16(device, p, wk, stream);
  }
}

}  // namespace trnopt

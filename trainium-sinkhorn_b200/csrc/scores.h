// Operators over an explicit score matrix S (rows x cols, row-major, unit column stride): internal declarations shared
// by score_log_probs.cu, score_balance.cu, score_route.cu and capi.cu.
#pragma once

#include <cuda_runtime.h>

#include "../../include/trnopt_cuda.h"

namespace trnopt {

struct LogProbsProblem {
  const void* scores;
  long long ld, rows;          // elements between rows; rows
  int cols;
  double temperature;
  const long long* targets;    // (rows, n_targets) column indices, negative = padding; nullptr with n_targets = 0
  int n_targets;
  int top;                     // best columns wanted per row
  void *log_prob, *entropy, *lse, *top_log_prob;   // float32 (float64 for float64 scores)
  long long* top_index;        // (rows, top)
  void *row_max, *log_sum;     // the row's largest score and log sum exp((S - max) / T): what the gradient reads
};

struct LogProbsGradProblem {
  const void* scores;
  long long ld, rows;
  int cols;
  double temperature;
  const long long* targets;
  int n_targets;
  const long long* top_index;
  int top;
  const void *row_max, *log_sum, *entropy;
  const void *d_log_prob, *d_entropy, *d_lse, *d_top;   // nullable
  void* grad;                  // (rows, cols) in the scores' type
  long long ld_grad;
};

struct BalanceProblem {
  const void* scores;
  long long ld;
  int rows, cols, iters;
  double eps;
  const float *a, *b, *g0;     // row masses, column masses, starting potential; nullable
  float *f, *g;
};

struct BalanceWork {
  unsigned* counter;       // arrivals at the barrier, 0 at the start
  unsigned long long* totals;  // (2, cols rounded up to 4): by parity, k_j in units of 2^-40, 0 at the start
  float* parts;            // (2, CTAs, cols rounded up to 4): the CTAs' column sums, and their maxima in the first iteration
  int* error_word;
  double log_cols, k_scale;  // log2 cols and cols / rows for uniform masses, where rows are summed without 1 / cols and
                           // columns without 1 / rows
};

struct RouteProblem {
  const void* scores;
  long long ld, rows;
  int cols, top, kind;
  const float* bias;
  int bias_on, groups, top_groups, group_top, renormalize;
  float scale;
  long long* index;            // (rows, top)
  float* weight;               // (rows, top)
  int* load;                   // (cols,) nullable
};

struct RouteGradProblem {
  const void* scores;
  long long ld, rows;
  int cols, top, kind, renormalize;
  float scale;
  const long long* index;
  const float* d_weight;
  void* grad;
  long long ld_grad;
};

cudaError_t log_probs_launch(int type, const LogProbsProblem& p, cudaStream_t stream);
cudaError_t log_probs_grad_launch(int type, const LogProbsGradProblem& p, cudaStream_t stream);
// balance, by the scores' type (score_balance_f32.cu, ...: one file each, for the compiler's time)
cudaError_t balance_launch_f32(int device, const BalanceProblem& p, const BalanceWork& wk, cudaStream_t stream);
cudaError_t balance_launch_f16(int device, const BalanceProblem& p, const BalanceWork& wk, cudaStream_t stream);
cudaError_t balance_launch_bf16(int device, const BalanceProblem& p, const BalanceWork& wk, cudaStream_t stream);
int balance_grid(int device, int rows, int cols);     // its CTAs
constexpr int kBalanceThreads = 512;
__host__ __device__ inline int lanes_per_row(int cols) {
  int l = 1;
  while (32 * l < cols) l *= 2;
  return l;
}
size_t balance_workspace_bytes(int device, int rows, int cols);
cudaError_t balance_launch(int device, int type, const BalanceProblem& p, void* ws, cudaStream_t stream);
cudaError_t route_launch(int type, const RouteProblem& p, cudaStream_t stream);
cudaError_t route_grad_launch(int type, const RouteGradProblem& p, cudaStream_t stream);

}  // namespace trnopt

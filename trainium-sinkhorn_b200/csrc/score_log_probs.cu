// Row softmax of a score matrix: log-probabilities of given columns, entropy, log-sum-exp and the best columns of
// each row, and the gradient. For row S, temperature T, m = max S, d_j = (S_j - m) / T:
//     s = sum_j exp(d_j),  log p_j = d_j - log s,  H = log s - sum_j exp(d_j) d_j / s,  lse = m / T + log s
//     dS_j = (1 / T) [ sum_t g_t (1[j = t] - p_j) + g_lse p_j - g_H p_j (log p_j + H) ]
// The difference S - m is taken before the scaling, so rows whose scores are all the type's lowest value are uniform
// rows and not overflow. Both terms of H are >= 0. A column of score -inf has p = 0 and adds nothing; a row without
// any other column has lse = log p = -inf, H = 0 and gradient 0; NaN or +inf in a row makes its values NaN.
// One CTA per row; sums in float32 (float64 for float64 scores).
#include <math.h>

#include "score_types.cuh"
#include "scores.h"

namespace trnopt {

namespace {

constexpr int LP_THREADS = 256;

// max that keeps a NaN
template <typename A>
__device__ __forceinline__ A max_nan(A a, A b) { return (a != a || a > b) ? a : b; }

template <typename A>
__device__ __forceinline__ A block_reduce_max(A v, A* sh) {
  for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sh[0];
  for (int w = 1; w < LP_THREADS / 32; ++w) v = max_nan(v, sh[w]);
  return v;
}

template <typename A>
__device__ __forceinline__ A block_reduce_sum(A v, A* sh) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sh[0];
  for (int w = 1; w < LP_THREADS / 32; ++w) v += sh[w];
  return v;
}

template <typename T>
__global__ void __launch_bounds__(LP_THREADS) log_probs_kernel(LogProbsProblem p) {
  using A = typename Acc<T>::type;
  __shared__ A sh[LP_THREADS / 32];
  __shared__ int shi[LP_THREADS / 32];
  const A inv_t = (A)(1.0 / p.temperature), inf = (A)INFINITY;
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* s = static_cast<const T*>(p.scores) + row * p.ld;
    A m = -inf;
    for (int j = threadIdx.x; j < p.cols; j += LP_THREADS) m = max_nan(m, widen(s[j]));
    m = block_reduce_max(m, sh);
    const bool empty = m == -inf;
    A sum = 0, down = 0;
    for (int j = threadIdx.x; j < p.cols; j += LP_THREADS) {
      const A x = widen(s[j]);
      if (x == -inf) continue;
      const A d = (x - m) * inv_t, e = exp(d);
      sum += e;
      down += e * d;
    }
    sum = block_reduce_sum(sum, sh);
    down = block_reduce_sum(down, sh);
    const A log_sum = empty ? -inf : log(sum);
    const bool none = log_sum != log_sum;
    if (threadIdx.x == 0) {
      static_cast<A*>(p.lse)[row] = empty ? -inf : m * inv_t + log_sum;
      static_cast<A*>(p.entropy)[row] = empty ? (A)0 : log_sum - down / sum;
      if (p.row_max) static_cast<A*>(p.row_max)[row] = m;
      if (p.log_sum) static_cast<A*>(p.log_sum)[row] = log_sum;
    }
    for (int t = threadIdx.x; t < p.n_targets; t += LP_THREADS) {
      const long long j = p.targets[row * p.n_targets + t];
      A v = 0;
      if (j >= p.cols) v = (A)NAN;
      else if (j >= 0) v = empty ? -inf : (widen(s[j]) - m) * inv_t - log_sum;
      static_cast<A*>(p.log_prob)[row * p.n_targets + t] = v;
    }
    // best columns: repeatedly the largest score after the last one taken, in (score desc, index asc) order
    A last = inf;
    int last_j = -1;
    for (int k = 0; k < p.top; ++k) {
      A best = -inf;
      int best_j = -1;
      if (!none)
        for (int j = threadIdx.x; j < p.cols; j += LP_THREADS) {
          const A x = widen(s[j]);
          if ((x < last || (x == last && j > last_j)) && x > best) { best = x; best_j = j; }
        }
      for (int o = 16; o > 0; o >>= 1) {
        const A ob = __shfl_xor_sync(0xffffffffu, best, o);
        const int oj = __shfl_xor_sync(0xffffffffu, best_j, o);
        if (ob > best || (ob == best && oj >= 0 && (best_j < 0 || oj < best_j))) { best = ob; best_j = oj; }
      }
      __syncthreads();
      if ((threadIdx.x & 31) == 0) { sh[threadIdx.x >> 5] = best; shi[threadIdx.x >> 5] = best_j; }
      __syncthreads();
      best = sh[0];
      best_j = shi[0];
      for (int w = 1; w < LP_THREADS / 32; ++w)
        if (sh[w] > best || (sh[w] == best && shi[w] >= 0 && (best_j < 0 || shi[w] < best_j))) {
          best = sh[w];
          best_j = shi[w];
        }
      if (threadIdx.x == 0) {
        p.top_index[row * p.top + k] = best_j;
        static_cast<A*>(p.top_log_prob)[row * p.top + k] =
            none ? (A)NAN : best_j < 0 ? -inf : (best - m) * inv_t - log_sum;
      }
      last = best;
      last_j = best_j < 0 ? p.cols : best_j;
    }
    __syncthreads();
  }
}

template <typename T>
__global__ void __launch_bounds__(LP_THREADS) log_probs_grad_kernel(LogProbsGradProblem p) {
  using A = typename Acc<T>::type;
  const A inv_t = (A)(1.0 / p.temperature), inf = (A)INFINITY;
  const int extra = p.n_targets + p.top;
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* s = static_cast<const T*>(p.scores) + row * p.ld;
    T* out = static_cast<T*>(p.grad) + row * p.ld_grad;
    const long long* tg = p.targets + row * p.n_targets;
    const long long* ti = p.top_index + row * p.top;
    const A* gt = p.d_log_prob ? static_cast<const A*>(p.d_log_prob) + row * p.n_targets : nullptr;
    const A* gk = p.d_top ? static_cast<const A*>(p.d_top) + row * p.top : nullptr;
    // entry q < n_targets is a given column, the others are the best columns
    auto column = [&](int q) { return q < p.n_targets ? tg[q] : ti[q - p.n_targets]; };
    auto upstream = [&](int q) { return q < p.n_targets ? (gt ? gt[q] : (A)0) : (gk ? gk[q - p.n_targets] : (A)0); };
    const A m = static_cast<const A*>(p.row_max)[row], log_sum = static_cast<const A*>(p.log_sum)[row];
    const bool empty = m == -inf;
    const A h = static_cast<const A*>(p.entropy)[row];
    const A gh = p.d_entropy ? static_cast<const A*>(p.d_entropy)[row] : (A)0;
    A total = p.d_lse ? -static_cast<const A*>(p.d_lse)[row] : (A)0;
    for (int q = 0; q < extra; ++q) {
      const long long j = column(q);
      if (j >= 0 && j < p.cols) total += upstream(q);
    }
    auto dense = [&](A x) {
      if (empty || x == -inf) return (A)0;
      const A lp = (x - m) * inv_t - log_sum;
      return -exp(lp) * (total + gh * (lp + h)) * inv_t;
    };
    for (int j = threadIdx.x; j < p.cols; j += LP_THREADS) narrow(dense(widen(s[j])), out + j);
    __syncthreads();
    for (int q = threadIdx.x; q < extra; q += LP_THREADS) {
      const long long j = column(q);
      if (j < 0 || j >= p.cols || empty) continue;
      bool first = true;                       // a column given more than once is written by its first entry
      for (int r = 0; r < q; ++r) first = first && column(r) != j;
      if (!first) continue;
      A g = upstream(q);
      for (int r = q + 1; r < extra; ++r)
        if (column(r) == j) g += upstream(r);
      narrow(dense(widen(s[j])) + g * inv_t, out + j);
    }
    __syncthreads();
  }
}

unsigned row_grid(long long rows) { return (unsigned)(rows < 65535 ? rows : 65535); }

}  // namespace

cudaError_t log_probs_launch(int type, const LogProbsProblem& p, cudaStream_t stream) {
  const unsigned grid = row_grid(p.rows);
  switch (type) {
    case TRNOPT_F32: log_probs_kernel<float><<<grid, LP_THREADS, 0, stream>>>(p); break;
    case TRNOPT_F16: log_probs_kernel<__half><<<grid, LP_THREADS, 0, stream>>>(p); break;
    case TRNOPT_BF16: log_probs_kernel<__nv_bfloat16><<<grid, LP_THREADS, 0, stream>>>(p); break;
    default: log_probs_kernel<double><<<grid, LP_THREADS, 0, stream>>>(p); break;
  }
  return cudaGetLastError();
}

cudaError_t log_probs_grad_launch(int type, const LogProbsGradProblem& p, cudaStream_t stream) {
  const unsigned grid = row_grid(p.rows);
  switch (type) {
    case TRNOPT_F32: log_probs_grad_kernel<float><<<grid, LP_THREADS, 0, stream>>>(p); break;
    case TRNOPT_F16: log_probs_grad_kernel<__half><<<grid, LP_THREADS, 0, stream>>>(p); break;
    case TRNOPT_BF16: log_probs_grad_kernel<__nv_bfloat16><<<grid, LP_THREADS, 0, stream>>>(p); break;
    default: log_probs_grad_kernel<double><<<grid, LP_THREADS, 0, stream>>>(p); break;
  }
  return cudaGetLastError();
}

}  // namespace trnopt

// Routing over a score matrix: each row's best columns and their weights, and the weights' gradient.
//     share_ij = softmax_j(S_i) or sigmoid(S_ij)
//     key_ij   = share_ij + bias_j (bias on the scores), S_ij + bias_j (bias on the logits: a balancing potential) or
//                S_ij (no bias)
//     groups of cols / groups neighbouring columns: a group's score is the sum of its group_top largest keys (without a
//     bias: shares); the top_groups best groups stay open (equal ones: the lower index)
//     index = the top best keys of the open columns (equal ones: the lower index)
//     weight = scale * share, or scale * share / sum of the chosen shares
// Columns of score -inf or biased key -inf are closed. Slots that no open column fills hold index -1 and weight 0. A
// row holding NaN or +inf chooses nothing: index -1, weight NaN.
// The order of keys is a comparison of values that may be a few float32 steps apart, so keys are float64; the weights
// are float32 from the logarithms of the shares (shares that underflow still give their ratio). One warp per row.
#include <math.h>

#include "score_types.cuh"
#include "scores.h"

namespace trnopt {

namespace {

constexpr int RT_WARPS = 4;
constexpr int RT_MAX_COLS = 1024;
constexpr unsigned kAll = 0xffffffffu;

__device__ __forceinline__ double warp_max(double v) {
  for (int o = 16; o > 0; o >>= 1) v = fmax(v, __shfl_xor_sync(kAll, v, o));
  return v;
}
template <typename A>
__device__ __forceinline__ A warp_sum(A v) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}
// the larger value, of equal ones the lower index; index -1 is no candidate
__device__ __forceinline__ void warp_best(double& v, int& j) {
  for (int o = 16; o > 0; o >>= 1) {
    const double ov = __shfl_xor_sync(kAll, v, o);
    const int oj = __shfl_xor_sync(kAll, j, o);
    if (oj >= 0 && (j < 0 || ov > v || (ov == v && oj < j))) { v = ov; j = oj; }
  }
}

// log sigmoid(x), exact for large |x|
__device__ __forceinline__ float log_sigmoid(float x) { return fminf(x, 0.f) - log1pf(expf(-fabsf(x))); }

template <typename T>
__global__ void __launch_bounds__(32 * RT_WARPS) route_kernel(RouteProblem p) {
  __shared__ double keys[RT_WARPS][RT_MAX_COLS];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int size = p.cols / p.groups;
  double* key = keys[w];
  for (long long row = (long long)blockIdx.x * RT_WARPS + w; row < p.rows; row += (long long)gridDim.x * RT_WARPS) {
    const T* s = static_cast<const T*>(p.scores) + row * p.ld;
    double m = -INFINITY, sum = 0.0;
    bool bad = false;
    for (int j = lane; j < p.cols; j += 32) {
      const float x = widen(s[j]);
      bad = bad || !(x < INFINITY) || (p.bias && p.bias[j] != p.bias[j]);
      m = fmax(m, (double)x);
    }
    bad = __any_sync(kAll, bad);
    m = warp_max(m);
    if (p.kind == TRNOPT_ROUTE_SOFTMAX && m > -INFINITY) {
      for (int j = lane; j < p.cols; j += 32) sum += exp((double)widen(s[j]) - m);
      sum = warp_sum(sum);
    }
    const bool on_scores = p.bias && p.bias_on == TRNOPT_ROUTE_BIAS_SCORES;
    auto share = [&](double x) { return p.kind == TRNOPT_ROUTE_SOFTMAX ? exp(x - m) / sum : 1.0 / (1.0 + exp(-x)); };
    if (!bad) {
      for (int j = lane; j < p.cols; j += 32) {
        const double x = widen(s[j]);
        double k = x;
        if (x > -INFINITY) {
          if (on_scores || (p.groups > 1 && !p.bias)) k = share(x);
          if (p.bias) k += (double)p.bias[j];
        }
        key[j] = k;
      }
      __syncwarp();
      if (p.groups > 1) {
        // lane g scores group g, then ranks it among all
        double top1 = -INFINITY, top2 = -INFINITY;
        if (lane < p.groups)
          for (int j = lane * size; j < (lane + 1) * size; ++j) {
            const double k = key[j];
            if (k > top1) { top2 = top1; top1 = k; }
            else if (k > top2) top2 = k;
          }
        const bool alive = top1 > -INFINITY;
        const double score = p.group_top == 2 && top2 > -INFINITY ? top1 + top2 : top1;
        int rank = 0;
        for (int g = 0; g < p.groups; ++g) {
          const double other = __shfl_sync(kAll, score, g);
          const bool other_alive = __shfl_sync(kAll, alive, g);
          rank += other_alive && (other > score || (other == score && g < lane));
        }
        __syncwarp();
        const unsigned open = __ballot_sync(kAll, lane < p.groups && alive && rank < p.top_groups);
        for (int j = lane; j < p.cols; j += 32) {
          if (!((open >> (j / size)) & 1)) key[j] = -INFINITY;
          else if (!p.bias) key[j] = widen(s[j]);        // without a bias the columns go by their scores themselves
        }
        __syncwarp();
      }
    }
    int mine = -1;                                        // lane k < top holds the k-th choice
    for (int k = 0; k < p.top && !bad; ++k) {
      double v = -INFINITY;
      int j = -1;
      for (int c = lane; c < p.cols; c += 32)
        if (key[c] > v) { v = key[c]; j = c; }
      warp_best(v, j);
      if (j < 0) break;
      if (lane == k) mine = j;
      if (lane == (j & 31)) key[j] = -INFINITY;
      __syncwarp();
    }
    float weight = 0.f;
    const float x = mine >= 0 ? widen(s[mine]) : 0.f;
    float lw = mine < 0 ? -INFINITY : p.kind == TRNOPT_ROUTE_SOFTMAX ? x - (float)m : log_sigmoid(x);
    if (p.renormalize) {
      float peak = lw;
      for (int o = 16; o > 0; o >>= 1) peak = fmaxf(peak, __shfl_xor_sync(kAll, peak, o));
      const float e = mine >= 0 ? expf(lw - peak) : 0.f, total = warp_sum(e);
      if (mine >= 0) weight = p.scale * (e / total);
    } else if (mine >= 0) {
      weight = p.scale * (p.kind == TRNOPT_ROUTE_SOFTMAX ? expf(lw) / (float)sum : expf(lw));
    }
    if (lane < p.top) {
      p.index[row * p.top + lane] = mine;
      p.weight[row * p.top + lane] = bad ? NAN : weight;
      if (p.load && mine >= 0) atomicAdd(p.load + mine, 1);
    }
    __syncwarp();
  }
}

template <typename T>
__global__ void __launch_bounds__(32 * RT_WARPS) route_grad_kernel(RouteGradProblem p) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  for (long long row = (long long)blockIdx.x * RT_WARPS + w; row < p.rows; row += (long long)gridDim.x * RT_WARPS) {
    const T* s = static_cast<const T*>(p.scores) + row * p.ld;
    T* out = static_cast<T*>(p.grad) + row * p.ld_grad;
    const int mine = lane < p.top ? (int)p.index[row * p.top + lane] : -1;
    const float d = mine >= 0 ? p.scale * p.d_weight[row * p.top + lane] : 0.f;
    const float x = mine >= 0 ? widen(s[mine]) : 0.f;
    const bool softmax = p.kind == TRNOPT_ROUTE_SOFTMAX;
    const bool any = __any_sync(kAll, mine >= 0);
    float grad = 0.f;
    if (p.renormalize || !softmax || !any) {
      for (int j = lane; j < p.cols; j += 32) narrow(0.f, out + j);
      const float other = softmax ? 1.f : 1.f / (1.f + expf(x));      // d log share / dS of a column by itself
      if (p.renormalize) {
        const float lw = mine < 0 ? -INFINITY : softmax ? x : log_sigmoid(x);
        float peak = lw;
        for (int o = 16; o > 0; o >>= 1) peak = fmaxf(peak, __shfl_xor_sync(kAll, peak, o));
        const float e = mine >= 0 ? expf(lw - peak) : 0.f;
        const float part = e / warp_sum(e), mean = warp_sum(mine >= 0 ? part * d : 0.f);
        grad = part * (d - mean) * other;
      } else {
        grad = d * expf(log_sigmoid(x)) * other;
      }
    } else {
      float m = -INFINITY, sum = 0.f;
      for (int j = lane; j < p.cols; j += 32) m = fmaxf(m, widen(s[j]));
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kAll, m, o));
      for (int j = lane; j < p.cols; j += 32) sum += expf(widen(s[j]) - m);
      sum = warp_sum(sum);
      const float share = mine >= 0 ? expf(x - m) / sum : 0.f, mean = warp_sum(share * d);
      for (int j = lane; j < p.cols; j += 32) narrow(-(expf(widen(s[j]) - m) / sum) * mean, out + j);
      grad = share * (d - mean);
    }
    __syncwarp();                                        // a chosen column's value follows the row's dense one
    if (mine >= 0) narrow(grad, out + mine);
  }
}

unsigned route_grid(long long rows) {
  const long long blocks = (rows + RT_WARPS - 1) / RT_WARPS;
  return (unsigned)(blocks < (1 << 20) ? blocks : (1 << 20));
}

}  // namespace

cudaError_t route_launch(int type, const RouteProblem& p, cudaStream_t stream) {
  if (p.load) {
    const cudaError_t e = cudaMemsetAsync(p.load, 0, sizeof(int) * p.cols, stream);
    if (e != cudaSuccess) return e;
  }
  if (p.rows == 0) return cudaSuccess;
  const unsigned grid = route_grid(p.rows);
  switch (type) {
    case TRNOPT_F32: route_kernel<float><<<grid, 32 * RT_WARPS, 0, stream>>>(p); break;
    case TRNOPT_F16: route_kernel<__half><<<grid, 32 * RT_WARPS, 0, stream>>>(p); break;
    default: route_kernel<__nv_bfloat16><<<grid, 32 * RT_WARPS, 0, stream>>>(p); break;
  }
  return cudaGetLastError();
}

cudaError_t route_grad_launch(int type, const RouteGradProblem& p, cudaStream_t stream) {
  if (p.rows == 0) return cudaSuccess;
  const unsigned grid = route_grid(p.rows);
  switch (type) {
    case TRNOPT_F32: route_grad_kernel<float><<<grid, 32 * RT_WARPS, 0, stream>>>(p); break;
    case TRNOPT_F16: route_grad_kernel<__half><<<grid, 32 * RT_WARPS, 0, stream>>>(p); break;
    default: route_grad_kernel<__nv_bfloat16><<<grid, 32 * RT_WARPS, 0, stream>>>(p); break;
  }
  return cudaGetLastError();
}

}  // namespace trnopt

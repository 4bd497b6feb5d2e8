// Sinkhorn on a score matrix: the potentials of the entropic transport plan
//     P_ij = a_i b_j exp((f_i + g_j + S_ij) / eps)
// between rows of mass a and columns of mass b, by the half-steps of the reference (src/trnopt/sinkhorn.py:108-119,
// with the cost -S held as a matrix):
//     f_i = -eps LSE_j(log b_j + (g_j + S_ij) / eps),   g_j = -eps LSE_i(log a_i + (f_i + S_ij) / eps).
// A row or column without mass to exchange (all its terms zero) takes potential 0. A row kernel (one warp per row), a
// column kernel (32 columns of a block of rows per CTA, online maxima) and its merge, per iteration.
#include <math.h>

#include "score_types.cuh"
#include "scores.h"

namespace trnopt {

namespace {

constexpr int BAL_ROWS = 256;    // rows of a column kernel's CTA

__device__ __forceinline__ void lse_add(float& m, float& l, float om, float ol) {
  const float n = om != om ? om : fmaxf(m, om);      // a NaN stays
  if (n == -INFINITY) return;
  l = l * expf(m - n) + ol * expf(om - n);
  m = n;
}

template <typename T>
__global__ void __launch_bounds__(256) balance_rows_kernel(BalanceProblem p, const float* g) {
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= p.rows) return;
  const T* s = static_cast<const T*>(p.scores) + (long long)row * p.ld;
  const float inv = (float)(1.0 / p.eps), lu = -logf((float)p.cols);
  float m = -INFINITY, l = 0.f;
  for (int j = lane; j < p.cols; j += 32) {
    const float x = (widen(s[j]) + (g ? g[j] : 0.f)) * inv + (p.b ? logf(p.b[j]) : lu);
    if (x != -INFINITY) lse_add(m, l, x, 1.f);
  }
  for (int o = 16; o > 0; o >>= 1)
    lse_add(m, l, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, l, o));
  if (lane == 0) p.f[row] = l == 0.f ? 0.f : (float)(-p.eps * ((double)m + log((double)l)));
}

template <typename T>
__global__ void __launch_bounds__(256) balance_cols_kernel(BalanceProblem p, float2* parts) {
  __shared__ float2 sh[8][33];
  const int j = blockIdx.x * 32 + (threadIdx.x & 31), w = threadIdx.x >> 5;
  const int r0 = blockIdx.y * BAL_ROWS, r1 = min(p.rows, r0 + BAL_ROWS);
  const float inv = (float)(1.0 / p.eps), lu = -logf((float)p.rows);
  float m = -INFINITY, l = 0.f;
  if (j < p.cols)
    for (int i = r0 + w; i < r1; i += 8) {
      const float x = (widen(static_cast<const T*>(p.scores)[i * p.ld + j]) + p.f[i]) * inv + (p.a ? logf(p.a[i]) : lu);
      if (x != -INFINITY) lse_add(m, l, x, 1.f);
    }
  sh[w][threadIdx.x & 31] = make_float2(m, l);
  __syncthreads();
  if (w == 0 && j < p.cols) {
    for (int k = 1; k < 8; ++k) lse_add(m, l, sh[k][threadIdx.x].x, sh[k][threadIdx.x].y);
    parts[(size_t)blockIdx.y * p.cols + j] = make_float2(m, l);
  }
}

__global__ void balance_merge_kernel(BalanceProblem p, const float2* parts, int n) {
  const int j = blockIdx.x * blockDim.x + threadIdx.x;
  if (j >= p.cols) return;
  float m = -INFINITY, l = 0.f;
  for (int k = 0; k < n; ++k) lse_add(m, l, parts[(size_t)k * p.cols + j].x, parts[(size_t)k * p.cols + j].y);
  p.g[j] = l == 0.f ? 0.f : (float)(-p.eps * ((double)m + log((double)l)));
}

template <typename T>
cudaError_t run(const BalanceProblem& p, float2* parts, cudaStream_t stream) {
  const int blocks = (p.rows + BAL_ROWS - 1) / BAL_ROWS;
  for (int it = 0; it < p.iters; ++it) {
    balance_rows_kernel<T><<<(p.rows + 7) / 8, 256, 0, stream>>>(p, it == 0 ? p.g0 : p.g);
    balance_cols_kernel<T><<<dim3((p.cols + 31) / 32, blocks), 256, 0, stream>>>(p, parts);
    balance_merge_kernel<<<(p.cols + 127) / 128, 128, 0, stream>>>(p, parts, blocks);
  }
  return cudaGetLastError();
}

}  // namespace

size_t balance_workspace_bytes(int, int rows, int cols) {
  return (size_t)((rows + BAL_ROWS - 1) / BAL_ROWS) * cols * sizeof(float2);
}

cudaError_t balance_launch(int, int type, const BalanceProblem& p, void* ws, cudaStream_t stream) {
  float2* parts = static_cast<float2*>(ws);
  switch (type) {
    case TRNOPT_F32: return run<float>(p, parts, stream);
    case TRNOPT_F16: return run<__half>(p, parts, stream);
    default: return run<__nv_bfloat16>(p, parts, stream);
  }
}

}  // namespace trnopt

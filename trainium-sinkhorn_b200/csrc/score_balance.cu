// Sinkhorn on a score matrix: the potentials of the entropic transport plan
//     P_ij = a_i b_j exp((f_i + g_j + S_ij) / eps)
// between rows of mass a and columns of mass b, by the half-steps of the reference (src/trnopt/sinkhorn.py:108-119,
// with the cost -S held as a matrix):
//     f_i = -eps LSE_j(log b_j + (g_j + S_ij) / eps),   g_j = -eps LSE_i(log a_i + (f_i + S_ij) / eps).
// A row or column without mass to exchange (all its terms zero) takes potential 0.
//
// Both half-steps of an iteration come from one exponential per score. In base 2, with c = log2 e / eps and the column
// potentials u_j = g_j c, a row's terms are e_j = 2^(S_ij c + u_j - m_i) and its sum l_i = sum_j b_j e_j, so
// f_i c = -(m_i + log2 l_i); the column sums k_j = sum_i a_i e_ij / l_i then give the next potentials,
// u_j <- u_j - log2 k_j. After an iteration every column's k_j would be 1, so the next one's lies between the smallest
// a_i / (row sum) and the largest, far from underflow; only the first iteration, from any g, keeps a running maximum per
// column instead. Potentials are held in float64 (their float32 copies are taken relative to the largest, which a row's
// maximum absorbs), the sums over rows in float32 per warp and float64 over the CTAs.
//
// One cooperative launch runs all iterations: a CTA owns a block of rows (which its L1 or the L2 holds after the first
// pass) and a warp takes kRows of them at a time, C columns per lane. Per iteration the CTAs exchange their column sums
// through global memory and one grid barrier, and each adds up all of them in the same order. Bound by the
// exponentials (16 per clock and SM) for many rows, by the barrier's latency for few.
#include <math.h>

#include "common.cuh"
#include "kernels.h"
#include "score_types.cuh"
#include "scores.h"

namespace trnopt {

namespace {

constexpr unsigned kAll = 0xffffffffu;

__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm("redux.sync.max.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "r"(kAll));
  return r;
}

// The sums over the warp of kRows values per lane, in every lane: the first steps halve the values a lane carries.
template <int kRows>
__device__ __forceinline__ void warp_sums(float (&v)[kRows]) {
  const int lane = threadIdx.x & 31;
  int o = 16;
#pragma unroll
  for (int n = kRows; n > 1; n /= 2, o /= 2) {
    const bool upper = lane & o;
#pragma unroll
    for (int k = 0; k < n / 2; ++k) {
      const float give = upper ? v[k] : v[k + n / 2], keep = upper ? v[k + n / 2] : v[k];
      v[k] = keep + __shfl_xor_sync(kAll, give, o);
    }
  }
  for (; o > 0; o /= 2) v[0] += __shfl_xor_sync(kAll, v[0], o);
  if (kRows > 1) {
    // value r sits in the lanes whose upper bits spell r
    const float mine = v[0];
    constexpr int kShift = kRows == 2 ? 4 : kRows == 4 ? 3 : 2;
#pragma unroll
    for (int r = 0; r < kRows; ++r) v[r] = __shfl_sync(kAll, mine, r << kShift);
  }
}

__device__ __forceinline__ void lse2_add(float& m, float& l, float om, float ol) {
  const float n = om != om ? om : fmaxf(m, om);      // a NaN stays
  if (n == -INFINITY) return;
  l = l * exp2f(m - n) + ol * exp2f(om - n);
  m = n;
}

// Arrive at the grid's barrier and wait until `target` arrivals have been made; false (on every thread) if that takes
// longer than the bound on waits.
__device__ __forceinline__ bool grid_barrier(unsigned* counter, unsigned target, int* error_word, int* flag) {
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    atomicAdd(counter, 1u);
    const unsigned long long t0 = globaltimer_ns();
    int ok = 1;
    unsigned seen;
    for (;;) {
      asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(seen) : "l"(counter) : "memory");
      if (seen >= target) break;
      if (globaltimer_ns() - t0 > kWaitLimitNs) {
        atomicOr(error_word, (int)kErrWaitTimeout);
        ok = 0;
        break;
      }
    }
    *flag = ok;
  }
  __syncthreads();
  return *flag != 0;
}

struct BalanceWork {
  unsigned* counter;       // arrivals at the barrier, 0 at the start
  float2* parts;           // (2, CTAs, cols): column sums (maximum and sum in the first iteration), by parity
  int* error_word;
};

template <int C> struct BalanceShape {
  static constexpr int kThreads = C == 32 ? 256 : 512;
  static constexpr int kRows = C <= 4 ? 4 : C == 8 ? 2 : 1;
};

// C columns per lane, kPair: in neighbouring pairs (2 lane + 64 k), else lane + 32 k.
template <typename T, int C, bool kPair>
__global__ void __launch_bounds__(BalanceShape<C>::kThreads, 1) balance_kernel(BalanceProblem p, BalanceWork wk) {
  constexpr int NT = BalanceShape<C>::kThreads, NW = NT / 32, kRows = BalanceShape<C>::kRows;
  extern __shared__ __align__(16) unsigned char smem[];
  // per-warp column sums, then the slices of the sum over the CTAs; the potentials u; whether a column has any term
  float2* red = reinterpret_cast<float2*>(smem);                    // (NW, cols)
  double* us = reinterpret_cast<double*>(red + (size_t)NW * p.cols);
  unsigned char* open = reinterpret_cast<unsigned char*>(us + p.cols);
  __shared__ int flag;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, cols = p.cols;
  const T* scores = static_cast<const T*>(p.scores);
  const double per_eps = 1.4426950408889634 / p.eps;
  const float c = (float)per_eps;
  const long long r0 = (long long)blockIdx.x * p.rows / gridDim.x, r1 = (long long)(blockIdx.x + 1) * p.rows / gridDim.x;
  auto column = [&](int k) { return kPair ? 2 * lane + 64 * (k / 2) + (k & 1) : lane + 32 * k; };

  float b[C], u[C];
  bool closed = false;                                      // a column of mass 0 is there
#pragma unroll
  for (int k = 0; k < C; ++k) {
    const int j = column(k);
    b[k] = j < cols ? (p.b ? p.b[j] : 1.f / (float)cols) : 0.f;
    closed = closed || (j < cols && b[k] == 0.f);
  }
  closed = __any_sync(kAll, closed);
  for (int j = tid; j < cols; j += NT) us[j] = p.g0 ? (double)p.g0[j] * per_eps : 0.0;
  __syncthreads();

  for (int it = 0; it < p.iters; ++it) {
    const bool first = it == 0, last = it == p.iters - 1;
    // float32 potentials relative to the largest
    double shift = -INFINITY;
#pragma unroll
    for (int k = 0; k < C; ++k) shift = fmax(shift, column(k) < cols ? us[column(k)] : -INFINITY);
    for (int o = 16; o > 0; o >>= 1) shift = fmax(shift, __shfl_xor_sync(kAll, shift, o));
    if (!(fabs(shift) < INFINITY)) shift = 0.0;
#pragma unroll
    for (int k = 0; k < C; ++k) u[k] = column(k) < cols ? (float)(us[column(k)] - shift) : -INFINITY;

    float sum[C], peak[C];                                  // column sums; their maxima in the first iteration
#pragma unroll
    for (int k = 0; k < C; ++k) { sum[k] = 0.f; peak[k] = -INFINITY; }
    for (long long row = r0 + (long long)w * kRows; row < r1; row += NW * kRows) {
      float z[kRows][C], m[kRows], l[kRows], a[kRows];
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const bool there = row + r < r1;
        const T* s = scores + (there ? row + r : row) * p.ld;
        a[r] = there ? (p.a ? p.a[row + r] : 1.f) : 0.f;
#pragma unroll
        for (int k = 0; k < C; k += kPair ? 2 : 1) {
          const int j = column(k);
          if constexpr (kPair) {
            float x0 = -INFINITY, x1 = -INFINITY;
            if (j < cols) load_pair(s + j, x0, x1);
            z[r][k] = x0;
            z[r][k + 1] = x1;
          } else {
            z[r][k] = j < cols ? widen(s[j]) : -INFINITY;
          }
        }
      }
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        m[r] = -INFINITY;
#pragma unroll
        for (int k = 0; k < C; ++k) {
          z[r][k] = fmaf(z[r][k], c, u[k]);
          m[r] = fmaxf(m[r], !closed || b[k] > 0.f ? z[r][k] : -INFINITY);
        }
        m[r] = warp_max(m[r]);
        const float shown = m[r] == -INFINITY ? 0.f : m[r];
        l[r] = 0.f;
#pragma unroll
        for (int k = 0; k < C; ++k) {
          z[r][k] -= shown;
          const float e = ex2_approx(z[r][k]);
          l[r] = fmaf(b[k], b[k] > 0.f ? e : 0.f, l[r]);
          if (!first) z[r][k] = e;
        }
      }
      warp_sums<kRows>(l);
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const bool empty = l[r] == 0.f;                     // f = 0: terms 2^(S c + u) as they are, less the shift
        if (last && lane == 0 && row + r < r1)
          p.f[row + r] = empty ? 0.f : (float)(-((double)(m[r] == -INFINITY ? 0.f : m[r]) + (double)log2f(l[r]) + shift) / per_eps);
        if (first) {
          // x = S c + f c + log2 a, in the gauge of u - shift: z - u - log2 l + log2 a
          const float off = (empty ? (float)shift : -log2f(l[r])) + log2f(a[r]);
#pragma unroll
          for (int k = 0; k < C; ++k) {
            const float x = z[r][k] - u[k] + off;
            if (column(k) < cols && x != -INFINITY) lse2_add(peak[k], sum[k], x, 1.f);
          }
        } else {
          const float weight = empty ? a[r] * exp2f((float)shift) : a[r] / l[r];
          if (a[r] != 0.f)
#pragma unroll
            for (int k = 0; k < C; ++k) sum[k] = fmaf(z[r][k], weight, sum[k]);
        }
      }
    }

    // column sums of the CTA's warps, then of all CTAs (in the same order everywhere)
    float2* mine = red + (size_t)w * cols;
#pragma unroll
    for (int k = 0; k < C; ++k)
      if (column(k) < cols) mine[column(k)] = make_float2(peak[k], sum[k]);
    __syncthreads();
    float2* parts = wk.parts + (size_t)(it & 1) * gridDim.x * cols;
    for (int j = tid; j < cols; j += NT) {
      float2 v = red[j];
      for (int k = 1; k < NW; ++k) {
        const float2 o = red[(size_t)k * cols + j];
        if (first) lse2_add(v.x, v.y, o.x, o.y);
        else v.y += o.y;
      }
      __stcg(parts + (size_t)blockIdx.x * cols + j, v);
    }
    if (!grid_barrier(wk.counter, (unsigned)(it + 1) * gridDim.x, wk.error_word, &flag)) {
      // gave up: no potentials
      for (long long i = r0 + tid; i < r1; i += NT) p.f[i] = NAN;
      if (blockIdx.x == 0)
        for (int j = tid; j < cols; j += NT) p.g[j] = NAN;
      return;
    }
    const double log_rows = p.a ? 0.0 : log2((double)p.rows);
    for (int j = tid; j < cols; j += NT) {
      double next;
      if (first) {
        float2 v = __ldcg(parts + j);
        for (int k = 1; k < (int)gridDim.x; ++k) {
          const float2 o = __ldcg(parts + (size_t)k * cols + j);
          lse2_add(v.x, v.y, o.x, o.y);
        }
        open[j] = v.y != 0.f;
        next = v.y == 0.f ? 0.0 : shift + log_rows - ((double)v.x + log2((double)v.y));
      } else {
        double k_j = 0.0;
        for (int k = 0; k < (int)gridDim.x; ++k) k_j += (double)__ldcg(&parts[(size_t)k * cols + j].y);
        // the same float32 potential that the sums were formed with
        const double before = (double)(float)(us[j] - shift) + shift;
        // (a sum that underflows, for masses beyond float32's range from one another, counts as 2^-126)
        next = open[j] ? before + log_rows - log2(k_j == 0.0 ? 0x1p-126 : k_j) : 0.0;
      }
      us[j] = next;
    }
    __syncthreads();
  }
  if (blockIdx.x == 0)
    for (int j = tid; j < cols; j += NT) p.g[j] = (float)(us[j] / per_eps);
}

size_t smem_bytes(int cols, int threads) { return (size_t)(threads / 32) * cols * sizeof(float2) + cols * (sizeof(double) + 1); }

int columns_per_lane(int cols) {
  int c = 1;
  while (32 * c < cols) c *= 2;
  return c;
}

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

// CTAs: one per SM, each with at least 128 rows.
int balance_grid(int device, int rows) {
  const int most = sm_count(device), want = (rows + 127) / 128;
  return want < most ? want : most;
}

template <typename T, int C, bool kPair>
cudaError_t launch(int device, const BalanceProblem& p, const BalanceWork& wk, cudaStream_t stream) {
  const size_t bytes = smem_bytes(p.cols, BalanceShape<C>::kThreads);
  static std::atomic<int> done[kMaxDevices];
  cudaError_t e = smem_attr_once(reinterpret_cast<const void*>(balance_kernel<T, C, kPair>), (int)bytes, done);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)balance_grid(device, p.rows));
  cfg.blockDim = dim3(BalanceShape<C>::kThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeCooperative;                // its CTAs wait for one another
  attr.val.cooperative = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, balance_kernel<T, C, kPair>, p, wk);
}

template <typename T>
cudaError_t launch(int device, const BalanceProblem& p, const BalanceWork& wk, cudaStream_t stream) {
  const bool pair = p.cols % 2 == 0 && p.ld % 2 == 0 && reinterpret_cast<uintptr_t>(p.scores) % (2 * sizeof(T)) == 0;
  switch (columns_per_lane(p.cols)) {
    case 1: return launch<T, 1, false>(device, p, wk, stream);
    case 2: return pair ? launch<T, 2, true>(device, p, wk, stream) : launch<T, 2, false>(device, p, wk, stream);
    case 4: return pair ? launch<T, 4, true>(device, p, wk, stream) : launch<T, 4, false>(device, p, wk, stream);
    case 8: return pair ? launch<T, 8, true>(device, p, wk, stream) : launch<T, 8, false>(device, p, wk, stream);
    case 16: return pair ? launch<T, 16, true>(device, p, wk, stream) : launch<T, 16, false>(device, p, wk, stream);
    default: return pair ? launch<T, 32, true>(device, p, wk, stream) : launch<T, 32, false>(device, p, wk, stream);
  }
}

constexpr size_t kCounterBytes = 256;

}  // namespace

size_t balance_workspace_bytes(int device, int rows, int cols) {
  return kCounterBytes + (size_t)2 * balance_grid(device, rows) * cols * sizeof(float2);
}

cudaError_t balance_launch(int device, int type, const BalanceProblem& p, void* ws, cudaStream_t stream) {
  BalanceWork wk{static_cast<unsigned*>(ws), reinterpret_cast<float2*>(static_cast<char*>(ws) + kCounterBytes),
                 device_error_word()};
  const cudaError_t e = cudaMemsetAsync(ws, 0, sizeof(unsigned), stream);
  if (e != cudaSuccess) return e;
  switch (type) {
    case TRNOPT_F32: return launch<float>(device, p, wk, stream);
    case TRNOPT_F16: return launch<__half>(device, p, wk, stream);
    default: return launch<__nv_bfloat16>(device, p, wk, stream);
  }
}

}  // namespace trnopt

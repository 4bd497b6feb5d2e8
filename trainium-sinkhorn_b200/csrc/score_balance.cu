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

#include <type_traits>

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
  float* parts;            // (2, 2, CTAs, cols rounded up to 4): by parity, the CTAs' column sums, and their maxima in the
                           // first iteration
  int* error_word;
};

template <int C> struct BalanceShape {
  static constexpr int kThreads = C == 32 ? 256 : 512;
  static constexpr int kRows = C <= 8 ? 4 : C == 16 ? 2 : 1;
};

// Shared memory for the warps' column sums, and then for the slices of the sum over the CTAs (NT quads of float64).
__host__ __device__ inline size_t exchange_bytes(int cols, int threads) {
  const size_t warps = (size_t)(threads / 32) * cols * sizeof(float2), slices = (size_t)threads * 4 * sizeof(double);
  return ((warps > slices ? warps : slices) + 15) & ~(size_t)15;
}

// C columns per lane, in runs of V neighbouring ones.
template <typename T, int C, int V>
__global__ void __launch_bounds__(BalanceShape<C>::kThreads, 1) balance_kernel(BalanceProblem p, BalanceWork wk) {
  constexpr int NT = BalanceShape<C>::kThreads, NW = NT / 32, kRows = BalanceShape<C>::kRows;
  extern __shared__ __align__(16) unsigned char smem[];
  // per-warp column sums, then the slices of the sum over the CTAs; the potentials u; whether a column has any term
  float2* red = reinterpret_cast<float2*>(smem);                    // (NW, cols)
  const int cols4 = (p.cols + 3) & ~3;
  double* us = reinterpret_cast<double*>(smem + exchange_bytes(p.cols, NT));
  unsigned char* open = reinterpret_cast<unsigned char*>(us + p.cols);
  __shared__ int flag;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, cols = p.cols;
  const T* scores = static_cast<const T*>(p.scores);
  const double per_eps = 1.4426950408889634 / p.eps, eps_per = p.eps * 0.6931471805599453;
  const float c = (float)per_eps;
  const long long r0 = (long long)blockIdx.x * p.rows / gridDim.x, r1 = (long long)(blockIdx.x + 1) * p.rows / gridDim.x;
  auto column = [&](int k) { return V * lane + 32 * V * (k / V) + k % V; };

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
    // the rows: kFirst with running maxima per column, kClosed where columns of mass 0 must not set a row's maximum
    auto pass = [&](auto first_, auto closed_) {
      constexpr bool kFirst = decltype(first_)::value, kClosed = decltype(closed_)::value;
      const T* at = scores + (r0 + (long long)w * kRows) * p.ld + V * lane;
      for (long long row = r0 + (long long)w * kRows; row < r1; row += NW * kRows, at += NW * kRows * p.ld) {
        float z[kRows][C], m[kRows], l[kRows];
        const bool whole = row + kRows <= r1;
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          const T* s = at + (whole || row + r < r1 ? r * p.ld : 0);
#pragma unroll
          for (int k = 0; k < C; k += V) {
            if (column(k) < cols) {
              load_scores<V>(s + 32 * k, z[r] + k);
            } else {
#pragma unroll
              for (int i = 0; i < V; ++i) z[r][k + i] = -INFINITY;
            }
          }
        }
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          float top = -INFINITY;
#pragma unroll
          for (int k = 0; k < C; ++k) {
            z[r][k] = fmaf(z[r][k], c, u[k]);
            top = fmaxf(top, !kClosed || b[k] > 0.f ? z[r][k] : -INFINITY);
          }
          top = warp_max(top);
          m[r] = top == -INFINITY ? 0.f : top;
          l[r] = 0.f;
          if constexpr (C % 2 == 0 && !kClosed) {
            uint64_t l2 = 0;
            const uint64_t m2 = pack2(-m[r], -m[r]);
#pragma unroll
            for (int k = 0; k < C; k += 2) {
              float x, y;
              unpack2(add2(pack2(z[r][k], z[r][k + 1]), m2), x, y);
              const float ex = ex2_approx(x), ey = ex2_approx(y);
              l2 = fma2(pack2(b[k], b[k + 1]), pack2(ex, ey), l2);
              z[r][k] = kFirst ? x : ex;
              z[r][k + 1] = kFirst ? y : ey;
            }
            float x, y;
            unpack2(l2, x, y);
            l[r] = x + y;
          } else {
#pragma unroll
            for (int k = 0; k < C; ++k) {
              z[r][k] -= m[r];
              const float e = ex2_approx(z[r][k]);
              l[r] = fmaf(b[k], !kClosed || b[k] > 0.f ? e : 0.f, l[r]);
              if (!kFirst) z[r][k] = e;
            }
          }
        }
        warp_sums<kRows>(l);
        if (last && lane < kRows && row + lane < r1) {
          float lr = l[0], mr = m[0];
#pragma unroll
          for (int r = 1; r < kRows; ++r) {
            lr = lane == r ? l[r] : lr;
            mr = lane == r ? m[r] : mr;
          }
          p.f[row + lane] = lr == 0.f ? 0.f : (float)(-((double)mr + (double)log2f(lr) + shift) * eps_per);
        }
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          const float a = !whole && row + r >= r1 ? 0.f : p.a ? __ldg(p.a + row + r) : 1.f;
          const bool empty = l[r] == 0.f;                   // f = 0: terms 2^(S c + u) as they are, less the shift
          if constexpr (kFirst) {
            // x = S c + f c + log2 a, in the gauge of u - shift: z - u - log2 l + log2 a
            const float off = (empty ? (float)shift : -log2f(l[r])) + log2f(a);
#pragma unroll
            for (int k = 0; k < C; ++k) {
              const float x = z[r][k] - u[k] + off;
              if (column(k) < cols && x != -INFINITY) lse2_add(peak[k], sum[k], x, 1.f);
            }
          } else if (a != 0.f) {
            const float weight = empty ? a * exp2f((float)shift) : __fdividef(a, l[r]);
            if constexpr (C % 2 == 0) {
              const uint64_t w2 = pack2(weight, weight);
#pragma unroll
              for (int k = 0; k < C; k += 2)
                unpack2(fma2(pack2(z[r][k], z[r][k + 1]), w2, pack2(sum[k], sum[k + 1])), sum[k], sum[k + 1]);
            } else {
#pragma unroll
              for (int k = 0; k < C; ++k) sum[k] = fmaf(z[r][k], weight, sum[k]);
            }
          }
        }
      }
    };
    if (first) pass(std::true_type{}, std::true_type{});
    else if (closed) pass(std::false_type{}, std::true_type{});
    else pass(std::false_type{}, std::false_type{});

    // column sums of the CTA's warps
    float2* mine = red + (size_t)w * cols;
#pragma unroll
    for (int k = 0; k < C; ++k)
      if (column(k) < cols) mine[column(k)] = make_float2(peak[k], sum[k]);
    __syncthreads();
    const size_t plane = (size_t)gridDim.x * cols4;
    float* sums = wk.parts + (size_t)(it & 1) * 2 * plane;
    float* peaks = sums + plane;
    for (int j = tid; j < cols; j += NT) {
      float2 v = red[j];
      for (int k = 1; k < NW; ++k) {
        const float2 o = red[(size_t)k * cols + j];
        if (first) lse2_add(v.x, v.y, o.x, o.y);
        else v.y += o.y;
      }
      __stcg(sums + (size_t)blockIdx.x * cols4 + j, v.y);
      if (first) __stcg(peaks + (size_t)blockIdx.x * cols4 + j, v.x);
    }
    if (!grid_barrier(wk.counter, (unsigned)(it + 1) * gridDim.x, wk.error_word, &flag)) {
      // gave up: no potentials
      for (long long i = r0 + tid; i < r1; i += NT) p.f[i] = NAN;
      if (blockIdx.x == 0)
        for (int j = tid; j < cols; j += NT) p.g[j] = NAN;
      return;
    }
    // of all CTAs, in the same order in each: four columns per thread, the CTAs in `slices` interleaved parts
    const int quads = cols4 / 4, slices = NT / quads, slice = tid / quads, quad = tid - slice * quads;
    double* part = reinterpret_cast<double*>(smem) + (size_t)slice * cols4 + 4 * quad;   // (`red` is free again)
    if (slice < slices) {
      if (first) {
        float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, l[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int k = slice; k < (int)gridDim.x; k += slices) {
          const float4 om = __ldcg(reinterpret_cast<const float4*>(peaks + (size_t)k * cols4) + quad);
          const float4 ol = __ldcg(reinterpret_cast<const float4*>(sums + (size_t)k * cols4) + quad);
          lse2_add(m[0], l[0], om.x, ol.x);
          lse2_add(m[1], l[1], om.y, ol.y);
          lse2_add(m[2], l[2], om.z, ol.z);
          lse2_add(m[3], l[3], om.w, ol.w);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) *reinterpret_cast<float2*>(part + e) = make_float2(m[e], l[e]);
      } else {
        double v[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll 16
        for (int k = slice; k < (int)gridDim.x; k += slices) {
          const float4 o = __ldcg(reinterpret_cast<const float4*>(sums + (size_t)k * cols4) + quad);
          v[0] += (double)o.x;
          v[1] += (double)o.y;
          v[2] += (double)o.z;
          v[3] += (double)o.w;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) part[e] = v[e];
      }
    }
    __syncthreads();
    const double log_rows = p.a ? 0.0 : log2((double)p.rows);
    for (int j = tid; j < cols; j += NT) {
      const double* at = reinterpret_cast<const double*>(smem) + j;
      double next;
      if (first) {
        float2 v = *reinterpret_cast<const float2*>(at);
        for (int k = 1; k < slices; ++k) {
          const float2 o = *reinterpret_cast<const float2*>(at + (size_t)k * cols4);
          lse2_add(v.x, v.y, o.x, o.y);
        }
        open[j] = v.y != 0.f;
        next = v.y == 0.f ? 0.0 : shift + log_rows - ((double)v.x + log2((double)v.y));
      } else {
        double k_j = 0.0;
        for (int k = 0; k < slices; ++k) k_j += at[(size_t)k * cols4];
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
    for (int j = tid; j < cols; j += NT) p.g[j] = (float)(us[j] * eps_per);
}

size_t smem_bytes(int cols, int threads) { return exchange_bytes(cols, threads) + cols * (sizeof(double) + 1); }

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

template <typename T, int C, int V>
cudaError_t launch(int device, const BalanceProblem& p, const BalanceWork& wk, cudaStream_t stream) {
  const size_t bytes = smem_bytes(p.cols, BalanceShape<C>::kThreads);
  static std::atomic<int> done[kMaxDevices];
  cudaError_t e = smem_attr_once(reinterpret_cast<const void*>(balance_kernel<T, C, V>), (int)bytes, done);
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
  return cudaLaunchKernelEx(&cfg, balance_kernel<T, C, V>, p, wk);
}

template <typename T>
cudaError_t launch(int device, const BalanceProblem& p, const BalanceWork& wk, cudaStream_t stream) {
  // the longest runs of columns per lane (up to 16 bytes) that the sizes and addresses allow
  auto runs = [&](int v) {
    return p.cols % v == 0 && p.ld % v == 0 && reinterpret_cast<uintptr_t>(p.scores) % (v * sizeof(T)) == 0;
  };
  constexpr int kLong = 16 / (int)sizeof(T);
  switch (columns_per_lane(p.cols)) {
    case 1: return launch<T, 1, 1>(device, p, wk, stream);
    case 2: return runs(2) ? launch<T, 2, 2>(device, p, wk, stream) : launch<T, 2, 1>(device, p, wk, stream);
    case 4: return runs(4) ? launch<T, 4, 4>(device, p, wk, stream)
                           : runs(2) ? launch<T, 4, 2>(device, p, wk, stream) : launch<T, 4, 1>(device, p, wk, stream);
    case 8: return runs(kLong) ? launch<T, 8, kLong>(device, p, wk, stream)
                               : runs(2) ? launch<T, 8, 2>(device, p, wk, stream) : launch<T, 8, 1>(device, p, wk, stream);
    case 16: return runs(kLong) ? launch<T, 16, kLong>(device, p, wk, stream)
                                : runs(2) ? launch<T, 16, 2>(device, p, wk, stream) : launch<T, 16, 1>(device, p, wk, stream);
    default: return runs(kLong) ? launch<T, 32, kLong>(device, p, wk, stream)
                                : runs(2) ? launch<T, 32, 2>(device, p, wk, stream) : launch<T, 32, 1>(device, p, wk, stream);
  }
}

constexpr size_t kCounterBytes = 256;

}  // namespace

size_t balance_workspace_bytes(int device, int rows, int cols) {
  return kCounterBytes + (size_t)4 * balance_grid(device, rows) * ((cols + 3) & ~3) * sizeof(float);
}

cudaError_t balance_launch(int device, int type, const BalanceProblem& p, void* ws, cudaStream_t stream) {
  BalanceWork wk{static_cast<unsigned*>(ws), reinterpret_cast<float*>(static_cast<char*>(ws) + kCounterBytes),
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

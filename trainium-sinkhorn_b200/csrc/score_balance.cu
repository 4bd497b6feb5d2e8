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
// column instead. Potentials are float32 relative to a column's after the first iteration (the common part, in float64,
// goes back at the end): they are differences of a few units, where the potentials themselves may be hundreds.
//
// One cooperative launch runs all iterations. A CTA owns a block of rows and keeps as many of them as fit in shared
// memory as they were read in the first pass (the rest come from L2 in every pass); a warp takes kRows of them at a
// time, C columns per lane, and a lane meets the same scores in every pass. Per iteration the CTAs exchange their column
// sums through global memory and one grid barrier, and each adds up all of them in the same order. Bound by the
// exponentials (16 per clock and SM) for many rows, by the barrier's latency for few; problems of up to
// 1024 rows of 32 columns (512 of 64, ...) stay in one CTA, without it.
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
    asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(counter) : "memory");
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

// Shared memory: the warps' column sums, later the slices of the sum over the CTAs (NT quads), and the potentials; after
// it the rows that are kept.
__host__ __device__ inline size_t exchange_bytes(int cols, int threads) {
  const size_t warps = (size_t)(threads / 32) * cols * sizeof(float2), slices = (size_t)threads * 4 * sizeof(float2);
  return ((warps > slices ? warps : slices) + 15) & ~(size_t)15;
}
__host__ __device__ inline size_t fixed_bytes(int cols, int threads) {
  return (exchange_bytes(cols, threads) + cols * (sizeof(float) + 1) + 15) & ~(size_t)15;
}
__host__ __device__ inline int row_bytes(int cols, int size) { return (cols * size + 15) & ~15; }

// C columns per lane, in runs of V neighbouring ones.
template <typename T, int C, int V>
__global__ void __launch_bounds__(BalanceShape<C>::kThreads, 1) balance_kernel(BalanceProblem p, BalanceWork wk,
                                                                           int kept_rows) {
  constexpr int NT = BalanceShape<C>::kThreads, NW = NT / 32, kRows = BalanceShape<C>::kRows;
  extern __shared__ __align__(16) unsigned char smem[];
  // per-warp column sums, then the slices of the sum over the CTAs; the potentials; whether a column has any term; rows
  float2* red = reinterpret_cast<float2*>(smem);                    // (NW, cols)
  float* us = reinterpret_cast<float*>(smem + exchange_bytes(p.cols, NT));
  unsigned char* open = reinterpret_cast<unsigned char*>(us + p.cols);
  T* kept = reinterpret_cast<T*>(smem + fixed_bytes(p.cols, NT));   // (kept_rows, pitch)
  __shared__ int flag;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, cols = p.cols, cols4 = (cols + 3) & ~3;
  const int pitch = row_bytes(cols, sizeof(T)) / (int)sizeof(T);
  const T* scores = static_cast<const T*>(p.scores);
  const double per_eps = 1.4426950408889634 / p.eps, eps_per = p.eps * 0.6931471805599453;
  const float c = (float)per_eps, per_rows = p.a ? 1.f : 1.f / (float)p.rows;
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
  // what float32 potentials are relative to: 0, or the given potential of column 0; later its potential after one iteration
  double shift = p.g0 && fabsf(p.g0[0]) < INFINITY ? (double)p.g0[0] * per_eps : 0.0;
  for (int j = tid; j < cols; j += NT) us[j] = p.g0 ? (float)((double)p.g0[j] * per_eps - shift) : 0.f;
  __syncthreads();

  for (int it = 0; it < p.iters; ++it) {
    const bool first = it == 0, last = it == p.iters - 1;
#pragma unroll
    for (int k = 0; k < C; ++k) u[k] = column(k) < cols ? us[column(k)] : -INFINITY;

    float sum[C], peak[C];                                  // column sums; their maxima in the first iteration
#pragma unroll
    for (int k = 0; k < C; ++k) { sum[k] = 0.f; peak[k] = -INFINITY; }
    // the rows: kFirst with running maxima per column, kClosed where columns of mass 0 must not set a row's maximum
    auto pass = [&](auto first_, auto closed_) {
      constexpr bool kFirst = decltype(first_)::value, kClosed = decltype(closed_)::value;
      const T* at = scores + (r0 + (long long)w * kRows) * p.ld + V * lane;
      T* here = kept + (size_t)w * kRows * pitch + V * lane;
      for (long long row = r0 + (long long)w * kRows; row < r1;
           row += NW * kRows, at += NW * kRows * p.ld, here += NW * kRows * pitch) {
        float z[kRows][C], m[kRows], l[kRows];
        const bool whole = row + kRows <= r1, keep = row - r0 + kRows <= kept_rows;
        if (!kFirst && keep) {
#pragma unroll
          for (int r = 0; r < kRows; ++r)
#pragma unroll
            for (int k = 0; k < C; k += V)
              if (column(k) < cols) {
                const Vec<T> v = read_any<V>(here + r * pitch + 32 * k);
#pragma unroll
                for (int i = 0; i < V; ++i) z[r][k + i] = v.get(i);
              } else {
#pragma unroll
                for (int i = 0; i < V; ++i) z[r][k + i] = -INFINITY;
              }
        } else {
#pragma unroll
          for (int r = 0; r < kRows; ++r) {
            const T* s = at + (whole || row + r < r1 ? r * p.ld : 0);
#pragma unroll
            for (int k = 0; k < C; k += V)
              if (column(k) < cols) {
                const Vec<T> v = read_global<V>(s + 32 * k);
                if (kFirst && keep) write_any<V>(here + r * pitch + 32 * k, v);
#pragma unroll
                for (int i = 0; i < V; ++i) z[r][k + i] = v.get(i);
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
          const bool empty = l[r] == 0.f;                   // f = 0: the terms 2^(S c + u) as they are
          if constexpr (kFirst) {
            // x = S c + f c + log2 a, in the gauge of u - shift: z - u - log2 l + log2 a
            const float off = (empty ? (float)shift : -log2f(l[r])) + log2f(a);
#pragma unroll
            for (int k = 0; k < C; ++k) {
              const float x = z[r][k] - u[k] + off;
              if (column(k) < cols && x != -INFINITY) lse2_add(peak[k], sum[k], x, 1.f);
            }
          } else if (empty) {
            if (a != 0.f)
#pragma unroll
              for (int k = 0; k < C; ++k)
                if (z[r][k] > 0.f) sum[k] += a * exp2f(log2f(z[r][k]) + (float)shift);
          } else if (a != 0.f) {
            const float weight = __fdividef(a, l[r]);
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
    const bool alone = gridDim.x == 1;
    const size_t plane = (size_t)gridDim.x * cols4;
    float* sums = wk.parts + (size_t)(it & 1) * 2 * plane;
    float* peaks = sums + plane;
    for (int j = tid; j < cols; j += NT) {
      float2 v = red[j];
      if (first) {
        for (int k = 1; k < NW; ++k) lse2_add(v.x, v.y, red[(size_t)k * cols + j].x, red[(size_t)k * cols + j].y);
      } else {
#pragma unroll
        for (int k = 1; k < NW; ++k) v.y += red[(size_t)k * cols + j].y;
      }
      if (alone) {
        red[j] = v;                                         // (row 0 of `red` is read by this thread alone)
      } else {
        __stcg(sums + (size_t)blockIdx.x * cols4 + j, v.y);
        if (first) __stcg(peaks + (size_t)blockIdx.x * cols4 + j, v.x);
      }
    }
    int slices = 1;
    if (!alone) {
      if (!grid_barrier(wk.counter, (unsigned)(it + 1) * gridDim.x, wk.error_word, &flag)) {
        // gave up: no potentials
        for (long long i = r0 + tid; i < r1; i += NT) p.f[i] = NAN;
        if (blockIdx.x == 0)
          for (int j = tid; j < cols; j += NT) p.g[j] = NAN;
        return;
      }
      // of all CTAs, in the same order in each: four columns per thread, the CTAs in `slices` interleaved parts
      const int quads = cols4 / 4, slice = tid / quads, quad = tid - slice * quads;
      slices = NT / quads;
      float2* part = red + (size_t)slice * cols4 + 4 * quad;            // (`red` is free again)
      if (slice < slices) {
        float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, v[4] = {0.f, 0.f, 0.f, 0.f};
        if (first) {
#pragma unroll 4
          for (int k = slice; k < (int)gridDim.x; k += slices) {
            const float4 om = __ldcg(reinterpret_cast<const float4*>(peaks + (size_t)k * cols4) + quad);
            const float4 ol = __ldcg(reinterpret_cast<const float4*>(sums + (size_t)k * cols4) + quad);
            lse2_add(m[0], v[0], om.x, ol.x);
            lse2_add(m[1], v[1], om.y, ol.y);
            lse2_add(m[2], v[2], om.z, ol.z);
            lse2_add(m[3], v[3], om.w, ol.w);
          }
        } else {
#pragma unroll 16
          for (int k = slice; k < (int)gridDim.x; k += slices) {
            const float4 o = __ldcg(reinterpret_cast<const float4*>(sums + (size_t)k * cols4) + quad);
            v[0] += o.x;
            v[1] += o.y;
            v[2] += o.z;
            v[3] += o.w;
          }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) part[e] = make_float2(m[e], v[e]);
      }
      __syncthreads();
    }
    for (int j = tid; j < cols; j += NT) {
      float2 v = red[j];
      if (first) {
        for (int k = 1; k < slices; ++k) lse2_add(v.x, v.y, red[(size_t)k * cols4 + j].x, red[(size_t)k * cols4 + j].y);
        // u after it, in float64 in the slices' place: the next float32 potentials are relative to column 0's
        open[j] = v.y != 0.f;
        reinterpret_cast<double*>(red)[j] =
            v.y == 0.f ? 0.0 : shift - ((double)v.x + (double)log2f(v.y * per_rows));
      } else {
        for (int k = 1; k < slices; ++k) v.y += red[(size_t)k * cols4 + j].y;
        // (a sum that underflows, for masses beyond float32's range from one another, counts as 2^-126)
        const float step = log2f(v.y == 0.f ? 1.17549435e-38f : v.y * per_rows);
        // the last potentials are not rounded to float32 before the common part goes back
        if (last && blockIdx.x == 0) p.g[j] = open[j] ? (float)(((double)us[j] - (double)step + shift) * eps_per) : 0.f;
        if (open[j]) us[j] -= step;
      }
    }
    __syncthreads();
    if (first) {
      const double* full = reinterpret_cast<const double*>(red);
      const double base = full[0];
      shift = fabs(base) < INFINITY ? base : 0.0;
      for (int j = tid; j < cols; j += NT) {
        us[j] = (float)(full[j] - shift);
        if (last && blockIdx.x == 0) p.g[j] = (float)(full[j] * eps_per);
      }
      __syncthreads();
    }
  }
}

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

// CTAs: one for problems of few rows, else one per SM with at least 64 rows each.
int balance_grid(int device, int rows, int cols) {
  if ((long long)rows * columns_per_lane(cols) <= 1024) return 1;
  const int most = sm_count(device), want = (rows + 63) / 64;
  return want < most ? want : most;
}

template <typename T, int C, int V>
cudaError_t launch(int device, const BalanceProblem& p, const BalanceWork& wk, cudaStream_t stream) {
  using Shape = BalanceShape<C>;
  const int grid = balance_grid(device, p.rows, p.cols);
  // the rows a CTA keeps: all of them, or what shared memory holds (227 KB less what the launch itself takes)
  const size_t fixed = fixed_bytes(p.cols, Shape::kThreads), most = 226 * 1024 - fixed;
  int kept = ((p.rows + grid - 1) / grid + Shape::kRows - 1) / Shape::kRows * Shape::kRows;
  const int fits = (int)(most / row_bytes(p.cols, sizeof(T))) / Shape::kRows * Shape::kRows;
  if (kept > fits) kept = fits;
  if (p.iters == 1) kept = 0;
  const size_t bytes = fixed + (size_t)kept * row_bytes(p.cols, sizeof(T));
  static std::atomic<int> done[kMaxDevices];
  cudaError_t e = smem_attr_once(reinterpret_cast<const void*>(balance_kernel<T, C, V>), (int)bytes, done);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(Shape::kThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeCooperative;                // its CTAs wait for one another
  attr.val.cooperative = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = grid > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, balance_kernel<T, C, V>, p, wk, kept);
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
  return kCounterBytes + (size_t)4 * balance_grid(device, rows, cols) * ((cols + 3) & ~3) * sizeof(float);
}

cudaError_t balance_launch(int device, int type, const BalanceProblem& p, void* ws, cudaStream_t stream) {
  BalanceWork wk{static_cast<unsigned*>(ws), reinterpret_cast<float*>(static_cast<char*>(ws) + kCounterBytes),
                 device_error_word()};
  if (balance_grid(device, p.rows, p.cols) > 1) {
    const cudaError_t e = cudaMemsetAsync(ws, 0, sizeof(unsigned), stream);
    if (e != cudaSuccess) return e;
  }
  switch (type) {
    case TRNOPT_F32: return launch<float>(device, p, wk, stream);
    case TRNOPT_F16: return launch<__half>(device, p, wk, stream);
    default: return launch<__nv_bfloat16>(device, p, wk, stream);
  }
}

}  // namespace trnopt

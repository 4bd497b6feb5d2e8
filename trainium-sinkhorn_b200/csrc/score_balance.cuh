// Sinkhorn on a score matrix: the potentials of the entropic transport plan
//     P_ij = a_i b_j exp((f_i + g_j + S_ij) / eps)
// between rows of mass a and columns of mass b, by the half-steps of the reference (src/trnopt/sinkhorn.py:108-119,
// with the cost -S held as a matrix):
//     f_i = -eps LSE_j(log b_j + (g_j + S_ij) / eps),   g_j = -eps LSE_i(log a_i + (f_i + S_ij) / eps).
// A row or column without mass to exchange (all its terms zero) takes potential 0.
//
// Both half-steps of an iteration come from one exponential per score. In base 2, with c = log2 e / eps and the column
// potentials u_j = g_j c, a row's terms are e_j = 2^(S_ij c + u_j - m_i) and its sum l_i = sum_j b_j e_j, so f_i c =
// -(m_i + log2 l_i); the column sums k_j = sum_i a_i e_ij / l_i then give the next potentials, u_j <- u_j - log2 k_j.
// After an iteration every column's k_j would be 1, so the next one's lies between the smallest a_i / (row sum) and the
// largest, far from underflow; only the first iteration, from any g, finds each column's maximum before its sum (and
// the last one, where columns of mass 0 need theirs). Potentials are pairs of float32, relative (after the first
// iteration) to the least of those that take part, and terms are formed from their high parts: differences of a few
// units, where the potentials themselves may be hundreds. Once a row's maximum or such a column's potential lies 2^10
// or more from 0 (finite masks, offsets), a CTA forms all its terms from the pairs, less their row's own constant:
// 65536 x 256 bfloat16 103 us an iteration in place of 11. A score more than float32's range (2.3e38 eps) below its
// row's largest is as good as -inf.
//
// One cooperative launch runs all iterations. A CTA owns a block of rows and keeps as many of them as fit in shared
// memory as they were read in the first pass (the rest come from L2 in every pass). L neighbouring lanes share a row,
// up to 32 columns each, so a row's maximum and sum take log2 L shuffles for the warp's 32 / L rows together, and a
// lane sums its columns over its rows in registers. Per iteration the CTAs add their column sums up in fixed point, one
// atomic addition of a 64-bit word per column and CTA: whole numbers, so their order does not matter, and the word
// counts the CTAs, so there is no other barrier. (Every CTA's sums in float32, behind a barrier and added in the same
// order by all, took 3 to 5 us of an iteration; they are left for iterations with maxima and for sums outside the fixed
// point's range.) What one CTA takes in two steps of its warps stays in one. Bound by the pass's instructions for many
// rows, by the exchange's latency for few. Measured per iteration: 65536 x 256 bfloat16 10.9 us (7 us the pass, of
// which 3.7 us are exponentials at 16 per clock and SM, the rest the exchange), 65536 x 16 2.7 us, 8192 x 64 3.4 us,
// 509 x 24 in one CTA 2.5 us; a call of one iteration, which passes twice and reads the scores from DRAM, 38 us for
// 65536 x 256.
#pragma once

#include <math.h>

#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "score_types.cuh"
#include "scores.h"

namespace trnopt {

namespace {

constexpr unsigned kAll = 0xffffffffu;

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
      if ((int)(seen - target) >= 0) break;                 // (the count may pass 2^32)
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

constexpr int NT = kBalanceThreads, NW = NT / 32;
// Terms' logarithms beyond this (a row's maximum, the potential of a column that takes part) would be off by more than 2^-14
// if they were formed in float32.
constexpr float kNear = 1024.f;

// Fixed-point sums k_j 2^40 over the CTAs (at most 255, counted in the top byte) serve from 2^-8, where 148 roundings are
// 2^-25 of them, to below 2^8. A part that is larger (or no number) adds 2^8 and so takes the sum out of that range.
constexpr unsigned long long kTotalLeast = 1ull << 32, kTotalMost = 1ull << 48, kTotalOne = 1ull << 56;

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// log2 k, to float32's relative accuracy also where k is close to 1: what converged potentials still move by is a
// difference that would otherwise be rounded the same way in every iteration.
__device__ __forceinline__ float log2_near_1(double k) {
  const double t = k - 1.0;
  if (!(fabs(t) < 0.015625)) return log2f((float)k);
  return (float)(1.4426950408889634 * (t * (1.0 - t * (0.5 - t * (1.0 / 3.0 - t * (0.25 - t * 0.2))))));
}

struct Plus {
  __device__ __forceinline__ float operator()(float x, float y) const { return x + y; }
};
struct Larger {
  __device__ __forceinline__ float operator()(float x, float y) const { return fmaxf(x, y); }
};

// Joins a warp's groups of L lanes: a lane gives half of its columns away at each step, while it has several. store(k, v) on
// the one lane that ends up with column k.
template <int L, int C, typename Op, typename Store>
__device__ __forceinline__ void fold_lanes(float (&acc)[C], Op op, Store store) {
  const int lane = threadIdx.x & 31;
  int from = 0, have = C;
  bool owner = true;
#pragma unroll
  for (int o = L; o < 32; o *= 2) {
    if (have > 1) {
      const bool upper = lane & o;
      have /= 2;
#pragma unroll
      for (int k = 0; k < C / 2; ++k)
        if (k < have) {
          const float give = upper ? acc[k] : acc[k + have], held = upper ? acc[k + have] : acc[k];
          acc[k] = op(held, __shfl_xor_sync(kAll, give, o));
        }
      from += upper ? have : 0;
    } else {
      acc[0] = op(acc[0], __shfl_xor_sync(kAll, acc[0], o));
      owner = owner && !(lane & o);
    }
  }
#pragma unroll
  for (int k = 0; k < C; ++k)
    if (owner && k < have) store(from + k, acc[k]);
}

// a + b, and what float32 rounds off (0 where the sum is infinite).
struct Two {
  float high, low;
};
__device__ __forceinline__ Two two_sum(float a, float b) {
  const float s = a + b, t = s - a;
  return {s, fabsf(s) < INFINITY ? (a - (s - t)) + (b - t) : 0.f};
}

// Whole numbers in the order of the values, and back.
__device__ __forceinline__ int order_of(float x) {
  const int b = __float_as_int(x);
  return b ^ ((b >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float value_of(int k) { return __int_as_float(k ^ ((k >> 31) & 0x7fffffff)); }

// Shared memory: the warps' column sums, later the slices of the sum over the CTAs (NT quads), and the potentials; after
// it the rows that are kept.
__host__ __device__ inline size_t exchange_bytes(int cols) {
  const size_t warps = (size_t)NW * cols * sizeof(float), slices = (size_t)NT * 4 * sizeof(float2);
  return ((warps > slices ? warps : slices) + 15) & ~(size_t)15;
}
__host__ __device__ inline size_t fixed_bytes(int cols) {
  const size_t pad = (size_t)lanes_per_row(cols) * 32;
  return (exchange_bytes(cols) + 4 * pad * sizeof(float) + cols * (2 * sizeof(double) + 2) + 15) & ~(size_t)15;
}
// A kept row: an odd number of 16-byte units, so that lanes on neighbouring rows meet different banks.
__host__ __device__ inline int row_bytes(int cols, int size) { return (((cols * size + 15) >> 4) | 1) << 4; }

// A lane's runs of a row whose first score (of the lane's) is at s: kFrom 0 from shared memory, 1 from global memory by 16
// bytes, 2 score by score. Columns past the last: 0.
template <typename T, int L, int C, int kFrom>
__device__ __forceinline__ void read_runs(Vec<T> (&v)[C / Vec<T>::kN], const T* s, int cols, int q) {
  constexpr int V = Vec<T>::kN;
#pragma unroll
  for (int r = 0; r < C / V; ++r) {
    const int at = r * L * V;
    v[r].q = make_uint4(0, 0, 0, 0);
    if (at < cols && (L == 1 || at + q * V < cols)) {
      if constexpr (kFrom == 0) {
        v[r] = *reinterpret_cast<const Vec<T>*>(s + at);
      } else if constexpr (kFrom == 1) {
        v[r] = read_global<V>(s + at);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (at + q * V + i < cols) v[r].set(i, s[at + i]);
      }
    }
  }
}

// What far_pass and far_scores take of balance_kernel (in shared memory).
template <typename T>
struct FarRows {
  const T *scores, *kept;          // the CTA's rows, and those that it keeps
  long long ld;
  int pitch, kept_rows, n, cols;
  const float *us, *ul, *peaks, *masses, *b;
  const unsigned char* out;
  float *f, *red;
  double per_eps, eps_per, log_cols, shift;
  float c, c_low;
  bool vectors;
};

// A pass over a warp's rows and its fold to `red` (the modes of balance_kernel), with the terms from pairs of float32. A row's
// own constant comes off first, so a row whose scores are all the type's lowest is a uniform one.
template <typename T, int L, int C>
__device__ __noinline__ void far_pass(const FarRows<T>& p, int mode, bool last) {
  constexpr int V = Vec<T>::kN, G = 32 / L;
  const int lane = threadIdx.x & 31, q = lane & (L - 1), group = lane / L;
  auto column = [&](int k) { return (k / V) * (L * V) + q * V + k % V; };
  unsigned closed = 0;                                      // columns that the row sums leave out
  if (mode != 0) {
#pragma unroll
    for (int k = 0; k < C; ++k)
      if (column(k) < p.cols && p.out[column(k)]) closed |= 1u << k;
  }
  auto counts = [&](int k) { return !(closed >> k & 1); };               // in the row's sum
  // (with mass: also one that starts from -inf, so that what is out of range below it is so in the first iteration, too)
  auto mass = [&](int k) { return counts(k) || !(p.b && p.b[column(k)] == 0.f); };
  float acc[C];
#pragma unroll
  for (int k = 0; k < C; ++k) acc[k] = mode == 1 ? -INFINITY : 0.f;
  for (int base = (threadIdx.x >> 5) * G; base < p.n; base += NW * G) {
    const int row = base + group;
    const bool there = row < p.n;
    Vec<T> v[C / V];
    const T* s = p.scores + (there ? row : p.n - 1) * p.ld + q * V;
    if (base + G <= p.kept_rows) read_runs<T, L, C, 0>(v, p.kept + row * p.pitch + q * V, p.cols, q);
    else if (p.vectors) read_runs<T, L, C, 1>(v, s, p.cols, q);
    else read_runs<T, L, C, 2>(v, s, p.cols, q);
    float top = -INFINITY;                                  // the row's constant
#pragma unroll
    for (int k = 0; k < C; ++k)
      if (column(k) < p.cols && p.us[column(k)] != -INFINITY && mass(k)) top = fmaxf(top, v[k / V].get(k % V));
#pragma unroll
    for (int o = 1; o < L; o *= 2) top = fmaxf(top, __shfl_xor_sync(kAll, top, o));
    if (top == -INFINITY) top = 0.f;
    // (S - top) c of the lane's k-th column as a high part and (added to `low`) what that is off by
    auto scaled = [&](int k, float& low) {
      const Two x = two_sum(v[k / V].get(k % V), -top);
      const float high = __fmul_rn(x.high, p.c);
      low += fabsf(high) < INFINITY ? fmaf(x.high, p.c, -high) + fmaf(x.high, p.c_low, x.low * p.c) : 0.f;
      return high;
    };
    // the largest term: to float32, as what it is off by cancels
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < C; ++k) {
      float low = 0.f;
      if (counts(k) && column(k) < p.cols) m = fmaxf(m, scaled(k, low) + p.us[column(k)]);
    }
#pragma unroll
    for (int o = 1; o < L; o *= 2) m = fmaxf(m, __shfl_xor_sync(kAll, m, o));
    if (m == -INFINITY) m = top = 0.f;                      // nothing in the sum
    float l = 0.f, d[C], less[C];                           // less: without the columns' potentials
#pragma unroll
    for (int k = 0; k < C; ++k) {
      const float u = column(k) < p.cols ? p.us[column(k)] : -INFINITY;
      d[k] = less[k] = -INFINITY;
      if (u != -INFINITY) {
        float low = 0.f;
        const float high = scaled(k, low);
        const Two z = two_sum(high, u), x = two_sum(high, -m);
        d[k] = (z.high - m) + (z.low + (low + p.ul[column(k)]));
        less[k] = (mode == 2 ? x.high - p.peaks[column(k)] : x.high) + (x.low + low);
      }
      d[k] = ex2_approx(d[k]);
      if (counts(k)) l += d[k];
    }
#pragma unroll
    for (int o = 1; o < L; o *= 2) l += __shfl_xor_sync(kAll, l, o);
    const float a = !there ? 0.f : p.masses ? __ldg(p.masses + row) : 1.f;
    const bool empty = l == 0.f;
    if (last && mode != 1 && q == 0 && there)
      p.f[row] = empty ? 0.f : (float)((p.log_cols - ((double)m + (double)top * p.per_eps + (double)log2f(l) + p.shift)) *
                                       p.eps_per);
    const float weight = empty ? 0.f : a / l, off = (empty ? (float)(p.shift - p.log_cols) : -log2f(l)) + log2f(a);
#pragma unroll
    for (int k = 0; k < C; ++k) {
      if (mode == 0) acc[k] = fmaf(d[k], weight, acc[k]);
      else if (mode == 1) acc[k] = fmaxf(acc[k], less[k] + off);
      else acc[k] += ex2_approx(less[k] + off);
    }
  }
  auto store = [&](int k, float v) {
    if (column(k) < p.cols) p.red[(threadIdx.x >> 5) * p.cols + column(k)] = v;
  };
  if (mode == 1) fold_lanes<L, C>(acc, Larger{}, store);
  else fold_lanes<L, C>(acc, Plus{}, store);
}

// Whether only c carries the scores of one of a warp's rows out of range, so that its float32 maximum is that of a row of -inf.
template <typename T, int L>
__device__ __forceinline__ bool far_scores(const FarRows<T>& p) {
  constexpr int G = 32 / L;
  const int lane = threadIdx.x & 31;
  bool found = false;
  __syncwarp();                                             // (kept rows: other lanes' runs, too)
  for (int base = (threadIdx.x >> 5) * G; base < p.n; base += NW * G) {
    const int row = min(base + lane / L, p.n - 1);
    const T* s = base + G <= p.kept_rows ? p.kept + row * p.pitch : p.scores + row * p.ld;
    float top = -INFINITY;
#pragma unroll 8
    for (int j = lane & (L - 1); j < p.cols; j += L)
      if (!(p.b && p.b[j] == 0.f)) top = fmaxf(top, widen(s[j]));
#pragma unroll
    for (int o = 1; o < L; o *= 2) top = fmaxf(top, __shfl_xor_sync(kAll, top, o));
    found = found || (top != -INFINITY && !(fabsf(top * p.c) < INFINITY));
  }
  return found;
}

// L lanes per row, C columns per lane in runs of 16 bytes (a kept row has whole runs, wherever it lies in global memory;
// `vectors`: it can be read there by runs, too).
// (C is 32, or 8 or 16 where a row of few columns has a lane of its own; u has places for 32 either way.)
template <typename T, int L, int C>
__global__ void __launch_bounds__(NT, 1) balance_kernel(BalanceProblem p, BalanceWork wk, int kept_rows, bool vectors) {
  constexpr int V = Vec<T>::kN, G = 32 / L;                                 // rows a warp takes at a time
  extern __shared__ __align__(16) unsigned char smem[];
  // the warps' column sums, then the slices of the sum over the CTAs; u + log2 b; log2 b; the CTA's column maxima in the
  // first iteration; whether a column has any term; the kept rows
  float* red = reinterpret_cast<float*>(smem);                      // (NW, cols)
  float2* slice_sums = reinterpret_cast<float2*>(smem);             // (slices, cols4)
  float* us = reinterpret_cast<float*>(smem + exchange_bytes(p.cols));
  float* peaks_s = us + L * 32;                                     // (u and the maxima have L x 32 places: -inf, 0)
  float* off_s = peaks_s + L * 32;
  float* ul = off_s + L * 32;                                       // what u + log2 b less `shift` is more than us
  double* per_b = reinterpret_cast<double*>(ul + L * 32);      // 1 / b, with the rows' and columns' counts in it
  double* lb = per_b + p.cols;
  unsigned char* open = reinterpret_cast<unsigned char*>(lb + p.cols);
  unsigned char* out = open + p.cols;                               // whether the rows' sums leave a column out
  T* kept = reinterpret_cast<T*>(smem + fixed_bytes(p.cols));       // (kept_rows, pitch)
  // whether a wait was in time; whether float32 is too coarse for a column that takes part; the least potential
  __shared__ int flag, far_columns, least;
  __shared__ FarRows<T> rows_s;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, q = lane & (L - 1), group = lane / L;
  const int cols = p.cols, cols4 = (cols + 3) & ~3, pitch = row_bytes(cols, sizeof(T)) / (int)sizeof(T);
  const double per_eps = 1.4426950408889634 / p.eps;
  const float c = (float)per_eps;
  const long long r0 = (long long)blockIdx.x * p.rows / gridDim.x, r1 = (long long)(blockIdx.x + 1) * p.rows / gridDim.x;
  const T* scores = static_cast<const T*>(p.scores) + r0 * p.ld + q * V;
  const float* masses = p.a ? p.a + r0 : nullptr;
  const int n = (int)(r1 - r0);
  auto column = [&](int k) { return (k / V) * (L * V) + q * V + k % V; };

  // Columns of mass 0 add nothing to the rows' sums, so their potentials matter to nobody else: they are found in the last
  // iteration, from its f, like the first iteration's from any g (every column's maximum before its sum: nothing keeps such
  // a column's terms below the rows' maxima).
  // (A column that starts from -inf is one of these in the first iteration.)
  bool some_closed = false, some_out = false;               // of mass 0; left out in the first iteration
  for (int j = tid; j < cols; j += NT) {
    const float b = p.b ? p.b[j] : 1.f;                     // (1 / cols each: log2 cols in a row's sum instead)
    some_closed = some_closed || b == 0.f;
    lb[j] = b == 0.f || b == 1.f ? 0.0 : log2((double)b);
    per_b[j] = b == 0.f ? wk.k_scale : wk.k_scale / (double)b;
    out[j] = b == 0.f || (p.g0 && p.g0[j] == -INFINITY);
    open[j] = !out[j];
    some_out = some_out || out[j];
  }
  for (int j = tid; j < L * 32; j += NT) {
    if (j >= cols) us[j] = -INFINITY;
    peaks_s[j] = off_s[j] = 0.f;
  }
  if (tid == 0) {
    flag = 1;
    far_columns = 0;
    least = order_of(INFINITY);
    rows_s = {scores - q * V, kept, p.ld, pitch, kept_rows, n, cols, us, ul, peaks_s, masses, p.b, out, p.f + r0, red, per_eps,
              p.eps * 0.6931471805599453, wk.log_cols, 0.0, c, (float)(per_eps - (double)c), vectors};
  }
  some_closed = __syncthreads_or(some_closed);
  some_out = __syncthreads_or(some_out);
  // What float32 potentials are relative to: 0, or the least one that takes part, by a given g, then by the potentials after
  // one iteration. So a column that a large finite score masks (its potential lies far above) does not cost the others their
  // accuracy.
  auto reference = [&](auto&& potential) {
    int mine = order_of(INFINITY);
    for (int j = tid; j < cols; j += NT) {
      const float u = (float)potential(j);
      if (open[j] && u > -INFINITY) mine = min(mine, order_of(u));
    }
    mine = __reduce_min_sync(kAll, mine);
    if (lane == 0 && mine < order_of(INFINITY)) atomicMin(&least, mine);
    __syncthreads();
    if (tid == 0) rows_s.shift = least < order_of(INFINITY) ? (double)value_of(least) : 0.0;
    __syncthreads();
  };
  auto hold = [&](int j, double u) {                        // u + log2 b of a column that takes part
    u -= rows_s.shift;
    us[j] = (float)u;
    ul[j] = fabsf(us[j]) < INFINITY ? (float)(u - (double)us[j]) : 0.f;
    if (open[j] && fabsf(us[j]) > kNear && fabsf(us[j]) < INFINITY) far_columns = 1;
  };
  if (p.g0) reference([&](int j) { return (double)p.g0[j] * per_eps + lb[j]; });
  for (int j = tid; j < cols; j += NT) {
    if (open[j]) hold(j, (p.g0 ? (double)p.g0[j] * per_eps : 0.0) + lb[j]);
    else us[j] = ul[j] = 0.f;
  }
  __syncthreads();
  auto closed_columns = [&]() {                             // the lane's columns that the rows' sums leave out
    unsigned closed = 0;
#pragma unroll
    for (int k = 0; k < C; ++k)
      if (column(k) < cols && out[column(k)]) closed |= 1u << k;
    return closed;
  };

  unsigned arrivals = 0;                                    // at the grid's barrier, up to the next one's end
  // The words of the fixed-point sums are never cleared: an iteration's sum is the difference to what the thread read two
  // iterations ago (a CTA adds to a word again only when every CTA has read the one in between, and so this one before).
  unsigned long long seen[2][2] = {{0, 0}, {0, 0}};
  int it = 0;
  // The iterations; kExact: with far_pass. The others leave off (true) once a term of the CTA's is too far from 0 for float32,
  // before the CTA has added its sums to the others', and kExact ones take over from that iteration on. (Two loops, as a call
  // of far_pass in this one would take registers from its passes: 65536 x 256 249 -> 270 us.)
  auto iterate = [&](auto exact_) {
    constexpr bool kExact = decltype(exact_)::value;
    for (; it < p.iters; ++it) {
      const bool first = it == 0, last = it == p.iters - 1, maxima = first || (last && some_closed);
      float acc[C];
      bool far = !kExact && far_columns;                      // (of this thread)
      bool empties = false;                                   // whether the thread has met rows with a maximum of -inf
      float farthest = 0.f;                                   // the largest |maximum| of its other rows
      // Modes: 0 column sums, without the columns of mass 0 (u = -inf); or, where the columns' maxima are found, 1 these and
      // then 2 the sums relative to them, of all columns (u = 0 for those that the rows' sums leave out).
      auto pass = [&](auto mode_, auto closed_) {
        constexpr int kMode = decltype(mode_)::value;
        constexpr bool kClosed = decltype(closed_)::value;
        const unsigned closed = kClosed ? closed_columns() : 0;
        uint64_t u2[C / 2], acc2[C / 2];                      // pairs of columns
#pragma unroll
        for (int k = 0; k < C; k += 2) {
          u2[k / 2] = pack2(us[column(k)], us[column(k + 1)]);
          acc2[k / 2] = kMode == 1 ? pack2(-INFINITY, -INFINITY) : 0;
        }
        const uint64_t c2 = pack2(c, c);
        for (int base = w * G; base < n; base += NW * G) {
          const int row = base + group;
          const bool there = row < n, keep = base + G <= kept_rows;
          const T* s = scores + (there ? row : n - 1) * p.ld;
          T* here = kept + (keep ? row * pitch + q * V : 0);
          uint64_t z2[C / 2];
          float m = -INFINITY, l = 0.f;
          Vec<T> v[C / V];
          // (columns past the last: 0, with u = -inf)
          if (keep && !(kMode == 1 && first)) {
            read_runs<T, L, C, 0>(v, here, cols, q);
          } else {
            if (vectors) read_runs<T, L, C, 1>(v, s, cols, q);
            else read_runs<T, L, C, 2>(v, s, cols, q);
            if (kMode == 1 && keep && first) {
#pragma unroll
              for (int r = 0; r < C / V; ++r)
                if (r * L * V + q * V < cols) *reinterpret_cast<Vec<T>*>(here + r * L * V) = v[r];
            }
          }
#pragma unroll
          for (int k = 0; k < C; k += 2) {
            z2[k / 2] = fma2(pack2(v[k / V].get(k % V), v[(k + 1) / V].get((k + 1) % V)), c2, u2[k / 2]);
            float x, y;
            unpack2(z2[k / 2], x, y);
            if (kClosed) {
              x = closed >> k & 1 ? -INFINITY : x;
              y = closed >> (k + 1) & 1 ? -INFINITY : y;
            }
            m = max3(m, x, y);
          }
#pragma unroll
          for (int o = 1; o < L; o *= 2) m = fmaxf(m, __shfl_xor_sync(kAll, m, o));
          if (kMode == 1) empties = empties || m == -INFINITY;
          m = m == -INFINITY ? 0.f : m;
          farthest = fmaxf(farthest, fabsf(m));
          {
            const uint64_t m2 = pack2(-m, -m);
            uint64_t l2 = 0;
#pragma unroll
            for (int k = 0; k < C; k += 2) {
              const uint64_t d2 = add2(z2[k / 2], m2);
              float x, y;
              unpack2(d2, x, y);
              const float ex = ex2_approx(x), ey = ex2_approx(y);
              const uint64_t e2 = pack2(ex, ey);
              if (kClosed) l2 = add2(pack2(closed >> k & 1 ? 0.f : ex, closed >> (k + 1) & 1 ? 0.f : ey), l2);
              else l2 = add2(e2, l2);
              z2[k / 2] = kMode == 0 ? e2 : d2;
            }
            float x, y;
            unpack2(l2, x, y);
            l = x + y;
          }
#pragma unroll
          for (int o = 1; o < L; o *= 2) l += __shfl_xor_sync(kAll, l, o);
          const float a = !there ? 0.f : masses ? __ldg(masses + row) : 1.f;
          const bool empty = l == 0.f;                        // f = 0
          if (kMode != 1 && last && q == 0 && there)
            p.f[(long long)blockIdx.x * p.rows / gridDim.x + row] =
                empty ? 0.f : (float)((wk.log_cols - ((double)m + (double)log2f(l) + rows_s.shift)) * rows_s.eps_per);
          if constexpr (kMode == 0) {
            const float weight = empty ? 0.f : a / l;         // (an empty row's terms are 0: no column of mass 0 is among them)
            const uint64_t w2 = pack2(weight, weight);
#pragma unroll
            for (int k = 0; k < C / 2; ++k) acc2[k] = fma2(z2[k], w2, acc2[k]);
          } else {
            // x = S c + f c + log2 a, in the gauge of u - shift: z - u - log2 l + log2 a (and log2 cols, as in mode 0); mode 2
            // takes it relative to the column's maximum, off_s = -u - maximum. (Columns with u = -inf: no number, passed over
            // by the maximum; z = -inf in the sums.)
            const float off = (empty ? (float)(rows_s.shift - wk.log_cols) : -log2f(l)) + log2f(a);
            const uint64_t o2 = pack2(off, off);
#pragma unroll
            for (int k = 0; k < C; k += 2) {
              float x, y, ax, ay;
              if constexpr (kMode == 1) {
                float ux, uy;
                unpack2(u2[k / 2], ux, uy);
                unpack2(add2(add2(z2[k / 2], pack2(-ux, -uy)), o2), x, y);
                unpack2(acc2[k / 2], ax, ay);
                acc2[k / 2] = pack2(fmaxf(ax, x), fmaxf(ay, y));
              } else {
                unpack2(add2(add2(z2[k / 2], pack2(off_s[column(k)], off_s[column(k + 1)])), o2), x, y);
                acc2[k / 2] = add2(acc2[k / 2], pack2(ex2_approx(x), ex2_approx(y)));
              }
            }
          }
        }
#pragma unroll
        for (int k = 0; k < C; k += 2) unpack2(acc2[k / 2], acc[k], acc[k + 1]);
      };
      // the warp's sums (or maxima) to `red`
      auto fold = [&](auto op) {
        fold_lanes<L, C>(acc, op, [&](int k, float v) {
          if (column(k) < cols) red[w * cols + column(k)] = v;
        });
      };
      if (maxima) {
        if (!first) {
          for (int j = tid; j < cols; j += NT)
            if (out[j]) us[j] = 0.f;
          __syncthreads();
        }
        if constexpr (kExact) {
          far_pass<T, L, C>(rows_s, 1, false);
          __syncthreads();
        } else {
          if (some_out) pass(std::integral_constant<int, 1>{}, std::true_type{});
          else pass(std::integral_constant<int, 1>{}, std::false_type{});
          fold(Larger{});
          bool out_of_range = false;                        // (the vote and what follows it: by the whole warp)
          if (first && __any_sync(kAll, empties)) out_of_range = far_scores<T, L>(rows_s);
          far = far || farthest > kNear || out_of_range;
          if (__syncthreads_or(far)) return true;
        }
        for (int j = tid; j < cols; j += NT) {
          float m = red[j];
          for (int k = 1; k < NW; ++k) m = fmaxf(m, red[k * cols + j]);
          m = fabsf(m) < INFINITY ? m : 0.f;
          peaks_s[j] = m;
          off_s[j] = us[j] == -INFINITY ? 0.f : -us[j] - m;
          far = far || (!(p.b && p.b[j] == 0.f) && fabsf(m) > kNear);       // (also of one that starts from -inf)
        }
        if constexpr (kExact) {
          __syncthreads();
          far_pass<T, L, C>(rows_s, 2, last);
        } else {
          if (__syncthreads_or(far)) return true;
          if (some_out) pass(std::integral_constant<int, 2>{}, std::true_type{});
          else pass(std::integral_constant<int, 2>{}, std::false_type{});
          fold(Plus{});
        }
        __syncthreads();
      } else if constexpr (kExact) {
        far_pass<T, L, C>(rows_s, 0, last);
        __syncthreads();
      } else {
        pass(std::integral_constant<int, 0>{}, std::false_type{});
        fold(Plus{});
        if (__syncthreads_or(far || farthest > kNear)) return true;
      }

      const bool alone = gridDim.x == 1;
      unsigned long long total[2];
      bool fixed = false;
      auto column_sum = [&](int j) {
        float v = red[j];
#pragma unroll
        for (int k = 1; k < NW; ++k) v += red[k * cols + j];
        return v;
      };
      auto gave_up = [&]() {                                  // no potentials
        it = p.iters;
        for (int i = tid; i < n; i += NT) rows_s.f[i] = NAN;
        if (blockIdx.x == 0)
          for (int j = tid; j < cols; j += NT) p.g[j] = NAN;
        return false;
      };
      if (alone) {
        for (int j = tid; j < cols; j += NT) red[j] = column_sum(j);       // (column j of `red` is this thread's alone)
      } else if (!maxima) {
        // in fixed point: a column's word counts the CTAs in its top byte, so whoever reads it knows when it has all of them
        unsigned long long* totals = wk.totals + (it & 1) * cols4;
        for (int j = tid; j < cols; j += NT) {
          const double k = (double)column_sum(j) * per_b[j];
          const bool in = k >= 0.0 && k < 0x1p8;
          atomicAdd(totals + j, kTotalOne + (in ? (unsigned long long)__double2ll_rn(k * 0x1p40) : kTotalMost));
        }
        const unsigned long long t0 = globaltimer_ns();
        auto complete = [&](int i) {                          // the thread's i-th word, once every CTA has added to it
          unsigned long long now;
          for (unsigned spin = 1;; ++spin) {
            asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(now) : "l"(totals + tid + i * NT) : "memory");
            if ((now - seen[it & 1][i]) / kTotalOne == gridDim.x) break;
            if (spin % 64 == 0 && globaltimer_ns() - t0 > kWaitLimitNs) {
              atomicOr(wk.error_word, (int)kErrWaitTimeout);
              flag = 0;
              break;
            }
          }
          return now;
        };
        // One lane per warp waits for its own first where many threads would wait: their reads hold up the sums that are to
        // come. Per iteration so / all at once: 65536 x 256 10.7 / 11.7 us, 65536 x 64 4.7 / 5.1 us, but 65536 x 16
        // 2.7 / 2.6 us, 8192 x 64 (32 CTAs) 3.5 / 3.3 us.
        if (cols * (int)gridDim.x > 4096) {
          if (lane == 0 && tid < cols) complete(0);
          __syncwarp();
        }
        fixed = true;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int j = tid + i * NT;
          if (j >= cols) break;
          const unsigned long long now = complete(i);
          total[i] = (now - seen[it & 1][i]) % kTotalOne;
          seen[it & 1][i] = now;
          fixed = fixed && (!open[j] || (total[i] >= kTotalLeast && total[i] < kTotalMost));
        }
        fixed = __syncthreads_and(fixed);                     // the same in every CTA
        if (!flag) return gave_up();
      }
      int slices = 1;
      if (!alone && !fixed) {
        // iterations with maxima, and sums out of that range: every CTA's float32 sums, behind a barrier of their own (and
        // where no fixed-point sums came before, behind one more: the other CTAs may still read the last ones)
        if (maxima && !first) {
          arrivals += gridDim.x;
          if (!grid_barrier(wk.counter, arrivals, wk.error_word, &flag)) return gave_up();
        }
        float* sums = wk.parts;
        float* peaks = sums + (size_t)gridDim.x * cols4;
        for (int j = tid; j < cols; j += NT) {
          const float v = column_sum(j);
          __stcg(sums + (size_t)blockIdx.x * cols4 + j, v);
          if (maxima) __stcg(peaks + (size_t)blockIdx.x * cols4 + j, v == 0.f ? -INFINITY : peaks_s[j]);
        }
        arrivals += gridDim.x;
        if (!grid_barrier(wk.counter, arrivals, wk.error_word, &flag)) return gave_up();
        // of all CTAs, in the same order in each: four columns per thread, the CTAs in `slices` interleaved parts
        const int quads = cols4 / 4, slice = tid / quads, quad = tid - slice * quads;
        slices = min(NT / quads, 16);                         // (few enough for the columns' threads to join)
        float2* part = slice_sums + (size_t)slice * cols4 + 4 * quad;     // (`red` is free again)
        if (slice < slices) {
          float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, v[4] = {0.f, 0.f, 0.f, 0.f};
          if (maxima) {
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
            constexpr int kBatch = 10;                        // loads in flight (148 CTAs in 16 slices: one round)
            for (int k0 = slice; k0 < (int)gridDim.x; k0 += slices * kBatch) {
              float4 o[kBatch];
#pragma unroll
              for (int i = 0; i < kBatch; ++i) {
                const int k = k0 + i * slices;
                o[i] = k < (int)gridDim.x ? __ldcg(reinterpret_cast<const float4*>(sums + (size_t)k * cols4) + quad)
                                          : make_float4(0.f, 0.f, 0.f, 0.f);
              }
#pragma unroll
              for (int i = 0; i < kBatch; ++i) {
                v[0] += o[i].x;
                v[1] += o[i].y;
                v[2] += o[i].z;
                v[3] += o[i].w;
              }
            }
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) part[e] = make_float2(m[e], v[e]);
        }
        __syncthreads();
      }
      double full[2];                                         // with maxima: u of the thread's columns (at most 2)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int j = tid + i * NT;
        if (j >= cols) break;
        float2 v = alone ? make_float2(peaks_s[j], red[j]) : fixed ? make_float2(0.f, 1.f) : slice_sums[j];
        if (maxima) {
          for (int k = 1; k < slices; ++k) {
            const float2 o = slice_sums[(size_t)k * cols4 + j];
            lse2_add(v.x, v.y, o.x, o.y);
          }
          open[j] = v.y != 0.f && !(p.b && p.b[j] == 0.f);    // takes part from here on
          full[i] = v.y == 0.f ? 0.0 : rows_s.shift - ((double)v.x + log2((double)v.y * wk.k_scale));
          if (last && blockIdx.x == 0) p.g[j] = (float)(full[i] * rows_s.eps_per);
        } else {
#pragma unroll 8
          for (int k = 1; k < slices; ++k) v.y += slice_sums[(size_t)k * cols4 + j].y;
          // k_j (a sum that underflows, for masses beyond float32's range from one another, counts as 2^-126)
          const float step = log2_near_1(fixed ? (double)total[i] * 0x1p-40 : v.y == 0.f ? 0x1p-126 : (double)v.y * per_b[j]);
          if (open[j]) {
            const Two u = two_sum(us[j], -step);
            const float low = ul[j] + u.low;
            us[j] = u.high + low;
            ul[j] = low - (us[j] - u.high);
            if (fabsf(us[j]) > kNear) far_columns = 1;
          }
          if (last && blockIdx.x == 0)
            p.g[j] = open[j] ? (float)(((double)us[j] + (double)ul[j] - lb[j] + rows_s.shift) * rows_s.eps_per) : 0.f;
        }
      }
      if (first) {
        if (tid == 0) {
          least = order_of(INFINITY);
          far_columns = 0;
        }
        __syncthreads();
        reference([&](int j) { return full[j < NT ? 0 : 1] + lb[j]; });
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int j = tid + i * NT;
          if (j >= cols) break;
          out[j] = p.b && p.b[j] == 0.f;
          if (out[j]) {
            us[j] = -INFINITY;
            ul[j] = 0.f;
          } else {
            hold(j, full[i] + lb[j]);                         // (of a column without terms, too: it has 0, and no terms)
          }
        }
      }
      __syncthreads();
    }
    return false;
  };
  if (iterate(std::false_type{})) iterate(std::true_type{});
}

template <typename T, int L, int C>
cudaError_t launch(int device, const BalanceProblem& p, const BalanceWork& wk, cudaStream_t stream) {
  const int grid = balance_grid(device, p.rows, p.cols);
  // the rows a CTA keeps: all of them, or what shared memory holds (227 KB less what the launch itself takes)
  constexpr int G = 32 / L;
  const size_t fixed = fixed_bytes(p.cols), most = 226 * 1024 - fixed;
  long long kept = (((long long)p.rows + grid - 1) / grid + G - 1) / G * G;
  const long long fits = (long long)(most / row_bytes(p.cols, sizeof(T))) / G * G;
  if (kept > fits) kept = fits;
  const size_t bytes = fixed + (size_t)kept * row_bytes(p.cols, sizeof(T));
  static std::atomic<int> done[kMaxDevices];
  cudaError_t e = smem_attr_once(reinterpret_cast<const void*>(balance_kernel<T, L, C>), (int)bytes, done);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeCooperative;                // its CTAs wait for one another
  attr.val.cooperative = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = grid > 1 ? 1 : 0;
  const bool vectors = p.cols % Vec<T>::kN == 0 && p.ld % Vec<T>::kN == 0 && reinterpret_cast<uintptr_t>(p.scores) % 16 == 0;
  return cudaLaunchKernelEx(&cfg, balance_kernel<T, L, C>, p, wk, (int)kept, vectors);
}

template <typename T>
cudaError_t launch(int device, const BalanceProblem& p, const BalanceWork& wk, cudaStream_t stream) {
  switch (lanes_per_row(p.cols)) {
    case 1: return p.cols <= 8 ? launch<T, 1, 8>(device, p, wk, stream)
                               : p.cols <= 16 ? launch<T, 1, 16>(device, p, wk, stream) : launch<T, 1, 32>(device, p, wk, stream);
    case 2: return launch<T, 2, 32>(device, p, wk, stream);
    case 4: return launch<T, 4, 32>(device, p, wk, stream);
    case 8: return launch<T, 8, 32>(device, p, wk, stream);
    case 16: return launch<T, 16, 32>(device, p, wk, stream);
    default: return launch<T, 32, 32>(device, p, wk, stream);
  }
}

}  // namespace

}  // namespace trnopt

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
// The order of keys is that of their 64-bit values. One warp per row holds float32 keys in registers, a run of columns
// per lane within a group; the keys that reach the (top + 1)-th largest of the lanes' best are a dozen or two, which are
// ranked in shared memory. Where neighbours in that order, or the last open and the first closed group, are closer than
// the float32 keys are exact, the candidates' (or the groups') keys are formed in float64 and ranked again. Keys that are
// the scores themselves are exact. Weights are float32 from the logarithms of the shares (shares that underflow still
// give their ratio). A persistent grid counts the load in shared memory. Bound by the selection's instructions: 32768 x 256 float32
// with 4 of 8 groups, a bias and 8 choices 50 us (958 instructions a row; 5.6 us the scores at the copy rate), plain softmax
// 31 us; 32768 x 64 bfloat16, 2 choices, 23 us.
#include <math.h>

#include <atomic>

#include "common.cuh"
#include "kernels.h"
#include "score_types.cuh"
#include "scores.h"

namespace trnopt {

namespace {

constexpr int RT_WARPS = 8;
constexpr int RT_LIST = 64;          // candidates of a row that are ranked

// Resident CTAs per SM, by the columns a lane holds: the persistent grid has as many.
constexpr int route_ctas(int columns) { return columns <= 8 ? 4 : 2; }

struct RouteSmem {
  uint64_t list[RT_WARPS][RT_LIST], best[RT_WARPS][32];     // (key, column) as whole numbers in their order
  float score[RT_WARPS][RT_LIST], best_score[RT_WARPS][32]; // the candidates' scores
  double exact[RT_WARPS][RT_LIST];                          // their keys in float64, where they are needed
};
constexpr unsigned kAll = 0xffffffffu;

__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm("redux.sync.max.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "r"(kAll));
  return r;
}
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

// Whole numbers in the order of the scores (-0 = +0); 0 is below every score's.
__device__ __forceinline__ uint32_t order(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}

// The key of a (key, column) pair; of 0, -inf.
__device__ __forceinline__ float key_of(uint64_t pair) {
  const uint32_t k = (uint32_t)(pair >> 32);
  return pair == 0 ? -INFINITY : __uint_as_float(k ^ ((k & 0x80000000u) ? 0x80000000u : 0xffffffffu));
}

// A value that the k largest of the warp's values reach: the k-th largest different one.
__device__ __forceinline__ float kth_largest(float v, int k) {
  float found = warp_max(v);
  for (int r = 1; r < k; ++r) {
    v = v == found ? -INFINITY : v;
    found = warp_max(v);
  }
  return found;
}

// A row's keys in float64: its share's constants, by the whole warp, then any column's key.
template <typename T>
struct ExactKeys {
  double m, sum;
  bool softmax, on_scores;
  __device__ __forceinline__ ExactKeys(const RouteProblem& p, const T* s) : m(-INFINITY), sum(0.0) {
    const int lane = threadIdx.x & 31;
    softmax = p.kind == TRNOPT_ROUTE_SOFTMAX;
    on_scores = p.bias && p.bias_on == TRNOPT_ROUTE_BIAS_SCORES;
    if (softmax && (on_scores || !p.bias)) {
      for (int j = lane; j < p.cols; j += 32) m = fmax(m, (double)widen(s[j]));
      m = warp_max(m);
      if (m > -INFINITY)
        for (int j = lane; j < p.cols; j += 32) sum += exp((double)widen(s[j]) - m);
      sum = warp_sum(sum);
    }
  }
  // `shares`: without a bias, the share (for the groups' scores) and not the score itself
  __device__ __forceinline__ double key(const RouteProblem& p, const T* s, int j, bool shares) const {
    const double x = widen(s[j]);
    if (!(x > -INFINITY)) return -INFINITY;
    double k = x;
    if (on_scores || (shares && !p.bias)) k = softmax ? exp(x - m) / sum : 1.0 / (1.0 + exp(-x));
    return p.bias ? k + (double)p.bias[j] : k;
  }
};

// Candidates list[0 .. n) ranked by their float64 keys, then by column, into best.
template <typename T>
__device__ __noinline__ void rank_exact(const RouteProblem& p, const T* s, const uint64_t* list, const float* score,
                                        double* exact, int n, uint64_t* best, float* best_score) {
  const int lane = threadIdx.x & 31;
  const ExactKeys<T> keys(p, s);
  for (int e = lane; e < n; e += 32) exact[e] = keys.key(p, s, (int)(0xffffffffu - (unsigned)list[e]), false);
  __syncwarp();
  for (int e = lane; e < n; e += 32) {
    const double k = exact[e];
    int rank = 0;
    for (int o = 0; o < n; ++o) rank += exact[o] > k || (exact[o] == k && (unsigned)list[o] > (unsigned)list[e]);
    if (rank < 32) {
      best[rank] = list[e];
      best_score[rank] = score[e];
    }
  }
  __syncwarp();
}

// Whether the lane's group stays open, by float64 scores; the lane's columns are first + k, k < n.
template <typename T>
__device__ __noinline__ bool open_exact(const RouteProblem& p, const T* s, int lanes, int first, int n) {
  const int group = (threadIdx.x & 31) / lanes;
  const ExactKeys<T> keys(p, s);
  double t1 = -INFINITY, t2 = -INFINITY;
  for (int k = 0; k < n; ++k) {
    const double x = keys.key(p, s, first + k, true);
    t2 = fmax(t2, fmin(t1, x));
    t1 = fmax(t1, x);
  }
  for (int o = 1; o < lanes; o *= 2) {
    const double o1 = __shfl_xor_sync(kAll, t1, o), o2 = __shfl_xor_sync(kAll, t2, o);
    t2 = fmax(fmin(t1, o1), fmax(t2, o2));
    t1 = fmax(t1, o1);
  }
  const double score = p.group_top == 2 && t2 > -INFINITY ? t1 + t2 : t1;
  int rank = 0;
  for (int g = 0; g < p.groups; ++g) {
    const double other = __shfl_sync(kAll, score, g * lanes);
    rank += other > score || (other == score && g < group);
  }
  return t1 > -INFINITY && rank < p.top_groups;
}

// A row's choices by 64-bit keys in shared memory: lane k < top gets the k-th column, or -1.
template <typename T>
__device__ __noinline__ int choose_exact(const RouteProblem& p, const T* s, double* key) {
  const int lane = threadIdx.x & 31, size = p.cols / p.groups;
  const ExactKeys<T> keys(p, s);
  for (int j = lane; j < p.cols; j += 32) key[j] = keys.key(p, s, j, p.groups > 1);
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
      else if (!p.bias) key[j] = widen(s[j]);              // without a bias the columns go by their scores themselves
    }
    __syncwarp();
  }
  int mine = -1;
  for (int k = 0; k < p.top; ++k) {
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
  __syncwarp();
  return mine;
}

// How the columns lie on the lanes: `lanes` (a power of two) for each group, `run` neighbouring columns on each.
struct RouteLayout {
  int lanes, run, size;
  bool vectors;                // runs are whole 16-byte (or shorter) vectors on their boundaries
  bool exact;                  // no such layout: every row by 64-bit keys
};

template <typename T, int C>
__global__ void __launch_bounds__(32 * RT_WARPS, route_ctas(C)) route_kernel(RouteProblem p, RouteLayout lay) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ RouteSmem sh;
  double* keys = reinterpret_cast<double*>(smem);                  // (RT_WARPS, cols), for rows by 64-bit keys
  int* counts = reinterpret_cast<int*>(keys + (size_t)RT_WARPS * p.cols);
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int group = lane / lay.lanes, in_group = (lane & (lay.lanes - 1)) * lay.run;
  const int first = group * lay.size + in_group;                    // the lane's columns: first + k, k < mine_n
  const int mine_n = group < p.groups ? max(0, min(lay.run, lay.size - in_group)) : 0;
  const bool softmax = p.kind == TRNOPT_ROUTE_SOFTMAX, on_scores = p.bias && p.bias_on == TRNOPT_ROUTE_BIAS_SCORES;
  const bool shares = on_scores || (p.groups > 1 && !p.bias);       // the choice looks at shares
  if (p.load) {
    for (int j = threadIdx.x; j < p.cols; j += 32 * RT_WARPS) counts[j] = 0;
    __syncthreads();
  }
  float bias[C];
  bool bad_bias = false;
#pragma unroll
  for (int k = 0; k < C; ++k) {
    bias[k] = p.bias && k < mine_n ? p.bias[first + k] : 0.f;
    bad_bias = bad_bias || bias[k] != bias[k];
  }
  if (lay.exact && p.bias)
    for (int j = lane; j < p.cols; j += 32) bad_bias = bad_bias || p.bias[j] != p.bias[j];
  bad_bias = __any_sync(kAll, bad_bias);

  constexpr int kV = C < Vec<T>::kN ? C : Vec<T>::kN;
  // Scores that come as vectors are fetched a row ahead where a lane holds few of them (of 8 they would spill: 32768 rows
  // of 64 columns 27 -> 23 us, of 256 columns 30 -> 36 us).
  constexpr bool kAhead = C <= 4;
  Vec<T> ahead[C / kV];
  auto fetch = [&](long long row) {
    if (lay.vectors && mine_n > 0 && row < p.rows) {
      const T* s = static_cast<const T*>(p.scores) + row * p.ld + first;
#pragma unroll
      for (int k = 0; k < C; k += kV) ahead[k / kV] = read_global<kV>(s + k);
    }
  };
  const long long stride = (long long)gridDim.x * RT_WARPS;
  if (kAhead) fetch((long long)blockIdx.x * RT_WARPS + w);
  for (long long row = (long long)blockIdx.x * RT_WARPS + w; row < p.rows; row += stride) {
    const T* s = static_cast<const T*>(p.scores) + row * p.ld;
    float x[C];
    if (lay.vectors) {
      if (!kAhead) fetch(row);
#pragma unroll
      for (int k = 0; k < C; ++k) x[k] = mine_n > 0 ? ahead[k / kV].get(k % kV) : -INFINITY;
      if (kAhead) fetch(row + stride);
    } else {
#pragma unroll
      for (int k = 0; k < C; ++k) x[k] = k < mine_n ? widen(s[first + k]) : -INFINITY;
    }
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < C; ++k) m = max_nan(m, x[k]);
    if (lay.exact)                                          // (the registers hold the first columns only)
      for (int j = lane; j < p.cols; j += 32) {
        m = max_nan(m, widen(s[j]));
      }
    const bool bad = __any_sync(kAll, !(m < INFINITY)) || bad_bias;
    m = warp_max(m);
    float sum = 0.f;
    if (softmax && (shares || !p.renormalize)) {
#pragma unroll
      for (int k = 0; k < C; ++k) sum += x[k] > -INFINITY ? ex2_approx((x[k] - m) * kLog2e) : 0.f;
      if (lay.exact) {
        sum = 0.f;
        for (int j = lane; j < p.cols; j += 32) sum += widen(s[j]) > -INFINITY ? ex2_approx((widen(s[j]) - m) * kLog2e) : 0.f;
      }
      sum = warp_sum(sum);
    }

    int mine = -1;                                          // lane k < top: the k-th choice, and its score
    float xm = 0.f;
    bool exact = lay.exact;
    if (!bad && !exact) {
      // keys, and how far two of them may be apart in float32 and still be in the other order in 64 bits: shares are off
      // by 2^-21 of themselves (2^-20 for a softmax, with its sum), a sum with a bias by 2^-24 of itself
      float key[C], tol = 0.f;
      if (!shares) {
#pragma unroll
        for (int k = 0; k < C; ++k) key[k] = x[k];
      } else if (softmax) {
        const float per_sum = 1.f / sum;
        tol = 4e-6f * per_sum;
#pragma unroll
        for (int k = 0; k < C; ++k) key[k] = ex2_approx((x[k] - m) * kLog2e) * per_sum;
      } else {
        tol = 4e-6f;
#pragma unroll
        for (int k = 0; k < C; ++k) key[k] = __fdividef(1.f, 1.f + ex2_approx(-x[k] * kLog2e));
      }
      if (p.bias) {
        float size = 0.f;
#pragma unroll
        for (int k = 0; k < C; ++k) {
          key[k] += bias[k];
          size = fmaxf(size, key[k] > -INFINITY ? fabsf(key[k]) : 0.f);
        }
        tol += 2.4e-7f * warp_max(size);
      }
      if (shares) {
#pragma unroll
        for (int k = 0; k < C; ++k) key[k] = x[k] == -INFINITY ? -INFINITY : key[k];
      }
      if (p.groups > 1) {
        float t1 = -INFINITY, t2 = -INFINITY;               // the group's two best, over its lanes
#pragma unroll
        for (int k = 0; k < C; ++k) {
          t2 = fmaxf(t2, fminf(t1, key[k]));
          t1 = fmaxf(t1, key[k]);
        }
        for (int o = 1; o < lay.lanes; o *= 2) {
          const float o1 = __shfl_xor_sync(kAll, t1, o), o2 = __shfl_xor_sync(kAll, t2, o);
          t2 = fmaxf(fminf(t1, o1), fmaxf(t2, o2));
          t1 = fmaxf(t1, o1);
        }
        const bool alive = t1 > -INFINITY;
        const float score = p.group_top == 2 && t2 > -INFINITY ? t1 + t2 : t1;
        int rank = 0;
        for (int g = 0; g < p.groups; ++g) {
          const float other = __shfl_sync(kAll, score, g * lay.lanes);        // (-inf: nothing open there)
          rank += other > score || (other == score && g < group);
        }
        bool open = alive && rank < p.top_groups;
        const float lowest = -warp_max(open ? -score : -INFINITY), highest = warp_max(open || !alive ? -INFINITY : score);
        if (lowest - highest <= 3.f * tol + 2.4e-7f * fabsf(lowest)) open = open_exact(p, s, lay.lanes, first, mine_n);
#pragma unroll
        for (int k = 0; k < C; ++k) key[k] = !open ? -INFINITY : p.bias ? key[k] : x[k];
      }
      const bool rounded = p.bias != nullptr;               // without a bias keys are scores from here on
      const int wanted = min(p.top + (rounded ? 1 : 0), 32);
      // at least `wanted` keys reach the wanted-th largest of the lanes' best ones: these go to shared memory
      float best = key[0];
#pragma unroll
      for (int k = 1; k < C; ++k) best = fmaxf(best, key[k]);
      // (closed columns are -inf; keys that rounding may have put below the bound are candidates, too)
      const float bound = fmaxf(kth_largest(best, wanted) - 2.f * tol, -3.4028235e38f);
      int n = 0;
#pragma unroll
      for (int k = 0; k < C; ++k) {
        const bool in = key[k] >= bound;
        const unsigned all = __ballot_sync(kAll, in);
        const int at = n + __popc(all & ((1u << lane) - 1));
        if (in && at < RT_LIST) {
          sh.list[w][at] = (uint64_t)order(key[k]) << 32 | (0xffffffffu - (unsigned)(first + k));
          if (kAhead) sh.score[w][at] = x[k];
        }
        n += __popc(all);
      }
      __syncwarp();
      uint64_t taken = 0;                                   // lane r < wanted: the r-th of them, 0 where there is none
      if (n <= RT_LIST) {
        // ranked by counting, a candidate or two per lane
        for (int e = lane; e < n; e += 32) {
          const uint64_t c = sh.list[w][e];
          int rank = 0;
#pragma unroll 4
          for (int o = 0; o < n; ++o) rank += sh.list[w][o] > c;
          if (rank < 32) {
            sh.best[w][rank] = c;
            if (kAhead) sh.best_score[w][rank] = sh.score[w][e];
          }
        }
        __syncwarp();
        if (lane < min(n, wanted)) taken = sh.best[w][lane];
        if (rounded) {
          // neighbours that float32 may have in the wrong order
          const float mine_key = key_of(taken), next = __shfl_down_sync(kAll, mine_key, 1);
          if (__any_sync(kAll, lane < wanted - 1 && next > -INFINITY && mine_key - next <= tol) || p.top == 32) {
            __syncwarp();
            rank_exact(p, s, sh.list[w], sh.score[w], sh.exact[w], n, sh.best[w], sh.best_score[w]);
            taken = lane < min(n, p.top) ? sh.best[w][lane] : 0;
          }
        }
        if (kAhead) xm = sh.best_score[w][lane];            // (elsewhere it is read again: x is not kept that long)
      } else if (rounded) {
        exact = true;                                       // more candidates than places
      } else {
        // many equal keys: the best one `wanted` times
        for (int r = 0; r < wanted; ++r) {
          uint64_t c = 0;
#pragma unroll
          for (int k = 0; k < C; ++k) {
            const uint64_t x = (uint64_t)order(key[k]) << 32 | (0xffffffffu - (unsigned)(first + k));
            c = key[k] > -INFINITY && x > c ? x : c;
          }
          for (int o = 16; o > 0; o >>= 1) {
            const uint64_t x = __shfl_xor_sync(kAll, c, o);
            c = x > c ? x : c;
          }
          if (c == 0) break;
          if (lane == r) { taken = c; xm = key_of(c); }
#pragma unroll
          for (int k = 0; k < C; ++k)
            if (first + k == (int)(0xffffffffu - (unsigned)c)) key[k] = -INFINITY;
        }
      }
      __syncwarp();
      if (taken != 0 && lane < p.top) mine = (int)(0xffffffffu - (unsigned)taken);
    }
    if (!bad && exact) {
      mine = choose_exact(p, s, keys + (size_t)w * p.cols);
      xm = mine >= 0 ? widen(s[mine]) : 0.f;
    }

    float weight = 0.f;
    if (!kAhead) xm = mine >= 0 ? widen(s[mine]) : 0.f;
    else if (mine < 0) xm = 0.f;
    const float lw = mine < 0 ? -INFINITY : softmax ? xm - m : log_sigmoid(xm);
    if (p.renormalize) {
      const float peak = warp_max(lw), e = mine >= 0 ? expf(lw - peak) : 0.f, total = warp_sum(e);
      if (mine >= 0) weight = p.scale * (e / total);
    } else if (mine >= 0) {
      weight = p.scale * (softmax ? expf(lw) / sum : expf(lw));
    }
    if (lane < p.top) {
      p.index[row * p.top + lane] = mine;
      p.weight[row * p.top + lane] = bad ? NAN : weight;
      if (p.load && mine >= 0) atomicAdd(counts + mine, 1);
    }
  }
  if (p.load) {
    __syncthreads();
    for (int j = threadIdx.x; j < p.cols; j += 32 * RT_WARPS) {
      if (gridDim.x == 1) p.load[j] = counts[j];
      else if (counts[j] != 0) atomicAdd(p.load + j, counts[j]);
    }
  }
}

// Gradient: a chosen column's value is scale * share * (d - mean) (renormalised: parts of the chosen ones' sum; a sigmoid:
// its own derivative), the others' 0, or for plain softmax weights -share * mean. One warp per row: the row's vectors, then
// the chosen columns over them.
template <typename T>
__global__ void __launch_bounds__(32 * RT_WARPS) route_grad_kernel(RouteGradProblem p) {
  constexpr int kN = Vec<T>::kN;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const bool softmax = p.kind == TRNOPT_ROUTE_SOFTMAX;
  for (long long row = (long long)blockIdx.x * RT_WARPS + w; row < p.rows; row += (long long)gridDim.x * RT_WARPS) {
    const T* s = static_cast<const T*>(p.scores) + row * p.ld;
    T* out = static_cast<T*>(p.grad) + row * p.ld_grad;
    const RowVectors<T> rv(out, p.cols);
    const long long index = lane < p.top ? p.index[row * p.top + lane] : -1;
    const int mine = index >= 0 && index < p.cols ? (int)index : -1;
    const float d = mine >= 0 ? p.scale * p.d_weight[row * p.top + lane] : 0.f;
    const float x = mine >= 0 ? widen(s[mine]) : 0.f;
    float grad = 0.f;
    if (p.renormalize || !softmax || !__any_sync(kAll, mine >= 0)) {
      for (int v = lane; v < (int)rv.count; v += 32) {
        const int j = (int)rv.column(v);
        if (rv.inside(v)) {
          *reinterpret_cast<uint4*>(out + j) = make_uint4(0, 0, 0, 0);
        } else {
          for (int e = max(j, 0); e < min(j + kN, p.cols); ++e) narrow(0.f, out + e);
        }
      }
      const float other = softmax ? 1.f : 1.f / (1.f + expf(x));      // d log share / dS of a column by itself
      if (p.renormalize) {
        const float lw = mine < 0 ? -INFINITY : softmax ? x : log_sigmoid(x);
        const float peak = warp_max(lw), e = mine >= 0 ? expf(lw - peak) : 0.f;
        const float total = warp_sum(e), part = mine >= 0 ? e / total : 0.f, mean = warp_sum(mine >= 0 ? part * d : 0.f);
        grad = part * (d - mean) * other;
      } else {
        grad = d * expf(log_sigmoid(x)) * other;
      }
    } else {
      float m = -INFINITY, sum = 0.f;
      for (int j = lane; j < p.cols; j += 32) m = fmaxf(m, widen(s[j]));
      m = warp_max(m);
      for (int j = lane; j < p.cols; j += 32) sum += ex2_approx((widen(s[j]) - m) * kLog2e);
      sum = warp_sum(sum);
      const float share = mine >= 0 ? expf(x - m) / sum : 0.f, mean = warp_sum(share * d), back = -mean / sum;
      for (int v = lane; v < (int)rv.count; v += 32) {
        const int j = (int)rv.column(v);
        Vec<T> r;
#pragma unroll
        for (int e = 0; e < kN; e += 2) {
          auto at = [&](int k) { return k >= 0 && k < p.cols ? ex2_approx((widen(s[k]) - m) * kLog2e) * back : 0.f; };
          r.set_pair(e, at(j + e), at(j + e + 1));
        }
        if (rv.inside(v)) {
          *reinterpret_cast<uint4*>(out + j) = r.q;
        } else {
#pragma unroll
          for (int e = 0; e < kN; ++e)
            if (j + e >= 0 && j + e < p.cols) out[j + e] = r.stored(e);
        }
      }
      grad = share * (d - mean);
    }
    __syncwarp();                                           // a chosen column's value follows the row's others
    if (mine >= 0) narrow(grad, out + mine);
  }
}

unsigned route_grid(long long rows) {
  const long long blocks = (rows + RT_WARPS - 1) / RT_WARPS;
  return (unsigned)(blocks < (1 << 20) ? blocks : (1 << 20));
}

template <typename T, int C>
cudaError_t launch(const RouteProblem& p, const RouteLayout& lay, cudaStream_t stream) {
  const size_t bytes = (size_t)RT_WARPS * p.cols * sizeof(double) + (size_t)p.cols * sizeof(int);
  static std::atomic<int> done[kMaxDevices];
  cudaError_t e = smem_attr_once(reinterpret_cast<const void*>(route_kernel<T, C>), (int)bytes, done);
  if (e != cudaSuccess) return e;
  // a persistent grid (the load is counted once per CTA)
  const long long blocks = (p.rows + RT_WARPS - 1) / RT_WARPS;
  const unsigned most = 148 * route_ctas(C), grid = (unsigned)(blocks < most ? blocks : most);
  if (p.load && grid > 1) {
    e = cudaMemsetAsync(p.load, 0, sizeof(int) * p.cols, stream);
    if (e != cudaSuccess) return e;
  }
  route_kernel<T, C><<<grid, 32 * RT_WARPS, bytes, stream>>>(p, lay);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch(const RouteProblem& p, cudaStream_t stream) {
  RouteLayout lay{};
  lay.size = p.cols / p.groups;
  lay.lanes = 32;
  for (int g = 1; g < p.groups; g *= 2) lay.lanes /= 2;
  lay.run = (lay.size + lay.lanes - 1) / lay.lanes;
  lay.exact = lay.run > 32;                                 // (few groups of many columns, not a power of two of them)
  if (lay.exact) { lay.lanes = 32; lay.run = 1; lay.size = p.cols < 32 ? p.cols : 32; }
  int c = 1;
  while (c < lay.run) c *= 2;
  const int v = c < Vec<T>::kN ? c : Vec<T>::kN;
  lay.vectors = !lay.exact && c == lay.run && lay.size % c == 0 && p.ld % v == 0 &&
                reinterpret_cast<uintptr_t>(p.scores) % (v * sizeof(T)) == 0;
  switch (c) {
    case 1: return launch<T, 1>(p, lay, stream);
    case 2: return launch<T, 2>(p, lay, stream);
    case 4: return launch<T, 4>(p, lay, stream);
    case 8: return launch<T, 8>(p, lay, stream);
    case 16: return launch<T, 16>(p, lay, stream);
    default: return launch<T, 32>(p, lay, stream);
  }
}

}  // namespace

cudaError_t route_launch(int type, const RouteProblem& p, cudaStream_t stream) {
  if (p.rows == 0) return p.load ? cudaMemsetAsync(p.load, 0, sizeof(int) * p.cols, stream) : cudaSuccess;
  switch (type) {
    case TRNOPT_F32: return launch<float>(p, stream);
    case TRNOPT_F16: return launch<__half>(p, stream);
    default: return launch<__nv_bfloat16>(p, stream);
  }
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

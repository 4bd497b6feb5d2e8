// Row softmax of a score matrix: log-probabilities of given columns, entropy, log-sum-exp and the best columns of
// each row, and the gradient. For row S, temperature T, m = max S, d_j = (S_j - m) / T:
//     s = sum_j exp(d_j),  log p_j = d_j - log s,  H = log s - sum_j exp(d_j) d_j / s,  lse = m / T + log s
//     dS_j = (1 / T) [ sum_t g_t (1[j = t] - p_j) + g_lse p_j - g_H p_j (log p_j + H) ]
// The difference S - m is taken before the scaling, so rows whose scores are all the type's lowest value are uniform
// rows and not overflow. Both terms of H are >= 0. A column of score -inf has p = 0 and adds nothing; a row without
// any other column has lse = log p = -inf, H = 0 and gradient 0; NaN or +inf in a row makes its values NaN.
// Sums in float32 (float64 for float64 scores).
//
// Forward: one pass over the scores. A row belongs to one CTA, or to the CTAs of a cluster when there are few rows;
// each thread holds 64 bytes of scores at a time (and the next 64 in flight), and keeps its own (m, s, sum e d),
// rescaled when its maximum rises. The best columns come out of the same pass: a bound below the K-th largest score is
// kept from the threads' running maxima (the K / warps-th largest of each warp's 32: at least K scores reach the
// smallest of these), raised after 1, 2, 4, 8, ... chunks, and the few scores above it are collected in a list that is
// ranked at the end. Where ties or ascending scores overflow the list, the chunk in registers and the list are cut to
// the K best by bisection.
#include <cooperative_groups.h>

#include "common.cuh"
#include "score_types.cuh"
#include "scores.h"

namespace trnopt {

namespace cg = cooperative_groups;

namespace {

constexpr unsigned kAll = 0xffffffffu;
constexpr int LP_VECS = 4;          // 16-byte vectors a thread holds of a chunk
constexpr int LP_LIST = 1024;       // candidates held for the best columns

// exp and log in the units of the sums: base 2 for float32, base e for float64. unit() turns such a logarithm into nats.
struct Base2 {
  static __device__ __forceinline__ float exp(float x) { return ex2_approx(x); }
  static __device__ __forceinline__ float log(float x) { return log2f(x); }
  static __device__ __forceinline__ float unit() { return 0.6931471805599453f; }
  static __device__ __forceinline__ float scale(double t) { return (float)(1.4426950408889634 / t); }
};
struct BaseE {
  static __device__ __forceinline__ double exp(double x) { return ::exp(x); }
  static __device__ __forceinline__ double log(double x) { return ::log(x); }
  static __device__ __forceinline__ double unit() { return 1.0; }
  static __device__ __forceinline__ double scale(double t) { return 1.0 / t; }
};
template <typename T> struct Base { using type = Base2; };
template <> struct Base<double> { using type = BaseE; };

// (S - m) c, at least -1e30: -inf scores (and -inf maxima) give exp() = 0 and a finite factor.
__device__ __forceinline__ float down(float x, float m, float c) { return fmaxf((x - m) * c, -1e30f); }
__device__ __forceinline__ double down(double x, double m, double c) { return fmax((x - m) * c, -1e30); }

// A softmax's running state: the largest score m, s = sum exp(d), t = sum exp(d) d.
template <typename A, typename B>
struct Sums {
  A m, s, t;
  __device__ __forceinline__ void raise(A to, A c) {          // to the larger maximum `to`
    const A d = down(m, to, c), w = B::exp(d);
    t = w * (t + s * d);
    s = w * s;
    m = to;
  }
  __device__ __forceinline__ void add(Sums o, A c) {
    const A to = max_nan(m, o.m);
    raise(to, c);
    o.raise(to, c);
    s += o.s;
    t += o.t;
  }
};

__device__ __forceinline__ float warp_max(float v) {
  for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(kAll, v, o));
  return v;
}
__device__ __forceinline__ double warp_max(double v) {
  for (int o = 16; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(kAll, v, o));
  return v;
}
template <typename A>
__device__ __forceinline__ A warp_sum(A v) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}

// Whole numbers in the order of the scores (-0 = +0), and back.
__device__ __forceinline__ uint32_t order(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ uint64_t order(double x) {
  const uint64_t b = (uint64_t)__double_as_longlong(x + 0.0);
  return b ^ ((uint64_t)((int64_t)b >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ float value(uint32_t k) {
  return __uint_as_float(k ^ ((k & 0x80000000u) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ double value(uint64_t k) {
  return __longlong_as_double((int64_t)(k ^ ((k >> 63) ? 0x8000000000000000ull : 0xffffffffffffffffull)));
}
__device__ __forceinline__ uint32_t warp_max_key(uint32_t k) { return __reduce_max_sync(kAll, k); }
__device__ __forceinline__ uint64_t warp_max_key(uint64_t k) {
  for (int o = 16; o > 0; o >>= 1) {
    const uint64_t x = __shfl_xor_sync(kAll, k, o);
    k = x > k ? x : k;
  }
  return k;
}

template <typename A>
struct Candidate {
  A x;
  int j;
};
template <typename A>
__device__ __forceinline__ bool better(A x, int j, A ox, int oj) { return x > ox || (x == ox && j < oj); }

template <typename A, int NW>
struct TopSmem {
  Candidate<A> list[LP_LIST], kept[LP_LIST];
  A bound[NW];
  int count, kept_count, wcount[NW];
};

template <typename A, int NW>
struct LogProbsSmem {
  A m[NW], s[NW], t[NW];
  Sums<A, typename Base<A>::type> part[8];                 // of a cluster's CTAs (written into the first one's)
};

// Number of threads' items over the CTA (every thread gets it).
template <typename A, int NW>
__device__ __forceinline__ int block_count(TopSmem<A, NW>& sh, int n) {
  n = __reduce_add_sync(kAll, n);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.wcount[threadIdx.x >> 5] = n;
  __syncthreads();
  int r = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) r += sh.wcount[w];
  return r;
}

// The K best of the list's first n candidates and the chunk in registers, as the new list: bisection on the K-th value,
// then on the column up to which columns of just that value are taken. Returns that value; all threads must call it.
template <typename T, typename A, int NW>
__device__ __noinline__ A cut_to_best(TopSmem<A, NW>& sh, const Vec<T> (&q)[LP_VECS], long long col0, int n, int top) {
  constexpr int NT = 32 * NW, kN = Vec<T>::kN, kOwn = LP_LIST / NT;
  using Key = decltype(order(A()));
  Candidate<A> own[kOwn];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    const int e = threadIdx.x + i * NT;
    own[i].x = e < n ? sh.list[e].x : (A)-INFINITY;
    own[i].j = e < n ? sh.list[e].j : 0;
  }
  auto each = [&](auto&& f) {
#pragma unroll
    for (int i = 0; i < kOwn; ++i) f(own[i].x, own[i].j);
#pragma unroll
    for (int i = 0; i < LP_VECS; ++i)
#pragma unroll
      for (int e = 0; e < kN; ++e) f(q[i].get(e), (int)(col0 + (long long)i * NT * kN + e));
  };
  Key k = 0;                                               // the largest key that at least `top` scores reach
  for (int bit = 8 * (int)sizeof(Key) - 1; bit >= 0; --bit) {
    const Key next = k | ((Key)1 << bit);
    const A bound = value(next);
    int c = 0;
    if (bound > (A)-INFINITY) {                            // (keys of NaN are above every score's)
      each([&](A x, int) { c += x >= bound; });
    } else {
      c = next <= order((A)-INFINITY) ? LP_LIST : 0;
    }
    if (block_count(sh, c) >= top) k = next;
  }
  const A kth = value(k);
  const bool all = !(kth > (A)-INFINITY);                  // fewer open columns than `top`: take them all
  int more = 0;
  each([&](A x, int) { more += x > (all ? (A)-INFINITY : kth); });
  const int wanted = all ? 0 : top - block_count(sh, more);
  int last = -1;                                           // columns of the K-th value are taken up to this one
  if (!all) {
    int low = 0, high = 0x7fffffff;
    while (low < high) {                                   // the smallest column that gives `wanted` of them
      const int mid = low + (high - low) / 2;
      int c = 0;
      each([&](A x, int j) { c += x == kth && j <= mid; });
      if (block_count(sh, c) >= wanted) high = mid;
      else low = mid + 1;
    }
    last = low;
  }
  __syncthreads();
  if (threadIdx.x == 0) sh.count = 0;
  __syncthreads();
  each([&](A x, int j) {
    if (all ? x > (A)-INFINITY : (x > kth || (x == kth && j <= last))) {
      const int at = atomicAdd(&sh.count, 1);
      if (at < LP_LIST) sh.list[at] = {x, j};
    }
  });
  __syncthreads();
  return all ? (A)-INFINITY : kth;
}

// The candidates of `in` ranked by (score, lower column): the `top` best into out (in order), the others dropped.
template <typename A>
__device__ __forceinline__ void rank_into(const Candidate<A>* in, int n, int top, int threads, Candidate<A>* out) {
  for (int e = threadIdx.x; e < n; e += threads) {
    const Candidate<A> c = in[e];
    int rank = 0;
    for (int o = 0; o < n; ++o) rank += better(in[o].x, in[o].j, c.x, c.j);
    if (rank < top) out[rank] = c;
  }
}

template <typename T, int NW, bool kTop>
__global__ void __launch_bounds__(32 * NW) log_probs_kernel(LogProbsProblem p, int parts) {
  using A = typename Acc<T>::type;
  using B = typename Base<T>::type;
  constexpr int NT = 32 * NW, kN = Vec<T>::kN;
  __shared__ LogProbsSmem<A, NW> sh;
  __shared__ __align__(16) unsigned char top_bytes[kTop ? sizeof(TopSmem<A, NW>) : 16];
  TopSmem<A, NW>& st = *reinterpret_cast<TopSmem<A, NW>*>(top_bytes);
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const long long row = blockIdx.x / parts;
  const int part = (int)(blockIdx.x % parts);
  const T* scores = static_cast<const T*>(p.scores) + row * p.ld;
  const RowVectors<T> rv(scores, p.cols);
  const long long per = (rv.count + parts - 1) / parts, v0 = part * per, v1 = min(rv.count, v0 + per);
  const A c = B::scale(p.temperature), inf = (A)INFINITY;

  // the first CTA answers for the row: its given columns' scores are fetched now
  A given = 0;
  long long given_j = -1;
  if (part == 0 && tid < p.n_targets) {
    given_j = p.targets[row * p.n_targets + tid];
    if (given_j >= 0 && given_j < p.cols) given = widen(scores[given_j]);
  }
  if (kTop) {
    if (tid == 0) st.count = st.kept_count = 0;
    if (tid < NW) st.bound[tid] = -inf;
    __syncthreads();
  }

  Sums<A, B> a{-inf, 0, 0};
  A bound = -inf;
  int listed = 0;                                           // candidates before this chunk
  const int each = (p.top + NW - 1) / NW;                   // scores that every warp vouches for
  Vec<T> q[LP_VECS];
#pragma unroll
  for (int i = 0; i < LP_VECS; ++i) q[i] = rv.load(v0 + i * NT + tid, v1);
  int chunk = 0;
  for (long long v = v0; v < v1; v += NT * LP_VECS, ++chunk) {
    Vec<T> next[LP_VECS];
    if (v + NT * LP_VECS < v1) {
#pragma unroll
      for (int i = 0; i < LP_VECS; ++i) next[i] = rv.load(v + (i + LP_VECS) * NT + tid, v1);
    }
    A peak = q[0].peak();
#pragma unroll
    for (int i = 1; i < LP_VECS; ++i) peak = max_nan(peak, q[i].peak());
    if (!(peak <= a.m)) a.raise(max_nan(peak, a.m), c);
#pragma unroll
    for (int i = 0; i < LP_VECS; ++i)
#pragma unroll
      for (int e = 0; e < kN; ++e) {
        const A d = down(q[i].get(e), a.m, c), x = B::exp(d);
        a.s += x;
        a.t += x * d;
      }
    if (kTop) {
      const bool refresh = (chunk & (chunk - 1)) == 0;
      if (refresh) {
        auto key = order(a.m);
        decltype(key) found = 0;
        for (int r = 0; r < each; ++r) {                    // the warp's each-th largest running maximum
          found = warp_max_key(key);
          const unsigned holds = __ballot_sync(kAll, key == found);
          if (lane == __ffs(holds) - 1) key = 0;
        }
        if (lane == 0) st.bound[w] = value(found);
        __syncthreads();
        A low = st.bound[0];
#pragma unroll
        for (int k = 1; k < NW; ++k) low = fmin(low, st.bound[k]);
        bound = fmax(bound, low);
      }
      // in a chunk that the bound knows of, scores equal to it may be among the K best; in a later one they may not
      if (refresh ? peak >= bound : peak > bound) {
#pragma unroll
        for (int i = 0; i < LP_VECS; ++i)
#pragma unroll
          for (int e = 0; e < kN; ++e) {
            const A x = q[i].get(e);
            if ((refresh ? x >= bound : x > bound) && x > -inf) {
              const int at = atomicAdd(&st.count, 1);
              if (at < LP_LIST) st.list[at] = {x, (int)(rv.column(v + i * NT + tid) + e)};
            }
          }
      }
      __syncthreads();
      int n = st.count;
      if (n > LP_LIST) {
        bound = fmax(bound, cut_to_best<T, A, NW>(st, q, rv.column(v + tid), listed, p.top));
        n = st.count;
      }
      __syncthreads();                                      // the count is read before the next chunk raises it
      listed = n;
    }
#pragma unroll
    for (int i = 0; i < LP_VECS; ++i) q[i] = next[i];
  }

  // the CTA's sums: a common maximum per warp, then over the warps
  {
    const A m = warp_max(a.m);
    a.raise(m, c);
    a.s = warp_sum(a.s);
    a.t = warp_sum(a.t);
    if (lane == 0) { sh.m[w] = a.m; sh.s[w] = a.s; sh.t[w] = a.t; }
  }
  if (kTop) {
    // candidates still above the last bound
    for (int e = tid; e < listed; e += NT) {
      const Candidate<A> cand = st.list[e];
      if (cand.x >= bound) st.kept[atomicAdd(&st.kept_count, 1)] = cand;
    }
  }
  __syncthreads();
  a = {sh.m[0], sh.s[0], sh.t[0]};
#pragma unroll
  for (int k = 1; k < NW; ++k) a.add({sh.m[k], sh.s[k], sh.t[k]}, c);

  Candidate<A>* best = nullptr;
  int n_best = 0;
  if (kTop) {
    n_best = min(st.kept_count, p.top);
    rank_into(st.kept, st.kept_count, p.top, NT, st.list);
    best = st.list;
    __syncthreads();
  }
  if (parts > 1) {
    // the cluster's CTAs bring their sums and best columns into the first one's shared memory
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();                                         // every CTA runs; the first one's list is ranked
    LogProbsSmem<A, NW>* sh0 = cluster.map_shared_rank(&sh, 0);
    if (tid == 0) sh0->part[part] = a;
    if (kTop) {
      TopSmem<A, NW>* st0 = cluster.map_shared_rank(&st, 0);
      for (int e = tid; e < p.top; e += NT)
        st0->kept[part * p.top + e] = e < n_best ? best[e] : Candidate<A>{-inf, 0x7fffffff - (part * p.top + e)};
    }
    cluster.sync();
    if (part != 0) return;
    for (int k = 1; k < parts; ++k) a.add(sh.part[k], c);
    if (kTop) {
      // empty slots (-inf, columns of their own) rank behind every candidate, each in a place of its own
      rank_into(st.kept, parts * p.top, p.top, NT, st.list);
      __syncthreads();
      n_best = p.top;
    }
  }

  const bool empty = a.m == -inf, bad = !(a.m < inf);
  const A inv_t = (A)(1.0 / p.temperature), log_s = bad ? (A)NAN : empty ? -inf : B::log(a.s) * B::unit();
  // in nats from the start: a lowest-value score may be finite here and not in base 2
  auto log_p = [&](A x) { return empty ? -inf : (x - a.m) * inv_t - log_s; };
  if (tid == 0) {
    static_cast<A*>(p.lse)[row] = empty ? -inf : a.m * inv_t + log_s;
    static_cast<A*>(p.entropy)[row] = empty ? (A)0 : log_s - a.t / a.s * B::unit();
    if (p.row_max) {
      static_cast<A*>(p.row_max)[row] = a.m;
      static_cast<A*>(p.log_sum)[row] = log_s;
    }
  }
  for (int k = tid; k < p.n_targets; k += NT) {
    if (k != tid) {
      given_j = p.targets[row * p.n_targets + k];
      if (given_j >= 0 && given_j < p.cols) given = widen(scores[given_j]);
    }
    static_cast<A*>(p.log_prob)[row * p.n_targets + k] =
        given_j < 0 ? (A)0 : given_j >= p.cols || bad ? (A)NAN : log_p(given);
  }
  if (kTop)
    for (int k = tid; k < p.top; k += NT) {
      const bool open = !bad && k < n_best && best[k].x > -inf;
      p.top_index[row * p.top + k] = open ? best[k].j : -1;
      static_cast<A*>(p.top_log_prob)[row * p.top + k] = bad ? (A)NAN : open ? log_p(best[k].x) : -inf;
    }
}

constexpr int LP_THREADS = 256;

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

// CTAs per row: a cluster where the rows alone leave SMs empty, as long as each CTA has a chunk of its own.
template <typename T, int NW>
int row_parts(const LogProbsProblem& p) {
  const long long chunk = 32LL * NW * LP_VECS * Vec<T>::kN;
  int parts = 1;
  while (parts < 8 && p.rows * parts < 148 * 2 && (long long)p.cols > chunk * parts) parts *= 2;
  return parts;
}

template <typename T, int NW, bool kTop>
cudaError_t launch(const LogProbsProblem& p, cudaStream_t stream) {
  const int parts = row_parts<T, NW>(p);
  const long long per = (1 << 30) / parts;                  // rows per launch: a grid's x stays below 2^31
  for (long long r = 0; r < p.rows; r += per) {
    LogProbsProblem q = p;
    q.rows = p.rows - r < per ? p.rows - r : per;
    const size_t size = sizeof(typename Acc<T>::type);
    auto at = [&](void* base, long long n) { return base ? static_cast<char*>(base) + n * size : nullptr; };
    q.scores = static_cast<const T*>(p.scores) + r * p.ld;
    q.targets = p.targets ? p.targets + r * p.n_targets : nullptr;
    q.log_prob = at(p.log_prob, r * p.n_targets);
    q.entropy = at(p.entropy, r);
    q.lse = at(p.lse, r);
    q.row_max = at(p.row_max, r);
    q.log_sum = at(p.log_sum, r);
    q.top_log_prob = at(p.top_log_prob, r * p.top);
    q.top_index = p.top_index ? p.top_index + r * p.top : nullptr;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(q.rows * parts));
    cfg.blockDim = dim3(32 * NW);
    cfg.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim = {(unsigned)parts, 1, 1};
    cfg.attrs = &attr;
    cfg.numAttrs = parts > 1 ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, log_probs_kernel<T, NW, kTop>, q, parts);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

template <typename T>
cudaError_t launch(const LogProbsProblem& p, cudaStream_t stream) {
  return p.top > 0 ? launch<T, 8, true>(p, stream) : launch<T, 8, false>(p, stream);
}

}  // namespace

cudaError_t log_probs_launch(int type, const LogProbsProblem& p, cudaStream_t stream) {
  switch (type) {
    case TRNOPT_F32: return launch<float>(p, stream);
    case TRNOPT_F16: return launch<__half>(p, stream);
    case TRNOPT_BF16: return launch<__nv_bfloat16>(p, stream);
    default: return launch<double>(p, stream);
  }
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

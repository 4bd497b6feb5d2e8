// Row softmax of a score matrix: log-probabilities of given columns, entropy, log-sum-exp and the best columns of
// each row, and the gradient. For row S, temperature T, m = max S, d_j = (S_j - m) / T:
//     s = sum_j exp(d_j),  log p_j = d_j - log s,  H = log s - sum_j exp(d_j) d_j / s,  lse = m / T + log s
//     dS_j = (1 / T) [ sum_t g_t (1[j = t] - p_j) + g_lse p_j - g_H p_j (log p_j + H) ]
// Both terms of H are >= 0. A column of score -inf has p = 0 and adds nothing; a row without any other column has
// lse = log p = -inf, H = 0 and gradient 0; NaN or +inf in a row makes its values NaN. Rows whose scores are all the
// type's lowest value are uniform rows. Sums in float32 (float64 for float64 scores).
//
// Forward: one pass over the scores. A row belongs to one CTA of 1 to 8 warps, or to the CTAs of a cluster when there are
// few rows; each thread works on 64 bytes of scores at a time, which it brings through shared memory itself (asynchronous
// copies, one or two more chunks in flight, no barrier), and keeps its own state: the largest score m, and with M = m c
// rounded (c = log2 e / T, or 1 / T in float64) the sums s = sum exp(x c - M) and t = sum exp(x c - M) (x c - M), both
// rescaled when m rises. M is a shift like any other, so its rounding cancels. Rows whose M is so large that it rounds by
// more than 1 (|m| / T beyond 1e7, 9e15 in float64) are summed again by the differences x - m.
// The best columns come out of the same pass: a bound below the K-th largest score is kept from the threads' running
// maxima (the K / warps-th largest of each warp's 32: at least K scores reach the smallest of these), raised after 1, 2,
// 4, 8, ... chunks, and each warp lists the few 16-byte vectors whose largest score reaches it. The K best scores lie in
// the K best vectors by (largest score, position): each of these holds a better score than any other vector does. So
// where ties or ascending scores overflow a list, the warp cuts it to its K best vectors by bisection, and at the end
// the vectors that still reach the bound are read again (from L2), and their scores ranked. Nothing but the first bound
// makes warps wait for one another. Bound by DRAM for many rows: 4096 x 131072 bfloat16 (1.07 GB) 174-198 us without best
// columns, 188-208 us with 5, by the scores, against 164 us at the copy rate of 6.55 TB/s; 1 x 131072 with 20, 12 us.
#include <cooperative_groups.h>

#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "score_types.cuh"
#include "scores.h"

namespace trnopt {

namespace cg = cooperative_groups;

namespace {

constexpr unsigned kAll = 0xffffffffu;
constexpr int LP_VECS = 4;          // 16-byte vectors a thread holds of a chunk
constexpr int LP_TOP = 64;          // most best columns
constexpr int LP_LIST = 96;         // vectors with candidates for them that a warp lists (more than LP_TOP)

// exp and log in the units of the sums: base 2 for float32, base e for float64. unit() turns such a logarithm into nats.
struct Base2 {
  static __device__ __forceinline__ float exp(float x) { return ex2_approx(x); }
  static __device__ __forceinline__ float log(float x) { return log2f(x); }
  static __device__ __forceinline__ float unit() { return 0.6931471805599453f; }
  static __device__ __forceinline__ float per_unit() { return 1.4426950408889634f; }
  static float scale(double t) { return (float)(1.4426950408889634 / t); }
  static __device__ __forceinline__ float wide() { return 0x1p24f; }       // shifts M beyond this are off by more than 1
};
struct BaseE {
  static __device__ __forceinline__ double exp(double x) { return ::exp(x); }
  static __device__ __forceinline__ double log(double x) { return ::log(x); }
  static __device__ __forceinline__ double unit() { return 1.0; }
  static __device__ __forceinline__ double per_unit() { return 1.0; }
  static double scale(double t) { return 1.0 / t; }
  static __device__ __forceinline__ double wide() { return 0x1p53; }
};
template <typename T> struct Base { using type = Base2; };
template <> struct Base<double> { using type = BaseE; };

// At least -1e30: differences to scores (or maxima) of -inf give exp() = 0 and a finite factor; NaN becomes -1e30 too.
__device__ __forceinline__ float floored(float d) { return fmaxf(d, -1e30f); }
__device__ __forceinline__ double floored(double d) { return fmax(d, -1e30); }

// A logarithm of p: from below where exp() is 0, so that its products with other numbers stay finite.
__device__ __forceinline__ float log_floored(float d) { return fmaxf(d, -200.f); }
__device__ __forceinline__ double log_floored(double d) { return fmax(d, -1000.0); }

// M: the rounded product itself, never contracted into what uses it.
__device__ __forceinline__ float shift(float m, float c) { return __fmul_rn(m, c); }
__device__ __forceinline__ double shift(double m, double c) { return __dmul_rn(m, c); }

// A softmax's running state: the largest score m; s and t relative to M = m c.
template <typename A, typename B>
struct Sums {
  A m, s, t;
  __device__ __forceinline__ void raise(A to, A c) {          // to the larger maximum `to`
    const A d = floored(shift(m, c) - shift(to, c)), w = B::exp(d);
    t = w > 0 ? w * (t + s * d) : 0;                          // (sums about an M of -inf are no numbers)
    s = w > 0 ? w * s : 0;
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

// The k-th largest (1 .. 32) of a warp's keys: by removal for the first ones, else by sorting the lanes.
template <typename K>
__device__ __forceinline__ K kth_key(K key, int k) {
  const int lane = threadIdx.x & 31;
  if (k <= 3) {
    K found = warp_max_key(key);
    for (int r = 1; r < k; ++r) {
      const unsigned holds = __ballot_sync(kAll, key == found);
      if (lane == __ffs(holds) - 1) key = 0;
      found = warp_max_key(key);
    }
    return found;
  }
#pragma unroll
  for (int size = 2; size <= 32; size *= 2)
#pragma unroll
    for (int o = size / 2; o > 0; o /= 2) {
      const K x = __shfl_xor_sync(kAll, key, o);
      const bool larger = ((lane & o) == 0) == ((lane & size) == 0);      // this lane keeps the larger key
      key = (x > key) == larger ? x : key;
    }
  return __shfl_sync(kAll, key, (k - 1) & 31);
}

// A score (or a vector's largest score) and its column (or the vector's number). Of two, the larger score comes first,
// of equal ones the lower number; float32 candidates carry both in one whole number.
template <typename A>
struct Candidate {
  double x;
  int j;
  Candidate() = default;
  __device__ __forceinline__ Candidate(double x_, int j_) : x(x_), j(j_) {}
  __device__ __forceinline__ double score() const { return x; }
  __device__ __forceinline__ int number() const { return j; }
  __device__ __forceinline__ bool before(const Candidate& o) const { return x > o.x || (x == o.x && j < o.j); }
};
template <>
struct Candidate<float> {
  uint64_t k;
  Candidate() = default;
  __device__ __forceinline__ Candidate(float x, int j) : k((uint64_t)order(x) << 32 | (0x7fffffffu - (uint32_t)j)) {}
  __device__ __forceinline__ float score() const { return value((uint32_t)(k >> 32)); }
  __device__ __forceinline__ int number() const { return (int)(0x7fffffffu - (uint32_t)k); }
  __device__ __forceinline__ bool before(const Candidate& o) const { return k > o.k; }
};

// Shared memory of a CTA of NW warps. The ring holds kStages chunks; after the scores it serves as `best` (the
// listed vectors, later the best columns) and `kept` (the scores of the K best vectors, or the best columns of each of a
// cluster's 8 CTAs). Where there are
// more than kRanked vectors, they are ranked and cut to K first.
template <typename T, int NW, bool kTop>
struct LogProbsSmem {
  using A = typename Acc<T>::type;
  static constexpr int kStages = NW == 8 ? 3 : 2, kRing = kStages * LP_VECS * 32 * NW * 16;
  static constexpr int kRanked = 64, kScores = kRanked * Vec<T>::kN;
  static constexpr int kBest = NW == 8 ? 8 * LP_TOP : LP_TOP;
  static constexpr int kKept = (kScores > kBest ? kScores : kBest) * (int)sizeof(Candidate<A>);
  static constexpr int kChosen = (NW * LP_LIST > kRanked ? NW * LP_LIST : kRanked) * (int)sizeof(Candidate<A>);
  union {
    uint4 ring[kRing / 16];
    unsigned char after[kTop ? (kRing > kKept + kChosen ? kRing : kKept + kChosen) : 16];
  };
  Candidate<A> list[kTop ? NW * LP_LIST : 1];
  volatile A bound[NW];
  int count[NW], kept_count, best_count;
  A m[NW], s[NW], t[NW];
  Sums<A, typename Base<T>::type> part[8];                   // of a cluster's CTAs (in the first one's)
  __device__ __forceinline__ Candidate<A>* kept() { return reinterpret_cast<Candidate<A>*>(after); }
  __device__ __forceinline__ Candidate<A>* best() { return reinterpret_cast<Candidate<A>*>(after + (kTop ? kKept : 0)); }
};

template <typename A>
struct Cut {
  int n;       // vectors left on the list
  A own;       // at least this many vectors reach it
};

// A warp's overflowing list, cut: the `top` best of its first n vectors and of the chunk (vectors mine[i * stride],
// numbers first + i * stride) by (largest score, lower number). Bisection on the K-th value, then on the number up to
// which vectors of just that value are taken.
template <typename T, typename A>
__device__ __noinline__ Cut<A> cut_list(const uint4* mine, int stride, int first, Candidate<A>* list, int* count,
                                        int n, A own, int top) {
  constexpr int kOld = LP_LIST / 32, kAllOf = kOld + LP_VECS;
  using Key = decltype(order(A()));
  const int lane = threadIdx.x & 31;
  A x[kAllOf];
  int j[kAllOf];
  Key key[kAllOf];
#pragma unroll
  for (int i = 0; i < kAllOf; ++i) {
    const int e = lane + i * 32, v = i - kOld;
    x[i] = v >= 0 ? Vec<T>{mine[v * stride]}.peak() : e < n ? list[e].score() : (A)-INFINITY;
    j[i] = v >= 0 ? first + v * stride : e < n ? list[e].number() : 0;
    key[i] = x[i] == x[i] ? order(x[i]) : 0;                 // (a row with NaN has no best columns)
  }
  Key k = 0;                                               // the largest key that at least `top` vectors reach
  for (int bit = 8 * (int)sizeof(Key) - 1; bit >= 0; --bit) {
    const Key next = k | ((Key)1 << bit);
    int reach = 0;
#pragma unroll
    for (int i = 0; i < kAllOf; ++i) reach += key[i] >= next;
    if ((int)__reduce_add_sync(kAll, reach) >= top) k = next;
  }
  int more = 0;
#pragma unroll
  for (int i = 0; i < kAllOf; ++i) more += key[i] > k;
  const int wanted = top - (int)__reduce_add_sync(kAll, more);
  int low = 0, high = 0x7fffffff;
  while (low < high) {                                     // the smallest number that gives `wanted` of them
    const int mid = low + (high - low) / 2;
    int reach = 0;
#pragma unroll
    for (int i = 0; i < kAllOf; ++i) reach += key[i] == k && j[i] <= mid;
    if ((int)__reduce_add_sync(kAll, reach) >= wanted) high = mid;
    else low = mid + 1;
  }
  __syncwarp();
  if (lane == 0) *count = 0;
  __syncwarp();
#pragma unroll
  for (int i = 0; i < kAllOf; ++i)
    if (x[i] > (A)-INFINITY && (key[i] > k || (key[i] == k && j[i] <= low))) {
      const int at = atomicAdd(count, 1);
      if (at < LP_LIST) list[at] = Candidate<A>(x[i], j[i]);
    }
  __syncwarp();
  return {min(*(volatile int*)count, LP_LIST), fmax(own, value(k))};
}

// The candidates of `in` ranked: the `top` first into out (in order), the others dropped.
template <typename A>
__device__ __forceinline__ void rank_into(const Candidate<A>* in, int n, int top, int threads, Candidate<A>* out) {
  for (int e = threadIdx.x; e < n; e += threads) {
    const Candidate<A> c = in[e];
    int rank = 0;
#pragma unroll 4
    for (int o = 0; o < n; ++o) rank += in[o].before(c);
    if (rank < top) out[rank] = c;
  }
}

// One chunk's sums relative to M: exp(d) and exp(d) d over the vectors, d = x c - M; kFloor for chunks with scores of
// -inf, whose d would make t no number.
template <typename T, typename A, typename B, bool kFloor>
__device__ __forceinline__ void chunk_sums(const Vec<T> (&q)[LP_VECS], A c, A M, A& s, A& t) {
  constexpr int kN = Vec<T>::kN;
  if constexpr (sizeof(A) == 4) {
    const uint64_t c2 = pack2(c, c), m2 = pack2(-M, -M);
    uint64_t s2 = 0, t2 = 0;                                // two sums each, of the even and the odd scores
#pragma unroll
    for (int i = 0; i < LP_VECS; ++i)
#pragma unroll
      for (int e = 0; e < kN; e += 2) {
        uint64_t d2 = fma2(pack2(q[i].get(e), q[i].get(e + 1)), c2, m2);
        float d0, d1;
        unpack2(d2, d0, d1);
        if (kFloor) {
          d0 = floored(d0);
          d1 = floored(d1);
          d2 = pack2(d0, d1);
        }
        const uint64_t x2 = pack2(B::exp(d0), B::exp(d1));
        s2 = add2(s2, x2);
        t2 = fma2(x2, d2, t2);
      }
    float a, b;
    unpack2(s2, a, b);
    s = a + b;
    unpack2(t2, a, b);
    t = a + b;
  } else {
    s = t = 0;
#pragma unroll
    for (int i = 0; i < LP_VECS; ++i)
#pragma unroll
      for (int e = 0; e < kN; ++e) {
        A d = fma(q[i].get(e), c, -M);
        if (kFloor) d = floored(d);
        const A x = B::exp(d);
        s += x;
        t = fma(x, d, t);
      }
  }
}

template <typename T, int NW, bool kTop>
__global__ void __launch_bounds__(32 * NW, (sizeof(T) == 8 ? 16 : 32) / NW)
    log_probs_kernel(LogProbsProblem p, int parts, typename Acc<T>::type c, typename Acc<T>::type inv_t) {
  using A = typename Acc<T>::type;
  using B = typename Base<T>::type;
  using Smem = LogProbsSmem<T, NW, kTop>;
  constexpr int NT = 32 * NW, kN = Vec<T>::kN, kChunk = NT * LP_VECS, kStages = Smem::kStages;
  extern __shared__ __align__(16) unsigned char smem_bytes[];
  Smem& sh = *reinterpret_cast<Smem*>(smem_bytes);
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const long long row = blockIdx.x / (unsigned)parts;
  const int part = (int)(blockIdx.x - (unsigned)row * (unsigned)parts);
  const T* scores = static_cast<const T*>(p.scores) + row * p.ld;
  const RowVectors<T> rv(scores, p.cols);
  // (parts is a power of two)
  const long long per = (rv.count + parts - 1) >> (31 - __clz(parts)), v0 = part * per, v1 = min(rv.count, v0 + per);
  const A inf = (A)INFINITY;

  uint4* mine = sh.ring + tid;                              // stage s, vector i: mine[(s * LP_VECS + i) * NT]
  auto fetch = [&](long long v, int stage) {                // the thread's vectors of the chunk at v, as one copy group
    uint4* to = mine + stage * LP_VECS * NT;
    if (v + kChunk <= v1 && rv.inside(v, kChunk)) {
      const T* at = scores + rv.column(v + tid);
#pragma unroll
      for (int i = 0; i < LP_VECS; ++i) copy_async16(to + i * NT, at + i * NT * kN);
    } else if (v < v1) {
#pragma unroll
      for (int i = 0; i < LP_VECS; ++i) {
        const long long at = v + i * NT + tid;
        if (at < v1 && rv.inside(at)) copy_async16(to + i * NT, scores + rv.column(at));
        else to[i * NT] = rv.load(at, v1).q;
      }
    }
    copy_async_commit();
  };
#pragma unroll
  for (int k = 0; k < kStages - 1; ++k) fetch(v0 + (long long)k * kChunk, k);

  // the first CTA answers for the row: its given columns' scores are fetched now
  A given = 0;
  long long given_j = -1;
  if (part == 0 && tid < p.n_targets) {
    given_j = p.targets[row * p.n_targets + tid];
    if (given_j >= 0 && given_j < p.cols) given = widen(scores[given_j]);
  }
  if (kTop) {
    if (tid == 0) sh.kept_count = sh.best_count = 0;
    if (tid < NW) { sh.bound[tid] = -inf; sh.count[tid] = 0; }
    __syncthreads();
  }

  Sums<A, B> a{-inf, 0, 0};
  // warps with scores to vouch for (all but those past the row's end), and how many each of them vouches for
  const int vouching = (int)max(1LL, min((long long)NW, (v1 - v0) / 32)), each = (p.top + vouching - 1) / vouching;
  A bound = -inf, own = -inf;                               // shared bound; the K-th of this warp's list once it was cut
  int listed = 0;                                           // vectors on the warp's list before this chunk
  auto refresh = [&]() {
    const auto key = kth_key(order(a.m), each);             // the warp's each-th largest running maximum
    if (lane == 0) sh.bound[w] = each <= 32 ? value(key) : -inf;
  };
  auto shared_bound = [&]() {
    A low = sh.bound[0];
    for (int k = 1; k < vouching; ++k) low = fmin(low, sh.bound[k]);
    bound = fmax(bound, low);
  };
  bool closed = false;                                      // whether the warp has met scores of -inf (or NaN)
  int chunk = 0, stage = 0;
  for (long long v = v0; v < v1; v += kChunk, ++chunk) {
    fetch(v + (long long)(kStages - 1) * kChunk, stage == 0 ? kStages - 1 : stage - 1);
    copy_async_wait<kStages - 1>();
    const uint4* from = mine + stage * LP_VECS * NT;
    Vec<T> q[LP_VECS];
#pragma unroll
    for (int i = 0; i < LP_VECS; ++i) q[i].q = from[i * NT];
    A peak = q[0].peak();
#pragma unroll
    for (int i = 1; i < LP_VECS; ++i) peak = max_nan(peak, q[i].peak());
    if (!(peak <= a.m)) a.raise(max_nan(peak, a.m), c);
    A s, t;
    if (!closed) {
      chunk_sums<T, A, B, false>(q, c, shift(a.m, c), s, t);
      closed = __any_sync(kAll, !(t == t));                 // from here on the warp floors its differences
    }
    if (closed) chunk_sums<T, A, B, true>(q, c, shift(a.m, c), s, t);
    a.s += s;
    a.t += t;
    if (kTop) {
      if ((chunk & (chunk - 1)) == 0) {
        refresh();
        if (chunk == 0) __syncthreads();                    // later bounds may be a refresh behind: still bounds
        else __syncwarp();
        shared_bound();
      }
      if (__any_sync(kAll, peak >= bound && peak > own)) {
#pragma unroll
        for (int i = 0; i < LP_VECS; ++i) {
          const A x = q[i].peak();
          if (x >= bound && x > own) {
            const int at = atomicAdd(&sh.count[w], 1);
            if (at < LP_LIST) sh.list[w * LP_LIST + at] = Candidate<A>(x, (int)(v + i * NT + tid));
          }
        }
        __syncwarp();
        const int n = *(volatile int*)&sh.count[w];
        if (n > LP_LIST) {
          const Cut<A> r = cut_list<T, A>(from, NT, (int)(v + tid), &sh.list[w * LP_LIST], &sh.count[w], listed, own,
                                          p.top);
          listed = r.n;
          own = r.own;
        } else {
          listed = n;
        }
      }
    }
    stage = stage + 1 == kStages ? 0 : stage + 1;
  }

  // the CTA's sums: a common maximum per warp, then over the warps
  {
    if (kTop) refresh();
    const A m = warp_max(a.m);
    a.raise(m, c);
    a.s = warp_sum(a.s);
    a.t = warp_sum(a.t);
    if (lane == 0) { sh.m[w] = a.m; sh.s[w] = a.s; sh.t[w] = a.t; }
  }
  __syncthreads();                                          // (and the ring is free)
  int n_best = 0;
  if (kTop) {
    // vectors that reach the last bounds
    shared_bound();
    for (int e = lane; e < listed; e += 32) {
      const Candidate<A> cand = sh.list[w * LP_LIST + e];
      if (cand.score() >= bound) sh.best()[atomicAdd(&sh.best_count, 1)] = cand;
    }
    __syncthreads();
    int n = sh.best_count;
    const Candidate<A>* vectors = sh.best();
    if (n > Smem::kRanked) {
      rank_into(sh.best(), n, p.top, NT, sh.list);
      vectors = sh.list;
      n = p.top;
      __syncthreads();
    }
    // their scores, read again
    for (int e = tid; e < n * kN; e += NT) {
      const long long j = rv.column(vectors[e / kN].number()) + e % kN;
      if (j < 0 || j >= p.cols) continue;
      const A x = widen(scores[j]);
      if (x >= bound && x > -inf) sh.kept()[atomicAdd(&sh.kept_count, 1)] = Candidate<A>(x, (int)j);
    }
    __syncthreads();
    n_best = min(sh.kept_count, p.top);
    rank_into(sh.kept(), sh.kept_count, p.top, NT, sh.best());
    __syncthreads();
  }
  a = {sh.m[0], sh.s[0], sh.t[0]};
#pragma unroll
  for (int k = 1; k < NW; ++k) a.add({sh.m[k], sh.s[k], sh.t[k]}, c);
  const Candidate<A>* best = sh.best();
  if (parts > 1) {
    // the cluster's CTAs bring their sums and best columns into the first one's shared memory
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();                                         // every CTA runs; the first one's `kept` is ranked
    Smem* sh0 = cluster.map_shared_rank(&sh, 0);
    if (tid == 0) sh0->part[part] = a;
    if (kTop)
      for (int e = tid; e < p.top; e += NT) {
        const int at = part * p.top + e;                    // empty slots: -inf, columns of their own
        sh0->kept()[at] = e < n_best ? best[e] : Candidate<A>(-inf, 0x7fffffff - at);
      }
    cluster.sync();
    if (part != 0) return;
    for (int k = 1; k < parts; ++k) a.add(sh.part[k], c);
    if (kTop) {
      rank_into(sh.kept(), parts * p.top, p.top, NT, sh.best());
      __syncthreads();
      n_best = p.top;
    }
  }

  const bool empty = a.m == -inf, bad = !(a.m < inf);
  A past = fma(a.m, c, -shift(a.m, c));                       // m c - M: s is relative to M, log_s below to m c
  if (!empty && !bad && !(fabs(shift(a.m, c)) <= B::wide())) {
    // M rounds m c by up to half its spacing, which may carry the terms out of range: s and t once more, by the differences
    // x - m
    past = 0;
    A s = 0, t = 0;
    for (long long j = tid; j < p.cols; j += NT) {
      const A d = floored((widen(scores[j]) - a.m) * c), x = B::exp(d);
      s += x;
      t += x * d;
    }
    s = warp_sum(s);
    t = warp_sum(t);
    __syncthreads();
    if (lane == 0) { sh.s[w] = s; sh.t[w] = t; }
    __syncthreads();
    a.s = a.t = 0;
    for (int k = 0; k < NW; ++k) { a.s += sh.s[k]; a.t += sh.t[k]; }
  }
  const A log_s = bad ? (A)NAN : empty ? -inf : (B::log(a.s) - past) * B::unit();
  // in nats from the start: a lowest-value score may be finite here and not in base 2
  auto log_p = [&](A x) { return empty ? -inf : (x - a.m) * inv_t - log_s; };
  if (tid == 0) {
    static_cast<A*>(p.lse)[row] = empty ? -inf : a.m * inv_t + log_s;
    static_cast<A*>(p.entropy)[row] = empty ? (A)0 : max_nan((A)0, (B::log(a.s) - a.t / a.s) * B::unit());
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
      const A x = k < n_best ? best[k].score() : -inf;
      const bool open = !bad && x > -inf;
      p.top_index[row * p.top + k] = open ? best[k].number() : -1;
      static_cast<A*>(p.top_log_prob)[row * p.top + k] = bad ? (A)NAN : open ? log_p(x) : -inf;
    }
}

// Gradient: a CTA of one warp takes `chunks` x 32 x LP_VECS vectors of one row, placed on the gradient's 16-byte
// boundaries, the next chunk on its way while one is worked on. With the row's m and log s a score needs no sum:
// p (A + B log p) / T, with A = -(g + g_H H), B = -g_H and g the sum of the upstream gradients of the row's given and best
// columns (less that of lse). Those columns are written once more, by the first entry that names them, with the entries that
// repeat it added in order. Bound by the two matrices' bytes: 8192 x 32768 bfloat16 (2 x 0.54 GB) 171 us, 164 us at the
// copy rate. (CTAs of 256 threads: 174 us, but 8192 x 1000 70 us against 12 us.) Named columns cost next to nothing up to
// some dozens, but grow with their square: 4096 x 1000 with 128 / 512 / 1024 targets a row 90 / 1,090 / 4,190 us.
template <typename T>
__global__ void __launch_bounds__(32, 32) log_probs_grad_kernel(LogProbsGradProblem p, int parts, int chunks,
                                                               typename Acc<T>::type c, typename Acc<T>::type inv_t) {
  using A = typename Acc<T>::type;
  using B = typename Base<T>::type;
  constexpr int NT = 32, kN = Vec<T>::kN, kChunk = NT * LP_VECS;
  const int lane = threadIdx.x;
  const long long row = blockIdx.x / (unsigned)parts;
  const long long v0 = (long long)(blockIdx.x - (unsigned)row * (unsigned)parts) * chunks * kChunk;
  const T* s = static_cast<const T*>(p.scores) + row * p.ld;
  T* out = static_cast<T*>(p.grad) + row * p.ld_grad;
  const RowVectors<T> rv(out, p.cols);
  if (v0 >= rv.count) return;
  const long long v1 = min(rv.count, v0 + (long long)chunks * kChunk);
  const long long first = rv.column(v0), end = rv.column(v1);                   // the CTA's columns
  const bool vectors = (reinterpret_cast<uintptr_t>(s + first) & 15) == 0;     // the scores' vectors fall together
  auto fetch = [&](Vec<T>(&q)[LP_VECS], long long v) {
    if (vectors && v + kChunk <= v1 && rv.inside(v, kChunk)) {
      const T* at = s + rv.column(v + lane);
#pragma unroll
      for (int i = 0; i < LP_VECS; ++i) q[i] = RowVectors<T>::read(at + i * NT * kN);
    } else {
#pragma unroll
      for (int i = 0; i < LP_VECS; ++i) {
        const long long at = v + i * NT + lane, j = rv.column(at);
        if (vectors && at < v1 && rv.inside(at)) {
          q[i] = RowVectors<T>::read(s + j);
        } else {
#pragma unroll
          for (int e = 0; e < kN; ++e)
            q[i].set(e, at < v1 && j + e >= 0 && j + e < p.cols ? s[j + e] : lowest_inf<T>());
        }
      }
    }
  };
  Vec<T> q[LP_VECS];
  fetch(q, v0);

  const A inf = (A)INFINITY;
  const int extra = p.n_targets + p.top;
  // entry k < n_targets is a given column, the others are the best columns
  const long long* tg = p.targets + row * p.n_targets;
  const long long* ti = p.top_index + row * p.top;
  const A* gt = p.d_log_prob ? static_cast<const A*>(p.d_log_prob) + row * p.n_targets : nullptr;
  const A* gk = p.d_top ? static_cast<const A*>(p.d_top) + row * p.top : nullptr;
  auto column = [&](int k) { return k < p.n_targets ? tg[k] : ti[k - p.n_targets]; };
  auto upstream = [&](int k) { return k < p.n_targets ? (gt ? gt[k] : (A)0) : (gk ? gk[k - p.n_targets] : (A)0); };
  const A m = static_cast<const A*>(p.row_max)[row], log_s = static_cast<const A*>(p.log_sum)[row];
  const A h = static_cast<const A*>(p.entropy)[row];
  const A gh = p.d_entropy ? static_cast<const A*>(p.d_entropy)[row] : (A)0;
  A total = 0;
  for (int k = lane; k < extra; k += 32) {
    const long long j = column(k);
    const A g = upstream(k);
    if (j >= 0 && j < p.cols) total += g;
  }
  total = warp_sum(total);
  if (p.d_lse) total -= static_cast<const A*>(p.d_lse)[row];
  const bool empty = m == -inf;
  const A ls = log_s * B::per_unit(), fa = -(total + gh * h), fb = -gh * B::unit();
  auto dense = [&](A x) {
    const A lp = log_floored(fma(x - m, c, -ls));
    return B::exp(lp) * fma(fb, lp, fa);                   // (times 1 / T last: a p of 0 stays 0 whatever T)
  };
  for (long long v = v0; v < v1; v += kChunk) {
    Vec<T> next[LP_VECS];
    if (v + kChunk < v1) fetch(next, v + kChunk);
#pragma unroll
    for (int i = 0; i < LP_VECS; ++i) {
#pragma unroll
      for (int e = 0; e < kN; e += 2) {
        if constexpr (sizeof(A) == 4) {
          float a, b;
          unpack2(fma2(add2(pack2(q[i].get(e), q[i].get(e + 1)), pack2(-m, -m)), pack2(c, c), pack2(-ls, -ls)), a, b);
          a = log_floored(a);
          b = log_floored(b);
          const uint64_t f = fma2(pack2(a, b), pack2(fb, fb), pack2(fa, fa));
          unpack2(mul2(mul2(pack2(B::exp(a), B::exp(b)), f), pack2(inv_t, inv_t)), a, b);
          q[i].set_pair(e, a, b);
        } else {
          q[i].set_pair(e, dense(q[i].get(e)) * inv_t, dense(q[i].get(e + 1)) * inv_t);
        }
      }
      if (empty) q[i].q = make_uint4(0, 0, 0, 0);
    }
    if (v + kChunk <= v1 && rv.inside(v, kChunk)) {
      T* at = out + rv.column(v + lane);
#pragma unroll
      for (int i = 0; i < LP_VECS; ++i) *reinterpret_cast<uint4*>(at + i * NT * kN) = q[i].q;
    } else {
#pragma unroll
      for (int i = 0; i < LP_VECS; ++i) {
        const long long at = v + i * NT + lane, j = rv.column(at);
        if (at >= v1) continue;
        if (rv.inside(at)) {
          *reinterpret_cast<uint4*>(out + j) = q[i].q;
        } else {
#pragma unroll
          for (int e = 0; e < kN; ++e)
            if (j + e >= 0 && j + e < p.cols) out[j + e] = q[i].stored(e);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < LP_VECS; ++i) q[i] = next[i];
  }
  if (extra == 0 || empty) return;
  __syncwarp();                                            // the named columns follow the CTA's others
  for (int k = lane; k < extra; k += NT) {
    const long long j = column(k);
    if (j < 0 || j >= p.cols || j < first || j >= end) continue;
    bool again = false;
    for (int r = 0; r < k; ++r) again = again || column(r) == j;
    if (again) continue;
    A g = upstream(k);
    for (int r = k + 1; r < extra; ++r)
      if (column(r) == j) g += upstream(r);
    narrow((g + dense(widen(s[j]))) * inv_t, out + j);
  }
}

// CTAs per row: a cluster where the rows alone leave SMs empty, up to two CTAs per SM and as long as each CTA has a chunk of
// its own. Measured with 1 / 2 / 4 / 8 CTAs per row, 131072 columns, 20 best: 1 row 21 / 16 / 12 / 12 us, 16 rows
// 21 / 16 / 14 / 13 us, 64 rows 22 / 16 / 15 / 19 us.
template <typename T, int NW>
int row_parts(const LogProbsProblem& p) {
  const long long chunk = 32LL * NW * LP_VECS * Vec<T>::kN;
  int parts = 1;
  if (NW == 8)
    while (parts < 8 && 2 * p.rows * parts <= 148 * 2 && (long long)p.cols > chunk * parts) parts *= 2;
  return parts;
}

template <typename T, int NW, bool kTop>
cudaError_t launch(const LogProbsProblem& p, cudaStream_t stream) {
  using Smem = LogProbsSmem<T, NW, kTop>;
  if (sizeof(Smem) > 48 * 1024) {
    static std::atomic<int> done[kMaxDevices];
    const cudaError_t e = smem_attr_once(reinterpret_cast<const void*>(log_probs_kernel<T, NW, kTop>), sizeof(Smem), done);
    if (e != cudaSuccess) return e;
  }
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
    cfg.dynamicSmemBytes = sizeof(Smem);
    cfg.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim = {(unsigned)parts, 1, 1};
    cfg.attrs = &attr;
    cfg.numAttrs = parts > 1 ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, log_probs_kernel<T, NW, kTop>, q, parts, Base<T>::type::scale(p.temperature),
                                             (typename Acc<T>::type)(1.0 / p.temperature));
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

template <typename T>
cudaError_t launch(const LogProbsProblem& p, cudaStream_t stream) {
  // The fewest warps per row that fill half of the SMs' 32 warp slots, and no more than the row has chunks for: what a
  // row costs besides its scores (ranking, joining sums) grows with its warps. Measured at 8 / 4 / 2 / 1 warps, bfloat16,
  // 5 best columns: 8192 x 32768 166 / 129 / 109 / 104 us, 8192 x 1000 115 / 59 / 33 / 18 us, 600 x 5000
  // 15 / 12 / 10 / 12 us, 300 x 131072 29 / 35 / 47 / 68 us. (600 x 5000 takes 4 warps by this rule, 2 us more than with 2.)
  // A warp vouches for 24 best columns at most (of its 32 lanes' maxima the 32nd is a poor bound): 2048 x 32000 with 64 best
  // columns 72 / 76 / 126 / 237 us.
  const long long warp_cols = 32LL * LP_VECS * Vec<T>::kN;
  int nw = 1;
  while (nw < 8 && (p.rows * nw < 148 * 16 || p.top > 24 * nw) && (long long)p.cols > nw * warp_cols) nw *= 2;
  if (nw == 1) return p.top > 0 ? launch<T, 1, true>(p, stream) : launch<T, 1, false>(p, stream);
  if (nw == 2) return p.top > 0 ? launch<T, 2, true>(p, stream) : launch<T, 2, false>(p, stream);
  if (nw == 4) return p.top > 0 ? launch<T, 4, true>(p, stream) : launch<T, 4, false>(p, stream);
  return p.top > 0 ? launch<T, 8, true>(p, stream) : launch<T, 8, false>(p, stream);
}

template <typename T>
cudaError_t grad_launch(const LogProbsGradProblem& p, cudaStream_t stream) {
  constexpr long long kCols = 32LL * LP_VECS * Vec<T>::kN;
  // (a row may start inside a vector, and then reach into one more chunk)
  const bool aligned = p.ld_grad % Vec<T>::kN == 0 && reinterpret_cast<uintptr_t>(p.grad) % 16 == 0;
  const long long all = ((long long)p.cols + (aligned ? 0 : Vec<T>::kN - 1) + kCols - 1) / kCols;
  // up to 4 chunks per CTA, which share the row's numbers, while that leaves 8 CTAs per SM: 8192 x 32768 with 1 / 4 / 16
  // chunks 241 / 171 / 177 us, 100 x 50000 8 / 8 / 12 us
  int chunks = 1;
  while (chunks < 4 && chunks < all && p.rows * ((all + 2 * chunks - 1) / (2 * chunks)) >= 148 * 8) chunks *= 2;
  const int parts = (int)((all + chunks - 1) / chunks);
  const long long per = (1LL << 30) / parts;
  const size_t size = sizeof(typename Acc<T>::type);
  for (long long r = 0; r < p.rows; r += per) {
    auto at = [&](const void* base, long long n) { return base ? static_cast<const char*>(base) + n * size : nullptr; };
    LogProbsGradProblem q = p;
    q.rows = p.rows - r < per ? p.rows - r : per;
    q.scores = static_cast<const T*>(p.scores) + r * p.ld;
    q.grad = static_cast<T*>(p.grad) + r * p.ld_grad;
    q.targets = p.targets ? p.targets + r * p.n_targets : nullptr;
    q.top_index = p.top_index ? p.top_index + r * p.top : nullptr;
    q.row_max = at(p.row_max, r);
    q.log_sum = at(p.log_sum, r);
    q.entropy = at(p.entropy, r);
    q.d_log_prob = at(p.d_log_prob, r * p.n_targets);
    q.d_entropy = at(p.d_entropy, r);
    q.d_lse = at(p.d_lse, r);
    q.d_top = at(p.d_top, r * p.top);
    log_probs_grad_kernel<T><<<(unsigned)(q.rows * parts), 32, 0, stream>>>(
        q, parts, chunks, Base<T>::type::scale(p.temperature), (typename Acc<T>::type)(1.0 / p.temperature));
  }
  return cudaGetLastError();
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
  switch (type) {
    case TRNOPT_F32: return grad_launch<float>(p, stream);
    case TRNOPT_F16: return grad_launch<__half>(p, stream);
    case TRNOPT_BF16: return grad_launch<__nv_bfloat16>(p, stream);
    default: return grad_launch<double>(p, stream);
  }
}

}  // namespace trnopt

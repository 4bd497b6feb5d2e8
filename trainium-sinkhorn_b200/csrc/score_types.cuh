// Loads and stores of the score types: float32, float16 and bfloat16 are worked on in float32, float64 in float64.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>
#include <stdint.h>

namespace trnopt {

template <typename T> struct Acc { using type = float; };
template <> struct Acc<double> { using type = double; };

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(__half x) { return __half2float(x); }
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ double widen(double x) { return x; }
// Rounded once to the stored type.
__device__ __forceinline__ void narrow(float v, float* p) { *p = v; }
__device__ __forceinline__ void narrow(float v, __half* p) { *p = __float2half_rn(v); }
__device__ __forceinline__ void narrow(float v, __nv_bfloat16* p) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void narrow(double v, double* p) { *p = v; }

// Asynchronous 16-byte copies into shared memory, waited for by the thread that made them.
__device__ __forceinline__ void copy_async16(void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from)
               : "memory");
}
__device__ __forceinline__ void copy_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft>                       // until at most kLeft of the thread's groups are outstanding
__device__ __forceinline__ void copy_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory");
}

// Two float32 operations in one instruction.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ double max_nan(double a, double b) { return (a != a || a > b) ? a : b; }   // (b NaN: b)

// Sixteen bytes of a row: kN scores.
template <typename T>
struct Vec {
  static constexpr int kN = 16 / (int)sizeof(T);
  uint4 q;

  __device__ __forceinline__ typename Acc<T>::type get(int i) const {      // i known at compile time
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    if constexpr (sizeof(T) == 2) {
      const uint32_t x = w[i / 2];
      if constexpr (sizeof(typename Acc<T>::type) == 4) return half_of(x, i & 1, (const T*)nullptr);
    } else if constexpr (sizeof(T) == 4) {
      return __uint_as_float(w[i]);
    } else {
      return __hiloint2double((int)w[2 * i + 1], (int)w[2 * i]);
    }
  }
  __device__ __forceinline__ void set(int i, T v) {
    uint32_t w[4] = {q.x, q.y, q.z, q.w};
    if constexpr (sizeof(T) == 2) {
      const uint32_t b = *reinterpret_cast<const uint16_t*>(&v);
      w[i / 2] = (i & 1) ? (w[i / 2] & 0xffffu) | (b << 16) : (w[i / 2] & 0xffff0000u) | b;
    } else if constexpr (sizeof(T) == 4) {
      w[i] = *reinterpret_cast<const uint32_t*>(&v);
    } else {
      const uint2 b = *reinterpret_cast<const uint2*>(&v);
      w[2 * i] = b.x;
      w[2 * i + 1] = b.y;
    }
    q = make_uint4(w[0], w[1], w[2], w[3]);
  }

  // Scores i and i + 1 (i even), rounded.
  __device__ __forceinline__ void set_pair(int i, typename Acc<T>::type a, typename Acc<T>::type b) {
    if constexpr (sizeof(T) == 2) {
      const uint32_t x = pair_of(a, b, (const T*)nullptr);
      if (i == 0) q.x = x;
      else if (i == 2) q.y = x;
      else if (i == 4) q.z = x;
      else q.w = x;
    } else {
      set(i, (T)a);
      set(i + 1, (T)b);
    }
  }
  __device__ __forceinline__ T stored(int i) const {
    T r;
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    if constexpr (sizeof(T) == 2) {
      const uint16_t b = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
      r = *reinterpret_cast<const T*>(&b);
    } else {
      r = (T)get(i);
    }
    return r;
  }

  // The largest of the kN scores, NaN if one is; two 16-bit scores at a time.
  __device__ __forceinline__ typename Acc<T>::type peak() const {
    if constexpr (sizeof(T) == 2) {
      return peak16((const T*)nullptr);
    } else {
      typename Acc<T>::type m = get(0);
#pragma unroll
      for (int i = 1; i < kN; ++i) m = max_nan(m, get(i));
      return m;
    }
  }

 private:
  static __device__ __forceinline__ uint32_t pair_of(float a, float b, const __nv_bfloat16*) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ uint32_t pair_of(float a, float b, const __half*) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float half_of(uint32_t x, int odd, const __nv_bfloat16*) {
    return __uint_as_float(odd ? x & 0xffff0000u : x << 16);
  }
  static __device__ __forceinline__ float half_of(uint32_t x, int odd, const __half*) {
    const __half2 h = *reinterpret_cast<const __half2*>(&x);
    return odd ? __high2float(h) : __low2float(h);
  }
  __device__ __forceinline__ float peak16(const __nv_bfloat16*) const {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&q);
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return max_nan(__low2float(m), __high2float(m));
  }
  __device__ __forceinline__ float peak16(const __half*) const {
    const __half2* h = reinterpret_cast<const __half2*>(&q);
    const __half2 m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
    return max_nan(__low2float(m), __high2float(m));
  }
};

template <typename T>
__device__ __forceinline__ T lowest_inf();
template <> __device__ __forceinline__ float lowest_inf<float>() { return -INFINITY; }
template <> __device__ __forceinline__ double lowest_inf<double>() { return -INFINITY; }
template <> __device__ __forceinline__ __half lowest_inf<__half>() { return __ushort_as_half(0xfc00); }
template <> __device__ __forceinline__ __nv_bfloat16 lowest_inf<__nv_bfloat16>() { return __ushort_as_bfloat16(0xff80); }

// A row of scores as 16-byte vectors: the row may start anywhere, so vector v holds the columns
// [v kN - shift, (v + 1) kN - shift) with `shift` the row start's distance (in scores) from the 16-byte boundary before
// it. Only vectors that lie wholly inside the row are read as such; columns outside it come back as -inf, and nothing
// outside it is read or written.
template <typename T>
struct RowVectors {
  const T* row;
  int shift, cols;
  long long count;

  __device__ __forceinline__ RowVectors(const T* r, int c) : row(r), cols(c) {
    shift = (int)((reinterpret_cast<uintptr_t>(r) & 15) / sizeof(T));
    count = ((long long)cols + shift + Vec<T>::kN - 1) / Vec<T>::kN;
  }
  __device__ __forceinline__ long long column(long long v) const { return v * Vec<T>::kN - shift; }
  __device__ __forceinline__ bool inside(long long v) const {
    return column(v) >= 0 && column(v) + Vec<T>::kN <= cols;
  }
  // whether the vectors [v, v + n) all lie wholly inside the row
  __device__ __forceinline__ bool inside(long long v, int n) const {
    return column(v) >= 0 && column(v + n) <= cols;
  }
  static __device__ __forceinline__ Vec<T> read(const T* at) {
    Vec<T> r;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
        : "=r"(r.q.x), "=r"(r.q.y), "=r"(r.q.z), "=r"(r.q.w)
        : "l"(at));
    return r;
  }
  __device__ __forceinline__ Vec<T> load(long long v, long long end) const {
    constexpr int kN = Vec<T>::kN;
    Vec<T> r;
    const long long j = column(v);
    if (v < end && inside(v)) {
      r = read(row + j);
    } else {
#pragma unroll
      for (int i = 0; i < kN; ++i)
        r.set(i, v < end && j + i >= 0 && j + i < cols ? row[j + i] : lowest_inf<T>());
    }
    return r;
  }
};

// V neighbouring scores (at most 16 bytes, on a boundary of V) in the first places of a vector, through the read-only
// cache.
template <int V, typename T>
__device__ __forceinline__ Vec<T> read_global(const T* p) {
  constexpr int kBytes = V * (int)sizeof(T);
  Vec<T> v;
  if constexpr (kBytes == 16) v.q = __ldg(reinterpret_cast<const uint4*>(p));
  else if constexpr (kBytes == 8) { const uint2 h = __ldg(reinterpret_cast<const uint2*>(p)); v.q.x = h.x; v.q.y = h.y; }
  else if constexpr (kBytes == 4) v.q.x = __ldg(reinterpret_cast<const uint32_t*>(p));
  else v.q.x = __ldg(reinterpret_cast<const uint16_t*>(p));
  return v;
}
}  // namespace trnopt

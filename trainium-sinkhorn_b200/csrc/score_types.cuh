// Loads and stores of the score types: float32, float16 and bfloat16 are worked on in float32, float64 in float64.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

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

}  // namespace trnopt

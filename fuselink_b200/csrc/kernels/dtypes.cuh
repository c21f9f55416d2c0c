// Element types of the training operators' arrays, and how kernels read and write them.
#pragma once
#include <cuda_runtime.h>

enum FlDtype { FL_BF16 = 0, FL_FP16 = 1, FL_FP32 = 2 };

#ifdef __CUDACC__
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace fl {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// N values that are loaded and stored as one access of N * sizeof(T) bytes
template <typename T, int N>
struct alignas(N * sizeof(T)) Pack {
  T v[N];
};

}  // namespace fl

// Calls f(T{}) with the element type of `dtype`
template <typename F>
static inline int fl_by_dtype(int dtype, F&& f) {
  switch (dtype) {
    case FL_BF16: return f(__nv_bfloat16{});
    case FL_FP16: return f(__half{});
    case FL_FP32: return f(float{});
  }
  return -1;
}
#endif

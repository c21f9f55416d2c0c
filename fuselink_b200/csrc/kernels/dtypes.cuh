// Element types of the training operators' arrays, and how kernels read and write them.
#pragma once
#include <cuda_runtime.h>

enum FlDtype { FL_BF16 = 0, FL_FP16 = 1, FL_FP32 = 2 };

#ifdef __CUDACC__
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>
#include <type_traits>

namespace fl {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// N values that are loaded and stored as one access of N * sizeof(T) bytes.  As bits: of a struct of 16-bit numbers each would be an access of its own.
template <int BYTES> struct RawBits;
template <> struct RawBits<16> { using type = uint4; };
template <> struct RawBits<8> { using type = uint2; };
template <> struct RawBits<4> { using type = uint32_t; };
template <> struct RawBits<2> { using type = uint16_t; };
template <> struct RawBits<1> { using type = uint8_t; };
template <typename T, int N>
struct Pack {
  typename RawBits<N * (int)sizeof(T)>::type raw;
  __device__ __forceinline__ void get(float* f) const {
    if constexpr (sizeof(T) == 4) {
      const float* x = reinterpret_cast<const float*>(&raw);
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = x[i];
    } else if constexpr (N == 1) {
      f[0] = to_f32(*reinterpret_cast<const T*>(&raw));
    } else {
      const uint32_t* x = reinterpret_cast<const uint32_t*>(&raw);
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
          f[2 * i] = __uint_as_float(x[i] << 16);
          f[2 * i + 1] = __uint_as_float(x[i] & 0xffff0000u);
        } else {
          const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&x[i]));
          f[2 * i] = y.x;
          f[2 * i + 1] = y.y;
        }
      }
    }
  }
  __device__ __forceinline__ void set(const float* f) {
    if constexpr (sizeof(T) == 4) {
      float* x = reinterpret_cast<float*>(&raw);
#pragma unroll
      for (int i = 0; i < N; ++i) x[i] = f[i];
    } else if constexpr (N == 1) {
      *reinterpret_cast<T*>(&raw) = from_f32<T>(f[0]);
    } else {
      uint32_t* x = reinterpret_cast<uint32_t*>(&raw);
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        if constexpr (std::is_same<T, __nv_bfloat16>::value) *reinterpret_cast<__nv_bfloat162*>(&x[i]) = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
        else *reinterpret_cast<__half2*>(&x[i]) = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      }
    }
  }
};

// Two at a time, each rounded as one alone would be
struct F2 {
  unsigned long long bits;
  __device__ __forceinline__ F2() {}
  __device__ __forceinline__ F2(float x, float y) { asm("mov.b64 %0, {%1, %2};" : "=l"(bits) : "f"(x), "f"(y)); }
  __device__ __forceinline__ void get(float& x, float& y) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(bits)); }
};
__device__ __forceinline__ F2 operator*(F2 a, F2 b) { F2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits)); return r; }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) { F2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits), "l"(c.bits)); return r; }
// A sum as a one + b, where `one` is an argument of the kernel: add.rn.f32x2 of a product, and fma.rn.f32x2 with a 1 that the compiler knows, became
// one rounding with it (46 of 16384 codes were another).
__device__ __forceinline__ F2 sum2(F2 a, F2 b, F2 one) { return fma2(a, one, b); }

__device__ __forceinline__ F2 plain_sum2(F2 a, F2 b) { F2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.bits) : "l"(a.bits), "l"(b.bits)); return r; }      // where one rounding in place of two does no harm

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

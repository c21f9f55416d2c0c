// One AdamW step over many tensors, with moments in fp32 or as 8-bit codes (adamw.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>
#include "dtypes.cuh"

#ifdef __cplusplus
extern "C" {
#endif

#define FL_ADAMW_BLOCK 256                       // values of a tensor that share a scale

typedef struct {
  void* param;                                   // [n]
  const void* grad;                              // [n], of the parameter's type
  void *m, *v;                                   // [n]: fp32, or e4m3 codes of the first moment and of the second one's root
  float *m_scale, *v_scale;                      // [(n + 255) / 256] with codes
  float* master;                                 // [n] fp32 copy of the parameter that the step works on
  long long* step;                               // steps that the tensor has had, below 2^40; the call adds one
  long long n;
} FlAdamwTensor;

typedef struct {
  double lr, beta1, beta2, eps, weight_decay;
  const float* lr_on_device;                     // in place of lr, or null
  int codes;                                     // moments as codes
  int master;                                    // every tensor has an fp32 copy
  int random;                                    // codes: one of the two around a value, by place, step and seed; else the nearest, for single steps
  uint32_t seed;
} FlAdamwArgs;

// dtype: FlDtype of parameters and gradients.  -1: sizes that the kernels do not take
int fl_adamw(int dtype, const FlAdamwTensor* tensors, long long count, const FlAdamwArgs* a, cudaStream_t stream);

#ifdef __cplusplus
}
#endif

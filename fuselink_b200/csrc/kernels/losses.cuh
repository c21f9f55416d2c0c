// Log-probabilities of given tokens, a clipped policy loss over them, and the logits' gradient of both (losses.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>
#include "dtypes.cuh"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct {
  const void* logits;                        // row r = (i, j), i < outer, j < inner, begins at i * outer_stride + j * inner_stride
  long long outer, inner, outer_stride, inner_stride, vocab;
  const long long* tokens;                   // [rows]; one outside the vocabulary gives NaN
  double temperature;
  float* logprobs;                           // [rows]; 0 where the weight is 0
  float* top;                                // [rows]: the row's largest logit, for the gradient; or null
  float* inverse;                            // [rows]: 1 / sum_j exp((x_j - top) / temperature); 0 where the weight is 0; with `top`
  // policy (loss not null)
  const float* old;                          // [rows]
  const float* advantages;                   // [rows]
  const float* reference;                    // [rows] or null
  const float* weights;                      // [rows] or null; rows of weight 0 are not read
  const float* total;                        // what the sums are divided by, or null: the weights' sum
  double kl, clip_low, clip_high;
  float *loss, *divergence, *clipped;        // one value each
  float* coefficient;                        // [rows]: derivative of the loss by the row's log-probability; or null
  void* dlogits;                             // for a derivative of 1, or null.  Its rows lie dlogits_outer and dlogits_inner apart, and every one
  long long dlogits_outer, dlogits_inner;    // begins as far behind a multiple of 16 bytes as the logits' row does
  void* scratch;                             // fl_policy_scratch() bytes
  // gradient
  const float* dlogprobs;                    // [rows]
  const float* upstream;                     // a factor of all dlogprobs, or null
  int unless_one;                            // do nothing where the factor is 1
} FlLossArgs;

// dtype: FlDtype of the logits.  -1: sizes that the kernels do not take
int fl_token_logprobs(int dtype, const FlLossArgs* a, cudaStream_t stream);       // logprobs, top, inverse
int fl_policy_loss(int dtype, const FlLossArgs* a, cudaStream_t stream);
int fl_logprobs_grad(int dtype, const FlLossArgs* a, cudaStream_t stream);        // dlogits from dlogprobs, tokens, top and inverse
long long fl_policy_scratch(void);

#ifdef __cplusplus
}
#endif

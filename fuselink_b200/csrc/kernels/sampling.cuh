// The next tokens by chance, from uniform numbers that the caller gives (see sampling.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>
#include "decoder.cuh"

// What a row is drawn by: an array with an entry per row, or, where that is null, one value for all of them.
struct FlSampleArgs {
  const void* logits; long long row_stride;    // [rows] of `vocab` elements of the type, row_stride elements apart
  int rows; long long vocab;
  const double* u64; const float* u32;         // [rows], one of the two; taken as 0 below 0 or where NaN, and as the largest number below 1 from 1 on
  const float* temperature; float temperature_all;    // 0, less or NaN: the greedy choice
  const int* top_k; int top_k_all;                    // 0 or less: off
  const float* top_p; float top_p_all;                // 1, more or NaN: off
  const float* min_p; float min_p_all;                // 0, less or NaN: off
  long long* tokens;                           // [rows]
  float* logprobs;                             // [rows]: of the token among those that were left; or null
};
constexpr long long FL_SAMPLE_MAX_VOCAB = 8ll * 65528;

// Tokens in the order of their logits, largest first and of equals the lowest index first; weight exp((logit - largest) / temperature).  The first
// top_k of them stay; of these the first ones whose weights make top_p of theirs; of these those of at least min_p times the largest weight;
// always one.  The token is the first whose weight brings the sum above u times the sum of those left.  -inf is never chosen, +inf only shares
// with +inf; a row of nothing but -inf gives token 0 and logprob -inf; a row with a NaN gives the first one, as the greedy choice does, and logprob NaN.
// Returns 0, a cudaError, or < 0 for arguments it does not take (-1 type, -2 sizes); nothing is launched then.
#ifdef __cplusplus
extern "C"
#endif
int fl_sample(int dtype, const FlSampleArgs* a, cudaStream_t stream);

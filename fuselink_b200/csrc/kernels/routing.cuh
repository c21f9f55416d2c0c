// Choice of a token's experts: scores, balance bias, groups, top-k, weights; and the gradient of the logits (routing.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>
#include "dtypes.cuh"

#ifdef __cplusplus
extern "C" {
#endif

#define FL_ROUTE_MAX_EXPERTS 1024
#define FL_ROUTE_MAX_TOPK 32
#define FL_ROUTE_MAX_GROUPS 32

enum FlRouteScore { FL_ROUTE_SOFTMAX = 0, FL_ROUTE_SIGMOID = 1 };

typedef struct {
  const void* logits;            // [tokens][experts], rows `stride` apart
  long long tokens, stride;
  int experts, topk, score;      // score: FlRouteScore
  int groups, topk_groups;       // consecutive experts in equal groups; those of the best topk_groups are chosen from
  int group_best;                // a group is as good as the sum of its 1 or 2 best
  int renormalize;               // weights sum to `scale`
  float scale;
  const float* bias;             // [experts], added to the scores for the choice alone; or null: the order is the logits'
  const float* offset;           // [experts], added to the logits; or null
  float* weights;                // [tokens][topk]
  int* chosen;                   // [tokens][topk], best first, of equals the lowest first
  int* load;                     // [experts]: tokens that chose each
  float* balance;                // E / (T k) sum_e load_e mean_t p_te / sum p_t, 0 without tokens; or null
  void* scratch;                 // fl_route_scratch() bytes, or null where that is 0
  // gradient
  const float* dweights;         // [tokens][topk] or null
  const float* dbalance;         // one value or null
  void* dlogits;                 // [tokens][experts]
} FlRouteArgs;

// dtype: FlDtype of the logits.  -1: sizes that the kernels do not take
int fl_route(int dtype, const FlRouteArgs* a, cudaStream_t stream);
int fl_route_grad(int dtype, const FlRouteArgs* a, cudaStream_t stream);
long long fl_route_scratch(long long tokens, int experts);

#ifdef __cplusplus
}
#endif

// Routing to experts.
//
//   p = softmax(l) or sigmoid(l);  c = p + bias;  a group's value = sum of its one or two largest c;  the best groups;  of their experts the
//   k largest c;  weights p / sum of the chosen p, times a factor;  load: how many tokens chose each expert;
//   balance = E / (T k) sum_e load_e mean_t (p_te / sum_e p_te).
//
// Equal values go to the lowest index, and a value and its neighbour may be as close as two numbers can be: the choice is made in 64 bits, where
// two ways to compute the same number all but never order them differently.  A NaN counts as the largest.  Without a bias the order is the
// logits' own.
//
// A warp per token; a lane holds N consecutive experts.
#include "routing.cuh"
#include <math.h>
#include "../common/fl_ptx.cuh"

namespace fl {
namespace routing {

constexpr int WARPS = 8, THREADS = WARPS * 32;
constexpr unsigned ALL = 0xffffffffu;

// order of numbers as order of whole numbers: 0 is less than any, NaN more than any
__device__ __forceinline__ unsigned long long key_of(double x) {
  if (x != x) return ~0ull;
  const unsigned long long b = (unsigned long long)__double_as_longlong(x + 0.0);
  return b >> 63 ? ~b : b | (1ull << 63);
}
__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(ALL, x, o);
  return x;
}
__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(ALL, x, o);
  return x;
}

struct Parts {
  int* load;       // [ctas][experts]
  float* share;    // [ctas][experts]
};
__host__ __device__ inline int ctas_of(long long tokens) {
  const long long n = (tokens + WARPS - 1) / WARPS;
  return (int)(n < 592 ? n : 592);
}
__host__ __device__ inline Parts parts_of(void* p, long long tokens, int experts) {
  return {(int*)p, (float*)((int*)p + (long long)ctas_of(tokens) * experts)};
}

// the lane's logits, in 64 bits; what is no expert is -inf
template <int N, typename T>
__device__ __forceinline__ void load_logits(double* l, const FlRouteArgs& a, long long t) {
  const T* row = (const T*)a.logits + t * a.stride;
  const int e0 = (threadIdx.x & 31) * N;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    l[i] = -INFINITY;
    if (e0 + i < a.experts) l[i] = (double)to_f32(row[e0 + i]) + (a.offset != nullptr ? (double)a.offset[e0 + i] : 0.0);
  }
}
// scores of the lane's experts; 0 for what is none, and for a token whose logits are all -inf
template <int N>
__device__ __forceinline__ void scores(double* p, const double* l, const FlRouteArgs& a) {
  const int e0 = (threadIdx.x & 31) * N;
  if (a.score == FL_ROUTE_SIGMOID) {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = e0 + i < a.experts ? 1.0 / (1.0 + exp(-l[i])) : 0.0;
    return;
  }
  double mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < N; ++i) mx = fmax(mx, l[i]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmax(mx, __shfl_xor_sync(ALL, mx, o));
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    p[i] = e0 + i < a.experts && !(mx == -INFINITY && l[i] == -INFINITY) ? exp(l[i] - mx) : 0.0;
    sum += p[i];
  }
  sum = warp_sum(sum);
#pragma unroll
  for (int i = 0; i < N; ++i) p[i] = sum == 0.0 ? 0.0 : p[i] / sum;
}

template <int N, typename T>
__global__ void __launch_bounds__(THREADS) route_kernel(const FlRouteArgs a) {
  extern __shared__ double choice[];             // [WARPS][experts]: c, for the groups
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e0 = lane * N, E = a.experts;
  int* load = reinterpret_cast<int*>(choice + (a.groups > 1 ? WARPS * E : 0));     // [experts]
  double* share = reinterpret_cast<double*>(load + (E + 1) / 2 * 2);               // [experts], where asked for
  for (int e = threadIdx.x; e < E; e += THREADS) load[e] = 0;
  __syncthreads();
  double mean[N];
#pragma unroll
  for (int i = 0; i < N; ++i) mean[i] = 0.0;
  for (long long t = (long long)blockIdx.x * WARPS + warp; t < a.tokens; t += (long long)gridDim.x * WARPS) {
    double l[N], p[N];
    unsigned long long key[N];
    load_logits<N, T>(l, a, t);
    scores<N>(p, l, a);
    if (a.balance != nullptr) {
      double sum = 0.0;
#pragma unroll
      for (int i = 0; i < N; ++i) sum += p[i];
      sum = warp_sum(sum);
#pragma unroll
      for (int i = 0; i < N; ++i) mean[i] += sum == 0.0 ? 0.0 : p[i] / sum;
    }
    unsigned groups = ALL;
    if (a.groups > 1) {
      double* c = choice + warp * E;
      const int size = E / a.groups;
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (e0 + i < E) c[e0 + i] = a.bias != nullptr ? p[i] + (double)a.bias[e0 + i] : p[i];
      __syncwarp();
      unsigned long long value = 0;
      if (lane < a.groups) {
        double best = 0.0, second = 0.0;
        unsigned long long kb = 0, ks = 0;
        for (int j = 0; j < size; ++j) {
          const double x = c[lane * size + j];
          const unsigned long long k = key_of(x);
          if (k > kb) { ks = kb; second = best; kb = k; best = x; }
          else if (k > ks) { ks = k; second = x; }
        }
        value = key_of(a.group_best == 2 ? best + second : best);
      }
      int rank = 0;
      for (int g = 0; g < a.groups; ++g) {
        const unsigned long long other = __shfl_sync(ALL, value, g);
        rank += other > value || (other == value && g < lane);
      }
      groups = __ballot_sync(ALL, lane < a.groups && rank < a.topk_groups);
      __syncwarp();
    }
    const int size = E / a.groups;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = e0 + i;
      const bool in = e < E && (a.groups == 1 || groups >> (e / size) & 1);
      key[i] = in ? key_of(a.bias != nullptr ? p[i] + (double)a.bias[e] : l[i]) : 0;
    }
    double total = 0.0, mine = 0.0;
    int my_expert = 0;
    for (int k = 0; k < a.topk; ++k) {
      unsigned long long best = 0;
      int at = 0;
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (key[i] > best) { best = key[i]; at = i; }
      unsigned long long top = best;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long other = __shfl_xor_sync(ALL, top, o);
        top = other > top ? other : top;
      }
      const int from = __ffs(__ballot_sync(ALL, best == top)) - 1;
      double score = 0.0;
      if (lane == from) {
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (i == at) { score = p[i]; key[i] = 0; }
        atomicAdd(&load[e0 + at], 1);
      }
      score = __shfl_sync(ALL, score, from);
      const int e = __shfl_sync(ALL, e0 + at, from);
      total += score;
      if (lane == k) { mine = score; my_expert = e; }
    }
    if (lane < a.topk) {
      double w = a.renormalize ? (total == 0.0 ? 0.0 : mine / total) : mine;
      a.weights[t * a.topk + lane] = (float)(w * (double)a.scale);
      a.chosen[t * a.topk + lane] = my_expert;
    }
  }
  __syncthreads();
  const Parts parts = parts_of(a.scratch, a.tokens, E);
  for (int e = threadIdx.x; e < E; e += THREADS) parts.load[(long long)blockIdx.x * E + e] = load[e];
  if (a.balance == nullptr) return;
  for (int w = 0; w < WARPS; ++w) {
    if (warp == w)
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (e0 + i < E) share[e0 + i] = w == 0 ? mean[i] : share[e0 + i] + mean[i];
    __syncthreads();
  }
  for (int e = threadIdx.x; e < E; e += THREADS) parts.share[(long long)blockIdx.x * E + e] = (float)share[e];
}

// one warp per expert and CTA-wide sum over the experts
__global__ void __launch_bounds__(1024) route_sum_kernel(const FlRouteArgs a) {
  __shared__ double term[FL_ROUTE_MAX_EXPERTS];
  const Parts parts = parts_of(a.scratch, a.tokens, a.experts);
  const int lane = threadIdx.x & 31, ctas = ctas_of(a.tokens), E = a.experts;
  for (int e = threadIdx.x >> 5; e < E; e += 32) {
    int n = 0;
    double s = 0.0;
    for (int b = lane; b < ctas; b += 32) {
      n += parts.load[(long long)b * E + e];
      if (a.balance != nullptr) s += (double)parts.share[(long long)b * E + e];
    }
    n = __reduce_add_sync(ALL, n);
    s = warp_sum(s);
    if (lane == 0) {
      a.load[e] = n;
      term[e] = s * n;
    }
  }
  if (a.balance == nullptr) return;
  __syncthreads();
  if (threadIdx.x < 32) {
    double s = 0.0;
    for (int e = lane; e < E; e += 32) s += term[e];
    s = warp_sum(s);
    if (lane == 0) *a.balance = a.tokens == 0 ? 0.f : (float)(s * E / ((double)a.tokens * a.tokens * a.topk));
  }
}

// With u_j = w_j / scale, D = sum_j dw_j w_j and q = p / sum p:
//   renormalised   dl_j = (scale dw_j - D) u_j (1 - p_j for a sigmoid)            for the chosen j, and nothing for the others
//   as they are    dl_j = dw_j w_j (1 - p_j)   or, softmax,  dw_j w_j - p_j D (the second part for all experts)
//   balance        dl_e += q_e (b_e - sum q b) (1 - p_e for a sigmoid),  b_e = d E load_e / (T^2 k)
template <int N, typename T>
__global__ void __launch_bounds__(THREADS) route_grad_kernel(const FlRouteArgs a) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e0 = lane * N, E = a.experts;
  const bool sigmoid = a.score == FL_ROUTE_SIGMOID;
  const float each = a.dbalance != nullptr ? (float)((double)*a.dbalance * E / ((double)a.tokens * a.tokens * a.topk)) : 0.f;
  const long long t = (long long)blockIdx.x * WARPS + warp;
  if (t >= a.tokens) return;
  float p[N], d[N];
  const T* row = (const T*)a.logits + t * a.stride;
  float mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    p[i] = -INFINITY;
    if (e0 + i < E) p[i] = to_f32(row[e0 + i]) + (a.offset != nullptr ? a.offset[e0 + i] : 0.f);
    mx = fmaxf(mx, p[i]);
  }
  float sum = 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(ALL, mx, o));
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (e0 + i >= E) p[i] = 0.f;
    else if (sigmoid) p[i] = 1.f / (1.f + expf(-p[i]));
    else p[i] = mx == -INFINITY && p[i] == -INFINITY ? 0.f : expf(p[i] - mx);
    sum += p[i];
  }
  sum = warp_sum(sum);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  if (!sigmoid)
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] *= inv;
  float dot = 0.f, mine = 0.f;
  int expert = -1;
  if (a.dweights != nullptr) {
    float w = 0.f, dw = 0.f;
    if (lane < a.topk) {
      w = a.weights[t * a.topk + lane];
      dw = a.dweights[t * a.topk + lane];
      expert = a.chosen[t * a.topk + lane];
    }
    dot = warp_sum(dw * w);
    mine = a.renormalize ? (a.scale * dw - dot) * (w / a.scale) : dw * w;
    if (lane >= a.topk || (a.renormalize && w == 0.f)) mine = 0.f;
  }
  float qb = 0.f;
  if (a.dbalance != nullptr) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      d[i] = e0 + i < E ? each * (float)a.load[e0 + i] : 0.f;
      qb += (sigmoid ? p[i] * inv : p[i]) * d[i];
    }
    qb = warp_sum(qb);
  }
  const float all = a.dweights != nullptr && !a.renormalize && !sigmoid ? dot : 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) d[i] = (a.dbalance != nullptr ? (sigmoid ? p[i] * inv : p[i]) * (d[i] - qb) : 0.f) - p[i] * all;
  if (a.dweights != nullptr)
    for (int k = 0; k < a.topk; ++k) {
      const int e = __shfl_sync(ALL, expert, k);
      const float v = __shfl_sync(ALL, mine, k);
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (e0 + i == e) d[i] += v;
    }
  T* out = (T*)a.dlogits + t * E;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (e0 + i < E) out[e0 + i] = from_f32<T>(sigmoid ? d[i] * (1.f - p[i]) : d[i]);
}

template <typename F>
static int by_experts(int experts, F&& f) {
  const int n = (experts + 31) / 32;
  if (n <= 1) return f(std::integral_constant<int, 1>{});
  if (n <= 2) return f(std::integral_constant<int, 2>{});
  if (n <= 4) return f(std::integral_constant<int, 4>{});
  if (n <= 8) return f(std::integral_constant<int, 8>{});
  if (n <= 16) return f(std::integral_constant<int, 16>{});
  return f(std::integral_constant<int, 32>{});
}

static bool bad(const FlRouteArgs* a) {
  return a->tokens < 0 || a->tokens >= INT32_MAX || a->experts < 1 || a->experts > FL_ROUTE_MAX_EXPERTS || a->topk < 1 || a->topk > FL_ROUTE_MAX_TOPK ||
         a->stride < a->experts || a->groups < 1 || a->groups > FL_ROUTE_MAX_GROUPS || a->experts % a->groups != 0 || a->topk_groups < 1 || a->topk_groups > a->groups ||
         a->topk > a->experts / a->groups * a->topk_groups || a->group_best < 1 || a->group_best > 2 || a->group_best > a->experts / a->groups ||
         (a->score != FL_ROUTE_SOFTMAX && a->score != FL_ROUTE_SIGMOID);
}

}  // namespace routing
}  // namespace fl

extern "C" long long fl_route_scratch(long long tokens, int experts, int balance) {
  return (long long)fl::routing::ctas_of(tokens) * experts * (balance ? 8 : 4);
}

extern "C" int fl_route(int dtype, const FlRouteArgs* a, cudaStream_t stream) {
  using namespace fl::routing;
  if (bad(a)) return -1;
  const int ctas = ctas_of(a->tokens);
  return fl_by_dtype(dtype, [&](auto type) {
    using T = decltype(type);
    return by_experts(a->experts, [&](auto width) {
      constexpr int N = decltype(width)::value;
      const int bytes = (a->groups > 1 ? WARPS * a->experts * 8 : 0) + (a->experts + 1) / 2 * 8 + (a->balance != nullptr ? a->experts * 8 : 0);
      if (ctas > 0) {
        if (bytes > 48 * 1024) {
          const cudaError_t e = cudaFuncSetAttribute(route_kernel<N, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
          if (e != cudaSuccess) return (int)e;
        }
        route_kernel<N, T><<<ctas, THREADS, bytes, stream>>>(*a);
      }
      route_sum_kernel<<<1, 1024, 0, stream>>>(*a);
      return (int)cudaGetLastError();
    });
  });
}

extern "C" int fl_route_grad(int dtype, const FlRouteArgs* a, cudaStream_t stream) {
  using namespace fl::routing;
  if (bad(a)) return -1;
  if (a->tokens == 0) return 0;
  return fl_by_dtype(dtype, [&](auto type) {
    using T = decltype(type);
    return by_experts(a->experts, [&](auto width) {
      constexpr int N = decltype(width)::value;
      route_grad_kernel<N, T><<<(unsigned)((a->tokens + WARPS - 1) / WARPS), THREADS, 0, stream>>>(*a);
      return (int)cudaGetLastError();
    });
  });
}

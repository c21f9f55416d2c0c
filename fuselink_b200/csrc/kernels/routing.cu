// Routing to experts.
//
//   p = softmax(l) or sigmoid(l);  c = p + bias;  a group's value = sum of its one or two largest c;  the best groups;  of their experts the
//   k largest c;  weights p / sum of the chosen p, times a factor;  load: how many tokens chose each expert;
//   balance = E / (T k) sum_e load_e mean_t (p_te / sum_e p_te).
//
// Equal values go to the lowest index, and a value and its neighbour may be as close as two numbers can be: the choice is that of 64 bits, where
// two ways to compute the same number all but never order them differently.  A NaN counts as the largest.  Without a bias the order is the
// logits' own.
//
// A warp per token; a lane holds N consecutive experts.  Scores are computed in fp32, with the hardware's exponential and reciprocal, and sorted as
// whole numbers whose lowest bits say which of the lane's experts it is; the k largest come from the lanes' lists one by one.  That is the choice of 64 bits
// wherever the values that decide it lie further apart than the errors of all this (2^-18 of the largest for 256 experts), or are the same number.  Elsewhere
// the warp does the token again in 64 bits (0.3% of tokens with fp32 logits of spread 1.7 over 256 experts in 8 groups).  So it does where such a value is -inf, whose key
// without its lowest bits is no number's: biases of -inf (65536 x 256: 375 to 425 us in place of 103 to 118), and fp32 logits of -inf that fill lanes (480 in place of 98).
//
// 65536 x 256, bias and groups: 104 us forward, 900 instructions a token, which is what bounds it; 48 us backward.  All of it in 64 bits: 398 us.
#include "routing.cuh"
#include <math.h>
#include "../common/fl_ptx.cuh"

namespace fl {
namespace routing {

constexpr unsigned ALL = 0xffffffffu;
constexpr int GRAD_WARPS = 8, GRAD_CTAS = 148 * 6;
constexpr int WARPS = 8;                         // of a CTA; a launch of one CTA has up to MOST_WARPS
template <int N> constexpr int MOST_WARPS = N <= 8 ? 16 : 8;
constexpr int CTAS = 148 * 4;
constexpr double UNIT = 4294967296.0;            // 2^32: shares are added up as whole numbers of 2^-32, so that the order makes no difference

// order of numbers as order of whole numbers: 0 is less than any, NaN more than any
__device__ __forceinline__ unsigned long long key_of(double x) {
  if (x != x) return ~0ull;
  const unsigned long long b = (unsigned long long)__double_as_longlong(x + 0.0);
  return b >> 63 ? ~b : b | (1ull << 63);
}
__device__ __forceinline__ double value_of(unsigned long long k) { return __longlong_as_double((long long)(k >> 63 ? k & ~(1ull << 63) : ~k)); }      // NaN for ~0
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

struct Totals {                                  // zeroed before the launch where there are several CTAs
  unsigned long long* share;                     // [experts]
  int* load;                                     // [experts]
  int* done;
  int* nan;
};
__host__ __device__ inline Totals totals_of(void* p, int experts) {
  Totals t;
  t.share = (unsigned long long*)p;
  t.load = (int*)(t.share + experts);
  t.done = t.load + experts;
  t.nan = t.done + 1;
  return t;
}

// whether rows can be read and written N values a lane
template <int N, typename T>
__device__ __forceinline__ bool whole(const void* p, long long stride, int experts) {
  constexpr int bytes = N * (int)sizeof(T) < 16 ? N * (int)sizeof(T) : 16;
  return experts % N == 0 && (((uintptr_t)p | (uintptr_t)(stride * (long long)sizeof(T))) & (bytes - 1)) == 0;
}
// the lane's logits; what is no expert is -inf
template <int N, typename T>
__device__ __forceinline__ void load_logits(float* l, const T* row, int e0, int experts, bool wide) {
  constexpr int M = N * (int)sizeof(T) <= 16 ? N : 16 / (int)sizeof(T);
  if (wide) {
#pragma unroll
    for (int i = 0; i < N; ++i) l[i] = -INFINITY;
    if (e0 < experts)
#pragma unroll
      for (int j = 0; j < N / M; ++j) reinterpret_cast<const Pack<T, M>*>(row + e0)[j].get(l + j * M);
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) l[i] = e0 + i < experts ? to_f32(row[e0 + i]) : -INFINITY;
}

struct Chosen {                                  // of lane k < topk: the k-th choice
  int expert;
  float weight;
};

__device__ __forceinline__ double logit64(const FlRouteArgs& a, float l, int e) { return (double)l + (a.offset != nullptr ? (double)a.offset[e] : 0.0); }

// the largest of the lanes' keys, by halves
__device__ __forceinline__ unsigned long long warp_max(unsigned long long k) {
  const uint32_t hi = __reduce_max_sync(ALL, (uint32_t)(k >> 32));
  return (unsigned long long)hi << 32 | __reduce_max_sync(ALL, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
}

// A token in 64 bits.  Seldom: its loops stay loops, since what such a token costs first of all is instructions that no cache has.  room: [experts] of
// the warp's own, where groups are not whole lanes.
template <int N, typename T>
__device__ __noinline__ Chosen choose_exactly(const FlRouteArgs& a, long long t, double* room) {
  const int lane = threadIdx.x & 31, e0 = lane * N, E = a.experts, size = E / a.groups, lanes = size / N, here = min(max(E - e0, 0), N);
  const T* row = (const T*)a.logits + t * a.stride;
  const bool sigmoid = a.score == FL_ROUTE_SIGMOID, in_lanes = size % N == 0 && (lanes & (lanes - 1)) == 0;
  double top = -INFINITY, sum = 0.0, total = 0.0;
  if (!sigmoid) {
#pragma unroll 1
    for (int i = 0; i < here; ++i) top = fmax(top, logit64(a, to_f32(row[e0 + i]), e0 + i));
#pragma unroll 1
    for (int o = 16; o > 0; o >>= 1) top = fmax(top, __shfl_xor_sync(ALL, top, o));
  }
  // scores: times their sum, for a softmax; 0 for a token whose logits are all -inf.  Twice through the lane's experts, then through the chosen one.
  unsigned long long key[N];
  double mine = 0.0;
  int expert = 0;
#pragma unroll 1
  for (int pass = sigmoid ? 1 : 0; pass < 3; ++pass) {
    if (pass == 2) {
      bool whole_lane = true;
      unsigned kept = ALL;
      if (a.topk_groups < a.groups) {
        unsigned long long best = 0, second = 0;
        const int group = in_lanes ? lane / lanes : lane, n = in_lanes ? N : group < a.groups ? size : 0;
        if (!in_lanes) __syncwarp();
#pragma unroll 1
        for (int j = 0; j < n; ++j) {
          const unsigned long long k = in_lanes ? key[j] : key_of(room[lane * size + j]);
          second = max(second, min(best, k));
          best = max(best, k);
        }
#pragma unroll 1
        for (int o = 1; in_lanes && o < lanes; o *= 2) {
          const unsigned long long b = __shfl_xor_sync(ALL, best, o), s = __shfl_xor_sync(ALL, second, o);
          second = max(max(second, s), min(best, b));
          best = max(best, b);
        }
        const unsigned long long v = group < a.groups ? key_of(a.group_best == 2 ? value_of(best) + value_of(second) : value_of(best)) : 0;
        int rank = 0;
#pragma unroll 1
        for (int g = 0; g < a.groups; ++g) {
          const unsigned long long other = __shfl_sync(ALL, v, in_lanes ? g * lanes : g);
          rank += other > v || (other == v && g < group);
        }
        const bool keep = group < a.groups && rank < a.topk_groups;
        if (in_lanes) whole_lane = keep;
        else kept = __ballot_sync(ALL, keep);
      }
#pragma unroll 1
      for (int i = 0; i < N; ++i) {
        const int e = e0 + i;
        if (i >= here || !whole_lane || !(kept >> (e / size) & 1)) key[i] = 0;
        else if (a.bias == nullptr) key[i] = key_of(logit64(a, to_f32(row[e]), e));
      }
#pragma unroll 1
      for (int k = 0; k < a.topk; ++k) {
        unsigned long long best = 0;
        int at = 0;
#pragma unroll 1
        for (int i = 0; i < N; ++i)
          if (key[i] > best) { best = key[i]; at = i; }
        const int from = __ffs(__ballot_sync(ALL, best == warp_max(best))) - 1;
        if (lane == from) key[at] = 0;
        const int e = __shfl_sync(ALL, e0 + at, from);
        if (lane == k) expert = e;
      }
    }
    const int n = pass < 2 ? here : lane < a.topk;
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      const int e = pass < 2 ? e0 + i : expert;
      const double l = logit64(a, to_f32(row[e]), e);
      const bool nothing = !sigmoid && top == -INFINITY && l == -INFINITY;
      const double y = exp(sigmoid ? -l : nothing ? -INFINITY : l - top);
      if (pass == 0) {
        sum += y;
        continue;
      }
      const double p = sigmoid ? 1.0 / (1.0 + y) : sum == 0.0 ? 0.0 : y / sum, c = a.bias != nullptr ? p + (double)a.bias[e] : p;
      mine = p;
      if (pass == 1) {
        key[i] = key_of(c);
        if (!in_lanes && a.topk_groups < a.groups) room[e] = c;
      }
    }
    if (pass == 0) sum = warp_sum(sum);
    if (pass == 1)
      for (int i = here; i < N; ++i) key[i] = 0;
    __syncwarp();
  }
  if (lane >= a.topk) mine = 0.0;
  total = warp_sum(mine);
  return Chosen{expert, (float)((a.renormalize ? (total == 0.0 ? 0.0 : mine / total) : mine) * (double)a.scale)};
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t key32(float x) {      // order of numbers as order of whole numbers; 0 is less than any
  const uint32_t b = __float_as_uint(x);
  return (int)b < 0 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value32(uint32_t k) { return __uint_as_float((int)k < 0 ? k & 0x7fffffffu : ~k); }
__device__ __forceinline__ float warp_max(float x) { return value32(__reduce_max_sync(ALL, key32(x))); }

// Scores of the lane's experts from their logits, in fp32, and the sum of all
template <int N>
__device__ __forceinline__ float scores32(float* p, const float* l, bool sigmoid) {
  constexpr float LOG2E = 1.4426950408889634f;
  float sum = 0.f;
  if (sigmoid) {
#pragma unroll
    for (int i = 0; i < N; ++i) sum += p[i] = rcp(1.f + ex2(l[i] * -LOG2E));
    return warp_sum(sum);
  }
  float top = l[0];
#pragma unroll
  for (int i = 1; i < N; ++i) top = fmaxf(top, l[i]);
  top = fmaxf(warp_max(top), -3.402823466e38f);  // of -inf alone: no differences of infinities
#pragma unroll
  for (int i = 0; i < N; ++i) sum += p[i] = ex2((l[i] - top) * LOG2E);
  sum = warp_sum(sum);
  const float inv = sum == 0.f ? 0.f : rcp(sum);
#pragma unroll
  for (int i = 0; i < N; ++i) p[i] *= inv;
  return sum == 0.f ? 0.f : 1.f;
}

// The lanes' experts as lists of keys, largest first
template <int N>
__device__ __forceinline__ void sort_down(uint32_t* k) {
#pragma unroll
  for (int size = 2; size <= N; size *= 2)
#pragma unroll
    for (int step = size / 2; step > 0; step /= 2)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int j = i ^ step;
        if (j > i) {
          const uint32_t hi = max(k[i], k[j]), lo = min(k[i], k[j]);
          const bool down = (i & size) == 0 || size == N;
          k[i] = down ? hi : lo;
          k[j] = down ? lo : hi;
        }
      }
}

// What a + b, rounded to s, has lost; 0 where s is no number
__device__ __forceinline__ float lost_of(float a, float b, float s) {
  const float c = s - a;
  return fabsf(s) < INFINITY ? (a - (s - c)) + (b - c) : 0.f;
}

// Weights of the lanes' choices, in fp32 from their own logits; false where fp32 does not do: what is not finite, and scores that all but vanish.  The exponential of
// a logit with its offset is one of the sum times one of what rounding took from it, which logits of 1000 would have 6e-5 of.
template <int N, typename T>
__device__ __forceinline__ bool weights32(Chosen& c, const FlRouteArgs& a, const T* row, const float* l) {
  const int lane = threadIdx.x & 31;
  const bool is = lane < a.topk;
  float x = is ? to_f32(row[c.expert]) : -INFINITY, lost = 1.f;
  if (a.offset != nullptr && is) {
    const float o = a.offset[c.expert], s = x + o;
    lost = expf(a.score == FL_ROUTE_SIGMOID ? -lost_of(x, o, s) : lost_of(x, o, s));
    x = s;
  }
  float e = 0.f, total = 1.f;
  if (a.score == FL_ROUTE_SIGMOID) {
    if (is) e = __fdividef(1.f, 1.f + expf(-x) * lost);
  } else {
    float top = x;                               // of all: a choice by other values may leave out the largest, beside which its scores may be nothing
    if (!a.renormalize || a.bias != nullptr || a.topk_groups < a.groups)
#pragma unroll
      for (int i = 0; i < N; ++i) top = fmaxf(top, l[i]);
    top = warp_max(top);
    if (x > -INFINITY) e = expf(x - top) * lost;
    if (!a.renormalize) {
      total = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (l[i] > -INFINITY) {
          float y = expf(l[i] - top);
          if (a.offset != nullptr) y *= expf(lost_of(to_f32(row[lane * N + i]), a.offset[lane * N + i], l[i]));
          total += y;
        }
      total = warp_sum(total);
    }
  }
  if (a.renormalize) total = warp_sum(e);
  e /= total;                                    // IEEE's: the only choice of all weighs `scale` and has no gradient
  c.weight = e * a.scale;
  return __all_sync(ALL, !is || x == -INFINITY || (e >= 1e-30f && e <= 1.f)) && total > 1e-30f && total < 1e30f;
}

// Whether values that are too near to be told apart by keys are the same number: the same logit with the same bias.  expert, mine: the lanes' choices and
// their keys, `edge` the last one's; lists: the lanes' keys, the first `taken` of which are chosen.
template <int N, typename T>
__device__ __noinline__ bool near_ones_equal(const FlRouteArgs& a, const T* row, int expert, uint32_t mine, uint32_t edge, float off, const uint32_t* lists, int taken) {
  constexpr uint32_t LOW = N - 1;
  const int lane = threadIdx.x & 31;
  bool sure = a.offset == nullptr;
  const bool is = lane < a.topk;
  const float my_l = is ? to_f32(row[expert]) : 0.f, my_b = is && a.bias != nullptr ? a.bias[expert] : 0.f, my_v = value32(mine & ~LOW);
  const float next_l = __shfl_down_sync(ALL, my_l, 1), next_b = __shfl_down_sync(ALL, my_b, 1), next_v = __shfl_down_sync(ALL, my_v, 1);
  if (lane < a.topk - 1) sure = sure && (my_v - next_v > off || (my_l == next_l && my_b == next_b));
  const float edge_v = value32(edge & ~LOW), edge_l = __shfl_sync(ALL, my_l, a.topk - 1), edge_b = __shfl_sync(ALL, my_b, a.topk - 1);
  for (int i = taken; i < N; ++i) {
    const uint32_t key = lists[i * 32 + lane];
    if (key == 0u || edge_v - value32(key & ~LOW) > off) break;
    const int e = lane * N + (int)(LOW - (key & LOW));
    sure = sure && to_f32(row[e]) == edge_l && (a.bias == nullptr || a.bias[e] == edge_b);
  }
  return __all_sync(ALL, sure);
}

// FULL: 32 N experts, so that every lane has N
template <int N, bool FULL, typename T>
__global__ void __launch_bounds__(MOST_WARPS<N> * 32, N <= 8 ? 2 : 1) route_kernel(const __grid_constant__ FlRouteArgs a) {
  // [warps][N + 1][32] lists of keys, 0 at the end, or what groups go by; [experts] loads; [experts] shares; [warps][experts] doubles, where groups are not whole lanes
  extern __shared__ __align__(16) float shared[];
  __shared__ double terms[MOST_WARPS<N>];
  __shared__ int last_one;
  constexpr uint32_t LOW = N - 1;                // a key's bits that say which of the lane's experts it is
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e0 = lane * N, E = FULL ? 32 * N : a.experts, warps = blockDim.x >> 5;
  const bool sigmoid = a.score == FL_ROUTE_SIGMOID, wide = whole<N, T>(a.logits, a.stride, E), some_groups = a.topk_groups < a.groups, biased = a.bias != nullptr;
  // the order of 16-bit logits is their keys' order: these lose nothing
  const bool as_they_are = !biased && a.offset == nullptr && sizeof(T) == 2, scored = biased || some_groups || a.balance != nullptr;
  float* values = shared + warp * 32 * (N + 1);  // more than there are experts
  uint32_t* lists = reinterpret_cast<uint32_t*>(values);
  int* load = reinterpret_cast<int*>(shared + warps * 32 * (N + 1));
  float* share = shared + warps * 32 * (N + 1) + E;
  double* room = reinterpret_cast<double*>(shared + warps * 32 * (N + 1) + 2 * E);
  const int size = E / a.groups, lanes = size / N, here = min(max(E - e0, 0), N);
  const bool in_lanes = size % N == 0 && (lanes & (lanes - 1)) == 0;
  for (int e = threadIdx.x; e < E; e += blockDim.x) load[e] = 0;
  float mean[N], bias[N], most = 0.f;
  bool numbers = true;                           // no NaN among the biases
#pragma unroll
  for (int i = 0; i < N; ++i) {
    mean[i] = 0.f;
    bias[i] = i >= here ? -INFINITY : biased ? a.bias[e0 + i] : 0.f;
    if (i < here && fabsf(bias[i]) < INFINITY) most = fmaxf(most, fabsf(bias[i]));      // an infinite one is far from all others
    numbers = numbers && bias[i] == bias[i];
  }
  most = 1.f + warp_max(most);                   // no score and no sum with its bias is larger
  __syncthreads();
  const long long step = (long long)gridDim.x * warps;
  for (long long t = (long long)blockIdx.x * warps + warp; t < a.tokens; t += step) {
    const T* row = (const T*)a.logits + t * a.stride;
    float l[N], c[N];                            // c: scores, then with the bias
    load_logits<N, T>(l, row, e0, E, wide);
    if (a.offset != nullptr)
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i < here) l[i] += a.offset[e0 + i];
    bool sure = numbers;
    if (scored) {
      const float sum = scores32<N>(c, l, sigmoid);
      sure = sure && sum == sum;                 // no NaN
      if (a.balance != nullptr) {
        const float inv = sum == 0.f ? 0.f : rcp(sum);
#pragma unroll
        for (int i = 0; i < N; ++i) mean[i] = fmaf(c[i], inv, mean[i]);
      }
#pragma unroll
      for (int i = 0; i < N; ++i) c[i] += bias[i];
    }
    // A softmax's scores are off by 2^-24 of the largest logit where an offset is added in fp32, their sum by as much, and two of them differ by both
    float spread = 0.f;
    if (a.offset != nullptr && !sigmoid) {
      uint32_t bits = 0u;
#pragma unroll
      for (int i = 0; i < N; ++i) bits = max(bits, fabsf(l[i]) < INFINITY ? __float_as_uint(l[i]) & 0x7fffffffu : 0u);
      spread = __uint_as_float(__reduce_max_sync(ALL, bits)) * 2.3841858e-7f;      // 2^-22
    }
    bool whole_lane = true;                      // whether the lane's experts are in a group that stays; else `kept` says it of each group
    unsigned kept = ALL;
    if (some_groups) {
      float best = c[0], second = -INFINITY;
      int group = lane;
      if (in_lanes) {
#pragma unroll
        for (int i = 1; i < N; ++i) {
          second = fmaxf(second, fminf(best, c[i]));
          best = fmaxf(best, c[i]);
        }
        for (int o = 1; o < lanes; o *= 2) {
          const float b = __shfl_xor_sync(ALL, best, o), s = __shfl_xor_sync(ALL, second, o);
          second = fmaxf(fmaxf(second, s), fminf(best, b));
          best = fmaxf(best, b);
        }
        group = lane / lanes;
      } else {
        __syncwarp();
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (i < here) values[e0 + i] = c[i];
        __syncwarp();
        best = -INFINITY;
        if (lane < a.groups)
          for (int j = 0; j < size; ++j) {
            const float x = values[lane * size + j];
            second = fmaxf(second, fminf(best, x));
            best = fmaxf(best, x);
          }
        __syncwarp();
      }
      // as keys whose lowest 5 bits put the first of equals before the others
      const bool is = group < a.groups;
      const uint32_t value = is ? (key32(a.group_best == 2 ? best + second : best) & ~31u) | (31 - group) : 0u;
      int rank = 0;
#pragma unroll 4
      for (int g = 0; g < a.groups; ++g) rank += __shfl_sync(ALL, value, in_lanes ? g * lanes : g) > value;
      const bool keep = is && rank < a.topk_groups;
      // the worst that stays against the best that goes
      const float least = value32(~__reduce_max_sync(ALL, keep ? ~value : 0u) & ~31u), other = value32(__reduce_max_sync(ALL, keep ? 0u : value) & ~31u);
      sure = sure && least - other > most * 3.0517578e-5f + spread;         // 2^-15: 2^-17 for the bits cut off of a sum of two, half as much for scores
      if (in_lanes) whole_lane = keep;
      else kept = __ballot_sync(ALL, keep);
    }
    float far = most;
    if (!biased) {
      uint32_t bits = 0u;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        c[i] = l[i];
        bits = max(bits, __float_as_uint(l[i]) & 0x7fffffffu);
      }
      sure = sure && bits <= 0x7f800000u;
      if (!as_they_are) {
        bits = 0u;
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (l[i] > -INFINITY) bits = max(bits, __float_as_uint(l[i]) & 0x7fffffffu);
        far = __uint_as_float(__reduce_max_sync(ALL, bits));
      }
    }
    uint32_t key[N];
#pragma unroll
    for (int i = 0; i < N; ++i) key[i] = (FULL || i < here) && whole_lane ? (key32(c[i] + 0.f) & ~LOW) | (LOW - i) : 0u;
    if (some_groups && !in_lanes) {
      for (int g = 0; g < a.groups; ++g)
        if (!(kept >> g & 1)) {
          const int from = g * size - e0;
#pragma unroll
          for (int i = 0; i < N; ++i)
            if (i >= from && i < from + size) key[i] = 0u;
        }
    }
    const float off = far * ((N + 8) * 2.3841858e-7f) + (biased ? spread : 0.f);      // (N + 8) 2^-22: N 2^-23 for the bits cut off, the rest for scores and sums
    sort_down<N>(key);
    uint32_t head = key[0], behind = N > 1 ? key[N > 1] : 0u, mine = 0u, last = 0u;
#pragma unroll
    for (int i = 0; i < N; ++i) lists[i * 32 + lane] = key[i];
    lists[N * 32 + lane] = 0u;
    int from_lane = 0, taken = 0;                // of this lane's
    for (int k = 0; k < a.topk; ++k) {
      const uint32_t cut = head & ~LOW;
      last = __reduce_max_sync(ALL, cut);
      const unsigned having = __ballot_sync(ALL, cut == last);
      const int from = __ffs(having) - 1;
      const uint32_t it = __shfl_sync(ALL, head, from);
      const bool me = cut == last && (having & ((1u << lane) - 1)) == 0u;
      if (lane == k) { mine = it; from_lane = from; }
      // the one behind is there before it is asked for; the next but one is loaded by all lanes
      head = me ? behind : head;
      taken += me;
      behind = lists[min(taken + 1, N) * 32 + lane];
    }
    Chosen chosen{from_lane * N + (int)(LOW - (mine & LOW)), 0.f};
    if (!as_they_are) {
      // neighbours among the chosen further apart than `off`, and the last of them from the rest
      const uint32_t next = __shfl_down_sync(ALL, mine, 1);
      const bool clear = (lane >= a.topk - 1 || value32(mine & ~LOW) - value32(next & ~LOW) > off) && (head == 0u || value32(last) - value32(head & ~LOW) > off);
      if (!__all_sync(ALL, clear) && __all_sync(ALL, sure)) sure = near_ones_equal<N, T>(a, row, chosen.expert, mine, last, off, lists, taken);
    }
    if (!(__all_sync(ALL, sure) && weights32<N, T>(chosen, a, row, l))) chosen = choose_exactly<N, T>(a, t, room + warp * E);
    if (lane < a.topk) {
      atomicAdd(&load[chosen.expert], 1);
      a.weights[t * a.topk + lane] = chosen.weight;
      a.chosen[t * a.topk + lane] = chosen.expert;
    }
  }
  __syncthreads();
  if (a.balance != nullptr)
    for (int w = 0; w < warps; ++w) {
      if (warp == w)
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (e0 + i < E) share[e0 + i] = w == 0 ? mean[i] : share[e0 + i] + mean[i];
      __syncthreads();
    }
  const Totals all = totals_of(a.scratch, E);
  const bool several = gridDim.x > 1;
  if (several) {
    for (int e = threadIdx.x; e < E; e += blockDim.x) {
      if (load[e] != 0) atomicAdd(&all.load[e], load[e]);
      if (a.balance == nullptr) continue;
      if (share[e] == share[e]) atomicAdd(&all.share[e], (unsigned long long)((double)share[e] * UNIT));
      else atomicOr(all.nan, 1);
    }
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last_one = atomicAdd(all.done, 1) == (int)gridDim.x - 1;
    __syncthreads();
    if (!last_one) return;
    __threadfence();
  }
  double term = 0.0;
  for (int e = threadIdx.x; e < E; e += blockDim.x) {
    const int n = several ? __ldcg(&all.load[e]) : load[e];
    a.load[e] = n;
    if (a.balance != nullptr) term += (several ? (double)__ldcg(&all.share[e]) / UNIT : (double)share[e]) * n;
  }
  if (a.balance == nullptr) return;
  term = warp_sum(term);
  if (lane == 0) terms[warp] = term;
  __syncthreads();
  if (threadIdx.x == 0) {
    double s = several && __ldcg(all.nan) != 0 ? (double)NAN : 0.0;
    for (int w = 0; w < warps; ++w) s += terms[w];
    *a.balance = a.tokens == 0 ? 0.f : (float)(s * E / ((double)a.tokens * a.tokens * a.topk));
  }
}

// With u_j = w_j / scale, D = sum_j dw_j w_j and q = p / sum p:
//   renormalised   dl_j = (scale dw_j - D) u_j (1 - p_j for a sigmoid)            for the chosen j, and nothing for the others
//   as they are    dl_j = dw_j w_j (1 - p_j)   or, softmax,  dw_j w_j - p_j D (the second part for all experts)
//   balance        dl_e += q_e (b_e - sum q b) (1 - p_e for a sigmoid),  b_e = d E load_e / (T^2 k)
// A row's part for all experts is written first, the few chosen then over it.  Where there is none (a renormalised choice, no balance term) the row is not read.
template <int N, typename T>
__global__ void __launch_bounds__(GRAD_WARPS * 32) route_grad_kernel(const FlRouteArgs a) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e0 = lane * N, E = a.experts;
  const bool sigmoid = a.score == FL_ROUTE_SIGMOID, wide = whole<N, T>(a.logits, a.stride, E), wide_out = whole<N, T>(a.dlogits, E, E);
  const float each = a.dbalance != nullptr ? (float)((double)*a.dbalance * E / ((double)a.tokens * a.tokens * a.topk)) : 0.f;
  float b[N];                                    // what the balance term asks of each expert, before a token's mean of it
#pragma unroll
  for (int i = 0; i < N; ++i) b[i] = a.dbalance != nullptr && e0 + i < E ? each * (float)a.load[e0 + i] : 0.f;
  for (long long t = (long long)blockIdx.x * GRAD_WARPS + warp; t < a.tokens; t += (long long)gridDim.x * GRAD_WARPS) {
    const T* row = (const T*)a.logits + t * a.stride;
    T* out = (T*)a.dlogits + t * E;
    float w = 0.f, dw = 0.f, x = 0.f, own_load = 0.f;
    int expert = 0;
    const bool is = lane < a.topk && a.dweights != nullptr;
    if (is) {
      w = a.weights[t * a.topk + lane];
      dw = a.dweights[t * a.topk + lane];
      expert = a.chosen[t * a.topk + lane];
    }
    float p[N], l[N];
    const bool whole_row = a.dbalance != nullptr || (!a.renormalize && !sigmoid);
    if (whole_row) {
      load_logits<N, T>(l, row, e0, E, wide);
      if (a.offset != nullptr)
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (e0 + i < E) l[i] += a.offset[e0 + i];
    }
    if (is) {
      x = to_f32(row[expert]) + (a.offset != nullptr ? a.offset[expert] : 0.f);
      if (a.dbalance != nullptr) own_load = (float)a.load[expert];
    }
    const float dot = warp_sum(__fmul_rn(dw, w));      // rounded as scale dw is below: of one choice the two are the same
    float qb = 0.f, inv = 0.f, top = 0.f;
    const float all = a.dweights != nullptr && !a.renormalize && !sigmoid ? dot : 0.f;
    if (whole_row) {
      float sum = 0.f;
      if (!sigmoid) {
        top = l[0];
#pragma unroll
        for (int i = 1; i < N; ++i) top = fmaxf(top, l[i]);
        top = fmaxf(warp_max(top), -3.402823466e38f);
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        p[i] = e0 + i >= E ? 0.f : sigmoid ? rcp(1.f + ex2(l[i] * -1.4426950408889634f)) : ex2((l[i] - top) * 1.4426950408889634f);
        sum += p[i];
      }
      sum = warp_sum(sum);
      inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
      for (int i = 0; i < N; ++i) qb += p[i] * b[i];
      qb = warp_sum(qb) * inv;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float q = p[i] * inv, y = q * (b[i] - qb - all);
        l[i] = sigmoid ? y * (1.f - p[i]) : y;
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) l[i] = 0.f;
    }
    if (wide_out) {
      constexpr int M = N * (int)sizeof(T) <= 16 ? N : 16 / (int)sizeof(T);
      if (e0 < E)
#pragma unroll
        for (int j = 0; j < N / M; ++j) {
          Pack<T, M> y;
          y.set(l + j * M);
          reinterpret_cast<Pack<T, M>*>(out + e0)[j] = y;
        }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (e0 + i < E) out[e0 + i] = from_f32<T>(l[i]);
    }
    if (a.dweights == nullptr) continue;
    __syncwarp();
    if (is) {
      // the chosen ones with the library's exponential: theirs are the large values
      float y = a.renormalize ? (w == 0.f ? 0.f : (__fmul_rn(a.scale, dw) - dot) * (w / a.scale)) : dw * w;
      const float e = sigmoid ? expf(-fabsf(x)) : 0.f, r = 1.f / (1.f + e);
      const float other = sigmoid ? (x >= 0.f ? e * r : r) : 1.f, own = sigmoid ? (x >= 0.f ? r : e * r) : expf(x - top);     // 1 - p and p of a sigmoid
      if (whole_row) y += (x == -INFINITY ? 0.f : own) * inv * (each * own_load - qb - all);
      out[expert] = from_f32<T>(y * (x != x ? x : other));
    }
  }
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

extern "C" long long fl_route_scratch(long long tokens, int experts) {
  return tokens <= (experts <= 256 ? fl::routing::MOST_WARPS<8> : fl::routing::MOST_WARPS<16>) ? 0 : (long long)experts * 12 + 8;
}

extern "C" int fl_route(int dtype, const FlRouteArgs* a, cudaStream_t stream) {
  using namespace fl::routing;
  if (bad(a)) return -1;
  return fl_by_dtype(dtype, [&](auto type) {
    using T = decltype(type);
    return by_experts(a->experts, [&](auto width) {
      constexpr int N = decltype(width)::value;
      const bool one = a->tokens <= MOST_WARPS<N>;
      const int warps = one ? (a->tokens > 0 ? (int)a->tokens : 1) : WARPS;
      const long long need = (a->tokens + WARPS - 1) / WARPS;
      const unsigned ctas = one ? 1u : (unsigned)(need < CTAS ? need : CTAS);
      const int size = a->experts / a->groups, lanes = size / N;
      const bool in_lanes = size % N == 0 && (lanes & (lanes - 1)) == 0;
      const int bytes = (warps * 32 * (N + 1) + 2 * a->experts) * 4 + (a->topk_groups < a->groups && !in_lanes ? warps * a->experts * 8 : 0);
      if (ctas > 1) {
        const cudaError_t e = cudaMemsetAsync(a->scratch, 0, (size_t)fl_route_scratch(a->tokens, a->experts), stream);
        if (e != cudaSuccess) return (int)e;
      }
      auto kernel = a->experts == 32 * N ? route_kernel<N, true, T> : route_kernel<N, false, T>;
      if (bytes > 40 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e != cudaSuccess) return (int)e;
      }
      kernel<<<ctas, warps * 32, bytes, stream>>>(*a);
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
      const long long need = (a->tokens + GRAD_WARPS - 1) / GRAD_WARPS;
      route_grad_kernel<N, T><<<(unsigned)(need < GRAD_CTAS ? need : GRAD_CTAS), GRAD_WARPS * 32, 0, stream>>>(*a);
      return (int)cudaGetLastError();
    });
  });
}

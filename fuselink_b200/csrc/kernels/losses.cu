// Log-probabilities of given tokens, the clipped policy loss, and the logits' gradient.
//
//   lp = x_tok / T - ln sum_j exp(x_j / T)                              dlp / dx_j = (1[j = tok] - p_j) / T
//   L  = sum_r w_r (-min(q A, clip(q, 1 - low, 1 + high) A) + k (exp(d) - d - 1)) / sum_r w_r,   q = exp(lp - old), d = reference - lp
//   dL / dlp_r = w_r / sum w (-q A where q A is the smaller, else 0;  + k (1 - exp(d)))
//
// A row's sum runs once over its logits in fp32, with the running maximum; what follows per row is one thread's, in 64 bits.  The policy loss
// knows dL / dlp as soon as it has the row's sum, so the kernel goes over the row once more right then, out of L2, and writes the
// gradient of a derivative of 1: the logits come from memory once.  Should the derivative turn out to be another number, the gradient is computed
// anew from the logits (fl_logprobs_grad), so that it is rounded once.
#include "losses.cuh"
#include <math.h>
#include "../common/fl_ptx.cuh"

namespace fl {
namespace losses {

constexpr int THREADS = 512, WARPS = THREADS / 32;
constexpr int CTAS = 148 * 4;
constexpr unsigned ALL = 0xffffffffu;
constexpr int AHEAD = 4;                           // vectors on their way per thread

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T> constexpr int PER = 16 / (int)sizeof(T);
template <typename T>
__device__ __forceinline__ int head_of(const T* row, long long vocab) {      // values in front of the first multiple of 16 bytes
  const int n = (int)((16 - ((uintptr_t)row & 15)) & 15) / (int)sizeof(T);
  return n < vocab ? n : (int)vocab;
}

struct Running {
  float top, sum;                                  // the largest logit so far, and the sum of 2^(unit (x - top))
  __device__ __forceinline__ void raise(float to, float unit) {
    if (to > top) {
      sum *= ex2((top - to) * unit);
      top = to;
    }
  }
};
__device__ __forceinline__ void merge(Running& a, const Running& b, float unit) {
  const float top = fmaxf(a.top, b.top);
  a.sum = a.sum * ex2((a.top - top) * unit) + b.sum * ex2((b.top - top) * unit);
  a.top = top;
}

// The row's running sum, the same in all threads.  It starts from the least finite number: a row's -inf then make no difference of infinities.
template <typename T>
__device__ __forceinline__ Running sum_row(const T* row, long long vocab, float unit, Running* shared) {
  constexpr int P = PER<T>;
  Running r{-3.402823466e38f, 0.f};
  const int head = head_of(row, vocab);
  const long long packs = (vocab - head) / P;
  const uint4* v = reinterpret_cast<const uint4*>(row + head);
  for (long long i = threadIdx.x; i < packs; i += THREADS * AHEAD) {
    uint4 x[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (i + j * THREADS < packs) x[j] = ld_v4(v + i + j * THREADS);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      if (i + j * THREADS >= packs) break;
      const T* y = reinterpret_cast<const T*>(&x[j]);
      float top = to_f32(y[0]);
#pragma unroll
      for (int k = 1; k < P; ++k) top = fmaxf(top, to_f32(y[k]));
      r.raise(top, unit);
#pragma unroll
      for (int k = 0; k < P; ++k) r.sum += ex2((to_f32(y[k]) - r.top) * unit);
    }
  }
  for (long long i = threadIdx.x; i < vocab - packs * P; i += THREADS) {
    const float x = to_f32(row[i < head ? i : packs * P + i]);
    r.raise(x, unit);
    r.sum += ex2((x - r.top) * unit);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) merge(r, Running{__shfl_xor_sync(ALL, r.top, o), __shfl_xor_sync(ALL, r.sum, o)}, unit);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = r;
  __syncthreads();
  r = shared[0];
#pragma unroll
  for (int w = 1; w < WARPS; ++w) merge(r, shared[w], unit);
  return r;
}

// out_j = factor (1[j = tok] - p_j)
template <typename T>
__device__ __forceinline__ void write_row(T* out, const T* row, long long vocab, float unit, float top, float inverse, float factor, long long tok) {
  constexpr int P = PER<T>;
  const int head = head_of(row, vocab);
  const long long packs = (vocab - head) / P;
  const float share = -factor * inverse;
  const bool none = factor == 0.f;                 // then nothing is read
  for (long long i = threadIdx.x; i < packs; i += THREADS * AHEAD) {
    uint4 x[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      x[j] = make_uint4(0, 0, 0, 0);
      if (i + j * THREADS < packs && !none) x[j] = ld_v4(reinterpret_cast<const uint4*>(row + head) + i + j * THREADS);
    }
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      if (i + j * THREADS >= packs) break;
      T* y = reinterpret_cast<T*>(&x[j]);
      const long long at = head + (i + j * THREADS) * P;
#pragma unroll
      for (int k = 0; k < P; ++k) {
        float d = none ? 0.f : ex2((to_f32(y[k]) - top) * unit) * share;
        if (at + k == tok) d += factor;
        y[k] = from_f32<T>(d);
      }
      st_v4(reinterpret_cast<uint4*>(out + head) + i + j * THREADS, x[j]);
    }
  }
  for (long long i = threadIdx.x; i < vocab - packs * P; i += THREADS) {
    const long long at = i < head ? i : packs * P + i;
    float d = none ? 0.f : ex2((to_f32(row[at]) - top) * unit) * share;
    if (at == tok) d += factor;
    out[at] = from_f32<T>(d);
  }
}

__device__ __forceinline__ double block_sum(double x, double* shared) {       // in a fixed order
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(ALL, x, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = x;
  __syncthreads();
  x = shared[0];
  for (int w = 1; w < WARPS; ++w) x += shared[w];
  return x;
}

struct Sums {
  double loss, divergence, clipped;
};

template <typename T>
__global__ void __launch_bounds__(THREADS) loss_kernel(const FlLossArgs a) {
  __shared__ Running shared[WARPS];
  __shared__ double sums[WARPS];
  __shared__ float said[2];
  const float unit = (float)(1.4426950408889634 / a.temperature);
  const long long rows = a.outer * a.inner;
  double total = (double)rows;
  if (a.loss != nullptr) {
    if (a.total != nullptr) total = *a.total;
    else if (a.weights != nullptr) {
      double w = 0.0;
      for (long long r = threadIdx.x; r < rows; r += THREADS) w += a.weights[r];
      total = block_sum(w, sums);
    }
  }
  Sums mine{0.0, 0.0, 0.0};
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* row = (const T*)a.logits + r / a.inner * a.outer_stride + r % a.inner * a.inner_stride;
    T* out = (T*)a.dlogits + r / a.inner * a.dlogits_outer + r % a.inner * a.dlogits_inner;
    const double w = a.weights != nullptr ? (double)a.weights[r] : 1.0;
    if (w == 0.0) {
      if (threadIdx.x == 0) {
        a.logprobs[r] = 0.f;
        if (a.top != nullptr) { a.top[r] = 0.f; a.inverse[r] = 0.f; }
        if (a.coefficient != nullptr) a.coefficient[r] = 0.f;
      }
      if (a.dlogits != nullptr) write_row<T>(out, row, a.vocab, unit, 0.f, 0.f, 0.f, -1);
      continue;
    }
    const Running s = sum_row<T>(row, a.vocab, unit, shared);
    const long long tok = a.tokens[r];
    if (threadIdx.x == 0) {
      const bool ok = tok >= 0 && tok < a.vocab;
      const double x = ok ? (double)to_f32(row[tok]) - (double)s.top : (double)NAN;
      const double lp = x / a.temperature - log((double)s.sum);
      a.logprobs[r] = (float)lp;
      if (a.top != nullptr) { a.top[r] = s.top; a.inverse[r] = 1.f / s.sum; }
      if (a.loss != nullptr) {
        const double adv = a.advantages[r], q = exp(lp - (double)a.old[r]);
        const double held = fmin(fmax(q, 1.0 - a.clip_low), 1.0 + a.clip_high) * adv, open = q * adv;
        double term = open <= held ? -open : -held, d = open <= held ? -open : 0.0;
        if (q != q) term = d = q;
        if (open > held) mine.clipped += w;
        if (a.reference != nullptr) {
          const double gap = (double)a.reference[r] - lp, more = expm1(gap);
          const double far = more < 1e300 ? more - gap : more;
          mine.divergence += w * far;
          term += a.kl * far;
          d -= a.kl * more;
        }
        mine.loss += w * term;
        said[0] = total == 0.0 ? 0.f : (float)(d * w / total);
        if (a.coefficient != nullptr) a.coefficient[r] = said[0];
      }
    }
    if (a.dlogits != nullptr) {
      __syncthreads();
      write_row<T>(out, row, a.vocab, unit, s.top, 1.f / s.sum, (float)((double)said[0] / a.temperature), tok);
    }
  }
  if (a.loss != nullptr && threadIdx.x == 0) {
    Sums* out = (Sums*)a.scratch;
    const double inv = total == 0.0 ? 0.0 : 1.0 / total;
    out[blockIdx.x] = Sums{mine.loss * inv, mine.divergence * inv, mine.clipped * inv};
  }
}

__global__ void __launch_bounds__(32) loss_sum_kernel(const FlLossArgs a, int ctas) {
  Sums s{0.0, 0.0, 0.0};
  for (int b = threadIdx.x; b < ctas; b += 32) {
    const Sums x = ((const Sums*)a.scratch)[b];
    s.loss += x.loss;
    s.divergence += x.divergence;
    s.clipped += x.clipped;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s.loss += __shfl_xor_sync(ALL, s.loss, o);
    s.divergence += __shfl_xor_sync(ALL, s.divergence, o);
    s.clipped += __shfl_xor_sync(ALL, s.clipped, o);
  }
  if (threadIdx.x == 0) {
    *a.loss = (float)s.loss;
    *a.divergence = (float)s.divergence;
    *a.clipped = (float)s.clipped;
  }
}

template <typename T>
__global__ void __launch_bounds__(THREADS) logprobs_grad_kernel(const FlLossArgs a) {
  const float up = a.upstream != nullptr ? *a.upstream : 1.f;
  if (a.unless_one && up == 1.f) return;
  const float unit = (float)(1.4426950408889634 / a.temperature);
  const long long rows = a.outer * a.inner;
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* row = (const T*)a.logits + r / a.inner * a.outer_stride + r % a.inner * a.inner_stride;
    T* out = (T*)a.dlogits + r / a.inner * a.dlogits_outer + r % a.inner * a.dlogits_inner;
    const long long tok = a.tokens[r];
    const float inverse = a.inverse[r];
    double g = (double)a.dlogprobs[r] * (double)up / a.temperature;
    if (inverse == 0.f) g = 0.0;                   // a row of weight 0
    else if (g != 0.0 && (tok < 0 || tok >= a.vocab)) g = NAN;
    write_row<T>(out, row, a.vocab, unit, a.top[r], inverse, (float)g, tok);
  }
}

static bool bad(const FlLossArgs* a) {
  return a->outer < 0 || a->inner < 0 || a->vocab < 1 || a->vocab >= INT32_MAX || (a->outer > 0 && a->inner >= INT32_MAX / a->outer) || !(a->temperature > 0.0) ||
         !(a->temperature < INFINITY);
}
// whether the gradient's rows lie to multiples of 16 bytes as the logits' rows do
static bool apart(const FlLossArgs* a, int size) {
  return (((uintptr_t)a->dlogits - (uintptr_t)a->logits) | (uintptr_t)((a->dlogits_outer - a->outer_stride) * size) | (uintptr_t)((a->dlogits_inner - a->inner_stride) * size)) & 15;
}
static int ctas_of(const FlLossArgs* a) { return (int)(a->outer * a->inner < CTAS ? a->outer * a->inner : CTAS); }

}  // namespace losses
}  // namespace fl

extern "C" long long fl_policy_scratch(void) { return fl::losses::CTAS * (long long)sizeof(fl::losses::Sums); }

extern "C" int fl_token_logprobs(int dtype, const FlLossArgs* a, cudaStream_t stream) {
  using namespace fl::losses;
  if (bad(a) || a->loss != nullptr || a->weights != nullptr || a->dlogits != nullptr) return -1;
  const int ctas = ctas_of(a);
  if (ctas == 0) return 0;
  return fl_by_dtype(dtype, [&](auto type) {
    loss_kernel<decltype(type)><<<ctas, THREADS, 0, stream>>>(*a);
    return (int)cudaGetLastError();
  });
}

extern "C" int fl_policy_loss(int dtype, const FlLossArgs* a, cudaStream_t stream) {
  using namespace fl::losses;
  if (bad(a) || a->loss == nullptr || a->scratch == nullptr || (a->dlogits != nullptr && apart(a, dtype == FL_FP32 ? 4 : 2))) return -1;
  const int ctas = ctas_of(a);
  return fl_by_dtype(dtype, [&](auto type) {
    if (ctas > 0) loss_kernel<decltype(type)><<<ctas, THREADS, 0, stream>>>(*a);
    loss_sum_kernel<<<1, 32, 0, stream>>>(*a, ctas);
    return (int)cudaGetLastError();
  });
}

extern "C" int fl_logprobs_grad(int dtype, const FlLossArgs* a, cudaStream_t stream) {
  using namespace fl::losses;
  if (bad(a) || apart(a, dtype == FL_FP32 ? 4 : 2)) return -1;
  const int ctas = ctas_of(a);
  if (ctas == 0) return 0;
  return fl_by_dtype(dtype, [&](auto type) {
    logprobs_grad_kernel<decltype(type)><<<ctas, THREADS, 0, stream>>>(*a);
    return (int)cudaGetLastError();
  });
}

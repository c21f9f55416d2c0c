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
#include <type_traits>
#include "../common/fl_ptx.cuh"

namespace fl {
namespace losses {

constexpr int SMS = 148;
constexpr int MOST_CTAS = SMS * 4;                 // 256 threads each, or half as many of 512
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

// 16 bytes of logits as pairs, and the largest of them
template <typename T> struct Logits;
template <> struct Logits<float> {
  static constexpr uint32_t NONE = 0xff800000u;    // -inf
  static __device__ __forceinline__ F2 pair(const uint4& x, int i) { return i == 0 ? F2(__uint_as_float(x.x), __uint_as_float(x.y)) : F2(__uint_as_float(x.z), __uint_as_float(x.w)); }
  static __device__ __forceinline__ uint4 larger(const uint4& a, const uint4& b) {
    return make_uint4(__float_as_uint(fmaxf(__uint_as_float(a.x), __uint_as_float(b.x))), __float_as_uint(fmaxf(__uint_as_float(a.y), __uint_as_float(b.y))),
                      __float_as_uint(fmaxf(__uint_as_float(a.z), __uint_as_float(b.z))), __float_as_uint(fmaxf(__uint_as_float(a.w), __uint_as_float(b.w))));
  }
  static __device__ __forceinline__ float largest(const uint4& x) {
    return fmaxf(fmaxf(__uint_as_float(x.x), __uint_as_float(x.y)), fmaxf(__uint_as_float(x.z), __uint_as_float(x.w)));
  }
};
template <typename T> struct Logits16 {
  static __device__ __forceinline__ uint32_t word(const uint4& x, int i) { return i == 0 ? x.x : i == 1 ? x.y : i == 2 ? x.z : x.w; }
};
template <> struct Logits<__nv_bfloat16> : Logits16<__nv_bfloat16> {
  static constexpr uint32_t NONE = 0xff80ff80u;
  static __device__ __forceinline__ F2 pair(const uint4& x, int i) { return F2(__uint_as_float(word(x, i) << 16), __uint_as_float(word(x, i) & 0xffff0000u)); }
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hmax2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ uint4 larger(const uint4& a, const uint4& b) { return make_uint4(larger(a.x, b.x), larger(a.y, b.y), larger(a.z, b.z), larger(a.w, b.w)); }
  static __device__ __forceinline__ float largest(const uint4& x) {
    const uint32_t m = larger(larger(x.x, x.y), larger(x.z, x.w));
    return fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
  }
};
template <> struct Logits<__half> : Logits16<__half> {
  static constexpr uint32_t NONE = 0xfc00fc00u;
  static __device__ __forceinline__ F2 pair(const uint4& x, int i) {
    const uint32_t w = word(x, i);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    return F2(f.x, f.y);
  }
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    const __half2 r = __hmax2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ uint4 larger(const uint4& a, const uint4& b) { return make_uint4(larger(a.x, b.x), larger(a.y, b.y), larger(a.z, b.z), larger(a.w, b.w)); }
  static __device__ __forceinline__ float largest(const uint4& x) {
    const uint32_t m = larger(larger(x.x, x.y), larger(x.z, x.w));
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&m));
    return fmaxf(f.x, f.y);
  }
};

struct Running {
  float top, sum;                                  // the largest logit so far, and the sum of 2^(unit (x - top))
};
__device__ __forceinline__ void merge(Running& a, const Running& b, float unit) {
  const float top = fmaxf(a.top, b.top);
  a.sum = a.sum * ex2((a.top - top) * unit) + b.sum * ex2((b.top - top) * unit);
  a.top = top;
}
// 2^(unit (x - top)) of both
__device__ __forceinline__ F2 powers(F2 x, F2 minus_top, F2 unit) {
  float a, b;
  (plain_sum2(x, minus_top) * unit).get(a, b);
  return F2(ex2(a), ex2(b));
}

// The row's running sum, the same in all threads.  It starts from the least finite number: a row's -inf then make no difference of infinities.
template <typename T, int THREADS>
__device__ __forceinline__ Running sum_row(const T* row, long long vocab, float unit, Running* shared) {
  constexpr int P = PER<T>;
  const int head = head_of(row, vocab);
  const int packs = (int)((vocab - head) / P);
  const uint4* v = reinterpret_cast<const uint4*>(row + head);
  const F2 unit2(unit, unit);
  float top = -3.402823466e38f;
  F2 sum(0.f, 0.f);
  for (int i = threadIdx.x; i < packs; i += THREADS * AHEAD) {
    uint4 x[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      constexpr uint32_t none = Logits<T>::NONE;
      x[j] = make_uint4(none, none, none, none);
      if (i + j * THREADS < packs) x[j] = ld_stream_v4(v + i + j * THREADS);
    }
    const float to = Logits<T>::largest(Logits<T>::larger(Logits<T>::larger(x[0], x[1]), Logits<T>::larger(x[2], x[3])));
    if (to > top) {
      const float fall = ex2((top - to) * unit);
      sum = sum * F2(fall, fall);
      top = to;
    }
    const F2 minus(-top, -top);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
#pragma unroll
      for (int k = 0; k < P / 2; ++k) sum = plain_sum2(sum, powers(Logits<T>::pair(x[j], k), minus, unit2));
  }
  float one, other;
  sum.get(one, other);
  Running r{top, one + other};
  for (long long i = threadIdx.x; i < vocab - (long long)packs * P; i += THREADS) {
    const float x = to_f32(row[i < head ? i : (long long)packs * P + i]), to = fmaxf(x, r.top);
    r.sum = r.sum * ex2((r.top - to) * unit) + ex2((x - to) * unit);
    r.top = to;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) merge(r, Running{__shfl_xor_sync(ALL, r.top, o), __shfl_xor_sync(ALL, r.sum, o)}, unit);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = r;
  __syncthreads();
  r = shared[0];
#pragma unroll
  for (int w = 1; w < THREADS / 32; ++w) merge(r, shared[w], unit);
  return r;
}

// out_j = factor (1[j = tok] - p_j).  The row is read from L2 for the most part, and what is written not kept there.
template <typename T, int THREADS>
__device__ __forceinline__ void write_row(T* out, const T* row, long long vocab, float unit, float top, float inverse, float factor, long long tok) {
  constexpr int P = PER<T>;
  const int head = head_of(row, vocab);
  const int packs = (int)((vocab - head) / P);
  const uint4* v = reinterpret_cast<const uint4*>(row + head);
  uint4* to = reinterpret_cast<uint4*>(out + head);
  const float share = -factor * inverse;
  if (factor == 0.f) {                             // nothing is read
    for (int i = threadIdx.x; i < packs; i += THREADS) st_cs_v4(to + i, make_uint4(0, 0, 0, 0));
    for (long long i = threadIdx.x; i < vocab - (long long)packs * P; i += THREADS) out[i < head ? i : (long long)packs * P + i] = from_f32<T>(0.f);
    return;
  }
  const F2 unit2(unit, unit), minus(-top, -top), share2(share, share);
  for (int i = threadIdx.x; i < packs; i += THREADS * AHEAD) {
    uint4 x[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (i + j * THREADS < packs) x[j] = ld_stream_v4(v + i + j * THREADS);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      if (i + j * THREADS >= packs) break;
      float f[P];
#pragma unroll
      for (int k = 0; k < P / 2; ++k) (powers(Logits<T>::pair(x[j], k), minus, unit2) * share2).get(f[2 * k], f[2 * k + 1]);
      Pack<T, P> y;
      y.set(f);
      st_cs_v4(to + i + j * THREADS, y.raw);
    }
  }
  for (long long i = threadIdx.x; i < vocab - (long long)packs * P; i += THREADS) {
    const long long at = i < head ? i : (long long)packs * P + i;
    out[at] = from_f32<T>(ex2((to_f32(row[at]) - top) * unit) * share);
  }
  // the token's own value, by the thread that has written it already
  if (tok >= 0 && tok < vocab) {
    const long long in = tok - head;
    const int owner = in < 0 ? (int)tok : in < (long long)packs * P ? (int)(in / P % THREADS) : (int)((tok - (long long)packs * P) % THREADS);
    if ((int)threadIdx.x == owner) out[tok] = from_f32<T>(fmaf(ex2((to_f32(row[tok]) - top) * unit), share, factor));
  }
}

template <int THREADS>
__device__ __forceinline__ double block_sum(double x, double* shared) {       // in a fixed order
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(ALL, x, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = x;
  __syncthreads();
  x = shared[0];
  for (int w = 1; w < THREADS / 32; ++w) x += shared[w];
  return x;
}

struct Sums {
  double loss, divergence, clipped;
};

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) loss_kernel(const FlLossArgs a) {
  __shared__ Running shared[THREADS / 32];
  __shared__ double sums[THREADS / 32];
  __shared__ float said[2];
  const float unit = (float)(1.4426950408889634 / a.temperature);
  const long long rows = a.outer * a.inner;
  double total = (double)rows;
  if (a.loss != nullptr) {
    if (a.total != nullptr) total = *a.total;
    else if (a.weights != nullptr) {
      double w = 0.0;
      for (long long r = threadIdx.x; r < rows; r += THREADS) w += a.weights[r];
      total = block_sum<THREADS>(w, sums);
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
      if (a.dlogits != nullptr) write_row<T, THREADS>(out, row, a.vocab, unit, 0.f, 0.f, 0.f, -1);
      continue;
    }
    const Running s = sum_row<T, THREADS>(row, a.vocab, unit, shared);
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
      write_row<T, THREADS>(out, row, a.vocab, unit, s.top, 1.f / s.sum, (float)((double)said[0] / a.temperature), tok);
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

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) logprobs_grad_kernel(const FlLossArgs a) {
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
    write_row<T, THREADS>(out, row, a.vocab, unit, a.top[r], inverse, (float)g, tok);
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
// Calls f(threads, CTAs).  256 threads a row, four rows an SM, where all rows that are in work stay in L2 until they are read again; 512, two rows an SM,
// where they would not, and where rows are so few that an SM has no more.
template <typename F>
static int by_rows(const FlLossArgs* a, int size, F&& f) {
  const long long rows = a->outer * a->inner;
  const bool wide = a->vocab * size > 96 * 1024 || rows <= 2 * SMS;
  const long long most = wide ? MOST_CTAS / 2 : MOST_CTAS;
  const int ctas = (int)(rows < most ? rows : most);
  return wide ? f(std::integral_constant<int, 512>{}, ctas) : f(std::integral_constant<int, 256>{}, ctas);
}

}  // namespace losses
}  // namespace fl

extern "C" long long fl_policy_scratch(void) { return fl::losses::MOST_CTAS * (long long)sizeof(fl::losses::Sums); }

extern "C" int fl_token_logprobs(int dtype, const FlLossArgs* a, cudaStream_t stream) {
  using namespace fl::losses;
  if (bad(a) || a->loss != nullptr || a->weights != nullptr || a->dlogits != nullptr) return -1;
  if (a->outer * a->inner == 0) return 0;
  return fl_by_dtype(dtype, [&](auto type) {
    using T = decltype(type);
    return by_rows(a, sizeof(T), [&](auto threads, int ctas) {
      constexpr int N = decltype(threads)::value;
      loss_kernel<T, N><<<ctas, N, 0, stream>>>(*a);
      return (int)cudaGetLastError();
    });
  });
}

extern "C" int fl_policy_loss(int dtype, const FlLossArgs* a, cudaStream_t stream) {
  using namespace fl::losses;
  if (bad(a) || a->loss == nullptr || a->scratch == nullptr || (a->dlogits != nullptr && apart(a, dtype == FL_FP32 ? 4 : 2))) return -1;
  return fl_by_dtype(dtype, [&](auto type) {
    using T = decltype(type);
    return by_rows(a, sizeof(T), [&](auto threads, int ctas) {
      constexpr int N = decltype(threads)::value;
      if (ctas > 0) loss_kernel<T, N><<<ctas, N, 0, stream>>>(*a);
      loss_sum_kernel<<<1, 32, 0, stream>>>(*a, ctas);
      return (int)cudaGetLastError();
    });
  });
}

extern "C" int fl_logprobs_grad(int dtype, const FlLossArgs* a, cudaStream_t stream) {
  using namespace fl::losses;
  if (bad(a) || apart(a, dtype == FL_FP32 ? 4 : 2)) return -1;
  if (a->outer * a->inner == 0) return 0;
  return fl_by_dtype(dtype, [&](auto type) {
    using T = decltype(type);
    return by_rows(a, sizeof(T), [&](auto threads, int ctas) {
      constexpr int N = decltype(threads)::value;
      logprobs_grad_kernel<T, N><<<ctas, N, 0, stream>>>(*a);
      return (int)cudaGetLastError();
    });
  });
}

// Log-probabilities of given tokens, the clipped policy loss, and the logits' gradient.
//
//   lp = x_tok / T - ln sum_j exp(x_j / T)                              dlp / dx_j = (1[j = tok] - p_j) / T
//   L  = sum_r w_r (-min(q A, clip(q, 1 - low, 1 + high) A) + k (exp(d) - d - 1)) / sum_r w_r,   q = exp(lp - old), d = reference - lp
//   dL / dlp_r = w_r / sum w (-q A where q A is the smaller, else 0;  + k (1 - exp(d)))
//
// A row's sum runs once over its logits in fp32, with the running maximum; what follows per row is one thread's, in 64 bits.  The policy loss
// knows dL / dlp as soon as it has the row's sum, so the kernel goes over the row once more right then, out of the caches as far as they go, and writes the
// gradient of a derivative of 1.  Should the derivative turn out to be another number, the gradient is computed
// anew from the logits (fl_logprobs_grad), so that it is rounded once.
//
// 8192 x 32000 bf16 with the gradient: 208 us, 0.70 of the measured copy rate; 4095 x 128256: 443 us.  Bound by exponentials (two a logit, 16 a cycle and SM: 56% of what the
// pipe could) and by what a row's two passes wait for one another.  Without the gradient 0.65 and 0.8.
#include "losses.cuh"
#include <math.h>
#include <type_traits>
#include "../common/fl_ptx.cuh"

namespace fl {
namespace losses {

constexpr int SMS = 148;
constexpr int MOST_CTAS = SMS * 32;
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

// 16 bytes of logits as fp32, and the largest of them
template <typename T> struct Logits;
template <> struct Logits<float> {
  static constexpr uint32_t NONE = 0xff800000u;    // -inf
  static __device__ __forceinline__ uint4 larger(const uint4& a, const uint4& b) {
    return make_uint4(__float_as_uint(fmaxf(__uint_as_float(a.x), __uint_as_float(b.x))), __float_as_uint(fmaxf(__uint_as_float(a.y), __uint_as_float(b.y))),
                      __float_as_uint(fmaxf(__uint_as_float(a.z), __uint_as_float(b.z))), __float_as_uint(fmaxf(__uint_as_float(a.w), __uint_as_float(b.w))));
  }
  static __device__ __forceinline__ float largest(const uint4& x) {
    return fmaxf(fmaxf(__uint_as_float(x.x), __uint_as_float(x.y)), fmaxf(__uint_as_float(x.z), __uint_as_float(x.w)));
  }
};
template <> struct Logits<__nv_bfloat16> {
  static constexpr uint32_t NONE = 0xff80ff80u;
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
template <> struct Logits<__half> {
  static constexpr uint32_t NONE = 0xfc00fc00u;
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
// log2(e) / temperature, not 0: -inf times it stays -inf
__device__ __forceinline__ float unit_of(double temperature) { return fmaxf((float)(1.4426950408889634 / temperature), 1.4e-45f); }
__device__ __forceinline__ float below(float x, float top, float unit) { return (0.5f * x - 0.5f * top) * (2.f * unit); }      // unit (x - top), of any two numbers
__device__ __forceinline__ Running merge(const Running& a, const Running& b, float unit) {
  const float top = fmaxf(a.top, b.top);
  return {top, a.sum * ex2(below(a.top, top, unit)) + b.sum * ex2(below(b.top, top, unit))};
}
// Exponents are unit x - base, one instruction for two, with base = unit top rounded.  While a row is summed, threads joined and maxima rise, sums are ones of 2^(unit x - base),
// which fall by the difference of two bases; the rounding's error comes in once, behind all that.  Where base is so large that it would matter (logits beyond `far`: 5.8e6
// times the temperature) exponents are taken one by one, as unit (x - top).
constexpr float LARGE = 8388608.f;                 // of a base; the error is 1/4 at most, of a thread without a value 1/2
__device__ __forceinline__ float far_of(double temperature) { return fminf((float)temperature * (0.69314718f * LARGE), 3.402823466e38f); }
__device__ __forceinline__ bool is_far(float top, float far) { return !(fabsf(top) < far); }
__device__ __forceinline__ Running merge_based(const Running& a, const Running& b, float unit) {
  const float top = fmaxf(a.top, b.top), base = __fmul_rn(top, unit);
  return {top, a.sum * ex2(__fmul_rn(a.top, unit) - base) + b.sum * ex2(__fmul_rn(b.top, unit) - base)};
}
__device__ __forceinline__ F2 powers(float x, float y, F2 unit, F2 minus) {
  float a, b;
  fma2(F2(x, y), unit, minus).get(a, b);
  return F2(ex2(a), ex2(b));
}

// The sum of a row of far logits.  Seldom: its loops stay loops.
template <typename T, int THREADS>
__device__ __forceinline__ Running sum_far_row(const T* row, long long vocab, float unit, Running* shared) {
  Running r{-3.402823466e38f, 0.f};
  for (long long i = threadIdx.x; i < vocab; i += THREADS) {
    const float x = to_f32(row[i]), to = fmaxf(x, r.top);
    r.sum = r.sum * ex2(below(r.top, to, unit)) + ex2(below(x, to, unit));
    r.top = to;
  }
#pragma unroll 1
  for (int o = 16; o > 0; o >>= 1) r = merge(r, Running{__shfl_xor_sync(ALL, r.top, o), __shfl_xor_sync(ALL, r.sum, o)}, unit);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = r;
  __syncthreads();
  r = shared[0];
#pragma unroll 1
  for (int w = 1; w < THREADS / 32; ++w) r = merge(r, shared[w], unit);
  return r;
}

// The row's running sum, the same in all threads.  It starts from a finite number: a row's -inf then make no difference of infinities, and a thread without a value
// has a sum of 0.
template <typename T, int THREADS>
__device__ __forceinline__ Running sum_row(const T* row, long long vocab, float unit, float far, Running* shared) {
  constexpr int P = PER<T>;
  const int head = head_of(row, vocab);
  const int packs = (int)((vocab - head) / P);
  const uint4* v = reinterpret_cast<const uint4*>(row + head);
  float top = -far;
  F2 sum(0.f, 0.f);
  const F2 unit2(unit, unit);
  for (int i = threadIdx.x; i < packs; i += THREADS * AHEAD) {
    uint4 x[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      constexpr uint32_t none = Logits<T>::NONE;
      x[j] = make_uint4(none, none, none, none);
      if (i + j * THREADS < packs) x[j] = ld_v4(v + i + j * THREADS);
    }
    const float to = Logits<T>::largest(Logits<T>::larger(Logits<T>::larger(x[0], x[1]), Logits<T>::larger(x[2], x[3])));
    if (to > top) {                                // the terms' new base is a rounded one too: they fall by the bases' difference, not by the logits'
      const float fall = ex2(__fmul_rn(top, unit) - __fmul_rn(to, unit));
      sum = sum * F2(fall, fall);
      top = to;
    }
    const float base = -__fmul_rn(top, unit);
    const F2 minus(base, base);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      float f[P];
      Pack<T, P>{x[j]}.get(f);
#pragma unroll
      for (int k = 0; k < P; k += 2) sum = plain_sum2(sum, powers(f[k], f[k + 1], unit2, minus));
    }
  }
  float one, other;
  sum.get(one, other);
  Running r{top, one + other};
  for (long long i = threadIdx.x; i < vocab - (long long)packs * P; i += THREADS) {
    const float x = to_f32(row[i < head ? i : (long long)packs * P + i]), to = fmaxf(x, r.top), higher = __fmul_rn(to, unit);
    r.sum = r.sum * ex2(__fmul_rn(r.top, unit) - higher) + ex2(fmaf(x, unit, -higher));
    r.top = to;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) r = merge_based(r, Running{__shfl_xor_sync(ALL, r.top, o), __shfl_xor_sync(ALL, r.sum, o)}, unit);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = r;
  __syncthreads();
  r = shared[0];
#pragma unroll
  for (int w = 1; w < THREADS / 32; ++w) r = merge_based(r, shared[w], unit);
  if (is_far(r.top, far)) return sum_far_row<T, THREADS>(row, vocab, unit, shared);      // or nothing above -far
  r.sum *= ex2(-fmaf(r.top, unit, -__fmul_rn(r.top, unit)));       // without the base's rounding
  return r;
}

// out_j = factor (1[j = tok] - p_j), from the row's end to its beginning: what was read last is in L1 and L2 still (of rows of 128256 bf16, 600 in work, L2 had
// lost 85% when they were read from the beginning again).  What is written is not kept.  inverse: 1 / sum_j 2^(unit (x_j - top))
template <typename T, int THREADS>
__device__ __forceinline__ void write_row(T* out, const T* row, long long vocab, float unit, float far, float top, float inverse, float factor, long long tok) {
  constexpr int P = PER<T>;
  const int head = head_of(row, vocab);
  const int packs = is_far(top, far) && factor != 0.f ? 0 : (int)((vocab - head) / P);
  const uint4* v = reinterpret_cast<const uint4*>(row + head);
  uint4* to = reinterpret_cast<uint4*>(out + head);
  if (factor == 0.f) {                             // nothing is read
    for (int i = threadIdx.x; i < packs; i += THREADS) st_cs_v4(to + i, make_uint4(0, 0, 0, 0));
    for (long long i = threadIdx.x; i < vocab - (long long)packs * P; i += THREADS) out[i < head ? i : (long long)packs * P + i] = from_f32<T>(0.f);
    return;
  }
  const float base = -(top * unit), share = -factor * inverse, fine = share * ex2(-fmaf(top, unit, base));      // the latter without the base's rounding
  const F2 unit2(unit, unit), minus(base, base), fine2(fine, fine);
  for (int i = (packs - 1) / (THREADS * AHEAD) * (THREADS * AHEAD) + (int)threadIdx.x; i >= 0; i -= THREADS * AHEAD) {
    uint4 x[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (i + j * THREADS < packs) x[j] = ld_v4(v + i + j * THREADS);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) {
      if (i + j * THREADS >= packs) break;
      float f[P];
      Pack<T, P>{x[j]}.get(f);
#pragma unroll
      for (int k = 0; k < P; k += 2) (powers(f[k], f[k + 1], unit2, minus) * fine2).get(f[k], f[k + 1]);
      Pack<T, P> y;
      y.set(f);
      st_cs_v4(to + i + j * THREADS, *reinterpret_cast<const uint4*>(&y.raw));
    }
  }
  for (long long i = threadIdx.x; i < vocab - (long long)packs * P; i += THREADS) {
    const long long j = i < head ? i : (long long)packs * P + i;
    out[j] = from_f32<T>(ex2(below(to_f32(row[j]), top, unit)) * share);
  }
  // the token's own value, by the thread that has written it already
  if (tok >= 0 && tok < vocab) {
    const long long in = tok - head;
    const int owner = in < 0 ? (int)tok : in < (long long)packs * P ? (int)(in / P % THREADS) : (int)((tok - (long long)packs * P) % THREADS);
    if ((int)threadIdx.x == owner) out[tok] = from_f32<T>(fmaf(ex2(below(to_f32(row[tok]), top, unit)), share, factor));
  }
}

struct Sums {
  double loss, divergence, clipped;
};
struct Scratch {
  double* total;                                   // the weights' sum
  Sums* sums;                                      // [CTAs]
};
__host__ __device__ inline Scratch scratch_of(void* p) { return {(double*)p, (Sums*)((char*)p + 256)}; }

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

__global__ void __launch_bounds__(1024) weights_kernel(const FlLossArgs a) {
  __shared__ double sums[32];
  grid_dep_launch();
  const long long rows = a.outer * a.inner;
  double w = 0.0;
#pragma unroll 8
  for (long long r = threadIdx.x; r < rows; r += 1024) w += a.weights[r];
  w = block_sum<1024>(w, sums);
  if (threadIdx.x == 0) *scratch_of(a.scratch).total = w;
}

// What one row adds to the loss, and the derivative of that by its log-probability; without the weight.  In 64 bits as far as numbers are taken from one another.
struct Term {
  double loss, divergence, slope;
  bool clipped;
};
__device__ __forceinline__ Term term_of(const FlLossArgs& a, double lp, float old, float advantage, float reference) {
  Term t{0.0, 0.0, 0.0, false};
  const float q = expf((float)(lp - (double)old)), A = advantage;
  const float held = fminf(fmaxf(q, (float)(1.0 - a.clip_low)), (float)(1.0 + a.clip_high)) * A, open = q * A;
  t.loss = open <= held ? -open : -held;
  t.slope = open <= held ? -open : 0.f;
  if (q != q) t.loss = t.slope = q;
  t.clipped = open > held;
  if (a.reference != nullptr) {
    const double gap = (double)reference - lp, more = expm1(gap);
    t.divergence = more < 1e300 ? more - gap : more;
    t.loss += a.kl * t.divergence;
    t.slope -= a.kl * more;
  }
  return t;
}

template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) loss_kernel(const FlLossArgs a) {
  __shared__ Running shared[THREADS / 32];
  __shared__ float said;
  const float unit = unit_of(a.temperature), far = far_of(a.temperature);
  const long long rows = a.outer * a.inner;
  const bool policy = a.loss != nullptr;
  double total = (double)rows;
  bool asked = false;
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
      if (a.dlogits != nullptr) write_row<T, THREADS>(out, row, a.vocab, unit, far, 0.f, 0.f, 0.f, -1);
      continue;
    }
    // asked for before the row, used behind it
    const long long tok = a.tokens[r];
    float old = 0.f, advantage = 0.f, reference = 0.f;
    if (threadIdx.x == 0 && policy) {
      old = a.old[r];
      advantage = a.advantages[r];
      if (a.reference != nullptr) reference = a.reference[r];
    }
    const Running s = sum_row<T, THREADS>(row, a.vocab, unit, far, shared);
    if (threadIdx.x == 0) {
      const bool ok = tok >= 0 && tok < a.vocab;
      const double x = ok ? (double)to_f32(row[tok]) - (double)s.top : (double)NAN;
      const double lp = x / a.temperature - log((double)s.sum);
      a.logprobs[r] = (float)lp;
      if (a.top != nullptr) { a.top[r] = s.top; a.inverse[r] = 1.f / s.sum; }
      if (policy) {
        const Term t = term_of(a, lp, old, advantage, reference);
        if (!asked) {
          asked = true;
          grid_dep_wait();                         // the weights' sum
          if (a.total != nullptr) total = *a.total;
          else if (a.weights != nullptr) total = *scratch_of(a.scratch).total;
          total = total == 0.0 ? 0.0 : 1.0 / total;
        }
        mine.loss += w * t.loss;
        mine.divergence += w * t.divergence;
        if (t.clipped) mine.clipped += w;
        said = total == 0.0 ? 0.f : (float)(t.slope * (w * total));
        if (a.coefficient != nullptr) a.coefficient[r] = said;
      }
    }
    if (a.dlogits != nullptr) {
      __syncthreads();
      write_row<T, THREADS>(out, row, a.vocab, unit, far, s.top, 1.f / s.sum, (float)((double)said / a.temperature), tok);
    }
  }
  if (policy && threadIdx.x == 0) {
    if (!asked) grid_dep_wait();                   // rows of weight 0 alone: whoever is done behind this launch knows the one in front to be done too
    scratch_of(a.scratch).sums[blockIdx.x] = asked ? Sums{mine.loss * total, mine.divergence * total, mine.clipped * total} : mine;
  }
}

__global__ void __launch_bounds__(256) loss_sum_kernel(const FlLossArgs a, int ctas) {
  __shared__ double sums[8];
  const Sums* parts = scratch_of(a.scratch).sums;
  Sums s{0.0, 0.0, 0.0};
#pragma unroll 4
  for (int b = threadIdx.x; b < ctas; b += 256) {
    s.loss += parts[b].loss;
    s.divergence += parts[b].divergence;
    s.clipped += parts[b].clipped;
  }
  s.loss = block_sum<256>(s.loss, sums);
  s.divergence = block_sum<256>(s.divergence, sums);
  s.clipped = block_sum<256>(s.clipped, sums);
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
  const float unit = unit_of(a.temperature), far = far_of(a.temperature);
  const long long rows = a.outer * a.inner;
  for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
    const T* row = (const T*)a.logits + r / a.inner * a.outer_stride + r % a.inner * a.inner_stride;
    T* out = (T*)a.dlogits + r / a.inner * a.dlogits_outer + r % a.inner * a.dlogits_inner;
    const long long tok = a.tokens[r];
    const float inverse = a.inverse[r];
    double g = (double)a.dlogprobs[r] * (double)up / a.temperature;
    if (inverse == 0.f) g = 0.0;                   // a row of weight 0
    else if (g != 0.0 && (tok < 0 || tok >= a.vocab)) g = NAN;
    write_row<T, THREADS>(out, row, a.vocab, unit, far, a.top[r], inverse, (float)g, tok);
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
// Calls f(threads, CTAs).  Short rows are a warp's or 128 threads' (32768 rows of 1000 bf16: 115 us with the gradient, 259 with 256 threads a row); others 256 threads',
// four an SM, whatever their length (1024 x 128256, two of 512: 15% slower); 512 where rows are so few that an SM has no more than two.
template <typename F>
static int by_rows(const FlLossArgs* a, int size, F&& f) {
  const long long rows = a->outer * a->inner, bytes = a->vocab * size;
  const int threads = bytes <= 8 * 1024 && rows > SMS * 8 ? 32 : bytes <= 24 * 1024 && rows > SMS * 4 ? 128 : rows > SMS * 2 ? 256 : 512;
  const long long most = SMS * (1024 / threads);
  const int ctas = (int)(rows < most ? rows : most);
  switch (threads) {
    case 32: return f(std::integral_constant<int, 32>{}, ctas);
    case 128: return f(std::integral_constant<int, 128>{}, ctas);
    case 256: return f(std::integral_constant<int, 256>{}, ctas);
    default: return f(std::integral_constant<int, 512>{}, ctas);
  }
}

}  // namespace losses
}  // namespace fl

extern "C" long long fl_policy_scratch(void) { return 256 + fl::losses::MOST_CTAS * (long long)sizeof(fl::losses::Sums); }

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
      if (ctas > 0) {
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[0].val.programmaticStreamSerializationAllowed = 1;
        cudaLaunchConfig_t c = {};
        c.gridDim = dim3(ctas); c.blockDim = dim3(N); c.stream = stream; c.attrs = at;
        if (a->weights != nullptr && a->total == nullptr) {
          weights_kernel<<<1, 1024, 0, stream>>>(*a);
          c.numAttrs = 1;                          // the rows begin beside that; what came before is behind both
        }
        cudaError_t e = cudaSuccess;
        // the ends of rows are read again out of L1 (8192 x 32000: 241 us without this, 231 with it; warps of their own have no use for it and want their CTAs' share)
        if (N == 256) e = cudaFuncSetAttribute(loss_kernel<T, N>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxL1);
        if (e == cudaSuccess) e = cudaLaunchKernelEx(&c, loss_kernel<T, N>, *a);
        if (e != cudaSuccess) return (int)e;
      }
      loss_sum_kernel<<<1, 256, 0, stream>>>(*a, ctas);
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

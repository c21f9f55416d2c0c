// AdamW over many tensors.
//
//   m = b1 m + (1 - b1) g      v = b2 v + (1 - b2) g^2      w = w (1 - lr decay) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Moments are kept in fp32, or as e4m3 codes of m and of sqrt(v) with a scale for each 256 values of a tensor: the smallest power of two,
// 2^-100 at least, that keeps their largest finite magnitude within 448.  The root halves the range that a code has to span, and a root above 0 keeps
// the smallest code at least: were it lost while m is not, the next steps would divide by eps.  Values that are not finite are kept
// as NaN.  The step itself uses m and v as they are before they become codes.  The roundings of m, v and the root are each IEEE's, without fused
// multiply-adds between them, so that the codes are the same wherever they are computed.
//
// Over many steps a value has to become one of the two codes around it, the upper one with a chance equal to its place between them.  Codes lie 6 to 12% of a value
// apart, while a step changes a root by 0.05% with b2 = 0.999: to the nearest code, which a call without a seed takes, all but the largest changes are rounded away at every step,
// for good.  The chance goes by a hash of the value's place, of the step's number and of the seed: adding its bits below those of the code carries into the code where it has to.
//
// Bound by memory in fp32: 22 bytes per bf16 weight, 28 with an fp32 copy of the weight as well (698 M weights: 2981 us, the measured copy rate).  With codes 10
// bytes, and by instructions (657 M weights: 59 a weight and 1480 us at random, 0.68 of the copy rate; 47 and 1370 to the nearest code;
// fp32 weights, or with copies, 0.9 in both).  A CTA takes 8192
// or 32768 values of one tensor; the tensors' addresses are kernel arguments, 400 tensors a launch, so that a captured step needs no copy of a table.
// The number of steps is on the device: every CTA of a tensor adds 2^40 to it when it has read it, and the last one puts the next number.
#include "adamw.cuh"
#include <cuda_fp8.h>
#include <math.h>
#include <string.h>
#include "../common/fl_ptx.cuh"

namespace fl {
namespace adamw {

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int BLOCK = FL_ADAMW_BLOCK, LEAST_CHUNK = 8192, MOST_CHUNK = 32768;
constexpr int MOST = 400, FEW = 32;              // tensors of a launch: 32 KB of arguments, or 2.5
constexpr unsigned ALL = 0xffffffffu;
constexpr long long ARRIVED = 1ll << 40;
enum Codes { NONE, NEAREST, RANDOM };              // how moments become codes

template <int CAP>
struct Launch {
  FlAdamwTensor t[CAP];
  int first[CAP];                                // chunks before the tensor's
  int count, chunk;                              // chunk: values of a CTA
  float b1, c1, b2, c2, eps, one;
  uint32_t seed;                                 // mixed
  double lr, decay, log_b1, log_b2;
  const float* lr_on_device;
};

// the smallest power of two, 2^-100 at least, that brings `bits` (of a finite number, not negative) within 448 = 1.75 * 2^8
__device__ __forceinline__ uint32_t scale_bits(uint32_t bits) {
  const int e = (int)(bits >> 23) + ((bits & 0x7fffffu) > 0x600000u) - 8;
  return (uint32_t)max(e, 27) << 23;
}
__device__ __forceinline__ uint32_t finite_bits(float x) {
  const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}
__device__ __forceinline__ float no_inf(float x) { return (__float_as_uint(x) & 0x7fffffffu) == 0x7f800000u ? NAN : x; }
__device__ __forceinline__ uint32_t codes_of2(float x, float y) {
  uint16_t c;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(c) : "f"(y), "f"(x));
  return c;
}
// 32 bits for each of four values, the first of which is at 4 q: draw(q, salt of the step), and what follows
constexpr uint32_t BY = 0x9e3779b9u, AND = 0x6a09e667u;      // 2^32 times the fractional parts of the golden section and of the root of 2
__host__ __device__ __forceinline__ uint32_t mix(uint32_t x) {
  x *= BY;
  x = (x ^ x >> 15) * AND;
  return x ^ x >> 16;
}
__device__ __forceinline__ uint32_t draw(long long place, uint32_t salt) { return mix(salt ^ (uint32_t)(place >> 2)); }
__device__ __forceinline__ uint32_t next_draw(uint32_t u) { return u * BY + AND; }
__device__ __forceinline__ uint32_t for_m(uint32_t u) { return u & 0xfffffu; }
__device__ __forceinline__ uint32_t for_root(uint32_t u) { return u >> 12; }
// x rounded to e4m3 by 20 bits.  Right from 2^-6 on, where a code has 3 bits behind the first
__device__ __forceinline__ float rounded_by(float x, uint32_t bits) { return __uint_as_float((__float_as_uint(x) + bits) & 0xfff00000u); }
// The same for all numbers: codes below 2^-6 are as far apart as those of the next power of two
__device__ __forceinline__ float any_rounded_by(float x, uint32_t bits) {
  const float size = fabsf(x), small = size < 0.015625f ? 0.015625f : 0.f;
  return x != x ? x : copysignf(__fsub_rn(rounded_by(__fadd_rn(size, small), bits), small), x);
}
// Codes of four values and roots, scaled by powers of two already.  No root above 0 becomes 0 by that: one is 2^-75 at least, its scale 2^56 at most.
__device__ __forceinline__ uint32_t not_lost(uint32_t rc, const float* root) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (root[i] > 0.f && (rc >> 8 * i & 0xffu) == 0u) rc |= 1u << 8 * i;         // the smallest in the place of 0, where the root is none
  return rc;
}
__device__ __forceinline__ uint32_t nearest_codes(const float* x) { return codes_of2(x[2], x[3]) << 16 | codes_of2(x[0], x[1]); }
__device__ __forceinline__ void any_codes(uint32_t& mc, uint32_t& rc, const float* m, const float* root, uint32_t u) {
  uint32_t x[2], y[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const uint32_t v = next_draw(u);
    x[j] = codes_of2(any_rounded_by(m[2 * j], for_m(u)), any_rounded_by(m[2 * j + 1], for_m(v)));
    y[j] = codes_of2(any_rounded_by(root[2 * j], for_root(u)), any_rounded_by(root[2 * j + 1], for_root(v)));
    u = next_draw(v);
  }
  mc = x[1] << 16 | x[0];
  rc = not_lost(y[1] << 16 | y[0], root);
}
__device__ __forceinline__ void values_of(float* x, uint32_t codes, float scale) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t two;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(two) : "h"((uint16_t)(codes >> 16 * h)));
    const float2 f = __half22float2(*reinterpret_cast<__half2*>(&two));
    x[2 * h] = f.x * scale;
    x[2 * h + 1] = f.y * scale;
  }
}

// four values from `at` on; those behind the end are 0
template <typename T>
__device__ __forceinline__ Pack<T, 4> load4(const void* p, long long at, long long n, bool wide) {
  Pack<T, 4> x;
  if (wide && at + 4 <= n) return *reinterpret_cast<const Pack<T, 4>*>((const T*)p + at);
  T* y = reinterpret_cast<T*>(&x.raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) y[i] = at + i < n ? ((const T*)p)[at + i] : T{};
  return x;
}
template <typename T>
__device__ __forceinline__ void store4(void* p, long long at, long long n, bool wide, const Pack<T, 4>& x) {
  if (wide && at + 4 <= n) {
    *reinterpret_cast<Pack<T, 4>*>((T*)p + at) = x;
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (at + i < n) ((T*)p)[at + i] = reinterpret_cast<const T*>(&x.raw)[i];
}

template <typename T>
__device__ __forceinline__ Pack<T, 4> pack(const float* f) {
  Pack<T, 4> x;
  x.set(f);
  return x;
}

__device__ __forceinline__ float rcp(float x) {   // 1 unit in the last place; 0 beyond 2^126
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// A lane's eight values of 256: consecutive ones, or, where some array has them in fp32, four and four that lie 128 apart, so that an access of the warp is
// without gaps.
template <typename T, bool APART>
struct Eight {
  static constexpr int M = APART ? 4 : sizeof(T) == 4 ? 4 : 8, LEAP = APART ? BLOCK / 2 : 4;
  Pack<T, M> p[8 / M];
  static __device__ __forceinline__ long long place(long long b) { return b + (threadIdx.x & 31) * (APART ? 4 : 8); }
  __device__ __forceinline__ void load(const T* from, long long b) {
#pragma unroll
    for (int j = 0; j < 8 / M; ++j) p[j] = *reinterpret_cast<const Pack<T, M>*>(from + place(b) + j * LEAP);
  }
  __device__ __forceinline__ void store(T* to, long long b) const {
#pragma unroll
    for (int j = 0; j < 8 / M; ++j) *reinterpret_cast<Pack<T, M>*>(to + place(b) + j * LEAP) = p[j];
  }
  __device__ __forceinline__ void get(float* f) const {
#pragma unroll
    for (int j = 0; j < 8 / M; ++j) p[j].get(f + j * M);
  }
  __device__ __forceinline__ void set(const float* f) {
#pragma unroll
    for (int j = 0; j < 8 / M; ++j) p[j].set(f + j * M);
  }
};
template <bool APART>
__device__ __forceinline__ uint2 load_codes(const void* from, long long b) {
  const uint8_t* at = (const uint8_t*)from + Eight<uint8_t, APART>::place(b);
  if (APART) return make_uint2(*reinterpret_cast<const uint32_t*>(at), *reinterpret_cast<const uint32_t*>(at + BLOCK / 2));
  return *reinterpret_cast<const uint2*>(at);
}
template <bool APART>
__device__ __forceinline__ void store_codes(void* to, long long b, uint2 c) {
  uint8_t* at = (uint8_t*)to + Eight<uint8_t, APART>::place(b);
  if (APART) {
    *reinterpret_cast<uint32_t*>(at) = c.x;
    *reinterpret_cast<uint32_t*>(at + BLOCK / 2) = c.y;
  } else {
    *reinterpret_cast<uint2*>(at) = c;
  }
}
__device__ __forceinline__ F2 values_of2(uint16_t codes) {
  uint32_t two;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(two) : "h"(codes));
  const float2 f = __half22float2(*reinterpret_cast<__half2*>(&two));
  return F2(f.x, f.y);
}
// 256 values with codes, whole and from multiples of 16 bytes on (codes: of 8).  What a lane has loaded of them:
template <typename T, bool MASTER>
struct Loaded {
  using W = typename std::conditional<MASTER, float, T>::type;
  static constexpr bool APART = sizeof(W) == 4;
  Eight<T, APART> g;
  Eight<W, APART> w;
  uint2 m, v;
  float ms, rs;
  __device__ __forceinline__ void load(const FlAdamwTensor& t, long long b) {
    g.load((const T*)t.grad, b);
    w.load(MASTER ? (const W*)t.master : (const W*)t.param, b);
    m = load_codes<APART>(t.m, b);
    v = load_codes<APART>(t.v, b);
    ms = t.m_scale[b / BLOCK];
    rs = t.v_scale[b / BLOCK];
  }
};
template <typename T, bool MASTER>
__device__ __forceinline__ void prefetch(const FlAdamwTensor& t, long long b) {
  bulk_prefetch_l2((const T*)t.grad + b, BLOCK * sizeof(T));
  if (MASTER) bulk_prefetch_l2(t.master + b, BLOCK * 4);
  else bulk_prefetch_l2((const T*)t.param + b, BLOCK * sizeof(T));
  bulk_prefetch_l2((const uint8_t*)t.m + b, BLOCK);
  bulk_prefetch_l2((const uint8_t*)t.v + b, BLOCK);
}
// Instructions go two values at a time where the hardware has that; the largest magnitudes are taken over numbers (a NaN is left out by itself), and
// infinities looked for only in them.
template <typename T, Codes CODES, bool MASTER, typename L>
__device__ __forceinline__ void step_codes(const Loaded<T, MASTER>& in, const FlAdamwTensor& t, const L& a, long long b, float first, float second, float keep, uint32_t salt) {
  constexpr bool APART = Loaded<T, MASTER>::APART;
  float g[8], w[8], m[8], root[8];
  const uint2 mc = in.m, vc = in.v;
  in.g.get(g);
  in.w.get(w);
  const float ms = in.ms, rs = in.rs;
  const F2 one(a.one, a.one);
  const F2 ms2(ms, ms), rs2(rs, rs), b1(a.b1, a.b1), c1(a.c1, a.c1), b2(a.b2, a.b2), c2(a.c2, a.c2), keep2(keep, keep), eps2(a.eps, a.eps), second2(second, second), first2(-first, -first);
  float m_most = 0.f, r_most = 0.f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t mw = j < 2 ? mc.x : mc.y, vw = j < 2 ? vc.x : vc.y;
    const F2 g2(g[2 * j], g[2 * j + 1]);
    const F2 r_old = values_of2((uint16_t)(vw >> 16 * (j & 1))) * rs2;
    const F2 m_new = sum2(values_of2((uint16_t)(mw >> 16 * (j & 1))) * ms2 * b1, g2 * c1, one), v_new = sum2(r_old * r_old * b2, g2 * g2 * c2, one);
    float v0, v1;
    v_new.get(v0, v1);
    m_new.get(m[2 * j], m[2 * j + 1]);
    root[2 * j] = __fsqrt_rn(v0);
    root[2 * j + 1] = __fsqrt_rn(v1);
    m_most = fmaxf(m_most, fmaxf(fabsf(m[2 * j]), fabsf(m[2 * j + 1])));
    r_most = fmaxf(r_most, fmaxf(root[2 * j], root[2 * j + 1]));
    float d0, d1;
    fma2(F2(root[2 * j], root[2 * j + 1]), second2, eps2).get(d0, d1);
    const F2 w2 = fma2(m_new * first2, F2(rcp(d0), rcp(d1)), F2(w[2 * j], w[2 * j + 1]) * keep2);
    w2.get(w[2 * j], w[2 * j + 1]);
  }
  Eight<T, APART> out;
  out.set(w);
  out.store((T*)t.param, b);
  if (MASTER) {
    Eight<float, APART> copy;
    copy.set(w);
    copy.store(t.master, b);
  }
  uint32_t mb = __reduce_max_sync(ALL, __float_as_uint(m_most)), rb = __reduce_max_sync(ALL, __float_as_uint(r_most));
  if (mb >= 0x7f800000u || rb >= 0x7f800000u) {  // infinities: no number decides a scale, and NaN is kept
    uint32_t most = 0, r = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      most = max(most, finite_bits(m[j]));
      r = max(r, finite_bits(root[j]));
      m[j] = no_inf(m[j]);
      root[j] = no_inf(root[j]);
    }
    mb = __reduce_max_sync(ALL, most);
    rb = __reduce_max_sync(ALL, r);
  }
  mb = scale_bits(mb);
  rb = scale_bits(rb);
  const float m_inv = __uint_as_float((254u << 23) - mb), r_inv = __uint_as_float((254u << 23) - rb);
  const F2 m_inv2(m_inv, m_inv), r_inv2(r_inv, r_inv);
  uint32_t mo[2], ro[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float p[4], q[4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int k = 4 * h + 2 * j;
      (F2(m[k], m[k + 1]) * m_inv2).get(p[2 * j], p[2 * j + 1]);
      (F2(root[k], root[k + 1]) * r_inv2).get(q[2 * j], q[2 * j + 1]);
    }
    if (CODES == NEAREST) {
      mo[h] = nearest_codes(p);
      ro[h] = nearest_codes(q);
      if ((ro[h] - 0x01010101u) & ~ro[h] & 0x80808080u) ro[h] = not_lost(ro[h], q);          // a code of 0 among the four
      continue;
    }
    const uint32_t drawn = draw(Eight<uint8_t, APART>::place(b) + h * (APART ? BLOCK / 2 : 4), salt);
    uint32_t x[2], y[2], u = drawn;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint32_t v = next_draw(u);
      x[j] = codes_of2(rounded_by(p[2 * j], for_m(u)), rounded_by(p[2 * j + 1], for_m(v)));
      y[j] = codes_of2(rounded_by(q[2 * j], for_root(u)), rounded_by(q[2 * j + 1], for_root(v)));
      u = next_draw(v);
    }
    mo[h] = x[1] << 16 | x[0];
    ro[h] = y[1] << 16 | y[0];
    // A code of up to 2^-6 (8) among the eight: a value that may lie below 2^-6, or a NaN, of which the bits may have made 0.  Then by the form for all numbers; one that was
    // 2^-6 at least is the same in both.
    if ((((mo[h] | 0x80808080u) - 0x09090909u) & ((ro[h] | 0x80808080u) - 0x09090909u) & 0x80808080u) != 0x80808080u) any_codes(mo[h], ro[h], p, q, drawn);
  }
  store_codes<APART>(t.m, b, make_uint2(mo[0], mo[1]));
  store_codes<APART>(t.v, b, make_uint2(ro[0], ro[1]));
  if ((threadIdx.x & 31) == 0) {
    t.m_scale[b / BLOCK] = __uint_as_float(mb);
    t.v_scale[b / BLOCK] = __uint_as_float(rb);
  }
}

template <typename T, Codes CODES, bool MASTER, int CAP>
__global__ void __launch_bounds__(THREADS, 4) adamw_kernel(const __grid_constant__ Launch<CAP> a) {
  __shared__ float shared[3];
  __shared__ uint32_t shared_salt;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int lo = 0, hi = a.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (a.first[mid] <= (int)blockIdx.x) lo = mid; else hi = mid - 1;
  }
  const FlAdamwTensor& t = a.t[lo];
  const int chunk = (int)blockIdx.x - a.first[lo], chunks = t.n > a.chunk ? (int)((t.n + a.chunk - 1) / a.chunk) : 1;
  if (threadIdx.x == 0) {
    const long long step = *reinterpret_cast<volatile long long*>(t.step) & (ARRIVED - 1);
    const double lr = a.lr_on_device != nullptr ? (double)*a.lr_on_device : a.lr;
    shared[0] = (float)(lr / -expm1((double)(step + 1) * a.log_b1));
    shared[1] = (float)(1.0 / sqrt(-expm1((double)(step + 1) * a.log_b2)));
    shared[2] = (float)(1.0 - lr * a.decay);
    if (CODES == RANDOM) shared_salt = mix((uint32_t)(step + 1) ^ a.seed);
    const unsigned long long before = atomicAdd(reinterpret_cast<unsigned long long*>(t.step), (unsigned long long)ARRIVED);
    if ((int)(before >> 40) == chunks - 1) atomicExch(reinterpret_cast<unsigned long long*>(t.step), (unsigned long long)(step + 1));
  }
  __syncthreads();
  const float first = shared[0], second = shared[1], keep = shared[2];
  const uint32_t salt = CODES == RANDOM ? shared_salt : 0u;
  uintptr_t bits = (uintptr_t)t.param | (uintptr_t)t.grad;
  bool wide = (bits & (4 * sizeof(T) - 1)) == 0;
  bits = (uintptr_t)t.m | (uintptr_t)t.v;
  wide = wide && (bits & (CODES ? 3 : 15)) == 0 && (!MASTER || ((uintptr_t)t.master & 15) == 0);
  const long long begin = (long long)chunk * a.chunk, end = min(t.n, begin + a.chunk);
  long long b = begin + warp * BLOCK;
  if constexpr (CODES != NONE) {
    const bool eights = (((uintptr_t)t.param | (uintptr_t)t.grad | (uintptr_t)t.master) & 15) == 0 && (((uintptr_t)t.m | (uintptr_t)t.v) & 7) == 0;
    // The next block's loads are on their way while one is computed.  Where weights are fp32 (or have a copy that is) the block behind it is asked into L2 as well: 285 M
    // weights 906 -> 770 us, with copies 979 -> 796; of 16-bit ones alone 588 -> 599, so there it is not.
    const bool far = Loaded<T, MASTER>::APART && (((uintptr_t)t.m | (uintptr_t)t.v) & 15) == 0 && lane == 0;
    if (eights && b + BLOCK <= end) {
      Loaded<T, MASTER> now, next;
      now.load(t, b);
      for (;;) {
        const long long to = b + WARPS * BLOCK;
        const bool more = to + BLOCK <= end;
        if (more) next.load(t, to);
        if (far && to + WARPS * BLOCK + BLOCK <= end) prefetch<T, MASTER>(t, to + WARPS * BLOCK);
        step_codes<T, CODES, MASTER>(now, t, a, b, first, second, keep, salt);
        b = to;
        if (!more) break;
        now = next;
      }
    }
  }
  for (; b < end; b += WARPS * BLOCK) {
    float m[2][4], root[2][4];
    uint32_t m_most = 0, r_most = 0;
    const float ms = CODES ? t.m_scale[b / BLOCK] : 1.f, rs = CODES ? t.v_scale[b / BLOCK] : 1.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const long long at = b + h * (BLOCK / 2) + lane * 4;
      const Pack<T, 4> g4 = load4<T>(t.grad, at, t.n, wide);
      float g[4], v[4], w[4];
      g4.get(g);
      if (CODES) {
        const Pack<uint8_t, 4> mc = load4<uint8_t>(t.m, at, t.n, wide), vc = load4<uint8_t>(t.v, at, t.n, wide);
        values_of(m[h], mc.raw, ms);
        values_of(v, vc.raw, rs);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __fmul_rn(v[i], v[i]);
      } else {
        load4<float>(t.m, at, t.n, wide).get(m[h]);
        load4<float>(t.v, at, t.n, wide).get(v);
      }
      if (MASTER) {
        load4<float>(t.master, at, t.n, wide).get(w);
      } else {
        load4<T>(t.param, at, t.n, wide).get(w);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        m[h][i] = __fadd_rn(__fmul_rn(m[h][i], a.b1), __fmul_rn(g[i], a.c1));
        v[i] = __fadd_rn(__fmul_rn(v[i], a.b2), __fmul_rn(__fmul_rn(g[i], g[i]), a.c2));
        root[h][i] = __fsqrt_rn(v[i]);
        w[i] = fmaf(-first * m[h][i], rcp(fmaf(root[h][i], second, a.eps)), w[i] * keep);
        if (CODES) {
          m_most = max(m_most, finite_bits(m[h][i]));
          r_most = max(r_most, finite_bits(root[h][i]));
        }
      }
      store4<T>(t.param, at, t.n, wide, pack<T>(w));
      if (MASTER) store4<float>(t.master, at, t.n, wide, pack<float>(w));
      if (!CODES) {
        store4<float>(t.m, at, t.n, wide, pack<float>(m[h]));
        store4<float>(t.v, at, t.n, wide, pack<float>(v));
      }
    }
    if (CODES) {
      const uint32_t mb = scale_bits(__reduce_max_sync(ALL, m_most)), rb = scale_bits(__reduce_max_sync(ALL, r_most));
      const float m_inv = __uint_as_float((254u << 23) - mb), r_inv = __uint_as_float((254u << 23) - rb);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const long long at = b + h * (BLOCK / 2) + lane * 4;
        uint32_t mc, rc;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          m[h][i] = no_inf(m[h][i]) * m_inv;
          root[h][i] = no_inf(root[h][i]) * r_inv;
        }
        if (CODES == NEAREST) {
          mc = nearest_codes(m[h]);
          rc = not_lost(nearest_codes(root[h]), root[h]);
        } else {
          any_codes(mc, rc, m[h], root[h], draw(at, salt));
        }
        store4<uint8_t>(t.m, at, t.n, wide, Pack<uint8_t, 4>{mc});
        store4<uint8_t>(t.v, at, t.n, wide, Pack<uint8_t, 4>{rc});
      }
      if (lane == 0) {
        t.m_scale[b / BLOCK] = __uint_as_float(mb);
        t.v_scale[b / BLOCK] = __uint_as_float(rb);
      }
    }
  }
}

template <typename T, Codes CODES, bool MASTER, int CAP>
static int launch(const FlAdamwTensor* t, int count, const FlAdamwArgs* a, cudaStream_t stream) {
  static thread_local Launch<CAP> l;
  long long all = 0, chunks = 0;
  for (int i = 0; i < count; ++i) all += t[i].n;
  // Each chunk begins with its tensor and its step, 2 us before the first value: with codes, which instructions bound, larger ones where there are many (285 M
  // bf16 weights: 604 us against 663); in fp32 the memory has enough to do with others' values (958 us against 1017).
  l.chunk = CODES && all / MOST_CHUNK > 148 * 16 ? MOST_CHUNK : LEAST_CHUNK;
  for (int i = 0; i < count; ++i) {
    l.t[i] = t[i];
    l.first[i] = (int)chunks;
    chunks += t[i].n > l.chunk ? (t[i].n + l.chunk - 1) / l.chunk : 1;
    if (chunks > INT32_MAX) return -1;
  }
  l.count = count;
  l.b1 = (float)a->beta1; l.c1 = (float)(1.0 - a->beta1);
  l.b2 = (float)a->beta2; l.c2 = (float)(1.0 - a->beta2);
  l.one = 1.f; l.eps = (float)a->eps; l.lr = a->lr; l.decay = a->weight_decay;
  l.log_b1 = log(a->beta1); l.log_b2 = log(a->beta2);
  l.lr_on_device = a->lr_on_device;
  l.seed = mix(a->seed);
  adamw_kernel<T, CODES, MASTER, CAP><<<(unsigned)chunks, THREADS, 0, stream>>>(l);
  return (int)cudaGetLastError();
}

template <typename T, Codes CODES, bool MASTER>
static int run(const FlAdamwTensor* t, long long count, const FlAdamwArgs* a, cudaStream_t stream) {
  for (long long i = 0; i < count;) {
    const int n = (int)(count - i < MOST ? count - i : MOST);
    const int rc = n <= FEW ? launch<T, CODES, MASTER, FEW>(t + i, n, a, stream) : launch<T, CODES, MASTER, MOST>(t + i, n, a, stream);
    if (rc != 0) return rc;
    i += n;
  }
  return 0;
}

}  // namespace adamw
}  // namespace fl

extern "C" int fl_adamw(int dtype, const FlAdamwTensor* t, long long count, const FlAdamwArgs* a, cudaStream_t stream) {
  using namespace fl::adamw;
  if (count < 0 || !(a->beta1 >= 0.0 && a->beta1 < 1.0 && a->beta2 >= 0.0 && a->beta2 < 1.0)) return -1;
  for (long long i = 0; i < count; ++i)
    if (t[i].n < 0 || t[i].n > (long long)LEAST_CHUNK * (1 << 22) || t[i].step == nullptr) return -1;
  return fl_by_dtype(dtype, [&](auto type) {
    using T = decltype(type);
    auto by_copies = [&](auto codes) {
      constexpr Codes CODES = decltype(codes)::value;
      if (!a->master) return run<T, CODES, false>(t, count, a, stream);
      if constexpr (sizeof(T) == 2) return run<T, CODES, true>(t, count, a, stream);
      else return -1;
    };
    if (!a->codes) return by_copies(std::integral_constant<Codes, NONE>{});
    return a->random ? by_copies(std::integral_constant<Codes, RANDOM>{}) : by_copies(std::integral_constant<Codes, NEAREST>{});
  });
}

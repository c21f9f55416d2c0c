// Sampling with temperature, top-k, top-p and min-p.
//
// All four limits keep a prefix of the tokens in the order of their logits, and so does drawing by a given number if the cumulative sums run in
// that order.  A 16-bit logit has at most 65536 values: a histogram of a row is the row sorted, equal logits have equal weights, and what is left
// is arithmetic on the occupied bins, in 64 bits at hardly a cost: a token decided by a sum that is off in the 24th bit would be another
// token in one of some hundred rows of a flat distribution over 10^5 entries.
//
// A cluster of CTAs per row.  Each counts its stretch of the row in shared memory (16-bit counters, 128 KB) and adds up counts and weights of 64 bins (a
// chunk) at a time; the first one adds up the CTAs' chunks through distributed shared memory.  There a warp finds the
// limits and the token's bin, by two votes over the sums of 1024 chunks and one over the 64 bins of a chunk each.  The CTA in whose stretch
// the token lies looks for it among its equals.  Bound by latency: one row of 128256 takes 14 us (26000 cycles: counting 4000, barriers of the cluster
// 3500 each, chunks 3500, searches 10000, the look among equals 2500); many rows by the shared memory's atomic additions, of which a warp's 32
// take some seven cycles: 192 rows 63 us (131 before logits were counted two at a time and weights computed eight at a time).
#include "sampling.cuh"
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>
#include "../common/fl_ptx.cuh"
#include "thin_gemm.cuh"

namespace fl {
namespace sampling {

constexpr int THREADS = 1024, WARPS = THREADS / 32, BINS = 65536, CHUNKS = 1024, PER_CHUNK = BINS / CHUNKS;

struct Shared {
  uint32_t hist[BINS / 2];                     // counters of bins 2 i and 2 i + 1
  double mass[CHUNKS];                         // of the chunk, then of all chunks up to it
  int count[CHUNKS];
  uint8_t occupied[CHUNKS];                    // whether the chunk has any
  double warp_mass[WARPS];
  int warp_count[WARPS];
  unsigned top, nan_at;                        // this CTA's first occupied bin and first NaN
  double min_total;                            // what min_p leaves: the number of tokens and their weight
  int min_left;
  int bin, rank;                               // what to look for; bin -1: nothing
  int found[8 * WARPS];                        // of its equals, by pass and warp
  int pass, where, left;                       // the pass and warp that has it, and its rank there
};

// bin of a logit: 0 is the largest number there could be, 65535 the smallest; -0 is 0
__device__ __forceinline__ unsigned bin_of(unsigned h) { return h == 0x8000u ? 0x7fffu : h & 0x8000u ? h : ~h & 0x7fffu; }
__device__ __forceinline__ uint32_t signs(uint32_t h) {          // 0xffff in the halves that are negative
  uint32_t m;
  asm("prmt.b32 %0, %1, 0, 0xbb99;" : "=r"(m) : "r"(h));
  return m;
}
template <typename T> struct Bits;
template <> struct Bits<__nv_bfloat16> {
  static constexpr unsigned INF = 0x7f80u;
  static __device__ __forceinline__ double value(unsigned h) { return (double)__uint_as_float(h << 16); }
};
template <> struct Bits<__half> {
  static constexpr unsigned INF = 0x7c00u;
  static __device__ __forceinline__ double value(unsigned h) { return (double)__half2float(__ushort_as_half((unsigned short)h)); }
};
template <typename T>
__device__ __forceinline__ double bin_value(unsigned bin) { return Bits<T>::value(bin & 0x8000u ? bin : ~bin & 0x7fffu); }

__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t ld_cluster_u8(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u8 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ double ld_cluster_f64(uint32_t addr) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void st_cluster_u32(uint32_t addr, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }

// e^x for x <= 0, to 2^-51 relatively; x below -700 counts as -700, which no sum over a row notices.  With x = n ln 2 + r, |r| <= ln 2 / 2, it is 2^n
// times the Taylor series of e^r, whose terms from r^14 / 14! on are below 2^-57.  Without a branch, so that a thread's bins go through side by
// side: with exp() the pass over the chunks took 9000 cycles.
__device__ __forceinline__ double exp_below_0(double x) {
  x = fmax(x, -700.0);
  const double n = rint(x * 1.4426950408889634);
  double r = fma(n, -0.6931471805599453, x);                   // ln 2 in two parts
  r = fma(n, -2.3190468138462996e-17, r);
  double p = 1.0 / 6227020800.0;
  p = fma(p, r, 1.0 / 479001600.0);
  p = fma(p, r, 1.0 / 39916800.0);
  p = fma(p, r, 1.0 / 3628800.0);
  p = fma(p, r, 1.0 / 362880.0);
  p = fma(p, r, 1.0 / 40320.0);
  p = fma(p, r, 1.0 / 5040.0);
  p = fma(p, r, 1.0 / 720.0);
  p = fma(p, r, 1.0 / 120.0);
  p = fma(p, r, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return p * __hiloint2double(((int)n + 1023) << 20, 0);       // 2^n
}

template <typename T>
struct Weights {
  double largest, per_temperature;             // 1 / temperature: one more rounding of 2^-53 and a division less per bin
  unsigned top;
  __device__ __forceinline__ double exponent(unsigned bin) const { return bin <= top ? 0.0 : (bin_value<T>(bin) - largest) * per_temperature; }
  // bins before the first occupied one count as that one's; from -inf's on there is nothing
  __device__ __forceinline__ double operator()(unsigned bin) const { return bin <= top ? 1.0 : bin >= (0x8000u | Bits<T>::INF) ? 0.0 : exp_below_0(exponent(bin)); }
};

struct Place { unsigned bin; int before, count; double mass_before, weight; };       // a bin, and what lies before it

// counts of bins bin0 and bin0 + 1 (bin0 even) in all CTAs
__device__ __forceinline__ uint2 two_bins(const Shared& s, unsigned bin0, int parts) {
  uint32_t w[8];
  const uint32_t at = smem_u32(&s.hist[bin0 / 2]);
#pragma unroll
  for (int p = 0; p < 8; ++p) w[p] = p < parts ? ld_cluster_u32(map_to_cta(at, p)) : 0u;       // all on their way before the first is needed
  uint2 n = make_uint2(0, 0);
#pragma unroll
  for (int p = 0; p < 8; ++p) { n.x += w[p] & 0xffffu; n.y += w[p] >> 16; }
  return n;
}
template <typename V>
__device__ __forceinline__ void scan_add(V& v, int lane) {                             // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V w = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += w;
  }
}

// The first bin that brings the count to `n` (by_count), or the weight to t, or above it (above).  A whole warp calls it.  Sums by chunk and by bin may
// differ in their last bit, so where none does it is the last occupied one of the chunk, or of those before it.
template <typename T>
__device__ __forceinline__ Place find(const Shared& s, const Weights<T>& weight, int parts, int lane, bool by_count, int n, double t, bool above) {
  auto reached = [&](int count, double mass) { return count > 0 && (by_count ? count >= n : above ? mass > t : mass >= t); };
  unsigned v = __ballot_sync(0xffffffffu, reached(s.count[lane * 32 + 31], s.mass[lane * 32 + 31]));
  const int group = v ? __ffs(v) - 1 : 31;
  v = __ballot_sync(0xffffffffu, reached(s.count[group * 32 + lane], s.mass[group * 32 + lane]));
  int chunk = group * 32 + (v ? __ffs(v) - 1 : 31);
  while (chunk > 0 && s.count[chunk] == s.count[chunk - 1]) --chunk;                  // an empty one, by a last bit
  Place at;
  at.before = chunk ? s.count[chunk - 1] : 0;
  at.mass_before = chunk ? s.mass[chunk - 1] : 0.0;
  const unsigned bin0 = chunk * PER_CHUNK + 2 * lane;
  const uint2 k = two_bins(s, bin0, parts);
  const double w0 = weight(bin0), w1 = weight(bin0 + 1);
  int c = k.x + k.y;
  double m = k.x * w0 + k.y * w1;
  scan_add(c, lane);
  scan_add(m, lane);
  const int c1 = at.before + c, c0 = c1 - (int)k.y;                                   // with the lane's bins
  const double m1 = at.mass_before + m, m0 = m1 - k.y * w1;
  const bool r0 = k.x && reached(c0, m0), r1 = k.y && reached(c1, m1);
  v = __ballot_sync(0xffffffffu, r0 || r1);
  const unsigned some = __ballot_sync(0xffffffffu, k.x || k.y);
  const int who = v ? __ffs(v) - 1 : some ? 31 - __clz(some) : 0;
  const bool second = v ? !r0 : k.y > 0;
  at.bin = __shfl_sync(0xffffffffu, second ? bin0 + 1 : bin0, who);
  at.count = __shfl_sync(0xffffffffu, (int)(second ? k.y : k.x), who);
  at.weight = __shfl_sync(0xffffffffu, second ? w1 : w0, who);
  at.before = __shfl_sync(0xffffffffu, second ? c1 - (int)k.y : c0 - (int)k.x, who);
  at.mass_before = __shfl_sync(0xffffffffu, second ? m1 - k.y * w1 : m0 - k.x * w0, who);
  return at;
}

template <typename T>
__global__ void __launch_bounds__(THREADS) sample_kernel(const FlSampleArgs a, int stretch) {
  extern __shared__ __align__(16) uint8_t smem[];
  Shared& s = *reinterpret_cast<Shared*>(smem);
  const int parts = gridDim.x, part = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.y;
  for (int i = tid; i < BINS / 8; i += THREADS) reinterpret_cast<uint4*>(s.hist)[i] = make_uint4(0, 0, 0, 0);
  s.count[tid] = 0;                                             // CHUNKS == THREADS
  s.mass[tid] = 0.0;
  s.occupied[tid] = 0;
  if (tid == 0) { s.top = BINS; s.nan_at = 0xffffffffu; }
  __syncthreads();
  grid_dep_launch();
  grid_dep_wait();
  const float temp = a.temperature ? a.temperature[row] : a.temperature_all;
  const bool greedy = !(temp > 0.f);

  // ---- count this CTA's stretch: a few logits up to a multiple of 16 bytes, vectors, a few behind them
  const unsigned short* x = reinterpret_cast<const unsigned short*>(a.logits) + (long long)row * a.row_stride;
  const long long begin = (long long)part * stretch;
  const int n = (int)max(min(begin + stretch, a.vocab) - begin, 0ll);
  x += begin;
  const int head = min((int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / 2, n), vecs = (n - head) / 8, tail = head + vecs * 8;
  const unsigned short* xv = x + head;
  constexpr uint32_t INF2 = Bits<T>::INF | Bits<T>::INF << 16;
  unsigned top = BINS, nan_at = 0xffffffffu;
  uint32_t tops = 0xffffffffu;                                  // two smallest bins
  auto take = [&](unsigned h, int at) {
    if ((h & 0x7fffu) > Bits<T>::INF) { nan_at = min(nan_at, (unsigned)(begin + at)); return; }
    if (h == (0x8000u | Bits<T>::INF)) return;                  // -inf weighs nothing
    const unsigned bin = bin_of(h);
    top = min(top, bin);
    if (!greedy) atomicAdd(&s.hist[bin >> 1], 1u << (16 * (bin & 1)));
  };
  if (tid < head) take(x[tid], tid);
  for (int i0 = tid; i0 < vecs; i0 += 4 * THREADS) {            // four vectors on their way at a time
    uint4 u[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (i0 + k * THREADS < vecs) u[k] = ld_stream_v4(xv + (i0 + k * THREADS) * 8);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (i0 + k * THREADS >= vecs) break;
      const uint32_t w[4] = {u[k].x, u[k].y, u[k].z, u[k].w};
      uint32_t finite = 0xffffffffu;                            // 0 in a half: an infinity or NaN among the eight
#pragma unroll
      for (int j = 0; j < 4; ++j) finite = __vminu2(finite, (w[j] & INF2) ^ INF2);
      if (greedy || (finite & 0xffffu) == 0 || finite >> 16 == 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int at = head + (i0 + k * THREADS) * 8 + 2 * j;
          take(w[j] & 0xffffu, at);
          take(w[j] >> 16, at + 1);
        }
      } else {                                                  // two at a time
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t zeros = __vcmpeq2(w[j], 0x80008000u), h = w[j] & ~zeros;          // -0 is 0
          const uint32_t bins = h ^ (~signs(h) & 0x7fff7fffu);              // positive ones are turned round
          tops = __vminu2(tops, bins);
          atomicAdd(&s.hist[(bins & 0xffffu) >> 1], bins & 1u ? 0x10000u : 1u);
          atomicAdd(&s.hist[bins >> 17], bins & 0x10000u ? 0x10000u : 1u);
        }
      }
    }
  }
  top = min(top, min(tops & 0xffffu, tops >> 16) == 0xffffu ? (unsigned)BINS : min(tops & 0xffffu, tops >> 16));
  if (tail + tid < n) take(x[tail + tid], tail + tid);          // at most seven
  top = __reduce_min_sync(0xffffffffu, top);
  nan_at = __reduce_min_sync(0xffffffffu, nan_at);
  if (lane == 0) { atomicMin(&s.top, top); atomicMin(&s.nan_at, nan_at); }
  __syncthreads();
  if (parts > 1) cluster_sync_all();

  const unsigned cta_top = lane < parts ? ld_cluster_u32(map_to_cta(smem_u32(&s.top), lane)) : BINS;              // a CTA's per lane
  const unsigned nans = lane < parts ? ld_cluster_u32(map_to_cta(smem_u32(&s.nan_at), lane)) : 0xffffffffu;
  top = __reduce_min_sync(0xffffffffu, cta_top);
  nan_at = __reduce_min_sync(0xffffffffu, nans);
  const int first_with_top = __ffs(__ballot_sync(0xffffffffu, cta_top == top)) - 1;
  if (greedy || nan_at != 0xffffffffu || top == BINS) {         // no weights are needed, and every CTA knows which one has the token
    const bool mine = nan_at == 0xffffffffu && top < BINS && part == first_with_top;
    if (part == 0 && tid == 0) {
      if (nan_at != 0xffffffffu || top == BINS) a.tokens[row] = nan_at == 0xffffffffu ? 0 : (long long)nan_at;
      if (a.logprobs) a.logprobs[row] = nan_at != 0xffffffffu ? NAN : top == BINS ? -INFINITY : 0.f;
    }
    if (tid == 0) { s.bin = mine ? (int)top : -1; s.rank = 0; }
    __syncthreads();
    if (parts > 1) cluster_sync_all();                          // s.top and s.nan_at have been read
  } else {
    Weights<T> weight;
    weight.top = top;
    weight.largest = bin_value<T>(top);
    weight.per_temperature = 1.0 / (double)temp;

    // ---- counts and weights of this CTA's chunks: eight lanes per chunk, eight bins per lane.  What CTAs read of one another is little, since that is
    // slow: with every counter read by the CTA that had its chunk this pass took 18000 cycles of a row's 55000.  Nine chunks of ten are empty, and
    // theirs are passed over with a load and a vote.
    uint4 h[CHUNKS / (4 * WARPS)];
#pragma unroll
    for (int i = 0; i < CHUNKS / (4 * WARPS); ++i) h[i] = *reinterpret_cast<const uint4*>(&s.hist[((i * WARPS + warp) * 32 + lane) * 4]);
#pragma unroll
    for (int i = 0; i < CHUNKS / (4 * WARPS); ++i) {
      const unsigned some = __ballot_sync(0xffffffffu, (h[i].x | h[i].y | h[i].z | h[i].w) != 0);
      if (some == 0) continue;
      const int chunk = (i * WARPS + warp) * 4 + lane / 8;
      const unsigned bin0 = chunk * PER_CHUNK + (lane & 7) * 8;
      const uint32_t w[4] = {h[i].x, h[i].y, h[i].z, h[i].w};
      int count = 0;
      // Eight neighbours are equally far apart (a chunk lies within a binade), so their weights fall by the same factor: two exponentials in place of eight.
      // Arithmetic in 64 bits is what this pass takes its time for.
      const unsigned first = max(bin0, min(top, bin0 + 7));     // there are none before the row's largest
      const double fall = exp_below_0((bin_value<T>(first + 1) - bin_value<T>(first)) * weight.per_temperature);
      double mass = 0.0;
#pragma unroll
      for (int j = 7; j >= 0; --j) {
        const int k = (int)(j & 1 ? w[j / 2] >> 16 : w[j / 2] & 0xffffu);
        count += k;
        if (bin0 + j >= first) mass = fma(mass, fall, (double)k);
      }
      mass *= weight(first);
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) {
        count += __shfl_xor_sync(0xffffffffu, count, o);
        mass += __shfl_xor_sync(0xffffffffu, mass, o);
      }
      if ((lane & 7) == 0 && count > 0) {
        s.count[chunk] = count;
        s.mass[chunk] = mass;
        s.occupied[chunk] = 1;
      }
    }
    __syncthreads();
    if (parts > 1) cluster_sync_all();

    // ---- the first CTA finds the token's bin
    double left_total = 1.0, exponent = 0.0;
    if (part == 0) {
      // the CTAs' chunks, added up in their order, and the sums up to each
      int count = s.count[tid];
      double mass = s.mass[tid];
      unsigned there = 0;
#pragma unroll
      for (int p = 1; p < 8; ++p)
        if (p < parts) there |= ld_cluster_u8(map_to_cta(smem_u32(&s.occupied[tid]), p)) << p;
      if (there) {
        unsigned c[8];
        double m[8];
#pragma unroll
        for (int p = 1; p < 8; ++p) {
          c[p] = there >> p & 1 ? ld_cluster_u32(map_to_cta(smem_u32(&s.count[tid]), p)) : 0u;
          m[p] = there >> p & 1 ? ld_cluster_f64(map_to_cta(smem_u32(&s.mass[tid]), p)) : 0.0;
        }
#pragma unroll
        for (int p = 1; p < 8; ++p) { count += c[p]; mass += m[p]; }
      }
      scan_add(count, lane);
      scan_add(mass, lane);
      if (lane == 31) { s.warp_count[warp] = count; s.warp_mass[warp] = mass; }
      __syncthreads();
      int c = lane < warp ? s.warp_count[lane] : 0;
      double m = lane < warp ? s.warp_mass[lane] : 0.0;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        c += __shfl_xor_sync(0xffffffffu, c, o);
        m += __shfl_xor_sync(0xffffffffu, m, o);
      }
      s.count[tid] = count + c;
      s.mass[tid] = mass + m;
      __syncthreads();
      const double min_p = a.min_p ? (double)a.min_p[row] : (double)a.min_p_all;
      if (warp == 1 && min_p > 0.0) {                           // beside the first warp's searches
        // the bins' weights fall: chunks whose first bin has at least min_p, and in the last of them its bins that do
        unsigned v = __ballot_sync(0xffffffffu, weight(lane * 32 * PER_CHUNK) >= min_p);
        int chunk = -1;
        if (v) {
          const int group = 31 - __clz(v);
          v = __ballot_sync(0xffffffffu, weight((group * 32 + lane) * PER_CHUNK) >= min_p);
          chunk = group * 32 + 31 - __clz(v);
        }
        int k = 0;
        double w = 0.0;
        if (chunk >= 0) {
          const unsigned bin0 = chunk * PER_CHUNK + 2 * lane;
          const uint2 n2 = two_bins(s, bin0, parts);
          const double w0 = weight(bin0), w1 = weight(bin0 + 1);
          if (w0 >= min_p) { k += n2.x; w += n2.x * w0; }
          if (w1 >= min_p) { k += n2.y; w += n2.y * w1; }
          k = __reduce_add_sync(0xffffffffu, k);
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
          if (chunk) { k += s.count[chunk - 1]; w += s.mass[chunk - 1]; }
        }
        if (lane == 0) {
          s.min_left = k < 1 ? 1 : k;
          s.min_total = k < 1 ? 1.0 : w;
        }
        asm volatile("bar.sync 1, 64;" ::: "memory");
      }
      if (warp == 0) {
        int left = s.count[CHUNKS - 1];                         // tokens that are left, and their weight
        double total = s.mass[CHUNKS - 1];
        const int top_k = a.top_k ? a.top_k[row] : a.top_k_all;
        if (top_k > 0 && top_k < left) {
          const Place at = find(s, weight, parts, lane, true, top_k, 0.0, false);
          left = top_k;
          total = at.mass_before + (top_k - at.before) * at.weight;
        }
        const double top_p = a.top_p ? (double)a.top_p[row] : (double)a.top_p_all;
        if (top_p < 1.0) {
          const double t = top_p * total;
          const Place at = find(s, weight, parts, lane, false, 0, t, false);
          const double want = ceil((t - at.mass_before) / at.weight);
          const int j = want >= at.count ? at.count : want < 1.0 ? 1 : (int)want;
          if (at.before + j < left) {
            left = at.before + j;
            total = at.mass_before + j * at.weight;
          }
        }
        if (min_p > 0.0) {
          asm volatile("bar.sync 1, 64;" ::: "memory");
          if (s.min_left < left) {
            left = s.min_left;
            total = s.min_total;
          }
        }
        double u = a.u64 ? a.u64[row] : (double)a.u32[row];
        u = u >= 0.0 ? fmin(u, 1.0 - 0x1p-53) : 0.0;
        const double t = u * total;
        Place at = find(s, weight, parts, lane, false, 0, t, true);
        const double want = floor((t - at.mass_before) / at.weight);
        int rank = want >= at.count - 1 ? at.count - 1 : want < 0.0 ? 0 : (int)want;
        if (at.before + rank >= left) {                         // a sum's last bit: the last of those left
          at = find(s, weight, parts, lane, true, left, 0.0, false);
          rank = left - 1 - at.before;
        }
        // the CTA that has it: lane p knows how many are in the CTAs up to p
        int upto = lane < parts ? (int)(ld_cluster_u32(map_to_cta(smem_u32(&s.hist[at.bin >> 1]), lane)) >> (16 * (at.bin & 1)) & 0xffffu) : 0;
        const int own = upto;
        scan_add(upto, lane);
        const unsigned v = __ballot_sync(0xffffffffu, lane < parts && upto > rank);
        const int owner = v ? __ffs(v) - 1 : parts - 1;
        if (lane < parts) {
          st_cluster_u32(map_to_cta(smem_u32(&s.rank), lane), (uint32_t)(rank - (upto - own)));
          st_cluster_u32(map_to_cta(smem_u32(&s.bin), lane), (uint32_t)(lane == owner ? (int)at.bin : -1));
        }
        left_total = total;
        exponent = weight.exponent(at.bin);
      }
    }
    __syncthreads();
    if (parts > 1) cluster_sync_all();                          // nobody reads another's memory behind this
    if (part == 0 && tid == 0 && a.logprobs) a.logprobs[row] = (float)(exponent - log(left_total));
  }
  if (s.bin < 0) return;

  // ---- the one of rank `rank` among the stretch's logits of this bin, in their order
  const unsigned want = (unsigned)s.bin;
  int rank = s.rank;
  unsigned v = __ballot_sync(0xffffffffu, lane < head && bin_of(x[min(lane, n - 1)]) == want);
  if (rank < __popc(v)) {
    if (warp == 0 && (v >> lane & 1) && __popc(v & ((1u << lane) - 1)) == rank) a.tokens[row] = begin + lane;
    return;
  }
  rank -= __popc(v);
  const uint32_t bits = want & 0x8000u ? want : ~want & 0x7fffu, two = bits | bits << 16, keep = bits == 0 ? 0x7fff7fffu : 0xffffffffu;    // 0 is also -0
  uint32_t is[2] = {0, 0};                                      // which of each pass's eight
#pragma unroll
  for (int k0 = 0; k0 < 8; k0 += 4) {                           // a stretch has at most eight vectors per thread
    uint4 u[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if ((k0 + k) * THREADS + tid < vecs) u[k] = ld_stream_v4(xv + ((k0 + k) * THREADS + tid) * 8);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint32_t m = 0;
      if ((k0 + k) * THREADS + tid < vecs) {
        const uint32_t w[4] = {u[k].x, u[k].y, u[k].z, u[k].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t e = __vcmpeq2(w[j] & keep, two);
          m |= (e & 1u | e >> 15 & 2u) << (2 * j);
        }
      }
      is[k0 / 4] |= m << (8 * k);
      const int found = __reduce_add_sync(0xffffffffu, __popc(m));
      if (lane == 0) s.found[(k0 + k) * WARPS + warp] = found;
    }
  }
  if (tid == 0) s.pass = -1;
  __syncthreads();
  if (warp == 0) {
    int f[8], sum = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) { f[j] = s.found[lane * 8 + j]; sum += f[j]; }
    int before = sum;
    scan_add(before, lane);
    const int all = __shfl_sync(0xffffffffu, before, 31);
    before -= sum;
    if (rank >= before && rank < before + sum) {
      int j = 0;
      while (j < 7 && rank >= before + f[j]) before += f[j++];
      s.pass = (lane * 8 + j) / WARPS;
      s.where = (lane * 8 + j) % WARPS;
      s.left = rank - before;
    }
    if (rank >= all) {                                          // behind the vectors
      const int at = tail + lane;
      v = __ballot_sync(0xffffffffu, at < n && bin_of(x[min(at, n - 1)]) == want);
      if ((v >> lane & 1) && __popc(v & ((1u << lane) - 1)) == rank - all) a.tokens[row] = begin + at;
    }
  }
  __syncthreads();
  if (s.pass < 0 || warp != s.where) return;
  const uint32_t m = is[s.pass / 4] >> (8 * (s.pass % 4)) & 255u;
  int before = __popc(m);
  scan_add(before, lane);
  before -= __popc(m);
  const int mine = s.left - before;
  if (mine >= 0 && mine < __popc(m)) {
    uint32_t r = m;
    for (int i = 0; i < mine; ++i) r &= r - 1;
    a.tokens[row] = begin + head + (long long)(s.pass * THREADS + tid) * 8 + __ffs(r) - 1;
  }
}

}  // namespace sampling
}  // namespace fl

// --------------------------------------------------------------------------------------------------------------------------
// host side
// --------------------------------------------------------------------------------------------------------------------------
template <typename T>
static int launch_sample(const FlSampleArgs& a, int parts, int stretch, bool early, cudaStream_t stream) {
  constexpr int smem = sizeof(fl::sampling::Shared);
  static bool set_on[64];                          // per device: a process may drive several GPUs
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  if (dev < 0 || dev >= 64) return -3;
  if (!set_on[dev]) {
    e = cudaFuncSetAttribute(fl::sampling::sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return (int)e;
    set_on[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(parts, a.rows, 1);
  cfg.blockDim = dim3(fl::sampling::THREADS, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = parts; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = early ? 2 : 1;
  return (int)cudaLaunchKernelEx(&cfg, fl::sampling::sample_kernel<T>, a, stretch);
}

extern "C" int fl_sample(int dtype, const FlSampleArgs* args, cudaStream_t stream) {
  FlSampleArgs a = *args;
  if (a.rows < 0 || a.vocab < 1 || a.vocab > FL_SAMPLE_MAX_VOCAB || (a.rows > 0 && a.logits == nullptr) || (a.u64 == nullptr) == (a.u32 == nullptr)) return -2;
  if (dtype != FL_DEC_BF16 && dtype != FL_DEC_FP16) return -1;
  // A counter has 16 bits, so a CTA takes 65528 logits at most; where SMs would be idle a row is cut finer, down to 4096.  A CTA takes the shared memory
  // of an SM, and a cluster those of one GPC, of which clusters of eight leave some over: they are for rows that all find room at once.
  int parts = 1;
  while (parts < 8 && (a.vocab > 65528ll * parts || (2ll * parts * a.rows <= (parts == 4 ? 96 : 148) && a.vocab >= 2ll * parts * 4096))) parts *= 2;
  const long long stretch = ((a.vocab + parts - 1) / parts + 7) / 8 * 8;
  const int rows = a.rows;
  const size_t step = 65535;                       // what a grid's second dimension takes
  for (size_t r = 0; r < (size_t)rows; r += step) {
    FlSampleArgs part = a;
    part.rows = (int)(rows - r < step ? rows - r : step);
    part.logits = reinterpret_cast<const uint16_t*>(a.logits) + (long long)r * a.row_stride;
    if (a.u64) part.u64 += r;
    if (a.u32) part.u32 += r;
    if (a.temperature) part.temperature += r;
    if (a.top_k) part.top_k += r;
    if (a.top_p) part.top_p += r;
    if (a.min_p) part.min_p += r;
    part.tokens += r;
    if (a.logprobs) part.logprobs += r;
    const int rc = dtype == FL_DEC_BF16 ? launch_sample<__nv_bfloat16>(part, parts, (int)stretch, rows <= FL_THIN_MAX_ROWS, stream)
                                        : launch_sample<__half>(part, parts, (int)stretch, rows <= FL_THIN_MAX_ROWS, stream);
    if (rc != 0) return rc;
  }
  return 0;
}

// Sampling with temperature, top-k, top-p and min-p.
//
// All four limits keep a prefix of the tokens in the order of their logits, and so does drawing by a given number if the cumulative sums run in
// that order.  A 16-bit logit has at most 65536 values: a histogram of a row is the row sorted, equal logits have equal weights, and what is left
// is arithmetic on the occupied bins, in 64 bits at hardly a cost: a token decided by a sum that is off in the 24th bit would be another
// token in one of some hundred rows of a flat distribution over 10^5 entries.
//
// A cluster of CTAs per row.  Each counts its stretch of the row in shared memory (16-bit counters, 128 KB); together they add the counters up
// through distributed shared memory, 64 bins (a chunk) per 8 lanes, and tell the first CTA each chunk's count and weight.  That one finds the
// limits and the token's bin: a scan over the 1024 chunks, then a warp's over the 64 bins of the one that matters.  The CTA in whose stretch
// the token lies looks for it among its equals.
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
  double warp_mass[WARPS];
  int warp_count[WARPS];
  unsigned top, nan_at;                        // this CTA's first occupied bin and first NaN
  unsigned first;                              // a search's answer
  int bin, rank;                               // what to look for; bin -1: nothing
  int below[WARPS];
};

// bin of a logit: 0 is the largest number there could be, 65535 the smallest; -0 is 0
__device__ __forceinline__ unsigned bin_of(unsigned h) { return h == 0x8000u ? 0x7fffu : h & 0x8000u ? h : ~h & 0x7fffu; }
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
__device__ __forceinline__ uint4 ld_cluster_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void st_cluster_u32(uint32_t addr, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }
__device__ __forceinline__ void st_cluster_f64(uint32_t addr, double v) { asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(addr), "d"(v) : "memory"); }

template <typename T>
struct Weights {
  double largest, temperature;
  unsigned top;
  __device__ __forceinline__ double exponent(unsigned bin) const { return bin <= top ? 0.0 : (bin_value<T>(bin) - largest) / temperature; }
  // bins before the first occupied one count as that one's; from -inf's on there is nothing
  __device__ __forceinline__ double operator()(unsigned bin) const { return bin <= top ? 1.0 : bin >= (0x8000u | Bits<T>::INF) ? 0.0 : exp(exponent(bin)); }
};

struct Place { unsigned bin; int before; double mass_before, weight; int count; };       // a bin, and what lies before it

template <typename T>
__global__ void __launch_bounds__(THREADS) sample_kernel(const FlSampleArgs a, int stretch) {
  extern __shared__ __align__(16) uint8_t smem[];
  Shared& s = *reinterpret_cast<Shared*>(smem);
  const int parts = gridDim.x, part = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row = blockIdx.y;
  for (int i = tid; i < BINS / 8; i += THREADS) reinterpret_cast<uint4*>(s.hist)[i] = make_uint4(0, 0, 0, 0);
  if (tid == 0) { s.top = BINS; s.nan_at = 0xffffffffu; }
  __syncthreads();
  grid_dep_launch();
  grid_dep_wait();

  // ---- count this CTA's stretch
  const unsigned short* x = reinterpret_cast<const unsigned short*>(a.logits) + (long long)row * a.row_stride;
  const long long begin = (long long)part * stretch, end = min(begin + stretch, a.vocab);
  unsigned top = BINS, nan_at = 0xffffffffu;
  auto take = [&](unsigned h, long long at) {
    if ((h & 0x7fffu) > Bits<T>::INF) { nan_at = min(nan_at, (unsigned)at); return; }
    if (h == (0x8000u | Bits<T>::INF)) return;                  // -inf weighs nothing
    const unsigned bin = bin_of(h);
    top = min(top, bin);
    atomicAdd(&s.hist[bin >> 1], 1u << (16 * (bin & 1)));
  };
  const long long head = min((long long)((16 - (reinterpret_cast<uintptr_t>(x + begin) & 15)) & 15) / 2, max(end - begin, 0ll));
  const long long vecs = max(end - begin - head, 0ll) / 8;
  if (begin + tid < begin + head) take(x[begin + tid], begin + tid);
  for (long long i = tid; i < vecs; i += THREADS) {
    const long long at = begin + head + i * 8;
    const uint4 u = ld_stream_v4(x + at);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      take(w[j] & 0xffffu, at + 2 * j);
      take(w[j] >> 16, at + 2 * j + 1);
    }
  }
  for (long long at = begin + head + vecs * 8 + tid; at < end; at += THREADS) take(x[at], at);
  top = __reduce_min_sync(0xffffffffu, top);
  nan_at = __reduce_min_sync(0xffffffffu, nan_at);
  if (lane == 0) { atomicMin(&s.top, top); atomicMin(&s.nan_at, nan_at); }
  __syncthreads();
  if (parts > 1) cluster_sync_all();

  for (int p = 0; p < parts; ++p) {
    top = min(top, ld_cluster_u32(map_to_cta(smem_u32(&s.top), p)));
    nan_at = min(nan_at, ld_cluster_u32(map_to_cta(smem_u32(&s.nan_at), p)));
  }
  const float temp = a.temperature ? a.temperature[row] : a.temperature_all;
  const bool greedy = !(temp > 0.f);
  Weights<T> weight;
  weight.top = top;
  weight.largest = top < BINS ? bin_value<T>(top) : 0.0;
  weight.temperature = greedy ? 1.0 : (double)temp;

  // ---- counts and weights of the chunks, to the first CTA
  const int mine = CHUNKS / parts;
  for (int c0 = 0; c0 < mine; c0 += THREADS / 8) {
    const int chunk = part * mine + c0 + tid / 8, bin0 = chunk * PER_CHUNK + (tid & 7) * 8;
    const bool in = c0 + tid / 8 < mine;
    unsigned n[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (in) {
      for (int p = 0; p < parts; ++p) {
        const uint4 u = ld_cluster_v4(map_to_cta(smem_u32(&s.hist[bin0 / 2]), p));
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) { n[2 * j] += w[j] & 0xffffu; n[2 * j + 1] += w[j] >> 16; }
      }
    }
    int count = 0;
    double mass = 0.0;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (n[j]) { count += n[j]; mass += n[j] * weight(bin0 + j); }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
      count += __shfl_xor_sync(0xffffffffu, count, o);
      mass += __shfl_xor_sync(0xffffffffu, mass, o);
    }
    if (in && (tid & 7) == 0) {
      st_cluster_u32(map_to_cta(smem_u32(&s.count[chunk]), 0), (uint32_t)count);
      st_cluster_f64(map_to_cta(smem_u32(&s.mass[chunk]), 0), mass);
    }
  }
  __syncthreads();
  if (parts > 1) cluster_sync_all();

  // ---- the first CTA finds the token's bin
  if (part == 0) {
    // sums up to each chunk
    int count = s.count[tid];
    double mass = s.mass[tid];
    const int own = count;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int c = __shfl_up_sync(0xffffffffu, count, o);
      const double m = __shfl_up_sync(0xffffffffu, mass, o);
      if (lane >= o) { count += c; mass += m; }
    }
    if (lane == 31) { s.warp_count[warp] = count; s.warp_mass[warp] = mass; }
    __syncthreads();
    int count_before = 0;
    double mass_before = 0.0;
    for (int w = 0; w < warp; ++w) { count_before += s.warp_count[w]; mass_before += s.warp_mass[w]; }
    count += count_before;
    mass += mass_before;
    s.count[tid] = count;
    s.mass[tid] = mass;
    __syncthreads();
    const int all = s.count[CHUNKS - 1];

    // The first bin that brings the count to `n`, or the weight to (`above`: above) t; every thread gets it.  Sums by chunk and by bin may differ
    // in their last bit, so where none does it is the last occupied one.
    auto find = [&](bool by_count, int n, double t, bool above) -> Place {
      if (tid == 0) s.first = 0xffffffffu;
      __syncthreads();
      const bool reached = own > 0 && (by_count ? count >= n : above ? mass > t : mass >= t);
      const unsigned vote = __ballot_sync(0xffffffffu, reached);
      if (vote && lane == 0) atomicMin(&s.first, (unsigned)(warp * 32 + __ffs(vote) - 1));
      __syncthreads();
      if (s.first == 0xffffffffu) {                             // s.first is the same for all, and read by all before it changes
        __syncthreads();
        const unsigned occupied = __ballot_sync(0xffffffffu, own > 0);
        if (tid == 0) s.first = 0;
        __syncthreads();
        if (occupied && lane == 0) atomicMax(&s.first, (unsigned)(warp * 32 + 31 - __clz(occupied)));
        __syncthreads();
      }
      const int chunk = (int)s.first;
      Place at;
      at.before = chunk ? s.count[chunk - 1] : 0;
      at.mass_before = chunk ? s.mass[chunk - 1] : 0.0;
      // two bins per lane, by every warp alike
      const int bin0 = chunk * PER_CHUNK + 2 * lane;
      unsigned n0 = 0, n1 = 0;
      for (int p = 0; p < parts; ++p) {
        const uint32_t w = ld_cluster_u32(map_to_cta(smem_u32(&s.hist[bin0 / 2]), p));
        n0 += w & 0xffffu;
        n1 += w >> 16;
      }
      const double w0 = n0 ? weight(bin0) : 0.0, w1 = n1 ? weight(bin0 + 1) : 0.0;
      int c = n0 + n1;
      double m = n0 * w0 + n1 * w1;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int cc = __shfl_up_sync(0xffffffffu, c, o);
        const double mm = __shfl_up_sync(0xffffffffu, m, o);
        if (lane >= o) { c += cc; m += mm; }
      }
      const int c0 = at.before + c - (int)n1, c1 = at.before + c;                      // counts and weights with the lane's bins
      const double m1 = at.mass_before + m, m0 = m1 - n1 * w1;
      const bool r0 = n0 && (by_count ? c0 >= n : above ? m0 > t : m0 >= t), r1 = n1 && (by_count ? c1 >= n : above ? m1 > t : m1 >= t);
      unsigned v = __ballot_sync(0xffffffffu, r0 || r1);
      const unsigned some = __ballot_sync(0xffffffffu, n0 || n1);
      const int who = v ? __ffs(v) - 1 : some ? 31 - __clz(some) : 0;
      const bool second = v ? !r0 : n1 > 0;
      const unsigned bin = second ? bin0 + 1 : bin0, nn = second ? n1 : n0;
      const double ww = second ? w1 : w0;
      const int bb = (second ? c1 : c0) - (int)nn;
      const double mb = (second ? m1 - n1 * w1 : m0 - n0 * w0);
      at.bin = __shfl_sync(0xffffffffu, bin, who);
      at.count = __shfl_sync(0xffffffffu, (int)nn, who);
      at.weight = __shfl_sync(0xffffffffu, ww, who);
      at.before = __shfl_sync(0xffffffffu, bb, who);
      at.mass_before = __shfl_sync(0xffffffffu, mb, who);
      __syncthreads();                                          // before s.first is used again
      return at;
    };

    int bin = -1, rank = 0;
    float logp = -INFINITY;
    if (nan_at == 0xffffffffu && all > 0) {
      if (greedy) {
        bin = (int)top;
        logp = 0.f;
      } else {
        int left = all;                                         // tokens that are left, and their weight
        double total = s.mass[CHUNKS - 1];
        const int k = a.top_k ? a.top_k[row] : a.top_k_all;
        if (k > 0 && k < left) {
          const Place at = find(true, k, 0.0, false);
          left = k;
          total = at.mass_before + (k - at.before) * at.weight;
        }
        const double top_p = a.top_p ? (double)a.top_p[row] : (double)a.top_p_all;
        const double min_p = a.min_p ? (double)a.min_p[row] : (double)a.min_p_all;
        if (top_p < 1.0) {
          const double t = top_p * total;
          const Place at = find(false, 0, t, false);
          const double want = ceil((t - at.mass_before) / at.weight);
          const int j = want >= at.count ? at.count : want < 1.0 ? 1 : (int)want;
          if (at.before + j < left) {
            left = at.before + j;
            total = at.mass_before + j * at.weight;
          }
        }
        if (min_p > 0.0) {
          // the bins' weights fall: the last chunk that has one of at least min_p, and in it the last such bin
          const bool some = own > 0 && weight(tid * PER_CHUNK) >= min_p;
          const unsigned v = __ballot_sync(0xffffffffu, some);
          if (tid == 0) s.first = 0;
          __syncthreads();
          if (v && lane == 0) atomicMax(&s.first, (unsigned)(warp * 32 + 32 - __clz(v)));
          __syncthreads();
          const int chunk = (int)s.first - 1;
          __syncthreads();
          int n = 0;
          double m = 0.0;
          if (chunk >= 0) {
            const int bin0 = chunk * PER_CHUNK + 2 * lane;
            unsigned n0 = 0, n1 = 0;
            for (int p = 0; p < parts; ++p) {
              const uint32_t w = ld_cluster_u32(map_to_cta(smem_u32(&s.hist[bin0 / 2]), p));
              n0 += w & 0xffffu;
              n1 += w >> 16;
            }
            const double w0 = weight(bin0), w1 = weight(bin0 + 1);
            if (n0 && w0 >= min_p) { n += n0; m += n0 * w0; }
            if (n1 && w1 >= min_p) { n += n1; m += n1 * w1; }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
              n += __shfl_xor_sync(0xffffffffu, n, o);
              m += __shfl_xor_sync(0xffffffffu, m, o);
            }
            if (chunk) { n += s.count[chunk - 1]; m += s.mass[chunk - 1]; }
          }
          if (n < left) {
            left = n;
            total = m;
          }
          if (left < 1) { left = 1; total = 1.0; }
        }
        double u = a.u64 ? a.u64[row] : (double)a.u32[row];
        u = u >= 0.0 ? fmin(u, 1.0 - 0x1p-53) : 0.0;
        const double t = u * total;
        Place at = find(false, 0, t, true);
        const double want = floor((t - at.mass_before) / at.weight);
        rank = want >= at.count - 1 ? at.count - 1 : want < 0.0 ? 0 : (int)want;
        if (at.before + rank >= left) {                         // a sum's last bit: the last of those left
          at = find(true, left, 0.0, false);
          rank = left - 1 - at.before;
        }
        bin = (int)at.bin;
        logp = (float)(weight.exponent(at.bin) - log(total));
      }
    }
    if (tid == 0) {
      int owner = 0;
      if (bin >= 0) {
        for (; owner < parts - 1; ++owner) {
          const int n = (int)(ld_cluster_u32(map_to_cta(smem_u32(&s.hist[bin >> 1]), owner)) >> (16 * (bin & 1)) & 0xffffu);
          if (rank < n) break;
          rank -= n;
        }
      } else {
        a.tokens[row] = nan_at == 0xffffffffu ? 0 : (long long)nan_at;
      }
      if (a.logprobs) a.logprobs[row] = nan_at == 0xffffffffu ? logp : NAN;
      for (int p = 0; p < parts; ++p) {
        st_cluster_u32(map_to_cta(smem_u32(&s.rank), p), (uint32_t)rank);
        st_cluster_u32(map_to_cta(smem_u32(&s.bin), p), (uint32_t)(p == owner ? bin : -1));
      }
    }
  }
  __syncthreads();
  if (parts > 1) cluster_sync_all();                            // nobody reads another's memory behind this
  if (s.bin < 0) return;

  // ---- the one of rank `rank` among the stretch's logits of this bin, in their order: a warp's piece, then a walk through it
  const unsigned want = (unsigned)s.bin;
  const long long n = end - begin, piece = ((n + WARPS - 1) / WARPS + 31) / 32 * 32;
  const long long p0 = begin + min(warp * piece, n), p1 = begin + min((warp + 1) * piece, n);
  int found = 0;
  for (long long at = p0 + lane; at < p1; at += 32) found += bin_of(x[at]) == want;
  found = __reduce_add_sync(0xffffffffu, found);
  if (lane == 0) s.below[warp] = found;
  __syncthreads();
  int rank = s.rank;
  for (int w = 0; w < warp; ++w) rank -= s.below[w];
  if (rank < 0 || rank >= found) return;
  for (long long at = p0; at < p1; at += 32) {
    const bool is = at + lane < p1 && bin_of(x[at + lane]) == want;
    const unsigned v = __ballot_sync(0xffffffffu, is);
    if (is && __popc(v & ((1u << lane) - 1)) == rank) a.tokens[row] = at + lane;
    rank -= __popc(v);
    if (rank < 0) return;
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
  // A counter has 16 bits, so a CTA takes 65528 logits at most; where SMs would be idle a row is cut finer, down to 4096.
  int parts = 1;
  while (parts < 8 && (a.vocab > 65528ll * parts || (2ll * parts * a.rows <= 148 && a.vocab >= 2ll * parts * 4096))) parts *= 2;
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

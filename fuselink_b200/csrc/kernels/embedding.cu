// Embedding lookup with a factor, and its gradient by sorted tokens.
//
//   out[t] = scale W[id_t]            dW[v] = scale sum over t with id_t = v, in the order of t, of dOut[t]
//
// Sums run in fp32 and in an order that the tokens alone decide (no floating-point atomics), so that the same batch gives the same bits; each
// value is rounded to the table's type once.  Both are bound by memory: the lookup reads and writes a row per token, the gradient reads one per
// token and writes all of the table, zeros for the most part.
//
// Gradient: embed_sort_kernel lists the tokens' places sorted by id, places of one id in order.  A CTA has a range of ids, counts its own ones
// (each warp a stretch of the batch, in counters of its own) and those below the range, which says where its stretch of the list begins
// without a word from the other CTAs.  embed_sum_kernel then takes 32 places of the list a CTA, however many ids they are of: rows of ids whose places
// are all among them are written at once, of the others (frequent words, padding) the CTA that is done last adds up the parts in their order, 32 at a
// time.  Other CTAs of the same launch have the copy engine write the rows of ids that do not occur, from zeros in shared memory.
// 8192 tokens, 32000 x 4096 bf16: lookup 15 us, sort 8, sums 58 to 64 (0.8 of the measured copy rate; an id's places all by one row of threads: 171, since one of
// 98 places keeps its threads busy for 23).
#include "embedding.cuh"
#include "../common/fl_ptx.cuh"

namespace fl {
namespace embedding {

constexpr int SORT_THREADS = 1024, SORT_WARPS = SORT_THREADS / 32;
constexpr int RANGE = 512;                       // ids of a sorting CTA
constexpr int BATCH = 8;                         // tokens on their way per sorting thread
constexpr int PART = 32;                         // places of a summing CTA, and parts that are added up at a time
constexpr int ZERO_IDS = 4;                      // ids that a warp looks at for rows of zeros (a table of 32000 x 4096 without tokens: 16 ids 66 us, 8 55, 4 50, 2 52)
constexpr int ZEROS = 8192;                      // bytes of zeros that a copy takes at most

template <typename I>
__device__ __forceinline__ long long token_at(const I* tokens, long long t, long long vocab) {
  const long long id = (long long)tokens[t];
  return id < 0 ? id + vocab : id;               // below -vocab it stays negative
}

// ------------------------------------------------------------------------------------------------------------------ lookup
// tpr threads per row, a power of two; each takes up to 4 packs of a row's stretch.  blockIdx.y: the stretch
template <typename T, int N, typename I>
__global__ void __launch_bounds__(128) embed_kernel(const FlEmbedArgs a, int tpr) {
  const long long t = (long long)blockIdx.x * (128 / tpr) + threadIdx.x / tpr;
  if (t >= a.n) return;
  const int packs = (int)(a.hidden / N), at = blockIdx.y * tpr * 4 + (threadIdx.x & (tpr - 1));
  const long long id = token_at((const I*)a.tokens, t, a.vocab);
  const bool ok = id >= 0 && id < a.vocab;
  if (!ok && a.status != nullptr && at == 0) *a.status = 1;
  const Pack<T, N>* row = reinterpret_cast<const Pack<T, N>*>((const T*)a.table + (ok ? id : 0) * a.table_stride);
  Pack<T, N>* out = reinterpret_cast<Pack<T, N>*>((T*)a.out + t * a.hidden);
  Pack<T, N> x[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (at + j * tpr < packs && ok) x[j] = row[at + j * tpr];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (at + j * tpr >= packs) break;
    float f[N];
    x[j].get(f);
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = ok ? f[i] * a.scale : 0.f;
    x[j].set(f);
    out[at + j * tpr] = x[j];
  }
}

// ------------------------------------------------------------------------------------------------------------------ sort
struct Scratch {
  int* first;       // [vocab + 1]: where an id's places begin in the list
  int2* list;       // [n]: place and id
  int* done;        // [2][parts][2][tiles]: parts (then groups of them) of an id that are there
  float* sums;      // [parts][2][columns]: of the id that a part begins with, and of the one that begins in it and goes on
};
__host__ __device__ inline long long up256(long long x) { return (x + 255) / 256 * 256; }
__host__ __device__ inline long long parts_of(long long n) { return (n + PART - 1) / PART; }
__host__ __device__ inline Scratch scratch_of(void* p, long long n, long long vocab, long long tiles) {
  char* c = (char*)p;
  Scratch s;
  s.first = (int*)c; c += up256((vocab + 1) * 4);
  s.list = (int2*)c; c += up256(n * 8);
  s.done = (int*)c; c += up256(parts_of(n) * 4 * tiles * 4);
  s.sums = (float*)c;
  return s;
}
// threads of a summing CTA, 16 bytes of a row each, and how many of their widths a row has
static int threads_of(long long hidden, int size) {
  int t = 32;
  while (t < 256 && t * 16 < hidden * size) t *= 2;
  return t;
}
static long long tiles_of(long long hidden, int size) { return (hidden * size + threads_of(hidden, size) * 16 - 1) / (threads_of(hidden, size) * 16); }

// exclusive sum over the block; total in *all
__device__ __forceinline__ int block_scan(int x, int* warp_sums, int* all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int y = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int z = __shfl_up_sync(0xffffffffu, y, o);
    if (lane >= o) y += z;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = y;
  __syncthreads();
  int before = 0, sum = 0;
  for (int w = 0; w < SORT_WARPS; ++w) {
    if (w == warp) before = sum;
    sum += warp_sums[w];
  }
  *all = sum;
  return before + y - x;
}

template <typename I>
__global__ void __launch_bounds__(SORT_THREADS) embed_sort_kernel(const FlEmbedArgs a, int tiles) {
  extern __shared__ int counters[];              // [SORT_WARPS][RANGE]
  __shared__ int warp_sums[SORT_WARPS];
  grid_dep_launch();
  const Scratch s = scratch_of(a.scratch, a.n, a.vocab, tiles);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long lo = (long long)blockIdx.x * RANGE, hi = lo + RANGE < a.vocab ? lo + RANGE : a.vocab;
  const I* tokens = (const I*)a.tokens;
  const int each = (int)((a.n + SORT_WARPS - 1) / SORT_WARPS + 31) / 32 * 32;
  const long long begin = (long long)warp * each, end = begin + each < a.n ? begin + each : a.n;
  int* mine = counters + warp * RANGE;
  // a token's id less the first of the range; what is no id at all becomes one behind it
  auto fetch = [&](int* x, long long t0) {
    long long id[BATCH];
#pragma unroll
    for (int j = 0; j < BATCH; ++j)
      if (t0 + j * 32 + lane < end) id[j] = token_at(tokens, t0 + j * 32 + lane, a.vocab);
#pragma unroll
    for (int j = 0; j < BATCH; ++j) x[j] = t0 + j * 32 + lane < end && id[j] >= 0 && id[j] < a.vocab ? (int)(id[j] - lo) : RANGE;
  };
  int x[BATCH];
  fetch(x, begin);                               // a warp of up to 256 tokens keeps them
  for (int i = lane; i < RANGE / 4; i += 32) reinterpret_cast<int4*>(mine)[i] = make_int4(0, 0, 0, 0);
  for (long long i = (long long)blockIdx.x * SORT_THREADS + threadIdx.x; i < parts_of(a.n) * 4 * tiles; i += (long long)gridDim.x * SORT_THREADS) s.done[i] = 0;
  __syncwarp();
  const int ids = (int)(hi - lo);
  int below = 0;
  for (long long t0 = begin; t0 < end; t0 += 32 * BATCH) {
    if (t0 > begin) fetch(x, t0);
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
      below += x[j] < 0;
      if (x[j] >= 0 && x[j] < ids) atomicAdd(&mine[x[j]], 1);
    }
  }
  __syncthreads();
  int base;
  block_scan(below, warp_sums, &base);
  int total = 0;
  if (threadIdx.x < RANGE)
#pragma unroll 8
    for (int w = 0; w < SORT_WARPS; ++w) total += counters[w * RANGE + threadIdx.x];
  int all;
  int first = base + block_scan(total, warp_sums, &all);
  if (threadIdx.x < RANGE) {
    if (threadIdx.x < ids) s.first[lo + threadIdx.x] = first;
#pragma unroll 8
    for (int w = 0; w < SORT_WARPS; ++w) {       // counters become where a warp's places of an id begin
      const int c = counters[w * RANGE + threadIdx.x];
      counters[w * RANGE + threadIdx.x] = first;
      first += c;
    }
  }
  if (threadIdx.x == 0 && hi == a.vocab) s.first[a.vocab] = base + all;
  __syncthreads();
  const bool kept = end - begin <= 32 * BATCH;
  for (long long t0 = begin; t0 < end; t0 += 32 * BATCH) {
    if (!kept) fetch(x, t0);
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
      const bool in = x[j] >= 0 && x[j] < ids;
      if (!__any_sync(0xffffffffu, in)) continue;
      const unsigned same = __match_any_sync(0xffffffffu, in ? x[j] : -1);
      const int rank = __popc(same & ((1u << lane) - 1));
      int at = 0;
      if (in) at = mine[x[j]] + rank;
      __syncwarp();
      if (in) {
        s.list[at] = make_int2((int)(t0 + j * 32 + lane), (int)lo + x[j]);
        if (rank == 0) mine[x[j]] = at + __popc(same);
      }
      __syncwarp();
    }
  }
}

// ------------------------------------------------------------------------------------------------------------------ sums
// A thread has W values of a row, 16 bytes in all, as W / N packs of N values, `apart` values from one another; AHEAD rows are on their way.
template <typename T, int N>
struct Way {
  static constexpr int W = 16 / (int)sizeof(T), C = W / N, AHEAD = C == 1 ? 8 : C == 2 ? 4 : 2;
  static __device__ __forceinline__ void load(Pack<T, N>* x, const T* row, long long col, int apart, long long hidden) {
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (col + c * apart < hidden) x[c] = *reinterpret_cast<const Pack<T, N>*>(row + col + c * apart);
  }
  static __device__ __forceinline__ void add(float* sum, const Pack<T, N>* x, long long col, int apart, long long hidden) {
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (col + c * apart < hidden) {
        float f[N];
        x[c].get(f);
#pragma unroll
        for (int k = 0; k < N; ++k) sum[c * N + k] += f[k];
      }
  }
  static __device__ __forceinline__ void store(T* row, const float* sum, float scale, long long col, int apart, long long hidden) {
#pragma unroll
    for (int c = 0; c < C; ++c)
      if (col + c * apart < hidden) {
        Pack<T, N> y;
        float f[N];
#pragma unroll
        for (int k = 0; k < N; ++k) f[k] = sum[c * N + k] * scale;
        y.set(f);
        *reinterpret_cast<Pack<T, N>*>(row + col + c * apart) = y;
      }
  }
};

// n zeros, by the copy engine as far as whole 16 bytes go
template <typename T>
__device__ __forceinline__ void put_zeros(T* to, long long n, const uint4* zeros) {
  while (n > 0 && ((uintptr_t)to & 15)) { *to++ = T{}; --n; }
  char* at = reinterpret_cast<char*>(to);
  long long bytes = n * (long long)sizeof(T);
  while (bytes >= 16) {
    const uint32_t k = (uint32_t)(bytes < ZEROS ? bytes & ~15ll : ZEROS);
    bulk_store(at, zeros, k);
    at += k;
    bytes -= k;
  }
  for (to = reinterpret_cast<T*>(at); bytes > 0; bytes -= sizeof(T)) *to++ = T{};
}

// The rows of ids without a place among ZERO_IDS for each warp: runs of them at a time.
template <typename T>
__device__ __forceinline__ void zero_rows(const FlEmbedArgs& a, const Scratch& s, unsigned block) {
  __shared__ __align__(128) uint4 zeros[ZEROS / 16];
  for (int i = threadIdx.x; i < ZEROS / 16; i += blockDim.x) zeros[i] = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  __syncthreads();
  const int lane = threadIdx.x & 31;
  const long long v0 = ((long long)block * (blockDim.x / 32) + threadIdx.x / 32) * ZERO_IDS;
  const int f = v0 + lane <= a.vocab && lane <= ZERO_IDS ? s.first[v0 + lane] : -1, next = __shfl_down_sync(0xffffffffu, f, 1);
  unsigned none = __ballot_sync(0xffffffffu, lane < ZERO_IDS && v0 + lane < a.vocab && f == next);
  if (lane != 0) return;
  while (none) {
    const int from = __ffs(none) - 1, n = __ffs(~(none >> from)) - 1;
    put_zeros((T*)a.dtable + (v0 + from) * a.hidden, n * a.hidden, zeros);
    none &= ~(((1u << n) - 1) << from);
  }
  tma_store_commit();
  tma_store_wait_read<0>();
}

// Whether the CTA is the last of `all` that come here with this counter; then it sees what they have written.
__device__ __forceinline__ bool last_of(int* counter, int all, int* shared) {
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) *shared = atomicAdd(counter, 1) == all - 1;
  __syncthreads();
  const bool last = *shared;
  if (last) __threadfence();
  return last;
}

// blockIdx.x: the zeros' CTAs, which then write for as long as the others sum; then a CTA per part and tile of blockDim.x * W columns.
template <typename T, int N>
__global__ void __launch_bounds__(256, 3) embed_sum_kernel(const FlEmbedArgs a, int zero_blocks, int tiles) {
  using way = Way<T, N>;
  __shared__ int2 list[PART + 2];                // the place before the part's, its own, the one behind them
  __shared__ int last_one;
  const Scratch s = scratch_of(a.scratch, a.n, a.vocab, tiles);
  grid_dep_wait();
  if (blockIdx.x < (unsigned)zero_blocks) {
    zero_rows<T>(a, s, blockIdx.x);
    return;
  }
  const int part = (blockIdx.x - zero_blocks) / tiles, tile = (blockIdx.x - zero_blocks) % tiles;
  const long long col = (long long)tile * blockDim.x * way::W + threadIdx.x * N, columns = (long long)tiles * blockDim.x * way::W;
  const int apart = blockDim.x * N, total = s.first[a.vocab], b = part * PART, n = min(PART, total - b);
  if (n <= 0) return;                            // tokens outside the vocabulary have no place
  for (int i = threadIdx.x; i < n + 2; i += blockDim.x) list[i] = b + i > 0 && b + i <= total ? s.list[b + i - 1] : make_int2(-1, -1);
  __syncthreads();
  const T* dout = (const T*)a.dout;
  T* dtable = (T*)a.dtable;
  float sum[way::W] = {};
  int begun = -1, goes_on = -1;                  // ids of which there is a part here: begun before, or at its beginning and going on; begun in it
  for (int i = 0; i < n; i += way::AHEAD) {
    Pack<T, N> x[way::AHEAD][way::C];
#pragma unroll
    for (int j = 0; j < way::AHEAD; ++j)
      if (i + j < n) way::load(x[j], dout + (long long)list[i + j + 1].x * a.hidden, col, apart, a.hidden);
#pragma unroll
    for (int j = 0; j < way::AHEAD; ++j) {
      if (i + j >= n) break;
      way::add(sum, x[j], col, apart, a.hidden);
      const int id = list[i + j + 1].y;
      if (i + j + 1 < n && list[i + j + 2].y == id) continue;
      const bool from_here = list[0].y != id, to_here = i + j + 1 < n || list[n + 1].y != id;
      if (from_here && to_here) {
        way::store(dtable + id * a.hidden, sum, a.scale, col, apart, a.hidden);
      } else if (!from_here || list[1].y == id) {
        begun = id;
        float* to = s.sums + (long long)part * 2 * columns + tile * blockDim.x * way::W + threadIdx.x;
#pragma unroll
        for (int k = 0; k < way::W; ++k) __stcg(to + k * blockDim.x, sum[k]);
      } else {
        goes_on = id;
        float* to = s.sums + ((long long)part * 2 + 1) * columns + tile * blockDim.x * way::W + threadIdx.x;
#pragma unroll
        for (int k = 0; k < way::W; ++k) __stcg(to + k * blockDim.x, sum[k]);
      }
#pragma unroll
      for (int k = 0; k < way::W; ++k) sum[k] = 0.f;
    }
  }
  const long long all_parts = parts_of(a.n);
  for (int which = 0; which < 2; ++which) {
    const int id = which == 0 ? begun : goes_on;
    if (id < 0) continue;
    const int from = s.first[id], p0 = from / PART, p1 = (s.first[id + 1] - 1) / PART, slot0 = from > p0 * PART;
    auto at = [&](int p) { return s.sums + ((long long)p * 2 + (p == p0 ? slot0 : 0)) * columns + tile * blockDim.x * way::W + threadIdx.x; };
    auto counter = [&](int level, int p) { return s.done + ((level * all_parts + p) * 2 + (p == p0 ? slot0 : 0)) * tiles + tile; };
    auto gather = [&](int first, int last, int step) {          // parts first, first + step (rounded down to step) ... last
#pragma unroll
      for (int k = 0; k < way::W; ++k) sum[k] = 0.f;
      for (int p = first; p <= last;) {
        float y[4][way::W];
        int q = p;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (q <= last)
#pragma unroll
            for (int k = 0; k < way::W; ++k) y[j][k] = __ldcg(at(q) + k * blockDim.x);
          q = (q / step + 1) * step;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (p <= last)
#pragma unroll
            for (int k = 0; k < way::W; ++k) sum[k] += y[j][k];
          p = (p / step + 1) * step;
        }
      }
    };
    const int g0 = max(part / PART * PART, p0), g1 = min(part / PART * PART + PART - 1, p1);
    if (!last_of(counter(0, g0), g1 - g0 + 1, &last_one)) continue;
    gather(g0, g1, 1);
    if (p0 / PART != p1 / PART) {
#pragma unroll
      for (int k = 0; k < way::W; ++k) __stcg(at(g0) + k * blockDim.x, sum[k]);
      if (!last_of(counter(1, p0), p1 / PART - p0 / PART + 1, &last_one)) continue;
      gather(p0, p1, PART);
    }
    way::store(dtable + id * a.hidden, sum, a.scale, col, apart, a.hidden);
  }
}

// the widest access that all rows allow, in values
template <typename T>
static int pack_of(long long hidden, long long stride, const void* p, const void* q) {
  const unsigned long long all = (unsigned long long)(uintptr_t)p | (uintptr_t)q | (unsigned long long)(hidden * sizeof(T)) | (unsigned long long)(stride * sizeof(T)) | 16;
  return (int)((all & -all) / sizeof(T));
}
template <typename T, typename F>
static int by_pack(int n, F&& f) {
  switch (n) {
    case 8: if constexpr (sizeof(T) == 2) return f(std::integral_constant<int, 8>{}); break;
    case 4: return f(std::integral_constant<int, 4>{});
    case 2: return f(std::integral_constant<int, 2>{});
    case 1: return f(std::integral_constant<int, 1>{});
  }
  return -1;
}

}  // namespace embedding
}  // namespace fl

using namespace fl::embedding;

static int embed_check(const FlEmbedArgs* a) {
  return a->n < 0 || a->n >= INT32_MAX || a->vocab < 1 || a->vocab >= INT32_MAX || a->hidden < 1 || a->hidden >= INT32_MAX ||
                 (a->token_bytes != 4 && a->token_bytes != 8) || a->vocab > (INT64_MAX >> 3) / a->hidden ? -1 : 0;
}

extern "C" long long fl_embed_scratch(long long n, long long vocab, long long hidden) {
  if (n < 0 || n >= INT32_MAX || vocab < 1 || vocab >= INT32_MAX || hidden < 1 || hidden >= INT32_MAX) return -1;
  const long long most = (hidden * 4 + 511) / 512;                       // tiles of 32 threads, fp32
  const Scratch s = scratch_of(nullptr, n, vocab, most);
  return (long long)((char*)s.sums - (char*)nullptr) + parts_of(n) * 2 * (hidden + 2048) * 4;
}

extern "C" int fl_embed(int dtype, const FlEmbedArgs* a, cudaStream_t stream) {
  if (embed_check(a) || a->table_stride < a->hidden) return -1;
  if (a->n == 0) return 0;
  return fl_by_dtype(dtype, [&](auto type) {
    using T = decltype(type);
    return by_pack<T>(pack_of<T>(a->hidden, a->table_stride, a->table, a->out), [&](auto width) {
      constexpr int N = decltype(width)::value;
      const long long packs = a->hidden / N;
      int tpr = 1;
      while (tpr < 128 && tpr * 4 < packs) tpr *= 2;
      const long long y = (packs + tpr * 4 - 1) / (tpr * 4), x = (a->n + 128 / tpr - 1) / (128 / tpr);
      if (y > 65535) return -1;
      const dim3 grid((unsigned)x, (unsigned)y);
      if (a->token_bytes == 8) embed_kernel<T, N, long long><<<grid, 128, 0, stream>>>(*a, tpr);
      else embed_kernel<T, N, int><<<grid, 128, 0, stream>>>(*a, tpr);
      return (int)cudaGetLastError();
    });
  });
}

extern "C" int fl_embed_grad(int dtype, const FlEmbedArgs* a, cudaStream_t stream) {
  if (embed_check(a)) return -1;
  return fl_by_dtype(dtype, [&](auto type) {
    using T = decltype(type);
    return by_pack<T>(pack_of<T>(a->hidden, a->hidden, a->dout, a->dtable), [&](auto width) {
      constexpr int N = decltype(width)::value;
      const int threads = threads_of(a->hidden, sizeof(T));
      const long long tiles = tiles_of(a->hidden, sizeof(T)), ranges = (a->vocab + RANGE - 1) / RANGE, ids = threads / 32 * ZERO_IDS,
                      zero_blocks = (a->vocab + ids - 1) / ids, blocks = zero_blocks + parts_of(a->n) * tiles;
      if (blocks > INT32_MAX) return -1;
      constexpr int bytes = SORT_WARPS * RANGE * 4;
      auto sort = a->token_bytes == 8 ? embed_sort_kernel<long long> : embed_sort_kernel<int>;
      cudaError_t e = cudaFuncSetAttribute(sort, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
      if (e != cudaSuccess) return (int)e;
      sort<<<(unsigned)ranges, SORT_THREADS, bytes, stream>>>(*a, (int)tiles);
      cudaLaunchAttribute at[1];
      at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
      at[0].val.programmaticStreamSerializationAllowed = 1;
      cudaLaunchConfig_t c = {};
      c.gridDim = dim3((unsigned)blocks); c.blockDim = dim3(threads); c.stream = stream; c.attrs = at; c.numAttrs = 1;
      e = cudaLaunchKernelEx(&c, embed_sum_kernel<T, N>, *a, (int)zero_blocks, (int)tiles);
      return (int)(e != cudaSuccess ? e : cudaGetLastError());
    });
  });
}

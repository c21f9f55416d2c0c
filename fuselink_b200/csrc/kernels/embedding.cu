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
// without a word from the other CTAs.  embed_sum_kernel then adds rows up: ids of up to 32 places by a warp each, up to 1024 by a CTA, and
// more of them (padding, say) by CTAs that take 1024 places each; the one that is done last adds up the parts in their order.
#include "embedding.cuh"
#include "../common/fl_ptx.cuh"

namespace fl {
namespace embedding {

constexpr int SORT_THREADS = 1024, SORT_WARPS = SORT_THREADS / 32;
constexpr int RANGE = 512;                       // ids of a sorting CTA
constexpr int SUM_WARPS = 8, SUM_THREADS = SUM_WARPS * 32;
constexpr int GROUP = 64;                        // ids of a summing CTA
constexpr int FEW = 32;                          // places of an id that a warp adds up alone
constexpr int MANY = 1024;                       // places that a CTA adds up alone
constexpr int AHEAD = 8;                         // rows on their way per warp

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
#pragma unroll
    for (int i = 0; i < N; ++i) x[j].v[i] = from_f32<T>(ok ? to_f32(x[j].v[i]) * a.scale : 0.f);
    out[at + j * tpr] = x[j];
  }
}

// ------------------------------------------------------------------------------------------------------------------ sort
struct Scratch {
  int* first;       // [vocab + 1]: where an id's places begin in the list
  int* places;      // [n]
  int* done;        // [parts][slices]: parts of an id of many places that are there
  float* parts;     // [parts][2][hidden]
};
__host__ __device__ inline long long up256(long long x) { return (x + 255) / 256 * 256; }
__host__ __device__ inline long long parts_of(long long n) { return n > MANY ? (n + MANY - 1) / MANY : 0; }
__host__ __device__ inline Scratch scratch_of(void* p, long long n, long long vocab, long long hidden) {
  char* c = (char*)p;
  Scratch s;
  s.first = (int*)c; c += up256((vocab + 1) * 4);
  s.places = (int*)c; c += up256(n * 4);
  s.done = (int*)c; c += up256(parts_of(n) * ((hidden + 31) / 32) * 4);
  s.parts = (float*)c;
  return s;
}

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
__global__ void __launch_bounds__(SORT_THREADS) embed_sort_kernel(const FlEmbedArgs a, int slices) {
  extern __shared__ int counters[];              // [SORT_WARPS][RANGE]
  __shared__ int warp_sums[SORT_WARPS];
  const Scratch s = scratch_of(a.scratch, a.n, a.vocab, a.hidden);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long lo = (long long)blockIdx.x * RANGE, hi = lo + RANGE < a.vocab ? lo + RANGE : a.vocab;
  const I* tokens = (const I*)a.tokens;
  for (int i = threadIdx.x; i < SORT_WARPS * RANGE; i += SORT_THREADS) counters[i] = 0;
  for (long long i = (long long)blockIdx.x * SORT_THREADS + threadIdx.x; i < parts_of(a.n) * slices; i += (long long)gridDim.x * SORT_THREADS) s.done[i] = 0;
  __syncthreads();
  const long long each = ((a.n + SORT_WARPS - 1) / SORT_WARPS + 31) / 32 * 32, begin = warp * each, end = begin + each < a.n ? begin + each : a.n;
  int* mine = counters + warp * RANGE;
  int below = 0;
  for (long long t = begin + lane; t < end; t += 32) {
    const long long id = token_at(tokens, t, a.vocab);
    below += id >= 0 && id < lo;
    if (id >= lo && id < hi) atomicAdd(&mine[id - lo], 1);
  }
  __syncthreads();
  int base;
  block_scan(below, warp_sums, &base);
  int total = 0;
  if (threadIdx.x < RANGE)
    for (int w = 0; w < SORT_WARPS; ++w) {       // counters become offsets of the warps within an id
      const int c = counters[w * RANGE + threadIdx.x];
      counters[w * RANGE + threadIdx.x] = total;
      total += c;
    }
  int all;
  const int first = base + block_scan(total, warp_sums, &all);
  if (threadIdx.x < RANGE) {
    for (int w = 0; w < SORT_WARPS; ++w) counters[w * RANGE + threadIdx.x] += first;
    if (lo + threadIdx.x < hi) s.first[lo + threadIdx.x] = first;
  }
  if (threadIdx.x == 0 && hi == a.vocab) s.first[a.vocab] = base + all;
  __syncthreads();
  for (long long t0 = begin; t0 < end; t0 += 32) {
    const long long t = t0 + lane, id = t < end ? token_at(tokens, t, a.vocab) : -1;
    const bool in = id >= lo && id < hi;
    if (__ballot_sync(0xffffffffu, in)) {
      const unsigned same = __match_any_sync(0xffffffffu, in ? (int)(id - lo) : -1);
      if (in) {
        const int rank = __popc(same & ((1u << lane) - 1));
        const int at = mine[id - lo] + rank;
        s.places[at] = (int)t;
        __syncwarp(same);
        if (rank == 0) mine[id - lo] = at + __popc(same);
      }
      __syncwarp();
    }
  }
}

// ------------------------------------------------------------------------------------------------------------------ sums
template <typename T, int N>
__device__ __forceinline__ void add_rows(float* sum, const T* dout, long long hidden, const int* places, int n, long long col, bool live) {
  for (int i = 0; i < n; i += AHEAD) {
    Pack<T, N> x[AHEAD];
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (i + j < n && live) x[j] = *reinterpret_cast<const Pack<T, N>*>(dout + (long long)places[i + j] * hidden + col);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j)
      if (i + j < n && live)
#pragma unroll
        for (int k = 0; k < N; ++k) sum[k] += to_f32(x[j].v[k]);
  }
}
template <typename T, int N>
__device__ __forceinline__ void put_row(T* to, const float* sum, float scale) {
  Pack<T, N> y;
#pragma unroll
  for (int k = 0; k < N; ++k) y.v[k] = from_f32<T>(sum[k] * scale);
  *reinterpret_cast<Pack<T, N>*>(to) = y;
}
// the warps' sums, added up in the warps' order by the first warp
template <int N>
__device__ __forceinline__ void join_warps(float* sum, float (*shared)[32 * N]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; ++k) shared[warp][k * 32 + lane] = sum[k];
  __syncthreads();
  if (warp == 0)
#pragma unroll
    for (int k = 0; k < N; ++k)
      for (int w = 1; w < SUM_WARPS; ++w) sum[k] += shared[w][k * 32 + lane];
}

// blockIdx.x: the ids' group, and behind the groups the parts of 1024 places; blockIdx.y: the slice of 32 * N columns
template <typename T, int N>
__global__ void __launch_bounds__(SUM_THREADS) embed_sum_kernel(const FlEmbedArgs a, int groups) {
  __shared__ float shared[SUM_WARPS][32 * N];
  __shared__ int first[GROUP + 1];
  __shared__ int last_one;
  const Scratch s = scratch_of(a.scratch, a.n, a.vocab, a.hidden);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long col = ((long long)blockIdx.y * 32 + lane) * N;
  const bool live = col < a.hidden;
  const T* dout = (const T*)a.dout;
  T* dtable = (T*)a.dtable;
  if (blockIdx.x < groups) {
    const long long v0 = (long long)blockIdx.x * GROUP;
    const int ids = (int)(a.vocab - v0 < GROUP ? a.vocab - v0 : GROUP);
    if (threadIdx.x <= ids) first[threadIdx.x] = s.first[v0 + threadIdx.x];
    __syncthreads();
    for (int r = warp; r < ids; r += SUM_WARPS) {
      const int n = first[r + 1] - first[r];
      if (n > FEW) continue;
      float sum[N] = {};
      add_rows<T, N>(sum, dout, a.hidden, s.places + first[r], n, col, live);
      if (live) put_row<T, N>(dtable + (v0 + r) * a.hidden + col, sum, a.scale);
    }
    for (int r = 0; r < ids; ++r) {
      const int n = first[r + 1] - first[r];
      if (n <= FEW || n > MANY) continue;
      const int each = (n + SUM_WARPS - 1) / SUM_WARPS, b = warp * each;
      float sum[N] = {};
      add_rows<T, N>(sum, dout, a.hidden, s.places + first[r] + b, max(0, min(each, n - b)), col, live);
      join_warps<N>(sum, shared);
      if (warp == 0 && live) put_row<T, N>(dtable + (v0 + r) * a.hidden + col, sum, a.scale);
    }
    return;
  }
  // places [b, e) of the list: those of ids with more than MANY, of which there are at most two here, the first's and the last's
  const int part = blockIdx.x - groups, total = s.first[a.vocab], b = part * MANY, e = min(b + MANY, total);
  if (b >= e) return;
  for (int which = 0; which < 2; ++which) {
    const int place = s.places[which == 0 ? b : e - 1];
    const long long id = a.token_bytes == 8 ? token_at((const long long*)a.tokens, place, a.vocab) : token_at((const int*)a.tokens, place, a.vocab);
    const int from = s.first[id], to = s.first[id + 1];
    if (to - from <= MANY) continue;
    if (which == 1 && from <= b) continue;                             // the same id as at the part's beginning
    const int p0 = max(from, b), n = min(to, e) - p0, each = (n + SUM_WARPS - 1) / SUM_WARPS, off = warp * each;
    float sum[N] = {};
    add_rows<T, N>(sum, dout, a.hidden, s.places + p0 + off, max(0, min(each, n - off)), col, live);
    join_warps<N>(sum, shared);
    if (warp == 0 && live)
#pragma unroll
      for (int k = 0; k < N; ++k) __stcg(&s.parts[((long long)part * 2 + which) * a.hidden + col + k], sum[k]);
    const int p_first = from / MANY, parts = (to - 1) / MANY - p_first + 1;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) last_one = atomicAdd(&s.done[(long long)p_first * gridDim.y + blockIdx.y], 1) == parts - 1;
    __syncthreads();
    if (!last_one) continue;
    __threadfence();
    const int per = (parts + SUM_WARPS - 1) / SUM_WARPS;
#pragma unroll
    for (int k = 0; k < N; ++k) sum[k] = 0.f;
    for (int i = warp * per; i < min((warp + 1) * per, parts); ++i) {
      const int slot = i == 0 && from > p_first * MANY;                // only in its first part may others stand before it
      if (live)
#pragma unroll
        for (int k = 0; k < N; ++k) sum[k] += __ldcg(&s.parts[((long long)(p_first + i) * 2 + slot) * a.hidden + col + k]);
    }
    join_warps<N>(sum, shared);
    if (warp == 0 && live) put_row<T, N>(dtable + id * a.hidden + col, sum, a.scale);
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
  const Scratch s = scratch_of(nullptr, n, vocab, hidden);
  return (long long)((char*)s.parts - (char*)nullptr) + parts_of(n) * 2 * hidden * 4;
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
      const long long slices = (a->hidden + 32 * N - 1) / (32 * N), groups = (a->vocab + GROUP - 1) / GROUP;
      if (slices > 65535) return -1;
      constexpr int bytes = SORT_WARPS * RANGE * 4;
      const unsigned ranges = (unsigned)((a->vocab + RANGE - 1) / RANGE);
      auto sort = a->token_bytes == 8 ? embed_sort_kernel<long long> : embed_sort_kernel<int>;
      cudaError_t e = cudaFuncSetAttribute(sort, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
      if (e != cudaSuccess) return (int)e;
      sort<<<ranges, SORT_THREADS, bytes, stream>>>(*a, (int)slices);
      embed_sum_kernel<T, N><<<dim3((unsigned)(groups + parts_of(a->n)), (unsigned)slices), SUM_THREADS, 0, stream>>>(*a, (int)groups);
      return (int)cudaGetLastError();
    });
  });
}

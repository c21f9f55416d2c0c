// A cache in 8 bits: e4m3 codes with one scale per page and KV head.
//
// Scales are powers of two.  A code's value is then exact, a page's codes follow a scale that grows with nothing lost but bits below
// e4m3's smallest number, and e4m3's precision does not depend on where in its binade the largest value lies.
#include "kv8.cuh"
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>
#include <initializer_list>
#include "../common/fl_ptx.cuh"
#include "thin_gemm.cuh"

namespace fl {
namespace kv8 {

template <typename T> struct Typed;
template <> struct Typed<__nv_bfloat16> {
  static __device__ __forceinline__ float2 f2(uint32_t w) { return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&w)); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
};
template <> struct Typed<__half> {
  static __device__ __forceinline__ float2 f2(uint32_t w) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
};
template <typename T>
__device__ __forceinline__ void unpack(uint4 u, float (&v)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = Typed<T>::f2(w[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
template <typename T>
__device__ __forceinline__ uint4 packed(const float (&v)[8]) {
  return make_uint4(Typed<T>::pack(v[0], v[1]), Typed<T>::pack(v[2], v[3]), Typed<T>::pack(v[4], v[5]), Typed<T>::pack(v[6], v[7]));
}

// two codes as halves, which hold every e4m3 value; the low byte becomes the low half
__device__ __forceinline__ uint32_t halves(uint32_t codes) {
  uint32_t h;
  asm("{.reg .b16 c, d; mov.b32 {c, d}, %1; cvt.rn.f16x2.e4m3x2 %0, c;}" : "=r"(h) : "r"(codes));
  return h;
}
// the code of a in the low byte, of b in the next; |a|, |b| within 448, or NaN
__device__ __forceinline__ uint32_t codes(float a, float b) {
  uint16_t c;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(c) : "f"(b), "f"(a));
  return c;
}
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) { return codes(a, b) | codes(c, d) << 16; }

// bits of the scale for a largest magnitude with these bits (see FlKv8): 448 = 1.75 * 2^8
__device__ __forceinline__ uint32_t scale_bits(uint32_t amax) {
  const int e = (int)(amax >> 23) - 8 + ((amax & 0x7fffffu) > 0x600000u ? 1 : 0);
  return (uint32_t)max(e, 27) << 23;
}

__device__ __forceinline__ void note(int* status, int what) {
  if (status != nullptr) *reinterpret_cast<volatile int*>(status) = what;
}

// the page at position `page` of request b's row, or -1
__device__ __forceinline__ int page_id(const FlKv8& kv, int b, int page) {
  int id = __ldg(kv.block_table + (long long)b * kv.table_stride + page);
  if (id < 0) id += kv.num_blocks;
  return id >= 0 && id < kv.num_blocks ? id : -1;
}

// ---- page write -----------------------------------------------------------------------------------------------------------
// Bound by memory: new tokens are read once, written once in the model's type and once in 8 bits.  A warp has one page of one head, of keys or
// of values: lane (t, c) takes columns 8 c .. 8 c + 7 of the first half of a token's row and the matching ones of the second (the pairs that the
// rotation mixes), 32 / (dim / 16) tokens at a time.  Four such steps, a page of 16 tokens, stay in registers between finding the largest
// magnitude and writing codes; larger pages are read again.
constexpr int STEPS = 4;

struct WriteArgs {
  const void* src; void* out; const void* bias; const float* rope; long long rope_rows;
  const long long* start; const long long* pos; const long long* counts;
  int batch, tokens, heads, reach;            // reach: pages that a request's tokens can lie in
  // pack: pages of 16 bits in place of rows
  const void* src_v; const int* src_table; int src_stride, src_blocks;
};

template <typename T>
struct Columns {                              // of one token: the two vectors that a lane takes
  uint4 lo, hi;
  __device__ __forceinline__ void turn(const T* bias, const float* cs, int half) {
    if (bias == nullptr && cs == nullptr) return;
    float a[8], b[8];
    unpack<T>(lo, a);
    unpack<T>(hi, b);
    if (bias != nullptr) {
      float e[8];
      unpack<T>(ld_v4(bias), e);
#pragma unroll
      for (int j = 0; j < 8; ++j) a[j] += e[j];
      unpack<T>(ld_v4(bias + half), e);
#pragma unroll
      for (int j = 0; j < 8; ++j) b[j] += e[j];
    }
    if (cs != nullptr) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {             // each product rounded, as separate operations would
        const float co = cs[j], si = cs[half + j], x = a[j], y = b[j];
        a[j] = __fsub_rn(__fmul_rn(x, co), __fmul_rn(y, si));
        b[j] = __fadd_rn(__fmul_rn(y, co), __fmul_rn(x, si));
      }
    }
    lo = packed<T>(a);
    hi = packed<T>(b);
  }
  __device__ __forceinline__ uint32_t amax() const {             // bits of the largest finite magnitude
    float a[8], b[8];
    unpack<T>(lo, a);
    unpack<T>(hi, b);
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      m = fmaxf(m, fabsf(a[j]) < INFINITY ? fabsf(a[j]) : 0.f);
      m = fmaxf(m, fabsf(b[j]) < INFINITY ? fabsf(b[j]) : 0.f);
    }
    return __float_as_uint(m);
  }
  static __device__ __forceinline__ uint2 code8(uint4 u, float inv) {
    float v[8];
    unpack<T>(u, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = fabsf(v[j]) < INFINITY ? v[j] * inv : NAN;
    return make_uint2(codes4(v[0], v[1], v[2], v[3]), codes4(v[4], v[5], v[6], v[7]));
  }
};

// One page of one head by one warp.  row(i): token i of the `n` that are new, i.e. its vector of this lane's columns; given(i, columns): what becomes
// of them besides.  again(i): the same after given().
template <typename T, typename Row, typename Given, typename Again>
__device__ __forceinline__ void write_page(uint8_t* page, float* scale, bool there, int lead, int n, int dim, Row row, Given given, Again again) {
  const int lane = threadIdx.x & 31, chunks = dim / 16, at_once = 32 / chunks, tk = lane / chunks, c = lane - tk * chunks;
  const bool on = tk < at_once;
  const int steps = (n + at_once - 1) / at_once;
  Columns<T> col[STEPS];
  uint32_t amax = 0;
  for (int s0 = 0; s0 < steps; s0 += STEPS) {
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const int i = (s0 + s) * at_once + tk;
      if (on && i < n) col[s] = row(i, c);
    }
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const int i = (s0 + s) * at_once + tk;
      if (on && i < n) {
        given(i, c, col[s]);
        amax = max(amax, col[s].amax());
      }
    }
  }
  if (!there) return;
  amax = __reduce_max_sync(0xffffffffu, amax);
  float sc = __uint_as_float(scale_bits(amax));
  if (lead > 0) {
    const float was = *scale;
    sc = fmaxf(sc, was);
    if (was != sc) {                            // the page's earlier codes follow
      const float f = was / sc;
      for (int i = lane * 16; i < lead * dim; i += 32 * 16) {
        const uint4 u = ld_v4(page + i);
        uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t h0 = halves(w[j]), h1 = halves(w[j] >> 16);
          const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&h0)), b = __half22float2(*reinterpret_cast<const __half2*>(&h1));
          w[j] = codes4(a.x * f, a.y * f, b.x * f, b.y * f);
        }
        st_v4(page + i, make_uint4(w[0], w[1], w[2], w[3]));
      }
    }
  }
  __syncwarp();                                 // every lane has read the scale
  if (lane == 0) *scale = sc;
  const float inv = __uint_as_float((254u << 23) - __float_as_uint(sc));      // 1 / 2^e
  for (int s0 = 0; s0 < steps; s0 += STEPS) {
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const int i = (s0 + s) * at_once + tk;
      if (on && i < n) {
        if (steps > STEPS) col[s] = again(i, c);
        uint8_t* p = page + (lead + i) * dim + 8 * c;
        *reinterpret_cast<uint2*>(p) = Columns<T>::code8(col[s].lo, inv);
        *reinterpret_cast<uint2*>(p + dim / 2) = Columns<T>::code8(col[s].hi, inv);
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(128) write_kernel(const WriteArgs a, const FlKv8 kv, long long page_units, long long units) {
  grid_dep_launch();
  grid_dep_wait();
  const int lane = threadIdx.x & 31, D = kv.dim, half = D / 2, chunks = D / 16, all = a.heads + 2 * kv.heads, bs = kv.block_size;
  const long long cap = (long long)kv.table_stride * bs;
  const T* src = reinterpret_cast<const T*>(a.src);
  T* out = reinterpret_cast<T*>(a.out);
  const T* bias = reinterpret_cast<const T*>(a.bias);
  for (long long u = (long long)blockIdx.x * 4 + (threadIdx.x >> 5); u < units; u += (long long)gridDim.x * 4) {
    if (u < page_units) {
      const bool is_v = u & 1;
      const long long r = u >> 1;
      const int kh = (int)(r % kv.heads), rest = (int)(r / kv.heads), pi = rest % a.reach, b = rest / a.reach;
      const long long st = a.start[b];
      const int n = a.counts ? (int)min(max(a.counts[b], 0ll), (long long)a.tokens) : a.tokens;
      // tokens [from, to) of the request's are in this page
      int from, to, lead, page;
      bool inside = st >= 0 && st + n <= cap;
      if (inside) {
        page = (int)st / bs + pi;
        lead = pi == 0 ? (int)st % bs : 0;
        from = pi == 0 ? 0 : page * bs - (int)st;
        to = min(n, (page + 1) * bs - (int)st);
      } else {                                  // no pages to write to: the rows are still turned
        page = 0; lead = 0;
        from = (int)min((long long)pi * bs, (long long)n);
        to = min(n, from + bs);
        if (n > 0 && lane == 0) note(kv.status, FL_DEC_BAD_POSITION);
      }
      if (from >= to) continue;
      const int id = inside ? page_id(kv, b, page) : -1;
      if (inside && id < 0 && lane == 0) note(kv.status, FL_DEC_BAD_PAGE);
      const int head = a.heads + (is_v ? kv.heads : 0) + kh;
      const long long turn = (a.pos ? a.pos[b] : st) + from;
      const long long first = ((long long)b * a.tokens + from) * all + head;
      const long long cell = ((long long)kv.layer * kv.num_blocks + max(id, 0)) * kv.heads + kh;
      uint8_t* dst = reinterpret_cast<uint8_t*>(is_v ? kv.v : kv.k) + cell * bs * D;
      const bool rotate = a.rope != nullptr && !is_v;
      const T* bias_h = bias ? bias + head * D : nullptr;
      write_page<T>(
          dst, (is_v ? kv.v_scale : kv.k_scale) + cell, id >= 0, lead, to - from, D,
          [&](int i, int c) {
            const T* p = src + (first + (long long)i * all) * D + 8 * c;
            return Columns<T>{ld_v4(p), ld_v4(p + half)};
          },
          [&](int i, int c, Columns<T>& col) {
            const float* cs = nullptr;
            if (rotate) {
              if (turn + i >= 0 && turn + i < a.rope_rows) cs = a.rope + (turn + i) * D + 8 * c;
              else note(kv.status, FL_DEC_BAD_POSITION);
            }
            col.turn(bias_h ? bias_h + 8 * c : nullptr, cs, half);
            T* p = out + (first + (long long)i * all) * D + 8 * c;
            st_v4(p, col.lo);
            st_v4(p + half, col.hi);
          },
          [&](int i, int c) {
            const T* p = out + (first + (long long)i * all) * D + 8 * c;
            return Columns<T>{ld_v4(p), ld_v4(p + half)};
          });
      continue;
    }
    // queries; and, where rows may be left out, those rows as they came
    const int per_row = (a.counts ? all : a.heads) * chunks;
    const long long item = (u - page_units) * 32 + lane;
    const long long n = item / per_row;
    if (n >= (long long)a.batch * a.tokens) continue;
    const int r = (int)(item - n * per_row), head = r / chunks, c = r - head * chunks;
    const int b = (int)(n / a.tokens), t = (int)(n - (long long)b * a.tokens);
    const bool in = a.counts == nullptr || t < a.counts[b];
    if (in && head >= a.heads) continue;
    if ((!in || (bias == nullptr && a.rope == nullptr)) && src == out) continue;
    const long long at = (n * all + head) * D + 8 * c;
    Columns<T> col{ld_v4(src + at), ld_v4(src + at + half)};
    if (in) {
      const long long turn = (a.pos ? a.pos[b] : a.start[b]) + t;
      const float* cs = nullptr;
      if (a.rope != nullptr) {
        if (turn >= 0 && turn < a.rope_rows) cs = a.rope + turn * D + 8 * c;
        else note(kv.status, FL_DEC_BAD_POSITION);
      }
      col.turn(bias ? bias + head * D + 8 * c : nullptr, cs, half);
    }
    st_v4(out + at, col.lo);
    st_v4(out + at + half, col.hi);
  }
}

template <typename T>
__global__ void __launch_bounds__(128) pack_kernel(const WriteArgs a, const FlKv8 kv, long long units) {
  const int D = kv.dim, half = D / 2, bs = kv.block_size;
  for (long long u = (long long)blockIdx.x * 4 + (threadIdx.x >> 5); u < units; u += (long long)gridDim.x * 4) {
    const bool is_v = u & 1;
    long long r = u >> 1;
    const int kh = (int)(r % kv.heads);
    r /= kv.heads;
    const int page = (int)(r % a.reach);
    r /= a.reach;
    const int b = (int)(r % a.batch), layer = (int)(r / a.batch);
    const long long len = a.start[b];
    if (len <= (long long)page * bs) continue;
    const bool lead_lane = (threadIdx.x & 31) == 0;
    if (page == 0 && len > (long long)a.reach * bs && lead_lane) note(kv.status, FL_DEC_BAD_POSITION);
    const int n = (int)min(len - (long long)page * bs, (long long)bs);
    int from = a.src_table[(long long)b * a.src_stride + page];
    if (from < 0) from += a.src_blocks;
    const int id = page_id(kv, b, page);
    if (from < 0 || from >= a.src_blocks || id < 0) {
      if (lead_lane) note(kv.status, FL_DEC_BAD_PAGE);
      continue;
    }
    const T* src = reinterpret_cast<const T*>(is_v ? a.src_v : a.src) + (((long long)layer * a.src_blocks + from) * bs * kv.heads + kh) * D;
    const long long cell = ((long long)layer * kv.num_blocks + id) * kv.heads + kh;
    auto row = [&](int i, int c) {
      const T* p = src + (long long)i * kv.heads * D + 8 * c;
      return Columns<T>{ld_v4(p), ld_v4(p + half)};
    };
    write_page<T>(reinterpret_cast<uint8_t*>(is_v ? kv.v : kv.k) + cell * bs * D, (is_v ? kv.v_scale : kv.k_scale) + cell, true, 0, n, D, row,
                  [](int, int, Columns<T>&) {}, row);
  }
}

// ---- attention over the pages -----------------------------------------------------------------------------------------------
// Bound by reading every code once.  A warp takes 16 tokens of a page and KV head at a time, straight from the pool into the fragments of
// m16n8k16 products in halves: the tokens are the rows of the first product (keys times queries) and the contraction of the second (values
// times weights), the query rows that share the KV head (heads of the group, and new tokens) the 8 NT columns of both, so that no product
// is spent on padding of a group of 8.  As in decoder.cu the orders that the products do not fix are chosen for 16-byte loads: lane t of a quad takes
// columns 16 t .. 16 t + 15 of each 64 of a key, lane group g columns DP / 8 g .. of a value.  Codes become halves exactly; queries are
// brought into their range by a power of two per row, which loses nothing that counts beside the row's largest (2^-40 of it); weights, at
// most 1, are rounded to 11 bits for the second product, their sum is not.  The page's scale meets the products' fp32 sums.
// A request's context is cut into chunks, a CTA each; where there is more than one, finish_kernel joins their (max, sum, output).
constexpr int WARPS = 4;
constexpr int PART = 2;                    // floats of a part besides its output: maximum, sum

struct AttArgs {
  const void* q; long long sb, st, sh;
  const long long* start; const long long* counts;
  int batch, tokens, heads, group, row_parts;
  int chunk;                               // units of 16 tokens per CTA
  int per_page;                            // units of a page
  int chunks;                              // parts that scratch holds per row
  float scale;                             // times log2 e
  void* out;
  float* part_o; float* part_s;            // [batch][heads * tokens][chunks][dim] and [..][PART]
  float* unit_s;                           // [batch][units][heads * tokens]: log2 of the unit's weights' sum; null: not asked for
  int units;                               // of a full table
};

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {              // an 8 x 8 matrix of halves over the warp
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t half2_of(float a, float b) {
  __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}
// over the lane groups (the rows of a product), for every quad lane
__device__ __forceinline__ float max_rows(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
}
__device__ __forceinline__ float sum_rows(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 4);
  v += __shfl_xor_sync(0xffffffffu, v, 8);
  return v + __shfl_xor_sync(0xffffffffu, v, 16);
}

template <int DP> struct Unit {               // 16 tokens on their way
  uint4 k[2][DP / 64];
  uint32_t v[4][DP / 32];
  float ks, vs;
  int live;                                   // tokens of it that the request has; 0: its page is not there
};

__device__ __forceinline__ int tokens_of(const long long* counts, int b, int tokens) {
  return counts ? (int)min(max(counts[b], 0ll), (long long)tokens) : tokens;
}
// slots that the request's new tokens see, the last one's own among them; at most the table's
__device__ __forceinline__ int seen_by_last(const AttArgs& a, const FlKv8& kv, int b) {
  const int n = tokens_of(a.counts, b, a.tokens);
  return n == 0 ? 0 : (int)min(max(a.start[b] + n, 0ll), (long long)kv.table_stride * kv.block_size);
}

template <typename T, int DP, int NT, bool MASS>
__global__ void __launch_bounds__(WARPS * 32) attention_kernel(const AttArgs a, const FlKv8 kv) {
  constexpr int KJ = DP / 64, MT = DP / 16, VB = DP / 8, ROWS = 8 * NT, LD = DP + 4;
  __shared__ __align__(16) float s_o[WARPS][ROWS][LD];
  __shared__ float s_m[WARPS][ROWS], s_l[WARPS][ROWS];
  grid_dep_launch();
  grid_dep_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int kh = blockIdx.x / a.row_parts, rp = blockIdx.x - kh * a.row_parts, b = blockIdx.y, z = blockIdx.z;
  const int D = kv.dim, bs = kv.block_size, all_rows = a.group * a.tokens, r0 = rp * ROWS;
  const int n_rows = min(ROWS, all_rows - r0), n_new = tokens_of(a.counts, b, a.tokens);
  const int len = seen_by_last(a, kv, b);
  const int pages = (len + bs - 1) / bs, units = pages * a.per_page;
  const int lo = z * a.chunk, hi = min(lo + a.chunk, units);
  if (z > 0 && lo >= units) return;
  // the warp's units
  const int mine = hi - lo, per = mine / WARPS, extra = mine % WARPS;
  const int first = lo + warp * per + min(warp, extra), last = first + per + (warp < extra ? 1 : 0);

  const uint8_t* kp = reinterpret_cast<const uint8_t*>(kv.k);
  const uint8_t* vp = reinterpret_cast<const uint8_t*>(kv.v);
  int ids = -1, ids_at = 0;                    // lane i: the page of unit ids_at + i
  auto look_up = [&](int u0) {
    ids_at = u0;
    ids = u0 + lane < last ? page_id(kv, b, (u0 + lane) / a.per_page) : -1;
  };
  auto load = [&](int u, Unit<DP>& x) {
    if (u >= ids_at + 32) look_up(u);
    const int id = __shfl_sync(0xffffffffu, ids, u - ids_at);
    const int page = u / a.per_page, s0 = (u - page * a.per_page) * 16;
    const int live = id < 0 ? 0 : min(min(bs - s0, len - page * bs - s0), 16);
    if (id < 0 && lane == 0) note(kv.status, FL_DEC_BAD_PAGE);
    x.live = live;
    const long long cell = ((long long)kv.layer * kv.num_blocks + max(id, 0)) * kv.heads + kh;
    const uint8_t* k = kp + (cell * bs + s0) * D;
    const uint8_t* v = vp + (cell * bs + s0) * D;
    x.ks = live > 0 ? __ldg(kv.k_scale + cell) : 0.f;
    x.vs = live > 0 ? __ldg(kv.v_scale + cell) : 0.f;
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int j = 0; j < KJ; ++j) {
        const int d = 64 * j + 16 * t;
        x.k[p][j] = make_uint4(0, 0, 0, 0);
        if (8 * p + g < live && d < D) x.k[p][j] = ld_stream_v4(k + (8 * p + g) * D + d);
      }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int tok = 2 * t + (i & 1) + 8 * (i >> 1);
#pragma unroll
      for (int w = 0; w < DP / 32; ++w) x.v[i][w] = 0;
      if (tok < live && VB * g < D) {
        if constexpr (DP == 128) {
          const uint4 w4 = ld_stream_v4(v + tok * D + VB * g);
          x.v[i][0] = w4.x; x.v[i][1] = w4.y; x.v[i][2] = w4.z; x.v[i][3] = w4.w;
        } else {
          asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(x.v[i][0]), "=r"(x.v[i][1]) : "l"(v + tok * D + VB * g));
        }
      }
    }
  };

  look_up(first);
  Unit<DP> now;
  if (first < last) load(first, now);

  // queries, as the second operand; a row's power of two is undone on its scores
  uint32_t qb[NT][KJ][8];
  float factor[NT][2];                         // of columns 2 t and 2 t + 1
  int sees[NT][2];                             // slots that the column's token sees
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = r0 + 8 * nt + g, tok = r / a.group, h = r - tok * a.group;
    const bool in = r < all_rows && tok < n_new;
    const T* q = reinterpret_cast<const T*>(a.q) + b * a.sb + tok * a.st + (long long)(kh * a.group + h) * a.sh;
    float f[KJ][16];
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < KJ; ++j) {
      const int d = 64 * j + 16 * t;
      uint4 u0 = make_uint4(0, 0, 0, 0), u1 = u0;
      if (in && d < D) {
        u0 = ld_v4(q + d);
        u1 = ld_v4(q + d + 8);
      }
      float v0[8], v1[8];
      unpack<T>(u0, v0);
      unpack<T>(u1, v1);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        f[j][i] = v0[i];
        f[j][8 + i] = v1[i];
        m = fmaxf(m, fabsf(v0[i]) < INFINITY ? fabsf(v0[i]) : 0.f);
        m = fmaxf(m, fabsf(v1[i]) < INFINITY ? fabsf(v1[i]) : 0.f);
      }
    }
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
    // largest magnitude to 2^14 .. 2^15; a row of magnitudes below 2^-100 stays below
    const int e = max((int)(__float_as_uint(m) >> 23), 27);           // 127 + exponent
    const float to = __uint_as_float((uint32_t)(268 - e) << 23), back = __uint_as_float((uint32_t)(e - 14) << 23);       // 2^(14 - exponent) and its inverse
#pragma unroll
    for (int j = 0; j < KJ; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) qb[nt][j][i] = half2_of(f[j][2 * i] * to, f[j][2 * i + 1] * to);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      factor[nt][c] = __shfl_sync(0xffffffffu, back, (2 * t + c) * 4) * a.scale;
      const int rc = r0 + 8 * nt + 2 * t + c, tc = rc / a.group;
      sees[nt][c] = rc < all_rows && tc < n_new ? max(min(len, (int)min(a.start[b] + tc + 1, (long long)len)), 0) : 0;
    }
  }

  float o[NT][MT][4], m[NT][2], l[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[nt][i][j] = 0.f;
#pragma unroll
    for (int c = 0; c < 2; ++c) { m[nt][c] = -INFINITY; l[nt][c] = 0.f; }
  }

#pragma unroll 1
  for (int u = first; u < last; ++u) {
    Unit<DP> x = now;
    if (u + 1 < last) load(u + 1, now);
    const int page = u / a.per_page, base = page * bs + (u - page * a.per_page) * 16;
    float s[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[nt][i] = 0.f;
#pragma unroll
    for (int j = 0; j < KJ; ++j) {
      const uint32_t w0[4] = {x.k[0][j].x, x.k[0][j].y, x.k[0][j].z, x.k[0][j].w};
      const uint32_t w1[4] = {x.k[1][j].x, x.k[1][j].y, x.k[1][j].z, x.k[1][j].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t a0 = halves(w0[i]), a2 = halves(w0[i] >> 16), a1 = halves(w1[i]), a3 = halves(w1[i] >> 16);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma(s[nt], a0, a1, a2, a3, qb[nt][j][2 * i], qb[nt][j][2 * i + 1]);
      }
    }
    uint32_t p0[NT], p1[NT];
    bool split = false;                        // some column sees part of the live tokens, another more
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float f[2], mn[2], add[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float k = factor[nt][c] * x.ks;
        const int ends = min(sees[nt][c] - base, x.live);
        split |= sees[nt][c] > 0 && ends < x.live;
        s[nt][c] = g < ends ? s[nt][c] * k : -INFINITY;
        s[nt][2 + c] = g + 8 < ends ? s[nt][2 + c] * k : -INFINITY;
        // 0 stands in for a maximum of -inf: a step of nothing else adds nothing.  A score that is NaN or +inf makes the sums NaN.
        const float before = m[nt][c];
        m[nt][c] = fmaxf(before, max_rows(fmaxf(s[nt][c], s[nt][2 + c])));
        mn[c] = m[nt][c] == -INFINITY ? 0.f : m[nt][c];
        f[c] = exp2f(before - mn[c]);
        s[nt][c] = exp2f(s[nt][c] - mn[c]);
        s[nt][2 + c] = exp2f(s[nt][2 + c] - mn[c]);
        add[c] = s[nt][c] + s[nt][2 + c];
        l[nt][c] = l[nt][c] * f[c] + add[c];
      }
      if (MASS) {
        const float s0 = sum_rows(add[0]), s1 = sum_rows(add[1]);
        if (g == 0) {
          float* w = a.unit_s + ((long long)b * a.units + u) * a.heads * a.tokens + kh * all_rows + r0 + 8 * nt + 2 * t;
          if (8 * nt + 2 * t < n_rows) w[0] = mn[0] + log2f(s0);
          if (8 * nt + 2 * t + 1 < n_rows) w[1] = mn[1] + log2f(s1);
        }
      }
      if (__any_sync(0xffffffffu, f[0] != 1.f || f[1] != 1.f)) {
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          o[nt][i][0] *= f[0]; o[nt][i][1] *= f[1];
          o[nt][i][2] *= f[0]; o[nt][i][3] *= f[1];
        }
      }
      p0[nt] = transposed(half2_of(s[nt][0], s[nt][1]));
      p1[nt] = transposed(half2_of(s[nt][2], s[nt][3]));
    }
    auto values = [&](auto takes) {
#pragma unroll
      for (int w = 0; w < DP / 32; ++w)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t sel = h ? 0x7362u : 0x5140u;
          const uint32_t u0 = __byte_perm(x.v[0][w], x.v[1][w], sel), u1 = __byte_perm(x.v[2][w], x.v[3][w], sel);
          const uint32_t a0 = halves(u0), a1 = halves(u0 >> 16), a2 = halves(u1), a3 = halves(u1 >> 16);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float c[4] = {0.f, 0.f, 0.f, 0.f};
            mma(c, a0, a1, a2, a3, p0[nt], p1[nt]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (takes(nt, i & 1)) o[nt][2 * w + h][i] += c[i] * x.vs;
          }
        }
    };
    if (a.tokens == 1 || !__any_sync(0xffffffffu, split)) {
      values([](int, int) { return true; });
    } else {
      // Among the last tokens a column's weight of 0 must not meet a value of a later token, which may be NaN: one new token at a time, with
      // the values behind it left out, and only its own columns take the sums.
      const Unit<DP> whole = x;
      const int t0 = r0 / a.group, t1 = min((r0 + n_rows - 1) / a.group, n_new - 1);
      for (int tok = t0; tok <= t1; ++tok) {
        const int ends = (int)min(a.start[b] + tok + 1, (long long)len) - base;
        if (ends <= 0) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int w = 0; w < DP / 32; ++w) x.v[i][w] = 2 * t + (i & 1) + 8 * (i >> 1) < ends ? whole.v[i][w] : 0;
        values([&](int nt, int c) { return (r0 + 8 * nt + 2 * t + c) / a.group == tok; });
      }
    }
  }

  // the warps' parts become one
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int row = 8 * nt + 2 * t + c;
      const float sum = sum_rows(l[nt][c]);
      if (g == 0) { s_m[warp][row] = m[nt][c]; s_l[warp][row] = sum; }
#pragma unroll
      for (int i = 0; i < MT; i += 2)
        *reinterpret_cast<float4*>(&s_o[warp][row][VB * g + 2 * i]) = make_float4(o[nt][i][c], o[nt][i][2 + c], o[nt][i + 1][c], o[nt][i + 1][2 + c]);
    }
  __syncthreads();
  const bool whole = units <= a.chunk;                       // of this request's context
  for (int i = threadIdx.x; i < n_rows * D; i += WARPS * 32) {
    const int row = i / D, d = i - row * D;
    float mm = -INFINITY, acc = 0.f, ll = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) mm = fmaxf(mm, s_m[w][row]);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float e = s_l[w][row] == 0.f ? 0.f : exp2f(s_m[w][row] - mm);       // a part without weight; not one whose sum is NaN
      acc += e * s_o[w][row][d];
      ll += e * s_l[w][row];
    }
    const int r = r0 + row, tok = r / a.group, h = kh * a.group + r - tok * a.group;
    const bool none = tok >= n_new || a.start[b] + tok < 0 || len == 0;
    if (whole) reinterpret_cast<T*>(a.out)[(((long long)b * a.tokens + tok) * a.heads + h) * D + d] = T(none ? 0.f : acc / ll);
    if (!whole || MASS) {
      const long long part = ((long long)b * a.heads * a.tokens + kh * all_rows + r) * a.chunks + z;
      if (!whole) a.part_o[part * D + d] = acc;
      if (d == 0) { a.part_s[part * PART] = mm; a.part_s[part * PART + 1] = ll; }
    }
  }
}

// Joins the chunks' parts: a CTA per row and request.  The first row_ctas CTAs of a request have its rows; the others, if weights are asked
// for, its pages, a warp each, whose lanes add up the rows' shares in an order that is always the same.
template <typename T>
__global__ void __launch_bounds__(128) finish_kernel(const AttArgs a, const FlKv8 kv, float* mass, int row_ctas, int page_ctas) {
  grid_dep_launch();
  grid_dep_wait();
  const int b = blockIdx.y, D = kv.dim, bs = kv.block_size, rows = a.heads * a.tokens, all_rows = a.group * a.tokens;
  const int len = seen_by_last(a, kv, b), units = (len + bs - 1) / bs * a.per_page;
  const int parts = (units + a.chunk - 1) / a.chunk;
  if ((int)blockIdx.x < row_ctas) {
    if (parts < 2) return;
    const int row = blockIdx.x, kh = row / all_rows, r = row - kh * all_rows, tok = r / a.group, h = kh * a.group + r - tok * a.group;
    const long long at = ((long long)b * rows + row) * a.chunks;
    float mm = -INFINITY;
    for (int z = 0; z < parts; ++z) mm = fmaxf(mm, a.part_s[(at + z) * PART]);
    for (int d = threadIdx.x; d < D; d += 128) {
      float acc = 0.f, ll = 0.f;
#pragma unroll 4
      for (int z = 0; z < parts; ++z) {
        const float pm = a.part_s[(at + z) * PART], pl = a.part_s[(at + z) * PART + 1], po = a.part_o[(at + z) * D + d];
        const float e = pl == 0.f ? 0.f : exp2f(pm - mm);
        acc += e * po;
        ll += e * pl;
      }
      const bool none = tok >= tokens_of(a.counts, b, a.tokens) || a.start[b] + tok < 0;
      reinterpret_cast<T*>(a.out)[(((long long)b * a.tokens + tok) * a.heads + h) * D + d] = T(none ? 0.f : acc / ll);
    }
    return;
  }
  if (mass == nullptr || len == 0) return;
  extern __shared__ float s_lse[];                           // log2 of every row's sum of weights; inf: a row that sees nothing
  for (int r = threadIdx.x; r < rows; r += 128) {
    const long long at = ((long long)b * rows + r) * a.chunks;
    const int tok = (r % all_rows) / a.group;
    float mm = -INFINITY, ll = 0.f;
    for (int z = 0; z < parts; ++z) mm = fmaxf(mm, a.part_s[(at + z) * PART]);
    for (int z = 0; z < parts; ++z) {
      const float pm = a.part_s[(at + z) * PART], pl = a.part_s[(at + z) * PART + 1];
      ll += pl == 0.f ? 0.f : exp2f(pm - mm) * pl;
    }
    const bool none = tok >= tokens_of(a.counts, b, a.tokens) || a.start[b] + tok < 0;
    s_lse[r] = none ? INFINITY : mm + log2f(ll);
  }
  __syncthreads();
  const int pages = units / a.per_page, lane = threadIdx.x & 31;
  for (int p = (blockIdx.x - row_ctas) * 4 + (threadIdx.x >> 5); p < pages; p += page_ctas * 4) {
    float sum = 0.f;
    for (int i = 0; i < a.per_page; ++i) {
      const float* w = a.unit_s + ((long long)b * a.units + p * a.per_page + i) * rows;
      for (int r = lane; r < rows; r += 32) sum += s_lse[r] == INFINITY ? 0.f : exp2f(w[r] - s_lse[r]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) mass[(long long)b * kv.table_stride + p] += sum;
  }
}

// ---- eviction ---------------------------------------------------------------------------------------------------------------
// Bound by the latency of one CTA per request: the number of pages that go is known, the weight up to which they go is found digit by
// digit (four histograms of 256), and one pass deals the row out in its order.
constexpr int EVICT_THREADS = 512;

// weights in an order that whole numbers have: NaN last, -0 as 0
__device__ __forceinline__ uint32_t evict_key(float m) {
  if (m != m) return 0xffffffffu;
  const uint32_t u = __float_as_uint(m == 0.f ? 0.f : m);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(EVICT_THREADS) evict_kernel(const float* mass, const int* table, const long long* lengths, int pages, int bs, int keep,
                                                              int recent, int sinks, float* mass_out, int* table_out, long long* lengths_out, int* gone) {
  __shared__ int hist[256];
  __shared__ uint32_t s_prefix;
  __shared__ int s_left, s_sum[2][EVICT_THREADS / 32];
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  mass += (long long)b * pages; table += (long long)b * pages;
  mass_out += (long long)b * pages; table_out += (long long)b * pages;
  const long long len = max(lengths[b], 0ll);
  const int used = (int)min(len / bs + (len % bs != 0), (long long)pages), extra = max(used - keep, 0);
  if (tid == 0) {
    lengths_out[b] = lengths[b] - (long long)extra * bs;
    gone[b] = extra;
  }
  const int lo = sinks, hi = used - recent;                    // hi - lo >= extra, since keep >= recent + sinks
  uint32_t prefix = 0;
  int left = extra;                                            // of those that go, among the weights that begin with the digits found
  if (extra > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = tid; i < 256; i += EVICT_THREADS) hist[i] = 0;
      __syncthreads();
      for (int i0 = lo; i0 < hi; i0 += EVICT_THREADS) {
        const int i = i0 + tid;
        const uint32_t key = i < hi ? evict_key(mass[i]) : 0;
        const bool in = i < hi && (shift == 24 || key >> (shift + 8) == prefix);
        const int digit = in ? (int)(key >> shift & 255) : 256;
        const unsigned same = __match_any_sync(0xffffffffu, digit);          // weights that no token ever saw are all alike
        if (in && lane == __ffs(same) - 1) atomicAdd(&hist[digit], __popc(same));
      }
      __syncthreads();
      if (warp == 0) {
        int n[8], sum = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) { n[j] = hist[lane * 8 + j]; sum += n[j]; }
        int before = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int v = __shfl_up_sync(0xffffffffu, before, o);
          if (lane >= o) before += v;
        }
        before -= sum;
        if (before < left && before + sum >= left) {
          int j = 0;
          while (j < 7 && before + n[j] < left) before += n[j++];
          s_prefix = prefix << 8 | (lane * 8 + j);
          s_left = left - before;
        }
      }
      __syncthreads();
      prefix = s_prefix;
      left = s_left;
    }
  }
  // positions below: kept pages from 0, those that go from used - extra
  int equal_before = 0, gone_before = 0;
  for (int i0 = 0; i0 < pages; i0 += EVICT_THREADS) {
    const int i = i0 + tid;
    float m = 0.f;
    int id = 0;
    if (i < pages) { m = mass[i]; id = table[i]; }
    const bool free = extra > 0 && i >= lo && i < hi;
    const uint32_t key = evict_key(m);
    const bool equal = free && key == prefix;
    const unsigned eq = __ballot_sync(0xffffffffu, equal);
    if (lane == 0) s_sum[0][warp] = __popc(eq);
    __syncthreads();
    int rank = equal_before + __popc(eq & ((1u << lane) - 1)), all_eq = 0;
#pragma unroll
    for (int w = 0; w < EVICT_THREADS / 32; ++w) {
      if (w < warp) rank += s_sum[0][w];
      all_eq += s_sum[0][w];
    }
    const bool goes = free && (key < prefix || (equal && rank < left));
    const unsigned go = __ballot_sync(0xffffffffu, goes);
    if (lane == 0) s_sum[1][warp] = __popc(go);
    __syncthreads();
    int out = gone_before + __popc(go & ((1u << lane) - 1)), all_go = 0;
#pragma unroll
    for (int w = 0; w < EVICT_THREADS / 32; ++w) {
      if (w < warp) out += s_sum[1][w];
      all_go += s_sum[1][w];
    }
    if (i < pages) {
      const int to = i >= used ? i : goes ? used - extra + out : i - out;
      table_out[to] = id;
      mass_out[to] = goes ? 0.f : m;
    }
    equal_before += all_eq;
    gone_before += all_go;
  }
}

}  // namespace kv8
}  // namespace fl

// --------------------------------------------------------------------------------------------------------------------------
// host side
// --------------------------------------------------------------------------------------------------------------------------
static bool aligned(std::initializer_list<const void*> pointers) {
  uintptr_t all = 0;
  for (const void* p : pointers) all |= reinterpret_cast<uintptr_t>(p);
  return (all & 15) == 0;
}
static bool sizes_fit(const FlKv8* kv) {
  return kv->dim % 16 == 0 && kv->dim >= 16 && kv->dim <= 128 && kv->heads >= 1 && kv->block_size >= 1 && kv->num_blocks >= 0 && kv->layers >= 1 &&
         kv->table_stride >= 0 && (long long)kv->table_stride * kv->block_size <= 0x3fffffffll;
}
static unsigned grid_of(long long warps) {
  const long long ctas = (warps + 3) / 4;
  return (unsigned)(ctas < 1 ? 1 : ctas > 148ll * 256 ? 148 * 256 : ctas);
}

#define FL_KV8_TYPES(dtype, ...)                                             \
  do {                                                                       \
    if ((dtype) == FL_DEC_BF16) { using T = __nv_bfloat16; __VA_ARGS__; }    \
    else if ((dtype) == FL_DEC_FP16) { using T = __half; __VA_ARGS__; }      \
    else return -1;                                                          \
  } while (0)

extern "C" int fl_kv8_write(int dtype, const void* qkv, void* out, const void* bias, const float* rope, long long rope_rows, const long long* start,
                            const long long* pos, const long long* counts, int batch, int tokens, int heads, const FlKv8* kv, cudaStream_t stream) {
  if (!sizes_fit(kv) || kv->layer < 0 || kv->layer >= kv->layers || batch < 0 || tokens < 0 || tokens > 0x3fffffff || heads < 0) return -2;
  if (!aligned({qkv, out, bias, rope, kv->k, kv->v})) return -4;
  if (batch == 0 || tokens == 0) return 0;
  fl::kv8::WriteArgs a = {};
  a.src = qkv; a.out = out; a.bias = bias; a.rope = rope; a.rope_rows = rope_rows;
  a.start = start; a.pos = pos; a.counts = counts; a.batch = batch; a.tokens = tokens; a.heads = heads;
  a.reach = (tokens + kv->block_size - 2) / kv->block_size + 1;
  const long long page_units = 2ll * batch * a.reach * kv->heads, rows = (long long)batch * tokens;
  if ((long long)batch * a.reach > 0x7fffffffll) return -2;
  const bool copy = qkv != out, q = copy || bias != nullptr || rope != nullptr;
  const long long items = q ? rows * (counts ? heads + 2 * kv->heads : heads) * (kv->dim / 16) : 0;
  const long long units = page_units + (items + 31) / 32;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid_of(units), 1, 1);
  cfg.blockDim = dim3(128, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = rows <= FL_THIN_MAX_ROWS ? 1 : 0;      // as the decoder's other passes
  FL_KV8_TYPES(dtype, return (int)cudaLaunchKernelEx(&cfg, fl::kv8::write_kernel<T>, a, *kv, page_units, units));
}

extern "C" int fl_kv8_pack(int dtype, const void* k_pool, const void* v_pool, int src_blocks, const int* src_table, int src_stride,
                           const long long* lengths, int batch, const FlKv8* kv, cudaStream_t stream) {
  if (!sizes_fit(kv) || batch < 0 || src_blocks < 0 || src_stride < 0) return -2;
  if (!aligned({k_pool, v_pool, kv->k, kv->v})) return -4;
  fl::kv8::WriteArgs a = {};
  a.src = k_pool; a.src_v = v_pool; a.src_table = src_table; a.src_stride = src_stride; a.src_blocks = src_blocks;
  a.start = lengths; a.batch = batch; a.reach = src_stride < kv->table_stride ? src_stride : kv->table_stride;
  const long long units = 2ll * kv->layers * batch * a.reach * kv->heads;
  if (units == 0) return 0;
  FL_KV8_TYPES(dtype, (fl::kv8::pack_kernel<T><<<grid_of(units), 128, 0, stream>>>(a, *kv, units)));
  return (int)cudaGetLastError();
}

// How a call is cut up: `chunk` units of 16 tokens per CTA, so that a full table gives every SM `resident` CTAs but a warp no fewer than two
// units; a table may be much longer than its contexts, so a chunk is never more than MOST units.
namespace {
constexpr int FEWEST = 2 * fl::kv8::WARPS, MOST = 64 * fl::kv8::WARPS;
struct Cut { int nt, row_parts, per_page, units, chunk, chunks; };
Cut cut_of(int batch, int tokens, int heads, const FlKv8* kv) {
  Cut c;
  const long long rows = (long long)heads / kv->heads * tokens;
  c.nt = rows > 8 ? 2 : 1;
  c.row_parts = (int)((rows + 8 * c.nt - 1) / (8 * c.nt));
  c.per_page = (kv->block_size + 15) / 16;
  c.units = kv->table_stride * c.per_page;
  const long long ctas = (long long)batch * kv->heads * c.row_parts, want = 148ll * (c.nt == 1 ? 3 : 2);
  long long parts = want / (ctas < 1 ? 1 : ctas);
  if (parts < 1) parts = 1;
  long long chunk = (c.units + parts - 1) / parts;
  if (chunk > MOST) chunk = MOST;
  if (chunk < FEWEST) chunk = FEWEST;
  while ((c.units + chunk - 1) / chunk > 65535) chunk *= 2;
  c.chunk = (int)chunk;
  c.chunks = (int)((c.units + chunk - 1) / chunk);
  if (c.chunks < 1) c.chunks = 1;
  return c;
}
long long up16(long long bytes) { return (bytes + 15) / 16 * 16; }

template <typename T, int DP, int NT>
int launch_attention(const fl::kv8::AttArgs& a, const FlKv8& kv, bool mass, dim3 grid, bool early, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(fl::kv8::WARPS * 32, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = early ? 1 : 0;
  return (int)cudaLaunchKernelEx(&cfg, mass ? fl::kv8::attention_kernel<T, DP, NT, true> : fl::kv8::attention_kernel<T, DP, NT, false>, a, kv);
}
}  // namespace

extern "C" long long fl_kv8_attention_scratch(int batch, int tokens, int heads, const FlKv8* kv, int mass) {
  if (!sizes_fit(kv) || batch < 1 || tokens < 1 || heads < 1 || heads % kv->heads) return 0;
  const Cut c = cut_of(batch, tokens, heads, kv);
  const long long rows = (long long)batch * heads * tokens;
  long long bytes = 0;
  if (c.chunks > 1) bytes += up16(rows * c.chunks * kv->dim * 4);
  if (c.chunks > 1 || mass) bytes += up16(rows * c.chunks * fl::kv8::PART * 4);
  if (mass) bytes += up16(rows * c.units * 4);
  return bytes;
}

extern "C" int fl_kv8_attention(int dtype, const void* q, long long stride_b, long long stride_t, long long stride_h, const long long* start,
                                const long long* counts, int batch, int tokens, int heads, float scale, const FlKv8* kv, void* out, float* mass,
                                void* scratch, cudaStream_t stream) {
  if (!sizes_fit(kv) || kv->layer < 0 || kv->layer >= kv->layers || batch < 0 || batch > 65535 || tokens < 0 || heads < 1 || heads % kv->heads ||
      (long long)heads * tokens > 0x3fffffffll || stride_b % 8 || stride_t % 8 || stride_h % 8)
    return -2;
  if (mass != nullptr && (long long)heads * tokens > 12 * 1024) return -2;         // rows whose sums a CTA keeps in shared memory
  if (!aligned({q, out, scratch, kv->k, kv->v})) return -4;
  if (batch == 0 || tokens == 0) return 0;
  const Cut c = cut_of(batch, tokens, heads, kv);
  const long long rows = (long long)batch * heads * tokens;
  if ((long long)kv->heads * c.row_parts > 0x7fffffffll || (c.chunks > 1 && (long long)heads * tokens > 0x7fffffffll)) return -2;
  fl::kv8::AttArgs a = {};
  a.q = q; a.sb = stride_b; a.st = stride_t; a.sh = stride_h;
  a.start = start; a.counts = counts; a.batch = batch; a.tokens = tokens; a.heads = heads; a.group = heads / kv->heads;
  a.row_parts = c.row_parts; a.chunk = c.chunk; a.per_page = c.per_page; a.chunks = c.chunks; a.units = c.units;
  a.scale = scale * 1.4426950408889634f;
  a.out = out;
  uint8_t* s = reinterpret_cast<uint8_t*>(scratch);
  if (c.chunks > 1) { a.part_o = reinterpret_cast<float*>(s); s += up16(rows * c.chunks * kv->dim * 4); }
  if (c.chunks > 1 || mass) { a.part_s = reinterpret_cast<float*>(s); s += up16(rows * c.chunks * fl::kv8::PART * 4); }
  if (mass) a.unit_s = reinterpret_cast<float*>(s);
  const dim3 grid(kv->heads * c.row_parts, batch, c.chunks);
  const bool early = (long long)batch * tokens <= FL_THIN_MAX_ROWS;
  int rc = 0;
#define FL_ATT(D, N) rc = launch_attention<T, D, N>(a, *kv, mass != nullptr, grid, early, stream)
  FL_KV8_TYPES(dtype, {
    if (kv->dim <= 64) { if (c.nt == 1) FL_ATT(64, 1); else FL_ATT(64, 2); }
    else { if (c.nt == 1) FL_ATT(128, 1); else FL_ATT(128, 2); }
  });
#undef FL_ATT
  if (rc != 0 || (c.chunks == 1 && mass == nullptr)) return rc;
  const int row_ctas = c.chunks > 1 ? heads * tokens : 0;
  const int pages = kv->table_stride, page_ctas = mass == nullptr ? 0 : pages < 4 ? 1 : pages / 4 > 64 ? 64 : pages / 4;
  if (row_ctas + page_ctas == 0) return 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(row_ctas + page_ctas, batch, 1);
  cfg.blockDim = dim3(128, 1, 1);
  cfg.dynamicSmemBytes = mass ? (size_t)heads * tokens * 4 : 0;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  FL_KV8_TYPES(dtype, return (int)cudaLaunchKernelEx(&cfg, fl::kv8::finish_kernel<T>, a, *kv, mass, row_ctas, page_ctas));
}

extern "C" int fl_kv8_evict(const float* mass, const int* table, const long long* lengths, int batch, int pages, int block_size, int keep, int recent,
                            int sinks, float* mass_out, int* table_out, long long* lengths_out, int* gone, cudaStream_t stream) {
  if (batch < 0 || pages < 0 || block_size < 1 || recent < 1 || sinks < 0 || (long long)recent + sinks > keep) return -2;
  if (batch == 0) return 0;
  fl::kv8::evict_kernel<<<batch, fl::kv8::EVICT_THREADS, 0, stream>>>(mass, table, lengths, pages, block_size, keep, recent, sinks, mass_out, table_out,
                                                                      lengths_out, gone);
  return (int)cudaGetLastError();
}

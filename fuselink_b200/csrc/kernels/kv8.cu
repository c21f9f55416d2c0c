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

// four codes as halves, which hold every e4m3 value: the first two, the last two
__device__ __forceinline__ uint2 halves(uint32_t codes) {
  uint2 h;
  asm("{.reg .b16 c, d; mov.b32 {c, d}, %2; cvt.rn.f16x2.e4m3x2 %0, c; cvt.rn.f16x2.e4m3x2 %1, d;}" : "=r"(h.x), "=r"(h.y) : "r"(codes));
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
  int id = __ldcg(kv.block_table + (long long)b * kv.table_stride + page);
  if (id < 0) id += kv.num_blocks;
  return id >= 0 && id < kv.num_blocks ? id : -1;
}

// ---- page write -----------------------------------------------------------------------------------------------------------
// Bound by memory: new tokens are read once, written once in the model's type and once in 8 bits.  A warp has one page of one head, of keys or
// of values: lane (t, c) takes columns 8 c .. 8 c + 7 of the first half of a token's row and the matching ones of the second (the pairs that the
// rotation mixes), 32 / (dim / 16) tokens at a time.  Four such steps, a page of 16 tokens, stay in registers between finding the largest
// magnitude and writing codes; larger pages are read again.  16 x 2048 tokens of 32 + 2 x 8 heads of 128: 254 us with a query's columns and angles
// looked up one by one, now 186 (136 of bytes); 5 x 389 ragged ones of 32 + 2 x 32 heads of 64: 18.5 us (7.0).  With 128 registers, for the four steps, an SM
// has 16 warps; 96 spill (253 us), two steps in registers and the others read again take 206, queries in a launch of their own 180 to 193.  A warp's
// next rows copied to shared memory while it works on these, by a grid that stays: 176 us, but 23.3 for the ragged ones.
constexpr int STEPS = 4;

struct WriteArgs {
  const void* src; void* out; const void* bias; const float* rope; long long rope_rows;
  const long long* start; const long long* pos; const long long* counts;
  int batch, tokens, heads, reach;            // reach: pages that a request's tokens can lie in
  int parts;                                  // warps that share a token's queries
  // pack: pages of 16 bits in place of rows
  const void* src_v; const int* src_table; int src_stride, src_blocks;
};

struct Angles {                               // of a lane's columns; read as what a kernel before may have written
  float co[8], si[8];
  __device__ __forceinline__ void load(const float* rope, int dim, int c) {
    const float4* a = reinterpret_cast<const float4*>(rope + 8 * c);
    const float4* b = reinterpret_cast<const float4*>(rope + dim / 2 + 8 * c);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 u = a[i], v = b[i];
      co[4 * i] = u.x; co[4 * i + 1] = u.y; co[4 * i + 2] = u.z; co[4 * i + 3] = u.w;
      si[4 * i] = v.x; si[4 * i + 1] = v.y; si[4 * i + 2] = v.z; si[4 * i + 3] = v.w;
    }
  }
};

template <typename T>
struct Columns {                              // of one token: the two vectors that a lane takes
  uint4 lo, hi;
  __device__ __forceinline__ void turn(const T* bias, const Angles* cs, int half) {
    if (bias == nullptr && cs == nullptr) return;
    float a[8], b[8];
    unpack<T>(lo, a);
    unpack<T>(hi, b);
    if (bias != nullptr) {
      float e[8];
      unpack<T>(*reinterpret_cast<const uint4*>(bias), e);
#pragma unroll
      for (int j = 0; j < 8; ++j) a[j] += e[j];
      unpack<T>(*reinterpret_cast<const uint4*>(bias + half), e);
#pragma unroll
      for (int j = 0; j < 8; ++j) b[j] += e[j];
    }
    if (cs != nullptr) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {             // each product rounded, as separate operations would
        const float co = cs->co[j], si = cs->si[j], x = a[j], y = b[j];
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
// of them; keep(i, columns): where they go besides.  again(i): the vector after given().
template <typename T, typename Row, typename Given, typename Keep, typename Again>
__device__ __forceinline__ void write_page(uint8_t* page, float* scale, bool there, int lead, int n, int dim, Row row, Given given, Keep keep, Again again) {
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
    // behind all of them, so that a step's angles and bias are on their way during the one before
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const int i = (s0 + s) * at_once + tk;
      if (on && i < n) keep(i, c, col[s]);
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
          const uint2 h = halves(w[j]);
          const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&h.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&h.y));
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
__global__ void __launch_bounds__(128, 4) write_kernel(const WriteArgs a, const FlKv8 kv, unsigned page_units, unsigned units) {
  grid_dep_launch();
  grid_dep_wait();
  const int lane = threadIdx.x & 31, D = kv.dim, half = D / 2, chunks = D / 16, all = a.heads + 2 * kv.heads, bs = kv.block_size;
  const long long cap = (long long)kv.table_stride * bs;
  const T* src = reinterpret_cast<const T*>(a.src);
  T* out = reinterpret_cast<T*>(a.out);
  const T* bias = reinterpret_cast<const T*>(a.bias);
  for (unsigned u = blockIdx.x * 4 + (threadIdx.x >> 5); u < units; u += gridDim.x * 4) {
    if (u < page_units) {
      const bool is_v = u & 1;
      const unsigned r = u >> 1, rest = r / kv.heads;
      const int kh = (int)(r - rest * kv.heads), b = (int)(rest / a.reach), pi = (int)(rest - (unsigned)b * a.reach);
      const long long st = a.start[b];
      const int n = a.counts ? (int)min(max(a.counts[b], 0ll), (long long)a.tokens) : a.tokens;
      // tokens [from, to) of the request's are in this page
      int from, to, lead, page;
      const bool inside = st >= 0 && st <= cap - n;             // in this order: st may be any number
      if (inside) {
        const int used = (int)st % bs;          // of the first page, before them
        page = (int)st / bs + pi;
        lead = pi == 0 ? used : 0;
        from = pi == 0 ? 0 : pi * bs - used;
        to = min(n, (pi + 1) * bs - used);
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
      const long long turn = min(a.pos ? a.pos[b] : st, a.rope_rows) + from;
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
            const T* bias_c = bias_h ? bias_h + 8 * c : nullptr;
            const bool there = rotate && turn + i >= 0 && turn + i < a.rope_rows;
            if (there) {
              Angles cs;
              cs.load(a.rope + (turn + i) * D, D, c);
              col.turn(bias_c, &cs, half);
            } else {
              if (rotate) note(kv.status, FL_DEC_BAD_POSITION);
              col.turn(bias_c, nullptr, half);
            }
          },
          [&](int i, int c, const Columns<T>& col) {
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
    // A token's queries, STEPS heads at a time for each lane, which has the same columns of all of them and so the same angles; of a row that is none of
    // the request's, everything as it came.
    const unsigned q = u - page_units, n = q / a.parts;
    const int part = (int)(q - n * a.parts), b = (int)(n / a.tokens), t = (int)(n - (unsigned)b * a.tokens);
    const bool in = a.counts == nullptr || t < a.counts[b];
    if ((!in || (bias == nullptr && a.rope == nullptr)) && src == out) continue;
    const int at_once = 32 / chunks, tk = lane / chunks, c = lane - tk * chunks, heads = in ? a.heads : all;
    if (tk >= at_once) continue;
    const long long turn = min(a.pos ? a.pos[b] : a.start[b], a.rope_rows) + t;
    const bool there = in && a.rope != nullptr && turn >= 0 && turn < a.rope_rows;
    if (in && a.rope != nullptr && !there) note(kv.status, FL_DEC_BAD_POSITION);
    Angles cs;
    if (there) cs.load(a.rope + turn * D, D, c);
    for (int h0 = part * STEPS * at_once + tk; h0 < heads; h0 += a.parts * STEPS * at_once) {
      Columns<T> col[STEPS];
      const long long at = ((long long)n * all + h0) * D + 8 * c;
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
        if (h0 + s * at_once < heads) {
          const T* p = src + at + (long long)s * at_once * D;
          col[s] = Columns<T>{ld_v4(p), ld_v4(p + half)};
        }
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
        if (h0 + s * at_once < heads) {
          if (in) col[s].turn(bias ? bias + (h0 + s * at_once) * D + 8 * c : nullptr, there ? &cs : nullptr, half);
        }
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
        if (h0 + s * at_once < heads) {
          T* p = out + at + (long long)s * at_once * D;
          st_v4(p, col[s].lo);
          st_v4(p + half, col[s].hi);
        }
    }
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
                  [](int, int, Columns<T>&) {}, [](int, int, const Columns<T>&) {}, row);
  }
}

// ---- attention over the pages -----------------------------------------------------------------------------------------------
// Bound by reading every code once.  A warp takes 16 tokens of a page and KV head at a time, straight from the pool into the fragments of
// m16n8k16 products in halves: the tokens are the rows of the first product (keys times queries) and the contraction of the second (values
// times weights), the query rows that share the KV head (heads of the group, and new tokens) the 8 NT columns of both, so that no product
// is spent on padding of a group of 8.  As in decoder.cu the orders that the products do not fix are chosen for 16-byte loads: lane t of a quad takes
// columns 16 t .. 16 t + 15 of each 64 of a key, lane group g columns DP / 8 g .. of a value.  Codes become halves exactly; queries are
// brought into their range by a power of two per row, which loses nothing that counts beside the row's largest (2^-40 of it).
//
// Weights times their page's scale of values meet the codes as halves, in a unit per row that follows the largest such product: what a page has no
// weight for takes no bits from the others, however large its values, and what lies below 2^-26 of the largest is lost.  A half has 11 bits.
// Where a KV head has four rows or fewer, the columns that are left have what is beyond them: 22 bits, and the output's error is that of sums in
// 32 bits.  Elsewhere the sum that the output is divided by is that of the weights as they were cut, so that what the cuts have in common cancels; as
// further products the bits beyond would cost 48 ragged requests of eight rows 64.5 us in place of 61.6, and the output is off by 1.650e-3 of its norm in
// place of 1.646e-3 (bf16; divided by the sum of uncut weights: 1.70e-3).  Weights of pages are of uncut sums.
//
// What a step of 16 tokens costs beside its 16 products and 64 conversions is kept out of the loop: the maximum that the weights refer to and the unit
// of the products only follow when a score is 2^8 or a page's scale 2^7 beyond them (a vote, not a reduction, per step).  With a maximum per step and a
// multiplication of every sum by the page's scale, and the codes on their way through registers, 16 x 2048 tokens of 8 KV heads of 128 took
// 25.6 us, now 17.5 (10.3 of bytes; 2 x 131072 tokens 101, 82 of bytes).  Codes are on their way through a ring in shared memory, two steps ahead
// of their use, which then never wait: of the 17.5 us some 9 go at the memory's rate, the others are launch, the first page ids and rows (4000 to
// 5000 cycles: a miss each, of pages anywhere in memory), and the joining of warps and CTAs (5000 cycles).
//
// A request's context is dealt out evenly over the warps of the CTAs in the grid's third dimension: a cluster of up to 8, which joins their (max, sum,
// output) through distributed shared memory, or more, whose parts finish_kernel joins.
constexpr int WARPS = 4;
constexpr int FEWEST = 2 * WARPS;          // steps that make a CTA worth having
constexpr int LONGEST = 64 * WARPS;        // steps beyond which a context is cut even where there are CTAs enough: ragged batches end together
constexpr int MOST_PARTS = 64;             // two for a lane of the kernel that joins them
constexpr int PART = 4;                    // floats of a part besides its output: maximum, sum of the weights as they meet the values, sum as they are
constexpr float LOWEST = -3e38f;           // a maximum of nothing: masked scores are -inf, which is below it
constexpr float SLACK = 8.f;               // log2 of the largest weight, whose reference only follows when a score is beyond it
constexpr float ROOM = 7.f;                // log2 of the largest page's scale in the column's unit: halves hold 2^(SLACK + ROOM)
constexpr float START = 3.f;               // log2 of the largest weight times its page's scale, in a unit that has just been chosen

struct AttArgs {
  const void* q; long long sb, st, sh;
  const long long* start; const long long* counts;
  int batch, tokens, heads, group, row_parts;
  int per_page;                            // steps of a page, or halves of steps
  int splits, clustered;                   // CTAs per request, KV head and rows; whether they are a cluster
  int early;                               // launched while the kernel before may still run
  float scale;                             // times log2 e
  void* out;
  float* part_o; float* part_s;            // [batch][heads * tokens][parts][dim] and [..][PART]; parts: splits, or 1 if they are a cluster
  float2* unit_s;                          // [batch][units][heads * tokens]: the weights' sum, and the maximum that they refer to; null: not asked for
  int units;                               // of a full table: steps, or halves of them
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
__device__ __forceinline__ float eleven_bits(float x, uint32_t keep = 0xffffe000u) { return __uint_as_float(__float_as_uint(x) & keep); }     // cut to what a half holds
__device__ __forceinline__ uint32_t half2_cut(float a, float b) {
  uint32_t r;
  asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}
__device__ __forceinline__ float exp2_fast(float x) {                     // the hardware's: 2^-22 off, relatively; 0 below 2^-126
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
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
__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}

__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}
// A warp's ring in shared memory.  Rows are 16 bytes further apart than they are long, so that the 16-byte (values of heads up to 64: 8-byte) reads of
// a product's rows meet different banks.
template <int DP> struct Ring {
  static constexpr int STAGES = DP == 128 ? 3 : 6;
  static constexpr int PITCH = DP + 16, KEYS = 16 * PITCH, SCALES = 2 * KEYS;
  static constexpr int STAGE = SCALES + 16;                    // 16 keys, 16 values, their scales
  static constexpr int BYTES = WARPS * STAGES * STAGE;
};
__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool there) {        // zeros where it is not there
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t to, const void* from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory"); }
__device__ __forceinline__ void copy4(uint32_t to, const void* from, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(there ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 lds_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint2 lds_v2(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ int tokens_of(const long long* counts, int b, int tokens) {
  return counts ? (int)min(max(counts[b], 0ll), (long long)tokens) : tokens;
}
// the request's first new slot; one behind the table as the table's end, so that sums with it fit
__device__ __forceinline__ long long start_of(const AttArgs& a, const FlKv8& kv, int b) { return min(a.start[b], (long long)kv.table_stride * kv.block_size); }
// slots that the request's new tokens see, the last one's own among them; at most the table's
__device__ __forceinline__ int seen_by_last(const AttArgs& a, const FlKv8& kv, int b) {
  const int n = tokens_of(a.counts, b, a.tokens);
  return n == 0 ? 0 : (int)min(max(start_of(a, kv, b) + n, 0ll), (long long)kv.table_stride * kv.block_size);
}

// parts' outputs are means (divided by their sums), so that joining them overflows nowhere
__device__ __forceinline__ float share(float m, float l, float mm) { return l == 0.f ? 0.f : exp2f(m - mm) * l; }      // 0: a part without weight; not one whose sum is NaN

// DP: head dimension rounded up to 64 or 128.  FULL: it is that, in pages of whole 16s.  HALVES: pages that are not, whose steps are two halves of up to
// eight tokens, from pages and with scales of their own: with steps of one page, pages of 8 took 1.9 times and pages of 5 three times as long.
template <typename T, int DP, int NT, bool BOTH, bool FULL, bool HALVES, bool MASS>
__global__ void __launch_bounds__(WARPS * 32, NT == 1 ? 4 : 2) attention_kernel(const AttArgs a, const FlKv8 kv) {
  using R = Ring<DP>;
  constexpr int KJ = DP / 64, MT = DP / 16, VB = DP / 8, ROWS = 8 * NT, LD = DP + 4;
  static_assert(WARPS * ROWS * LD * 4 <= R::BYTES, "the warps' parts take the rings' place");
  extern __shared__ __align__(16) uint8_t s_ring[];
  auto s_o = reinterpret_cast<float(*)[ROWS][LD]>(s_ring);
  __shared__ float s_m[WARPS][ROWS], s_l[WARPS][ROWS], s_x[WARPS][ROWS], s_cm[ROWS], s_cl[ROWS], s_cx[ROWS];
  grid_dep_launch();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int kh = blockIdx.x / a.row_parts, rp = blockIdx.x - kh * a.row_parts, b = blockIdx.y, z = blockIdx.z;
  const int D = FULL ? DP : kv.dim, bs = kv.block_size, all_rows = a.group * a.tokens, r0 = rp * ROWS;
  const int n_rows = min(ROWS, all_rows - r0);
  static_assert(!BOTH || NT == 1, "half of the only eight columns");
  constexpr int COL = BOTH ? 3 : 7;            // a column's row, of eight
  constexpr bool EXACT = MASS && !BOTH;        // the weights' sums are kept apart from the sums of the weights as they meet the values
  // The warp's units: every nw-th.  Which pages these are does not depend on the context's length, nor do the queries, so that all three are on
  // their way side by side.
  const int nw = a.splits * WARPS, first = z * WARPS + warp;
  constexpr int H = HALVES ? 2 : 1;            // parts of a unit that have a page of their own, each of SIZE tokens at most
  constexpr int SIZE = 16 / H;
  struct Ids { int of[H]; };
  auto look_up = [&](int u0) {                 // lane i: the pages of unit u0 + i nw
    Ids ids;
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const int part = (u0 + lane * nw) * H + h;
      ids.of[h] = part < a.units ? page_id(kv, b, a.per_page == 1 ? part : part / a.per_page) : -1;
    }
    return ids;
  };
  if (a.early) {
    // a look ahead, before the wait for the kernel that writes queries and the new tokens' pages: the first units asked into L2, a line per
    // lane.  Whatever it finds only says what is worth having there; all of it is read again behind the wait.
    const long long n = min(__ldcg(a.start + b), (long long)kv.table_stride * bs) + a.tokens, bytes = (long long)SIZE * D;
    const Ids ahead = look_up(first);
#pragma unroll
    for (int i = 0; i < R::STAGES - 1; ++i)
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const int part = (first + i * nw) * H + h, id = __shfl_sync(0xffffffffu, ahead.of[h], i);
        const int page = a.per_page == 1 ? part : part / a.per_page, s0 = (part - page * a.per_page) * SIZE;
        const long long byte = (lane & 15) * 128;
        if (id >= 0 && (long long)page * bs + s0 < n && byte < bytes && s0 * D + byte < (long long)bs * D) {
          const long long cell = ((long long)kv.layer * kv.num_blocks + id) * kv.heads + kh;
          prefetch_l2(reinterpret_cast<const uint8_t*>(lane < 16 ? kv.k : kv.v) + (cell * bs + s0) * D + byte);
          if ((lane & 15) == 0) prefetch_l2((lane ? kv.v_scale : kv.k_scale) + cell);
        }
      }
  }
  grid_dep_wait();
  Ids ids = look_up(first);
  const long long start = start_of(a, kv, b);
  const int n_new = tokens_of(a.counts, b, a.tokens);
  uint4 q_raw[NT][KJ][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int r = r0 + 8 * nt + (g & COL), tok = a.tokens == 1 ? 0 : r / a.group, h = r - tok * a.group;
    const T* q = reinterpret_cast<const T*>(a.q) + b * a.sb + tok * a.st + (long long)(kh * a.group + h) * a.sh;
#pragma unroll
    for (int j = 0; j < KJ; ++j) {
      const int d = DP == 128 ? 32 * t + 16 * j : 16 * t;
      q_raw[nt][j][0] = q_raw[nt][j][1] = make_uint4(0, 0, 0, 0);
      if (r < all_rows && d < D) {
        q_raw[nt][j][0] = ld_v4(q + d);
        q_raw[nt][j][1] = ld_v4(q + d + 8);
      }
    }
  }
  const int len = n_new == 0 ? 0 : (int)min(max(start + n_new, 0ll), (long long)kv.table_stride * bs);
  const int units = ((len + bs - 1) / bs * a.per_page + H - 1) / H;
  const int mine = first < units ? (units - first + nw - 1) / nw : 0;

  // this lane's 16 bytes of a row, in every PASS-th row
  constexpr int PIECES = DP / 16, PASS = 32 / PIECES;
  const int row0 = lane / PIECES, piece = lane % PIECES;
  const uint8_t* kp = reinterpret_cast<const uint8_t*>(kv.k) + row0 * D + 16 * piece;
  const uint8_t* vp = reinterpret_cast<const uint8_t*>(kv.v) + row0 * D + 16 * piece;
  const uint32_t ring = smem_u32(s_ring) + warp * R::STAGES * R::STAGE, cell0 = ring + row0 * R::PITCH + 16 * piece;
  const long long pool0 = (long long)kv.layer * kv.num_blocks;
  const bool column = FULL || 16 * piece < D;
  if (!column) {                               // columns that there are not: zeros, once
    for (int s = 0; s < R::STAGES; ++s)
      for (int i = 0; i < 32; i += PASS)
        asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(cell0 + s * R::STAGE + i * R::PITCH), "r"(0u) : "memory");
  }
  // where a unit's parts begin, and tokens of them that the request has (none or fewer: it has not got that far)
  struct Place { int base[H], live[H], s0[H]; };
  auto place = [&](int u) {
    Place p;
#pragma unroll
    for (int h = 0; h < H; ++h) {
      int page = u * H + h;
      p.s0[h] = 0;
      if (a.per_page > 1) { const int part = page; page /= a.per_page; p.s0[h] = (part - page * a.per_page) * SIZE; }
      p.base[h] = page * bs + p.s0[h];
      p.live[h] = min(min(bs - p.s0[h], len - p.base[h]), SIZE);
    }
    return p;
  };
  auto fetch = [&](int i, int stage) {         // the warp's i-th unit; every lane calls it, i by i; an empty group behind the last
    if (i < mine) {
      const int u = first + i * nw;
      if (i > 0 && i % 32 == 0) ids = look_up(u);
      Place p = place(u);
#pragma unroll
      for (int h = 0; h < H; ++h) {
        const int id = __shfl_sync(0xffffffffu, ids.of[h], i % 32);
        if (id < 0 && p.live[h] > 0 && lane == 0) note(kv.status, FL_DEC_BAD_PAGE);
        if (id < 0) p.live[h] = 0;
        const long long cell = (pool0 + max(id, 0)) * kv.heads + kh, at = (cell * bs + p.s0[h]) * D;
        const uint32_t to = cell0 + stage * R::STAGE + h * SIZE * R::PITCH;
        if (column) {
          const uint8_t *k = kp + at, *v = vp + at;
          if (p.live[h] == SIZE) {
#pragma unroll
            for (int j = 0; j < SIZE; j += PASS) {
              copy16(to + j * R::PITCH, k + j * D);
              copy16(to + R::KEYS + j * R::PITCH, v + j * D);
            }
          } else {
#pragma unroll
            for (int j = 0; j < SIZE; j += PASS) {
              const bool there = j + row0 < p.live[h];           // the addresses of others may be anything
              copy16(to + j * R::PITCH, there ? k + j * D : reinterpret_cast<const uint8_t*>(kv.k), there);
              copy16(to + R::KEYS + j * R::PITCH, there ? v + j * D : reinterpret_cast<const uint8_t*>(kv.v), there);
            }
          }
        }
        if (lane < 2) copy4(ring + stage * R::STAGE + R::SCALES + 8 * h + 4 * lane, (lane ? kv.v_scale : kv.k_scale) + cell, id >= 0);
      }
    }
    copies_commit();
  };

#pragma unroll
  for (int s = 0; s < R::STAGES - 1; ++s) fetch(s, s);

  // queries, as the second operand; a row's power of two is undone on its scores
  uint32_t qb[NT][KJ][8];
  float factor[NT][2];                         // of columns 2 t and 2 t + 1
  int sees[NT][2], fewest = len;               // slots that the column's token sees; the fewest of any that sees some
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float f[KJ][16];
    float m = 0.f;
    if (MASS) {
      // rows that are no token's count as zeros: whatever stands in them would move the references of the columns beside them, by a rounding
      const int row = r0 + 8 * nt + (g & COL), tok = a.tokens == 1 ? 0 : row / a.group;
      if (tok >= n_new || start + tok < 0) {
#pragma unroll
        for (int j = 0; j < KJ; ++j) q_raw[nt][j][0] = q_raw[nt][j][1] = make_uint4(0, 0, 0, 0);
      }
    }
#pragma unroll
    for (int j = 0; j < KJ; ++j) {
      float v0[8], v1[8];
      unpack<T>(q_raw[nt][j][0], v0);
      unpack<T>(q_raw[nt][j][1], v1);
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
    const int e = max((int)(__float_as_uint(m) >> 23), 27);                     // 127 + exponent
    const float to = __uint_as_float((uint32_t)(268 - e) << 23), back = __uint_as_float((uint32_t)(e - 14) << 23);       // 2^(14 - exponent) and its inverse
#pragma unroll
    for (int j = 0; j < KJ; ++j)
#pragma unroll
      for (int i = 0; i < 8; ++i) qb[nt][j][i] = half2_of(f[j][2 * i] * to, f[j][2 * i + 1] * to);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      factor[nt][c] = __shfl_sync(0xffffffffu, back, (2 * t + c) * 4) * a.scale;
      const int rc = r0 + 8 * nt + (2 * t + c & COL), tc = a.tokens == 1 ? 0 : rc / a.group;
      sees[nt][c] = rc < all_rows && tc < n_new ? max((int)min(start + tc + 1, (long long)len), 0) : 0;
      if (sees[nt][c] > 0) fewest = min(fewest, sees[nt][c]);
    }
  }
  fewest = __reduce_min_sync(0xffffffffu, fewest);

  // A column's sums: weights 2^(score - m) in l (lx: before they were cut), the same times values in o, in units of 2^down.  m and down are whole numbers,
  // so that neither reference leaves a rounding behind when it moves.
  float o[NT][MT][4], m[NT][2], l[NT][2], lx[NT][2], down[NT][2];
  const uint32_t rest = t < 2 ? 0u : 0xffffe000u;              // BOTH: the bits of a weight that are not this column's
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[nt][i][j] = 0.f;
#pragma unroll
    for (int c = 0; c < 2; ++c) { m[nt][c] = LOWEST; l[nt][c] = lx[nt][c] = 0.f; down[nt][c] = LOWEST; }
  }

  int stage = 0;
#pragma unroll 1
  for (int i = 0; i < mine; ++i) {
    copies_wait<R::STAGES - 2>();
    __syncwarp();                                // every lane's copies of this unit are there, and the last unit has been read
    const uint32_t at = ring + stage * R::STAGE;
    const int u = first + i * nw;
    fetch(i + R::STAGES - 1, stage == 0 ? R::STAGES - 1 : stage - 1);
    stage = stage + 1 == R::STAGES ? 0 : stage + 1;
    const Place p = place(u);
    int base[H], live[H];
    float ks[H], vs[H];
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const uint2 scales = lds_v2(at + R::SCALES + 8 * h);
      ks[h] = __uint_as_float(scales.x);
      vs[h] = __uint_as_float(scales.y);
      base[h] = p.base[h];
      live[h] = ks[h] == 0.f ? 0 : p.live[h];    // 0: a page that is not there
    }
    float s[NT][4], s2[NT][4];                   // two chains of products
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[nt][i] = s2[nt][i] = 0.f;
#pragma unroll
    for (int j = 0; j < KJ; ++j) {
      const uint32_t from = at + g * R::PITCH + (DP == 128 ? 32 * t + 16 * j : 16 * t);
      const uint4 u0 = lds_v4(from), u1 = lds_v4(from + 8 * R::PITCH);
      const uint32_t k0[4] = {u0.x, u0.y, u0.z, u0.w}, k1[4] = {u1.x, u1.y, u1.z, u1.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint2 h0 = halves(k0[i]), h1 = halves(k1[i]);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma(i & 1 ? s2[nt] : s[nt], h0.x, h1.x, h0.y, h1.y, qb[nt][j][2 * i], qb[nt][j][2 * i + 1]);
      }
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[nt][i] += s2[nt][i];
    uint32_t v[4][DP / 32];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t from = at + R::KEYS + (2 * t + (i & 1) + 8 * (i >> 1)) * R::PITCH + VB * g;
      if constexpr (DP == 128) {
        const uint4 w = lds_v4(from);
        v[i][0] = w.x; v[i][1] = w.y; v[i][2] = w.z; v[i][3] = w.w;
      } else {
        const uint2 w = lds_v2(from);
        v[i][0] = w.x; v[i][1] = w.y;
      }
    }
    // tokens g and g + 8: the unit's only part, or one each
    constexpr int H1 = H - 1;
    const bool seen = base[0] + SIZE <= fewest && base[H1] + SIZE <= fewest;         // by every column
    if (!seen || live[0] < SIZE || live[H1] < SIZE) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          s[nt][c] = g < min(sees[nt][c] - base[0], live[0]) ? s[nt][c] : -INFINITY;
          s[nt][2 + c] = g + 8 - 8 * H1 < min(sees[nt][c] - base[H1], live[H1]) ? s[nt][2 + c] : -INFINITY;
        }
    }
    float page_unit[H];                          // log2 of the values' scale
#pragma unroll
    for (int h = 0; h < H; ++h) page_unit[h] = (float)((int)(__float_as_uint(vs[h]) >> 23) - 127);
    float wt[NT][4];                             // weights, first their logarithms
    bool beyond = false;
    // -inf stays -inf whatever it meets: a factor of 0 (an underflow, or no page) would make it NaN
    auto by = [&](int nt, int i) { return fmaxf(factor[nt][i & 1] * ks[i >> 1 ? H1 : 0], 0x1p-126f); };
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 4; ++i) wt[nt][i] = fmaf(s[nt][i], by(nt, i), -m[nt][i & 1]);
#pragma unroll
      for (int c = 0; c < 2; ++c) beyond |= fmaxf(wt[nt][c], wt[nt][2 + c]) > SLACK || fmaxf(page_unit[0], page_unit[H1]) - down[nt][c] > ROOM;
    }
    if (__any_sync(0xffffffffu, beyond)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float f[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float from = m[nt][c], was = down[nt][c];
          const float s0 = s[nt][c] * by(nt, c), s1 = s[nt][2 + c] * by(nt, 2 + c);
          m[nt][c] = fmaxf(from, ceilf(max_rows(fmaxf(s0, s1))));
          wt[nt][c] = s0 - m[nt][c];
          wt[nt][2 + c] = s1 - m[nt][c];
          const float fall = from - m[nt][c], e = exp2_fast(fall);
          l[nt][c] *= e;
          if (EXACT) lx[nt][c] *= e;
          down[nt][c] = fmaxf(was + fall, ceilf(max_rows(fmaxf(wt[nt][c] + page_unit[0], wt[nt][2 + c] + page_unit[H1]))) - START);
          f[c] = exp2_fast(was - down[nt][c] + fall);
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          o[nt][i][0] *= f[0]; o[nt][i][1] *= f[1];
          o[nt][i][2] *= f[0]; o[nt][i][3] *= f[1];
        }
      }
    }
    uint32_t p0[NT], p1[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float add[2], w[4];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          wt[nt][2 * h + c] = exp2_fast(wt[nt][2 * h + c]);
          w[2 * h + c] = BOTH ? wt[nt][2 * h + c] : eleven_bits(wt[nt][2 * h + c]);
        }
        add[c] = wt[nt][c] + wt[nt][2 + c];
        l[nt][c] += w[c] + w[2 + c];
        if (EXACT) lx[nt][c] += add[c];
        // a page whose values are so much larger than what counts has no weight beyond the smallest numbers
        const float u0 = exp2_fast(fminf(page_unit[0] - down[nt][c], 126.f)), u1 = HALVES ? exp2_fast(fminf(page_unit[H1] - down[nt][c], 126.f)) : u0;
        w[c] *= u0;
        w[2 + c] *= u1;
      }
      if (BOTH) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] -= eleven_bits(w[i], rest);
      }
      p0[nt] = transposed(half2_cut(w[0], w[1]));
      p1[nt] = transposed(half2_cut(w[2], w[3]));
      if (MASS) {
        auto keep = [&](int part, float s0, float s1) {
          s0 = sum_rows(s0);
          s1 = sum_rows(s1);
          if (g == 0 && part < a.units) {
            float2* w = a.unit_s + ((long long)b * a.units + part) * a.heads * a.tokens + kh * all_rows + r0 + 8 * nt + 2 * t;
            if (8 * nt + 2 * t < n_rows) w[0] = make_float2(s0, m[nt][0]);
            if (8 * nt + 2 * t + 1 < n_rows) w[1] = make_float2(s1, m[nt][1]);
          }
        };
        if (HALVES) {
          keep(2 * u, wt[nt][0], wt[nt][1]);
          keep(2 * u + 1, wt[nt][2], wt[nt][3]);
        } else {
          keep(u, add[0], add[1]);
        }
      }
    }
    auto values = [&](auto each) {
#pragma unroll
      for (int w = 0; w < DP / 32; ++w)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t sel = h ? 0x7362u : 0x5140u;
          const uint32_t u0 = __byte_perm(v[0][w], v[1][w], sel), u1 = __byte_perm(v[2][w], v[3][w], sel);
          const uint2 h0 = halves(u0), h1 = halves(u1);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) each(nt, 2 * w + h, h0.x, h0.y, h1.x, h1.y);
        }
    };
    if (a.tokens == 1 || seen) {
      values([&](int nt, int i, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) { mma(o[nt][i], a0, a1, a2, a3, p0[nt], p1[nt]); });
    } else {
      // Among the last tokens a column's weight of 0 must not meet a value of a later token, which may be NaN: one new token at a time, with
      // the values behind it left out (the last one first, so that each leaves out more), and only its own columns take the sums.
      const int t0 = r0 / a.group, t1 = min((r0 + n_rows - 1) / a.group, n_new - 1);
      for (int tok = t1; tok >= t0; --tok) {
        const int sees_now = (int)min(start + tok + 1, (long long)len);
        if (sees_now <= base[0]) break;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int w = 0; w < DP / 32; ++w)
            if (2 * t + (i & 1) + (HALVES ? 0 : 8 * (i >> 1)) >= sees_now - base[HALVES ? i >> 1 : 0]) v[i][w] = 0;
        values([&](int nt, int i, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
          float c[4] = {0.f, 0.f, 0.f, 0.f};
          mma(c, a0, a1, a2, a3, p0[nt], p1[nt]);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if ((r0 + 8 * nt + (2 * t + (j & 1) & COL)) / a.group == tok) o[nt][i][j] += c[j];
        });
      }
    }
  }
  copies_wait<0>();
  __syncthreads();                               // the rings' memory is free

  // the warps' parts become one
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int row = 8 * nt + 2 * t + c;
      const float sum = sum_rows(l[nt][c]), f = sum == 0.f ? 0.f : 1.f / sum, unit = exp2f(down[nt][c]);
      if (g == 0) { s_m[warp][row] = m[nt][c]; s_l[warp][row] = sum; }
      if (EXACT) {
        const float x = sum_rows(lx[nt][c]);
        if (g == 0) s_x[warp][row] = x;
      }
      auto mean = [&](float v) { return v * f * unit; };
#pragma unroll
      for (int i = 0; i < MT; i += 2)
        *reinterpret_cast<float4*>(&s_o[warp][row][VB * g + 2 * i]) = make_float4(mean(o[nt][i][c]), mean(o[nt][i][2 + c]), mean(o[nt][i + 1][c]), mean(o[nt][i + 1][2 + c]));
    }
  __syncthreads();
  // Four columns of a row per thread.  `joined4` adds up the warps' means by what they count for in the CTA's.
  const long long row_at = (long long)b * a.heads * a.tokens + kh * all_rows + r0;
  const int pieces = D / 4;
  auto joined4 = [&](int row, int d, float& mm, float& ll, float& xx) {
    float w[WARPS];
    mm = LOWEST;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) mm = fmaxf(mm, s_m[i][row]);
    ll = xx = 0.f;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) { w[i] = share(s_m[i][row], s_l[i][row], mm); ll += w[i]; }
    if (EXACT) {
#pragma unroll
      for (int i = 0; i < WARPS; ++i) xx += share(s_m[i][row], s_x[i][row], mm);
    } else {
      xx = ll;
    }
    const float f = ll == 0.f ? 0.f : 1.f / ll;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < WARPS; ++i) {
      float4 v = *reinterpret_cast<const float4*>(&s_o[i][row][d]);
      if (BOTH) {
        const float4 more = *reinterpret_cast<const float4*>(&s_o[i][row + 4][d]);
        v.x += more.x; v.y += more.y; v.z += more.z; v.w += more.w;
      }
      const float k = w[i] * f;
      acc.x += k * v.x; acc.y += k * v.y; acc.z += k * v.z; acc.w += k * v.w;
    }
    return acc;
  };
  auto result = [&](int row, int d, float mm, float ll, float xx, float4 acc) {
    const int r = r0 + row, tok = a.tokens == 1 ? 0 : r / a.group, h = kh * a.group + r - tok * a.group;
    const bool none = tok >= n_new || start + tok < 0 || len == 0;
    if (none) acc = make_float4(0.f, 0.f, 0.f, 0.f);
    else if (ll == 0.f) acc = make_float4(NAN, NAN, NAN, NAN);
    *reinterpret_cast<uint2*>(reinterpret_cast<T*>(a.out) + (((long long)b * a.tokens + tok) * a.heads + h) * D + d) =
        make_uint2(Typed<T>::pack(acc.x, acc.y), Typed<T>::pack(acc.z, acc.w));
    if (MASS && d == 0) {
      float* p = a.part_s + (row_at + row) * (a.clustered ? 1 : a.splits) * PART;
      *reinterpret_cast<float4*>(p) = make_float4(mm, ll, xx, 0.f);
    }
  };
  if (!a.clustered || a.splits == 1) {
    for (int i = threadIdx.x; i < n_rows * pieces; i += WARPS * 32) {
      const int row = i / pieces, d = 4 * (i - row * pieces);
      float mm, ll, xx;
      const float4 acc = joined4(row, d, mm, ll, xx);
      if (a.splits == 1) {
        result(row, d, mm, ll, xx, acc);
      } else {
        const long long part = (row_at + row) * a.splits + z;
        *reinterpret_cast<float4*>(a.part_o + part * D + d) = acc;
        if (d == 0) *reinterpret_cast<float4*>(a.part_s + part * PART) = make_float4(mm, ll, xx, 0.f);
      }
    }
    return;
  }
  for (int i = threadIdx.x; i < n_rows * pieces; i += WARPS * 32) {
    const int row = i / pieces, d = 4 * (i - row * pieces);
    float mm, ll, xx;
    const float4 acc = joined4(row, d, mm, ll, xx);
    *reinterpret_cast<float4*>(&s_o[0][row][d]) = acc;         // read and written by this thread alone
    if (d == 0) { s_cm[row] = mm; s_cl[row] = ll; s_cx[row] = xx; }
  }
  __syncwarp();
  cluster_sync_all();
  for (int i = z * WARPS * 32 + threadIdx.x; i < n_rows * pieces; i += a.splits * WARPS * 32) {
    const int row = i / pieces, d = 4 * (i - row * pieces);
    const uint32_t am = smem_u32(&s_cm[row]), al = smem_u32(&s_cl[row]), ao = smem_u32(&s_o[0][row][d]);
    float pm[8], pl[8], px[8], mm = LOWEST, ll = 0.f;
    float4 po[8], acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int x = 0; x < 8; ++x)
      if (x < a.splits) {
        pm[x] = ld_cluster_f32(map_to_cta(am, x));
        pl[x] = ld_cluster_f32(map_to_cta(al, x));
        if (EXACT) px[x] = ld_cluster_f32(map_to_cta(smem_u32(&s_cx[row]), x));
        po[x] = ld_cluster_f32x4(map_to_cta(ao, x));
      }
#pragma unroll
    for (int x = 0; x < 8; ++x)
      if (x < a.splits) mm = fmaxf(mm, pm[x]);
#pragma unroll
    for (int x = 0; x < 8; ++x)
      if (x < a.splits) { pl[x] = share(pm[x], pl[x], mm); ll += pl[x]; }
    float xx = EXACT ? 0.f : ll;
    if (EXACT) {
#pragma unroll
      for (int x = 0; x < 8; ++x)
        if (x < a.splits) xx += share(pm[x], px[x], mm);
    }
    const float f = ll == 0.f ? 0.f : 1.f / ll;
#pragma unroll
    for (int x = 0; x < 8; ++x)
      if (x < a.splits) {
        const float k = pl[x] * f;
        acc.x += k * po[x].x; acc.y += k * po[x].y; acc.z += k * po[x].z; acc.w += k * po[x].w;
      }
    result(row, d, mm, ll, xx, acc);
  }
  __syncwarp();
  cluster_sync_all();                            // nobody leaves while its part is being read
}

struct Joined { float m, sum, w0, w1; };       // of a row's parts: their maximum and sum; what parts `lane` and `lane` + 32 count for in it
template <int SUM>                              // which of the parts' sums
__device__ __forceinline__ Joined joined(const AttArgs& a, long long at, int parts, int lane) {
  Joined j;
  float m[2] = {LOWEST, LOWEST}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (lane + 32 * i < parts) {
      const float4 p = *reinterpret_cast<const float4*>(a.part_s + (at + lane + 32 * i) * PART);
      m[i] = p.x;
      l[i] = SUM == 1 ? p.y : p.z;
    }
  j.m = fmaxf(m[0], m[1]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) j.m = fmaxf(j.m, __shfl_xor_sync(0xffffffffu, j.m, o));
  j.w0 = share(m[0], l[0], j.m);
  j.w1 = share(m[1], l[1], j.m);
  j.sum = j.w0 + j.w1;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) j.sum += __shfl_xor_sync(0xffffffffu, j.sum, o);
  return j;
}

// Joins parts that are no cluster's: a CTA per row and request.  The first row_ctas CTAs of a request have its rows; the others, if weights are asked
// for, its pages, a warp each, whose lanes add up the rows' shares in an order that is always the same.
template <typename T>
__global__ void __launch_bounds__(128) finish_kernel(const AttArgs a, const FlKv8 kv, float* mass, int row_ctas, int page_ctas) {
  grid_dep_launch();
  grid_dep_wait();
  const int b = blockIdx.y, D = kv.dim, bs = kv.block_size, rows = a.heads * a.tokens, all_rows = a.group * a.tokens;
  const int len = seen_by_last(a, kv, b), units = (len + bs - 1) / bs * a.per_page;
  const int parts = a.clustered ? 1 : a.splits, lane = threadIdx.x & 31;
  if ((int)blockIdx.x < row_ctas) {
    const int row = blockIdx.x, kh = row / all_rows, r = row - kh * all_rows, tok = r / a.group, h = kh * a.group + r - tok * a.group;
    const long long at = ((long long)b * rows + row) * parts;
    const Joined j = joined<1>(a, at, parts, lane);
    const float f = j.sum == 0.f ? 0.f : 1.f / j.sum;
    const bool none = tok >= tokens_of(a.counts, b, a.tokens) || start_of(a, kv, b) + tok < 0;
    const int d = threadIdx.x;
    const float* part = a.part_o + at * D + min(d, D - 1);
    float acc = 0.f;
    for (int z0 = 0; z0 < parts; z0 += 16) {                   // sixteen on their way at a time
      float v[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = z0 + i < parts ? part[(z0 + i) * D] : 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) acc += __shfl_sync(0xffffffffu, z0 < 32 ? j.w0 : j.w1, (z0 + i) & 31) * f * v[i];
    }
    if (d < D) reinterpret_cast<T*>(a.out)[(((long long)b * a.tokens + tok) * a.heads + h) * D + d] = T(none ? 0.f : j.sum == 0.f ? NAN : acc);
    return;
  }
  if (mass == nullptr || len == 0) return;
  extern __shared__ float2 s_row[];                          // of every row: the maximum, and 1 / its sum of weights (0: a row that sees nothing)
  const int n_new = tokens_of(a.counts, b, a.tokens);
  auto keep = [&](int r, float m, float sum) {
    const int tok = (r % all_rows) / a.group;
    s_row[r] = make_float2(m, tok >= n_new || start_of(a, kv, b) + tok < 0 ? 0.f : sum == 0.f ? NAN : 1.f / sum);
  };
  if (parts == 1) {
    for (int r = threadIdx.x; r < rows; r += 128) {
      const float* p = a.part_s + ((long long)b * rows + r) * PART;
      keep(r, p[0], p[2]);
    }
  } else {
    for (int r = threadIdx.x >> 5; r < rows; r += 4) {
      const Joined j = joined<2>(a, ((long long)b * rows + r) * parts, parts, lane);
      if (lane == 0) keep(r, j.m, j.sum);
    }
  }
  __syncthreads();
  const int pages = units / a.per_page;
  for (int p = (blockIdx.x - row_ctas) * 4 + (threadIdx.x >> 5); p < pages; p += page_ctas * 4) {
    float sum = 0.f;
    for (int i = 0; i < a.per_page; ++i) {
      const float2* w = a.unit_s + ((long long)b * a.units + p * a.per_page + i) * rows;
      for (int r = lane; r < rows; r += 32) {
        const float2 row = s_row[r];
        if (row.y != 0.f) sum += w[r].x * exp2_fast(w[r].y - row.x) * row.y;         // what a row that sees nothing left may be NaN
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) mass[(long long)b * kv.table_stride + p] += sum;
  }
}

// ---- eviction ---------------------------------------------------------------------------------------------------------------
// Bound by the latency of one CTA per request.  How many pages go is known; the weight up to which they go is found digit by digit (histograms of 256, up
// to the digit whose whole counter goes), and the row is dealt out in its order.  Threads keep their weights in registers, so that memory is read once: one
// each of up to 1024 pages (16 rows of 145: 12.5 us with eight each, 3.4 with one), eight each of more (64 rows of 8192: 28 us with one page per thread and
// pass, 14.3 with a vote per page in every digit and two rankings, now 9.6, of which instructions take half); rows of more than 8192 go by in
// pieces of that, once for every digit (4 rows of 40000: 52 us).
constexpr int EVICT_THREADS = 1024, EVICT_WARPS = EVICT_THREADS / 32, EVICT_EACH = 8;

// weights in an order that whole numbers have: NaN last, -0 as 0
__device__ __forceinline__ uint32_t evict_key(float m) {
  if (m != m) return 0xffffffffu;
  const uint32_t u = __float_as_uint(m == 0.f ? 0.f : m);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

template <int EACH> struct EvictShared {
  int hist[4][256];                                                            // one per digit
  uint8_t kind[EACH * EVICT_THREADS];                                          // of the piece's pages
  unsigned short to[EACH * EVICT_THREADS];                                     // how many go before the page, and whether it does
  unsigned before[EVICT_WARPS];                                                // a warp's pages below the limit, and from bit 16 on those equal to it
  int digit, left, whole;
};
constexpr unsigned EVICT_BELOW = 1, EVICT_EQUAL = 2, EVICT_OUT = 0x8000;

template <int EACH>
__global__ void __launch_bounds__(EVICT_THREADS) evict_kernel(const float* mass, const int* table, const long long* lengths, int pages, int bs, int keep,
                                                              int recent, int sinks, float* mass_out, int* table_out, long long* lengths_out, int* gone) {
  __shared__ __align__(16) EvictShared<EACH> s;
  const int b = blockIdx.x, threads = blockDim.x, piece_size = threads * EACH, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  mass += (long long)b * pages; table += (long long)b * pages;
  mass_out += (long long)b * pages; table_out += (long long)b * pages;
  const long long given = lengths[b];
  float m[EACH];
  int id[EACH];
  auto place = [&](unsigned piece, int k) { return piece + (unsigned)(k * threads + tid); };
  auto load = [&](unsigned piece, bool ids) {
#pragma unroll
    for (int k = 0; k < EACH; ++k) m[k] = place(piece, k) < (unsigned)pages ? mass[place(piece, k)] : 0.f;
    if (!ids) return;
#pragma unroll
    for (int k = 0; k < EACH; ++k) id[k] = place(piece, k) < (unsigned)pages ? table[place(piece, k)] : 0;
  };
  load(0, true);
  for (int i = tid; i < 4 * 256; i += threads) s.hist[0][i] = 0;
  const long long len = max(given, 0ll);
  // (a division in 64 bits would cost each warp as much as a digit)
  const long long full = len <= 0x7fffffffll ? (long long)((unsigned)len / (unsigned)bs) : len / bs;
  const int used = (int)min(full + (full * bs != len), (long long)pages), extra = max(used - keep, 0);
  if (tid == 0) {
    lengths_out[b] = given - (long long)extra * bs;
    gone[b] = extra;
  }
  // pages that may go: from `lo` on, `free_pages` of them; at least `extra`, since keep >= recent + sinks
  const unsigned lo = sinks, free_pages = extra > 0 ? used - recent - sinks : 0;
  uint32_t key[EACH];
  unsigned free = 0;                                           // of the thread's
  auto look = [&](unsigned piece) {
    free = 0;
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
      key[k] = evict_key(m[k]);
      free |= (place(piece, k) - lo < free_pages ? 1u : 0u) << k;
    }
  };
  look(0);
  __syncthreads();
  uint32_t prefix = 0;
  int shift = 32, left = extra;                                // of those that go, among the weights that begin with the digits found
  bool whole = extra == 0;                                     // all of them do: further digits say nothing
  while (shift > 0 && !whole) {
    shift -= 8;
    int* hist = s.hist[shift / 8];
    for (unsigned piece = 0; piece < (unsigned)pages; piece += piece_size) {
      if (pages > piece_size) { load(piece, false); look(piece); }
      // weights that no token ever saw are all alike: a warp's additions to one counter cost no more than others (adding them up first, 12.3 us)
#pragma unroll
      for (int k = 0; k < EACH; ++k)
        if ((free >> k & 1) && (shift == 24 || key[k] >> (shift + 8) == prefix)) atomicAdd(&hist[key[k] >> shift & 255], 1);
    }
    __syncthreads();
    if (warp == 0) {
      const int4 h0 = reinterpret_cast<const int4*>(hist)[2 * lane], h1 = reinterpret_cast<const int4*>(hist)[2 * lane + 1];
      const int n[8] = {h0.x, h0.y, h0.z, h0.w, h1.x, h1.y, h1.z, h1.w};
      const int sum = n[0] + n[1] + n[2] + n[3] + n[4] + n[5] + n[6] + n[7];
      int before = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, before, o);
        if (lane >= o) before += v;
      }
      before -= sum;
      if (before < left && before + sum >= left) {
        int j = 0, equals = n[0];
#pragma unroll
        for (int q = 0; q < 7; ++q)
          if (j == q && before + n[q] < left) { before += n[q]; ++j; equals = n[q + 1]; }
        s.digit = lane * 8 + j;
        s.left = left - before;
        s.whole = equals == left - before;
      }
    }
    __syncthreads();
    prefix = prefix << 8 | (uint32_t)s.digit;
    left = s.left;
    whole = s.whole;
  }
  // Kept pages go to the front, those that go to used - extra and on.  A thread ranks neighbours, so that a warp has one sum and not one per page of a thread;
  // what a page is and where it goes change their order through shared memory.
  unsigned below_before = 0, equal_before = 0;
  auto going = [&](unsigned below, unsigned equal) { return below + min(equal, (unsigned)left); };          // of those that are equal the first `left` go
  for (unsigned piece = 0; piece < (unsigned)pages; piece += piece_size) {
    if (pages > piece_size) { load(piece, true); look(piece); }
    const unsigned gone_before = going(below_before, equal_before);
    unsigned to[EACH] = {};
    if (extra > 0) {
      unsigned kind[EACH], own = 0;
#pragma unroll
      for (int k = 0; k < EACH; ++k) {
        const uint32_t digits = key[k] >> shift;
        kind[k] = !(free >> k & 1) ? 0 : digits < prefix ? EVICT_BELOW : digits == prefix ? EVICT_EQUAL : 0;
      }
      if constexpr (EACH > 1) {
        static_assert(EACH == 8, "a vector of eight bytes and one of eight halves");
#pragma unroll
        for (int k = 0; k < EACH; ++k) s.kind[k * threads + tid] = (uint8_t)kind[k];
        __syncthreads();
        const uint2 v = reinterpret_cast<const uint2*>(s.kind)[tid];
#pragma unroll
        for (int k = 0; k < EACH; ++k) kind[k] = (k < 4 ? v.x : v.y) >> (k % 4 * 8) & 255;
      }
#pragma unroll
      for (int k = 0; k < EACH; ++k) {
        kind[k] = (kind[k] & EVICT_BELOW) | (kind[k] & EVICT_EQUAL) << 15;             // as the sums have them
        own += kind[k];
      }
      unsigned upto = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      if (lane == 31) s.before[warp] = upto;
      __syncthreads();
      unsigned all = lane * 32 < threads ? s.before[lane] : 0, others = lane < warp ? all : 0;
      all = __reduce_add_sync(0xffffffffu, all);
      others = __reduce_add_sync(0xffffffffu, others);
      upto += others - own;                                    // of the piece, before the thread's
#pragma unroll
      for (int k = 0; k < EACH; ++k) {
        const unsigned equals = equal_before + (upto >> 16);
        const bool out = kind[k] == 1 || (kind[k] != 0 && equals < (unsigned)left);
        to[k] = going(below_before + (upto & 0xffffu), equals) - gone_before + (out ? EVICT_OUT : 0);
        upto += kind[k];
      }
      below_before += all & 0xffffu;
      equal_before += all >> 16;
      if constexpr (EACH > 1) {
        reinterpret_cast<uint4*>(s.to)[tid] = make_uint4(to[0] | to[1] << 16, to[2] | to[3] << 16, to[4] | to[5] << 16, to[6] | to[7] << 16);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < EACH; ++k) to[k] = s.to[k * threads + tid];
      }
    }
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
      const unsigned i = place(piece, k);
      if (i >= (unsigned)pages) continue;
      const bool out = to[k] & EVICT_OUT;
      const unsigned rank = gone_before + (to[k] & (EVICT_OUT - 1));
      const unsigned at = i >= (unsigned)used ? i : out ? used - extra + rank : i - rank;
      table_out[at] = id[k];
      mass_out[at] = out ? 0.f : m[k];
    }
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
         kv->table_stride >= 0 && (long long)kv->table_stride * kv->block_size <= 0x3fffffffll && (long long)kv->block_size * kv->dim <= 0x7fffffffll;
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
  a.reach = (int)(((long long)tokens + kv->block_size - 2) / kv->block_size + 1);
  const long long page_units = 2ll * batch * a.reach * kv->heads, rows = (long long)batch * tokens;
  const bool q = qkv != out || bias != nullptr || rope != nullptr;
  const int per_warp = fl::kv8::STEPS * (32 / (kv->dim / 16));       // heads
  a.parts = heads <= per_warp ? 1 : (heads + per_warp - 1) / per_warp;
  const long long units = page_units + (q ? rows * a.parts : 0);
  if (units > 0x7fffffffll || (long long)(heads + 2 * kv->heads) * kv->dim > 0x7fffffffll) return -2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid_of(units), 1, 1);
  cfg.blockDim = dim3(128, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = rows <= FL_THIN_MAX_ROWS ? 1 : 0;      // as the decoder's other passes
  FL_KV8_TYPES(dtype, return (int)cudaLaunchKernelEx(&cfg, fl::kv8::write_kernel<T>, a, *kv, (unsigned)page_units, (unsigned)units));
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

// How a call is cut up: enough CTAs for the SMs (four of NT = 1, two of NT = 2 each), as a cluster where 8 per request and KV head are enough.
namespace {
struct Cut { int nt, row_parts, per_page, units, splits; bool both, halves, clustered; };
Cut cut_of(int batch, int tokens, int heads, const FlKv8* kv) {
  Cut c;
  const long long rows = (long long)heads / kv->heads * tokens;
  c.nt = rows > 8 ? 2 : 1;
  c.both = rows <= 4;
  c.row_parts = (int)((rows + 8 * c.nt - 1) / (8 * c.nt));
  c.halves = kv->block_size % 16 != 0;
  const int size = c.halves ? 8 : 16;
  c.per_page = (kv->block_size + size - 1) / size;
  c.units = kv->table_stride * c.per_page;
  const int steps = c.halves ? (c.units + 1) / 2 : c.units;
  const long long ctas = (long long)batch * kv->heads * c.row_parts, want = 148ll * (c.nt == 1 ? 4 : 2);
  const long long most = (steps + fl::kv8::FEWEST - 1) / fl::kv8::FEWEST;
  long long splits = want / (ctas < 1 ? 1 : ctas);
  const long long even = (steps + fl::kv8::LONGEST - 1) / fl::kv8::LONGEST;
  if (splits < even) splits = even;
  if (splits > most) splits = most;
  if (splits > fl::kv8::MOST_PARTS) splits = fl::kv8::MOST_PARTS;
  if (splits < 1) splits = 1;
  c.splits = (int)splits;
  c.clustered = splits <= 8;
  return c;
}
long long up16(long long bytes) { return (bytes + 15) / 16 * 16; }

template <typename T, int DP, int NT, bool BOTH, bool FULL, bool HALVES, bool MASS>
int launch_attention(const fl::kv8::AttArgs& a, const FlKv8& kv, dim3 grid, bool early, cudaStream_t stream) {
  constexpr int smem = fl::kv8::Ring<DP>::BYTES;
  static bool set_on[64];                          // per device: a process may drive several GPUs
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  if (dev < 0 || dev >= 64) return -3;
  if (!set_on[dev]) {
    e = cudaFuncSetAttribute(fl::kv8::attention_kernel<T, DP, NT, BOTH, FULL, HALVES, MASS>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return (int)e;
    set_on[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.dynamicSmemBytes = smem;
  cfg.gridDim = grid;
  cfg.blockDim = dim3(fl::kv8::WARPS * 32, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = 1; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = a.clustered ? a.splits : 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = early ? 2 : 1;
  return (int)cudaLaunchKernelEx(&cfg, fl::kv8::attention_kernel<T, DP, NT, BOTH, FULL, HALVES, MASS>, a, kv);
}
template <typename T, int DP>
int launch_attention(const fl::kv8::AttArgs& a, const FlKv8& kv, const Cut& c, bool mass, dim3 grid, bool early, cudaStream_t stream) {
#define FL_ATT(N, B, F, S) return mass ? launch_attention<T, DP, N, B, F, S, true>(a, kv, grid, early, stream) : launch_attention<T, DP, N, B, F, S, false>(a, kv, grid, early, stream)
#define FL_ATT_ROWS(F, S) do { if (c.both) FL_ATT(1, true, F, S); if (c.nt == 1) FL_ATT(1, false, F, S); FL_ATT(2, false, F, S); } while (0)
  if (c.halves) FL_ATT_ROWS(false, true);
  if (kv.dim == DP) FL_ATT_ROWS(true, false);
  FL_ATT_ROWS(false, false);
#undef FL_ATT_ROWS
#undef FL_ATT
}
}  // namespace

// Requests beyond a grid's second dimension, and those whose scratch would be more than this, go in launches one after the other, which share the
// scratch: weights cost 8 bytes per row and unit of the table, 4 MB per request of 64 heads and 8192 pages of 16.
constexpr int MOST_REQUESTS = 65535;
constexpr long long MOST_SCRATCH = 256ll << 20;

static long long scratch_of(const Cut& c, int batch, int tokens, int heads, const FlKv8* kv, bool mass) {
  const long long rows = (long long)batch * heads * tokens, parts = c.clustered ? 1 : c.splits;
  long long bytes = 0;
  if (!c.clustered) bytes += up16(rows * parts * kv->dim * 4);
  if (!c.clustered || mass) bytes += up16(rows * parts * fl::kv8::PART * 4);
  if (mass) bytes += up16(rows * c.units * 8);
  return bytes;
}
static int at_once(int batch, int tokens, int heads, const FlKv8* kv, bool mass) {
  int n = batch < MOST_REQUESTS ? batch : MOST_REQUESTS;
  while (n > 1 && scratch_of(cut_of(n, tokens, heads, kv), n, tokens, heads, kv, mass) > MOST_SCRATCH) n = (n + 1) / 2;
  return n;
}

extern "C" long long fl_kv8_attention_scratch(int batch, int tokens, int heads, const FlKv8* kv, int mass) {
  if (!sizes_fit(kv) || batch < 1 || tokens < 1 || heads < 1 || heads % kv->heads) return 0;
  const int n = at_once(batch, tokens, heads, kv, mass != 0);
  const long long whole = scratch_of(cut_of(n, tokens, heads, kv), n, tokens, heads, kv, mass != 0);
  const long long rest = batch % n == 0 ? 0 : fl_kv8_attention_scratch(batch % n, tokens, heads, kv, mass);
  return whole > rest ? whole : rest;
}

extern "C" int fl_kv8_attention(int dtype, const void* q, long long stride_b, long long stride_t, long long stride_h, const long long* start,
                                const long long* counts, int batch, int tokens, int heads, float scale, const FlKv8* kv, void* out, float* mass,
                                void* scratch, cudaStream_t stream) {
  if (!sizes_fit(kv) || kv->layer < 0 || kv->layer >= kv->layers || batch < 0 || tokens < 0 || heads < 1 || heads % kv->heads ||
      (long long)heads * tokens > 0x3fffffffll || stride_b % 8 || stride_t % 8 || stride_h % 8 || !(scale >= 0.f && scale < INFINITY))
    return -2;
  if (mass != nullptr && (long long)heads * tokens > FL_KV8_MASS_ROWS) return -2;   // a CTA of the kernel that adds them up keeps each one's sum in shared memory
  if (!aligned({q, out, scratch, kv->k, kv->v})) return -4;
  if (batch == 0 || tokens == 0) return 0;
  const int once = at_once(batch, tokens, heads, kv, mass != nullptr);
  if (batch > once) {
    if (dtype != FL_DEC_BF16 && dtype != FL_DEC_FP16) return -1;
    for (long long b = 0; b < batch; b += once) {
      FlKv8 part = *kv;
      part.block_table += b * kv->table_stride;
      const int n = (int)(batch - b < once ? batch - b : once);
      const int rc = fl_kv8_attention(dtype, (const uint8_t*)q + 2 * b * stride_b, stride_b, stride_t, stride_h, start + b, counts ? counts + b : nullptr, n, tokens, heads,
                                      scale, &part, (uint8_t*)out + 2 * b * tokens * heads * kv->dim, mass ? mass + b * kv->table_stride : nullptr, scratch, stream);
      if (rc != 0) return rc;
    }
    return 0;
  }
  const Cut c = cut_of(batch, tokens, heads, kv);
  const long long rows = (long long)batch * heads * tokens, parts = c.clustered ? 1 : c.splits;
  fl::kv8::AttArgs a = {};
  a.q = q; a.sb = stride_b; a.st = stride_t; a.sh = stride_h;
  a.start = start; a.counts = counts; a.batch = batch; a.tokens = tokens; a.heads = heads; a.group = heads / kv->heads;
  a.row_parts = c.row_parts; a.per_page = c.per_page; a.splits = c.splits; a.clustered = c.clustered; a.units = c.units;
  a.scale = scale * 1.4426950408889634f;
  a.out = out;
  uint8_t* s = reinterpret_cast<uint8_t*>(scratch);
  if (!c.clustered) { a.part_o = reinterpret_cast<float*>(s); s += up16(rows * parts * kv->dim * 4); }
  if (!c.clustered || mass) { a.part_s = reinterpret_cast<float*>(s); s += up16(rows * parts * fl::kv8::PART * 4); }
  if (mass) a.unit_s = reinterpret_cast<float2*>(s);
  const dim3 grid(kv->heads * c.row_parts, batch, c.splits);
  const bool early = (long long)batch * tokens <= FL_THIN_MAX_ROWS;
  a.early = early;
  int rc = 0;
  FL_KV8_TYPES(dtype, rc = kv->dim <= 64 ? launch_attention<T, 64>(a, *kv, c, mass != nullptr, grid, early, stream)
                                         : launch_attention<T, 128>(a, *kv, c, mass != nullptr, grid, early, stream));
  if (rc != 0 || (c.clustered && mass == nullptr)) return rc;
  const int row_ctas = c.clustered ? 0 : heads * tokens;
  const int pages = kv->table_stride, most = 8 * 148 / batch;                 // eight CTAs per SM, if there is a page for each warp of theirs
  const int page_ctas = mass == nullptr ? 0 : pages < 4 || most < 1 ? 1 : pages / 4 > most ? most : pages / 4;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(row_ctas + page_ctas, batch, 1);
  cfg.blockDim = dim3(128, 1, 1);
  cfg.dynamicSmemBytes = mass ? (size_t)heads * tokens * sizeof(float2) : 0;
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
  const int each = pages <= fl::kv8::EVICT_THREADS ? 1 : fl::kv8::EVICT_EACH;
  const long long wanted = ((long long)pages + each - 1) / each;
  const int threads = wanted > fl::kv8::EVICT_THREADS ? fl::kv8::EVICT_THREADS : wanted < 32 ? 32 : (int)(wanted + 31) / 32 * 32;
  if (each == 1) fl::kv8::evict_kernel<1><<<batch, threads, 0, stream>>>(mass, table, lengths, pages, block_size, keep, recent, sinks, mass_out, table_out, lengths_out, gone);
  else fl::kv8::evict_kernel<fl::kv8::EVICT_EACH><<<batch, threads, 0, stream>>>(mass, table, lengths, pages, block_size, keep, recent, sinks, mass_out, table_out, lengths_out, gone);
  return (int)cudaGetLastError();
}

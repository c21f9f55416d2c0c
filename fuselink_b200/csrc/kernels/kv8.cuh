// A paged cache of keys and values in 8 bits, and what a decoder does with it (see kv8.cu): writing, attention, eviction.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>
#include "decoder.cuh"

// Codes are e4m3, [layers][num_blocks][heads][block_size][dim]; every (page, head) has a scale, [layers][num_blocks][heads], a power of two: the
// smallest, 2^-100 at least, that keeps the page's largest finite magnitude within 448.  A value that is not finite is stored as NaN.
struct FlKv8 {
  void* k; void* v;
  float* k_scale; float* v_scale;
  const int* block_table; int table_stride;   // [batch][table_stride] page ids; negative ones count from the end
  int layer, layers, num_blocks, block_size, heads, dim;
  int* status;                                 // FlDecStatus, or null
};

constexpr int FL_KV8_MASS_ROWS = 6 * 1024;   // new tokens times heads of a call that asks for pages' weights

// dim: a multiple of 16, at most 128; a page of a head at most 2^31 - 1 codes, a table at most 2^30 - 1 slots.  Tensors start at a multiple of 16 bytes.  Calls return 0, a cudaError, or < 0 for arguments they do
// not take (-1 type, -2 sizes, -4 addresses); nothing is launched then.
#ifdef __cplusplus
extern "C" {
#endif
// qkv [batch][tokens][heads + 2 kv.heads][dim]: bias [(heads + 2 kv.heads) * dim] added, queries and keys rotated (rope: [rope_rows][dim],
// cosines then sines), into `out` (which may be qkv).  Keys and values of token t of request b also go to slot start[b] + t of its pages; what the
// page held behind the last one written is no longer valid.  counts: tokens per request (null: all of them); rows behind them are left
// as they are.  pos: what the first token is rotated by (null: start).
int fl_kv8_write(int dtype, const void* qkv, void* out, const void* bias, const float* rope, long long rope_rows, const long long* start,
                 const long long* pos, const long long* counts, int batch, int tokens, int heads, const FlKv8* kv, cudaStream_t stream);
// The first lengths[b] tokens of request b, from a pool of 16-bit pages [layers][src_blocks][block_size][heads][dim] (FL_KV_LBSHD), of all layers
// (kv->layer is not looked at).
int fl_kv8_pack(int dtype, const void* k_pool, const void* v_pool, int src_blocks, const int* src_table, int src_stride, const long long* lengths,
                int batch, const FlKv8* kv, cudaStream_t stream);
// out [batch][tokens][heads * dim] = softmax(scale q k^T) v of tokens start[b] .. start[b] + counts[b] - 1 (counts null: `tokens` of them) over the
// slots up to their own; zeros where there is none.  scale: finite, not negative.  q: element strides of (request, token, head).  mass (or null): [batch][table_stride], += the
// weights' sum over this call's tokens and heads, page by page; tokens * heads is at most FL_KV8_MASS_ROWS then.
// scratch: fl_kv8_attention_scratch() bytes, from a multiple of 16 on: what one request needs (with weights 8 bytes per token, head and 16 slots of the table, or
// part of a page), or 256 MiB at most.
long long fl_kv8_attention_scratch(int batch, int tokens, int heads, const FlKv8* kv, int mass);
int fl_kv8_attention(int dtype, const void* q, long long stride_b, long long stride_t, long long stride_h, const long long* start,
                     const long long* counts, int batch, int tokens, int heads, float scale, const FlKv8* kv, void* out, float* mass, void* scratch,
                     cudaStream_t stream);
// Per request: of its ceil(lengths / block_size) pages the lightest of those from `sinks` on that are not among the last `recent` go, until
// `keep` are left (of equals the earlier one; NaN weighs most).  Kept pages move up in their order, then come those that went, in theirs, with
// mass 0, then the rest of the row.  Inputs and outputs do not overlap.
int fl_kv8_evict(const float* mass, const int* table, const long long* lengths, int batch, int pages, int block_size, int keep, int recent, int sinks,
                 float* mass_out, int* table_out, long long* lengths_out, int* gone, cudaStream_t stream);
#ifdef __cplusplus
}
#endif

// Rows of an embedding table times a factor, and the table's gradient from the rows' gradients (embedding.cu).
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>
#include "dtypes.cuh"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct {
  const void* tokens;            // [n] int64 (token_bytes 8) or int32 (4); a negative one counts from the vocabulary's end
  int token_bytes;
  long long n, vocab, hidden;    // hidden: values of a row
  const void* table;             // [vocab][hidden], rows table_stride apart (forward)
  long long table_stride;
  void* out;                     // [n][hidden] (forward)
  const void* dout;              // [n][hidden] (gradient)
  void* dtable;                  // [vocab][hidden] (gradient); every row is written
  void* scratch;                 // fl_embed_scratch() bytes (gradient)
  float scale;
  int* status;                   // word that a token outside the vocabulary sets to 1, or null; such a token gives zeros and no gradient
} FlEmbedArgs;

// dtype: FlDtype of table, out, dout and dtable.  -1: sizes that the kernels do not take
int fl_embed(int dtype, const FlEmbedArgs* a, cudaStream_t stream);
int fl_embed_grad(int dtype, const FlEmbedArgs* a, cudaStream_t stream);
long long fl_embed_scratch(long long n, long long vocab, long long hidden);    // bytes; -1: too large

#ifdef __cplusplus
}
#endif

/*
 * C ABI of the operators that a decoder runs between its quantized linears, in libdinoml_b200_gguf.so: a paged cache of keys and
 * values in 8 bits (write, read, attention over it) and the root-mean-square norm with the residual's addition.
 *
 * Conventions are those of dinoml_b200_gguf.h: device pointers, `stream` a cudaStream_t as void*, 0 = ok, 1 = null pointer, 2 = non-positive
 * dimension, 4 = launch failure, 6 = unsupported dtype or cache type, 7 = alignment, 8 = size outside what the kernels take; a message is
 * available from dino_get_last_error().  What only the device sees (block table, lengths, starts, begins) is checked there: an entry that
 * points outside of the cache or of the rows is left out of the operation, and dinoml_b200_gguf_device_status() answers 10.  16 there: a wait
 * inside of an attention kernel gave up, and its results are not to be used; reading the status empties the workspaces' counters.
 */
#ifndef DINOML_B200_DECODER_H_
#define DINOML_B200_DECODER_H_

#include <stdint.h>

#include "dinoml_b200_gguf.h"

#ifdef __cplusplus
extern "C" {
#endif

enum DinoB200KvType { DINOML_B200_KV_INT8 = 1, DINOML_B200_KV_E4M3 = 2 };

/* A cache: `blocks` blocks of `block_size` tokens.  k, v: uint8[blocks][kv_heads][block_size][head_dim] (int8 or float8 e4m3), 16-byte
 * aligned; k_scale, v_scale: float[blocks][kv_heads].  A stored value stands for q * scale.  e4m3's codes for NaN are no values (a write gives none): a key
 * with one makes the rows that see it NaN, a value may do so to its channel of rows of the call that do not.  block_size is 16, 32, 64 or 128, head_dim 64, 128
 * or 256. */
typedef struct DinoB200KvCache {
  void* k;
  void* v;
  float* k_scale;
  float* v_scale;
  int type; /* DinoB200KvType */
  int blocks, kv_heads, block_size, head_dim;
} DinoB200KvCache;

/* Which tokens a call is about.  Position p of sequence b is in slot p % block_size of block block_table[b * table_stride + p / block_size].
 * Rows of the call's dense tensors are packed: sequence b has rows starts[b] .. starts[b + 1] - 1; with
 * starts null every sequence has one row.  lengths[b] counts the tokens of the sequence, those of the call's rows among them: row starts[b] + j
 * is position lengths[b] - (starts[b + 1] - starts[b]) + j.  Rows at negative positions (an idle slot has length 0) are
 * nobody's, and so are those before starts[0] and behind starts[sequences] (a padded batch): they are not written to the cache, and zero in what a read or the
 * attention gives. */
typedef struct DinoB200KvBatch {
  const int* block_table;
  int64_t table_stride; /* elements */
  int table_blocks;     /* entries per sequence */
  const int* lengths;
  const int* starts;
  int sequences, rows;
} DinoB200KvBatch;

/* Quantizes the rows of k and v ([rows][kv_heads][head_dim], `dtype` as in dinoml_b200_gguf.h, strides in elements, head_dim contiguous) into the
 * cache.  The scale s of a block and head only grows while the block fills: s = max(s, a) with a from the largest |x| of the new tokens,
 * a = |x| * (1/127) for int8 and the smallest power of two with |x| <= 448 a for e4m3; tokens that are in the block already are brought to the
 * new scale; the token in slot 0 starts the block anew.  New values are round-to-nearest-even of x / s.  A block and head with an infinity or a NaN
 * among its new tokens gets the scale NaN and so reads as NaN.  One call writes a block for one sequence only. */
DINOML_B200_API int dinoml_b200_kv_cache_write(const DinoB200KvCache* cache, const DinoB200KvBatch* batch, const void* k, const void* v, int dtype,
                                               int64_t k_row_stride, int64_t k_head_stride, int64_t v_row_stride, int64_t v_head_stride, void* stream);

/* Dense keys and values k_out, v_out [rows][kv_heads][head_dim] (contiguous, 16-byte aligned) of a range of every sequence: row starts[b] + j is position
 * begins[b] + j (begins null: 0).  lengths is not read. */
DINOML_B200_API int dinoml_b200_kv_cache_read(const DinoB200KvCache* cache, const DinoB200KvBatch* batch, const int* begins, void* k_out, void* v_out, int dtype,
                                              void* stream);

/* out[row][head] = softmax(scale * q[row][head] K^T) V over the positions max(0, p - window + 1) .. p of the row's own sequence (window 0: 0 .. p),
 * p its position; head h reads cached head h / (heads / kv_heads).  q: [rows][heads][head_dim], strides in elements, head_dim contiguous; out
 * contiguous.  A row that sees nothing is zero.  Scores, softmax statistics and sums are float32.  The library keeps the workspace of sequences
 * that several CTAs share: one per device and stream, and for captured calls one per capture and stream, which is made during the capture and given back when the graph
 * is destroyed.  So a graph may be replayed on any stream, beside other graphs and beside calls on the stream that it was captured on; two graphs that are
 * instantiated from one capture have one workspace and must not overlap.  Run a call once before the first capture: kernels are loaded then. */
DINOML_B200_API int dinoml_b200_kv_cache_attention(const DinoB200KvCache* cache, const DinoB200KvBatch* batch, const void* q, void* out, int dtype, int heads,
                                                   int64_t q_row_stride, int64_t q_head_stride, float scale, int window, void* stream);

/* t = x + residual (residual null: t = x), y = t / sqrt(mean(t^2) + eps) * weight, over rows of `width` values, in float32 with one rounding at the end.
 * x, residual, total (t rounded to dtype, null: not stored; may be residual or x itself): [rows][width] in `dtype`; weight: [width] in weight_dtype (float32 or
 * `dtype`).  y: [rows][width] in `dtype`, or with q8_0 != 0 rows of GGUF Q8_0 blocks (34 bytes per 32 values: a float16 scale d = max|y| * (1/127), 32 int8
 * round(y / d)); width is then a multiple of 32. */
DINOML_B200_API int dinoml_b200_rms_norm(const void* x, const void* residual, const void* weight, void* y, void* total, int dtype, int weight_dtype, int rows,
                                         int width, float eps, int q8_0, void* stream);

/* The workspaces that the library keeps for a stream of the caller's (those of the attention and of the linears) are emptied and wait for another stream, or are
 * freed.  Waits for the stream; call it before the stream is destroyed, and after the graphs with linears that were captured on it.  Workspaces of streams that are not released live as long as the process. */
DINOML_B200_API int dinoml_b200_release_stream(void* stream);

#ifdef __cplusplus
}
#endif
#endif /* DINOML_B200_DECODER_H_ */

// extern "C" surface of the embedding, the rotation, the pool of blocks and the choice of tokens (include/dinoml_b200_decoder.h).
#include "../../include/dinoml_b200_decoder.h"
#include "decoder_entry.h"

namespace b200gguf {
int embedding(const void* tokens, int token_bytes, const void* table, int64_t vocabulary, void* out, int qtype, int dtype, int64_t count, int64_t width, float scale,
              cudaStream_t s);
int rotary(const DinoB200Heads* q, const DinoB200Heads* k, const int* positions, const double* frequencies, int pairs, int dtype, int weight_dtype, int rows, int head_dim,
           float eps, float magnitude, int interleaved, cudaStream_t s);
int sample(const void* logits, int64_t row_stride, int dtype, int rows, int vocabulary, const float* uniforms, const DinoB200SampleSettings* settings, int* tokens,
           float* probabilities, cudaStream_t s);
namespace kv {
int pool_step(const DinoB200KvPool* pool, const int* new_tokens, const int* drop, int rows, int* lengths, int* starts, int* positions, int* slots, cudaStream_t s);
}  // namespace kv
}  // namespace b200gguf

using namespace b200gguf;

extern "C" {

int dinoml_b200_embedding(const void* tokens, int token_bytes, const void* table, int64_t vocabulary, void* out, int qtype, int dtype, int64_t count, int64_t width,
                          float scale, void* stream) {
  return entry("dinoml_b200_embedding",
               [&] { return embedding(tokens, token_bytes, table, vocabulary, out, qtype, dtype, count, width, scale, static_cast<cudaStream_t>(stream)); });
}

int dinoml_b200_rotary(const DinoB200Heads* q, const DinoB200Heads* k, const int* positions, const double* frequencies, int pairs, int dtype, int weight_dtype, int rows,
                       int head_dim, float eps, float magnitude, int interleaved, void* stream) {
  return entry("dinoml_b200_rotary", [&] {
    return rotary(q, k, positions, frequencies, pairs, dtype, weight_dtype, rows, head_dim, eps, magnitude, interleaved, static_cast<cudaStream_t>(stream));
  });
}

int dinoml_b200_kv_pool_step(const DinoB200KvPool* pool, const int* new_tokens, const int* drop, int rows, int* lengths, int* starts, int* positions, int* slots,
                             void* stream) {
  return entry("dinoml_b200_kv_pool_step", [&] { return kv::pool_step(pool, new_tokens, drop, rows, lengths, starts, positions, slots, static_cast<cudaStream_t>(stream)); });
}

int dinoml_b200_sample(const void* logits, int64_t row_stride, int dtype, int rows, int vocabulary, const float* uniforms, const DinoB200SampleSettings* settings, int* tokens,
                       float* probabilities, void* stream) {
  return entry("dinoml_b200_sample", [&] {
    return sample(logits, row_stride, dtype, rows, vocabulary, uniforms, settings, tokens, probabilities, static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"

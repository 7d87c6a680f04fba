// extern "C" surface of the operators between the quantized linears (include/dinoml_b200_decoder.h).
#include "../../include/dinoml_b200_decoder.h"
#include "gguf_common.cuh"

namespace b200gguf {
int set_error(int rc, const char* where);
void stream_release_scratch(cudaStream_t s);
void umma_release_scratch(cudaStream_t s);
void attention_release_scratch(cudaStream_t s);
namespace kv {
int cache_write(const DinoB200KvCache* cache, const DinoB200KvBatch* batch, const void* k, const void* v, int dtype, int64_t k_row_stride,
                int64_t k_head_stride, int64_t v_row_stride, int64_t v_head_stride, cudaStream_t s);
int cache_read(const DinoB200KvCache* cache, const DinoB200KvBatch* batch, const int* begins, void* k_out, void* v_out, int dtype, cudaStream_t s);
int cache_attention(const DinoB200KvCache* cache, const DinoB200KvBatch* batch, const void* q, void* out, int dtype, int heads, int64_t q_row_stride,
                    int64_t q_head_stride, float scale, int window, cudaStream_t s);
}  // namespace kv
namespace norm {
int rms_norm(const void* x, const void* residual, const void* weight, void* y, void* total, int dtype, int weight_dtype, int rows, int width, float eps, int q8_0,
             cudaStream_t s);
}  // namespace norm
}  // namespace b200gguf

using namespace b200gguf;

// The workspaces' bookkeeping and the messages allocate on the host: no exception leaves an entry.
template <typename F> static int entry(const char* where, F f) noexcept {
  try {
    return set_error(f(), where);
  } catch (...) {
  }
  try {
    return set_error(RC_LAUNCH, where);
  } catch (...) {
    return RC_LAUNCH;
  }
}

extern "C" {

int dinoml_b200_kv_cache_write(const DinoB200KvCache* cache, const DinoB200KvBatch* batch, const void* k, const void* v, int dtype, int64_t k_row_stride,
                               int64_t k_head_stride, int64_t v_row_stride, int64_t v_head_stride, void* stream) {
  return entry("dinoml_b200_kv_cache_write", [&] {
    return kv::cache_write(cache, batch, k, v, dtype, k_row_stride, k_head_stride, v_row_stride, v_head_stride, static_cast<cudaStream_t>(stream));
  });
}

int dinoml_b200_kv_cache_read(const DinoB200KvCache* cache, const DinoB200KvBatch* batch, const int* begins, void* k_out, void* v_out, int dtype, void* stream) {
  return entry("dinoml_b200_kv_cache_read", [&] { return kv::cache_read(cache, batch, begins, k_out, v_out, dtype, static_cast<cudaStream_t>(stream)); });
}

int dinoml_b200_kv_cache_attention(const DinoB200KvCache* cache, const DinoB200KvBatch* batch, const void* q, void* out, int dtype, int heads,
                                   int64_t q_row_stride, int64_t q_head_stride, float scale, int window, void* stream) {
  return entry("dinoml_b200_kv_cache_attention", [&] {
    return kv::cache_attention(cache, batch, q, out, dtype, heads, q_row_stride, q_head_stride, scale, window, static_cast<cudaStream_t>(stream));
  });
}

int dinoml_b200_rms_norm(const void* x, const void* residual, const void* weight, void* y, void* total, int dtype, int weight_dtype, int rows, int width,
                         float eps, int q8_0, void* stream) {
  return entry("dinoml_b200_rms_norm",
               [&] { return norm::rms_norm(x, residual, weight, y, total, dtype, weight_dtype, rows, width, eps, q8_0, static_cast<cudaStream_t>(stream)); });
}

int dinoml_b200_release_stream(void* stream) {
  return entry("dinoml_b200_release_stream", [&]() -> int {
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (cudaStreamSynchronize(s) != cudaSuccess) return RC_LAUNCH;
    stream_release_scratch(s);
    umma_release_scratch(s);
    attention_release_scratch(s);
    return RC_OK;
  });
}

}  // extern "C"

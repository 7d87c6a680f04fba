// Attention over the 8-bit cache (layout: kv_cache.cuh): one warp per row and head, one pass over the positions with the running maximum and sum
// of the softmax.
#include "kv_cache.cuh"

namespace b200gguf {
namespace kv {

template <typename T, int TYPE>
__global__ void __launch_bounds__(256) kv_attention_kernel(Cache c, Batch p, const T* q, T* out, int heads, int64_t row_stride, int64_t head_stride, float scale,
                                                           int window) {
  using Q = Quant<TYPE>;
  const int64_t unit = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const int row = int(unit / heads), head = int(unit % heads);
  if (row >= p.rows) return;
  int b = row;
  if (p.starts != nullptr) b = last_at_most(p.sequences, row, [&](int i) { return int64_t(__ldg(p.starts + i)); });
  const Rows rows = rows_of(p, b);
  const int position = __ldg(p.lengths + b) - rows.count + row - rows.first;
  const bool mine = row >= rows.first && row < rows.first + rows.count;
  const int end = int(min(int64_t(position) + 1, int64_t(p.table_blocks) << c.block_log2));      // of what the table can reach
  if (mine && end <= position) flag_range(p.status);
  const int kv_head = head / (heads / c.heads), per = c.dim / 32;
  float x[8], acc[8];
  for (int i = 0; i < per; ++i) {
    x[i] = to_float<T>(q[row * row_stride + head * head_stride + lane + 32 * i]);
    acc[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  int block = -1, id = -1;
  for (int at = window > 0 ? max(0, position - window + 1) : 0; mine && at < end; ++at) {
    if (at >> c.block_log2 != block) {
      block = at >> c.block_log2;
      id = block_at(p, c.blocks, b, block);
    }
    if (id < 0) continue;
    const int64_t bh = int64_t(id) * c.heads + kv_head;
    const int64_t offset = ((bh << c.block_log2) + (at & ((1 << c.block_log2) - 1))) * c.dim + lane;
    float s = 0.f;
    for (int i = 0; i < per; ++i) s += x[i] * Q::up(c.data[0][offset + 32 * i]);
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    s *= c.scale[0][bh] * scale;
    const float next = fmaxf(m, s), keep = m == -INFINITY ? 0.f : expf(m - next), w = expf(s - next);
    m = next;
    l = l * keep + w;
    for (int i = 0; i < per; ++i) acc[i] = acc[i] * keep + w * (c.scale[1][bh] * Q::up(c.data[1][offset + 32 * i]));
  }
  const float inverse = l == 0.f ? 0.f : 1.f / l;
  for (int i = 0; i < per; ++i) out[(int64_t(row) * heads + head) * c.dim + lane + 32 * i] = from_float<T>(acc[i] * inverse);
}

int cache_attention(const DinoB200KvCache* cache, const DinoB200KvBatch* batch, const void* q, void* out, int dtype, int heads, int64_t q_row_stride,
                    int64_t q_head_stride, float scale, int window, cudaStream_t s) {
  Cache c;
  Batch p;
  if (int rc = cache_view(cache, &c)) return rc;
  if (q == nullptr || out == nullptr) return RC_NULL;
  if (heads <= 0) return RC_DIMS;
  if (heads % c.heads != 0 || window < 0) return RC_RANGE;
  if (int rc = batch_view(batch, true, &p)) return rc;
  return with_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & (sizeof(T) - 1)) != 0) return RC_ALIGN;
    const int64_t ctas = (int64_t(p.rows) * heads + 7) / 8;
    if (ctas > INT32_MAX) return RC_RANGE;
    auto launch = [&](auto kern) {
      kern<<<unsigned(ctas), 256, 0, s>>>(c, p, static_cast<const T*>(q), static_cast<T*>(out), heads, q_row_stride, q_head_stride, scale, window);
      return cudaGetLastError() == cudaSuccess ? RC_OK : RC_LAUNCH;
    };
    return cache->type == DINOML_B200_KV_INT8 ? launch(kv_attention_kernel<T, DINOML_B200_KV_INT8>) : launch(kv_attention_kernel<T, DINOML_B200_KV_E4M3>);
  });
}

}  // namespace kv
}  // namespace b200gguf

// Host side of attention over the 8-bit cache: checks, workspaces, which kernel takes a call.  The kernels are in kv_attention_few.cuh and kv_attention_many.cuh.
#include "captured_sets.h"
#include "kv_attention.cuh"

namespace b200gguf {
namespace kv {

// (Never destroyed: a graph may be dropped while the process ends.)
static AttnWorkspaces& workspaces() {
  static AttnWorkspaces* all = new AttnWorkspaces;
  return *all;
}
// Rows (tokens x heads of a cached head) of a sequence up to which the kernel of few rows takes it: it reads the cache once for 16 rows, the other one once for
// 256, at a lower rate.  Measured (few, many; 64 sequences, 8 cached heads, int8): heads of 128, 4000 tokens, 16 rows 173 and 372 us, 32 rows 301 and 373, 36 rows 425 and 374,
// 64 rows 557 and 378; of 64, 2000 tokens, 32 rows 128 and 184, 48 rows 175 and 184, 64 rows 222 and 184; of 256, 2000 tokens, 16 rows 231 and 226, 20 rows 321 and 230 (where
// both take the same the kernel of few rows is kept: its weights have no smallest one); float32, heads of 128, 2000 tokens, 16 rows 129 and 193, 32 rows 216 and 204.
static int few_rows(int dim) { return dim == 256 ? 16 : 32; }

float* attention_scratch(size_t floats, int ctas, cudaStream_t s, int** arrived) {
  int dev = -1;
  if (ctas > AttnScratch::kMaxWorkers || cudaGetDevice(&dev) != cudaSuccess) return nullptr;
  return workspaces().get(dev, s, floats, arrived);
}

void attention_reset() {
  int dev = -1;
  if (cudaGetDevice(&dev) == cudaSuccess) workspaces().reset(dev);
}

int cache_attention(const DinoB200KvCache* cache, const DinoB200KvBatch* batch, const void* q, void* out, int dtype, int heads, int64_t q_row_stride,
                    int64_t q_head_stride, float scale, int window, cudaStream_t s) {
  AttnParams a = {};
  if (int rc = cache_view(cache, &a.c)) return rc;
  if (q == nullptr || out == nullptr) return RC_NULL;
  if (heads <= 0) return RC_DIMS;
  if (heads % a.c.heads != 0 || window < 0) return RC_RANGE;
  if (dtype != DINO_F16 && dtype != DINO_BF16 && dtype != DINO_F32) return RC_DTYPE;
  if ((reinterpret_cast<uintptr_t>(q) & (dtype == DINO_F32 ? 3 : 1)) != 0 || (reinterpret_cast<uintptr_t>(out) & 15) != 0) return RC_ALIGN;
  a.group = heads / a.c.heads;
  a.by_group.set(uint32_t(a.group));
  if ((int64_t(a.c.blocks) * a.c.heads) << a.c.block_log2 > INT32_MAX) return RC_RANGE;      // rows of the copies' coordinates
  if (int rc = batch_view(batch, true, &a.p)) return rc;
  if (int64_t(a.p.rows) * a.group > INT32_MAX) return RC_RANGE;
  a.q = q;
  a.out = out;
  a.row_stride = q_row_stride;
  a.head_stride = q_head_stride;
  a.scale = scale * kLog2e;
  a.window = window;
  a.heads = heads;
  a.dtype = dtype;
  // Sequences with few rows go to one kernel, those with many to the other; which there are only the device knows, so a call with rows enough is both.
  const int64_t all_rows = int64_t(a.p.rows) * a.group, rows = (all_rows + a.p.sequences - 1) / a.p.sequences;
  const bool tensor = dtype != DINO_F32 || a.c.dim != 256;                   // (two terms of 256 values do not fit into shared memory)
  const int64_t most = a.p.starts == nullptr ? a.group : all_rows;          // rows of a sequence
  a.min_rows = 0;
  a.max_rows = tensor ? few_rows(a.c.dim) : INT32_MAX;
  // One tile of eight rows or two (one reading of the cache for 9 to 16 rows), by the mean rows of a sequence, or of a single token where the mean says that there are
  // prompts, beside which single tokens are what is most common.  Measured (one, two; 32 sequences of 4000 tokens, 8 cached
  // heads, int8, single tokens): heads of 64, 8 rows 46 and 59 us, 12 rows 81 and 60; of 128, 8 rows 61 and 83, 12 rows 103 and 86, float32 12 rows 132 and 104.
  // Heads of 256 have no second tile: its sums leave a quarter of an SM two warps, 8 rows 113 and 239, 16 rows 202 and 251, float32 251 and 325.
  // 64 single tokens of 4 rows and a prompt of 512: 137 and 160 us; 32 chunks of 3 tokens and a prompt of 512 (where this rule is wrong) 178 and 160.
  const int64_t usual = rows > few_rows(a.c.dim) ? a.group : rows;
  const int tiles = usual <= 8 || a.c.dim == 256 ? 1 : 2;
  if (a.p.starts != nullptr || most <= a.max_rows) {
    const int rc = cache->type == DINOML_B200_KV_INT8 ? attention_few_int8(a, tiles, s) : attention_few_e4m3(a, tiles, s);
    if (rc != RC_OK || most <= a.max_rows) return rc;
  }
  a.min_rows = a.max_rows + 1;
  a.max_rows = INT32_MAX;
  return attention_many(a, cache->type, s);
}

}  // namespace kv

void attention_release_scratch(cudaStream_t s) { kv::workspaces().release(s); }

}  // namespace b200gguf

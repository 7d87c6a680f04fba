// Write and read of the 8-bit cache of keys and values (layout: kv_cache.cuh).
#include <mutex>

#include "kv_attention.cuh"

namespace b200gguf {
namespace kv {

static __device__ int g_kv_status;

static int* status_ptr() {
  static int* ptr[kGemvMaxDevices] = {};
  static std::mutex mu;
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kGemvMaxDevices) return nullptr;
  std::lock_guard<std::mutex> lock(mu);
  if (ptr[dev] == nullptr) {
    void* p = nullptr;
    if (cudaGetSymbolAddress(&p, g_kv_status) != cudaSuccess) return nullptr;
    ptr[dev] = static_cast<int*>(p);
  }
  return ptr[dev];
}

int cache_view(const DinoB200KvCache* c, Cache* out) {
  if (c == nullptr || c->k == nullptr || c->v == nullptr || c->k_scale == nullptr || c->v_scale == nullptr) return RC_NULL;
  if (c->blocks <= 0 || c->kv_heads <= 0 || c->block_size <= 0 || c->head_dim <= 0) return RC_DIMS;
  if (c->type != DINOML_B200_KV_INT8 && c->type != DINOML_B200_KV_E4M3) return RC_DTYPE;
  int log2 = 4;
  while (log2 < 7 && (1 << log2) != c->block_size) ++log2;
  if ((1 << log2) != c->block_size || (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)) return RC_RANGE;
  if (((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15) != 0) return RC_ALIGN;
  *out = {{static_cast<uint8_t*>(c->k), static_cast<uint8_t*>(c->v)}, {c->k_scale, c->v_scale}, c->blocks, c->kv_heads, c->head_dim, log2};
  return RC_OK;
}

int batch_view(const DinoB200KvBatch* b, bool needs_lengths, Batch* out) {
  if (b == nullptr || b->block_table == nullptr || (needs_lengths && b->lengths == nullptr)) return RC_NULL;
  if (b->sequences <= 0 || b->rows <= 0 || b->table_blocks <= 0) return RC_DIMS;
  if (b->table_stride < b->table_blocks && b->sequences > 1) return RC_RANGE;
  if (b->starts == nullptr && b->rows != b->sequences) return RC_RANGE;
  int* status = status_ptr();
  if (status == nullptr) return RC_LAUNCH;
  *out = {b->block_table, b->lengths, b->starts, b->table_stride, b->table_blocks, b->sequences, b->rows, status};
  return RC_OK;
}

// ---- write ------------------------------------------------------------------------------------------------------------------
// A unit is the new tokens of one sequence in one block, for one head of K or of V: the only writer of that block and head, so the scale and the
// tokens that are there already need no atomics.  NT threads work on a unit (a warp where a call brings a token or two, a CTA where it brings
// whole blocks).
struct Source {
  const void* x[2];
  int64_t row_stride[2], head_stride[2];
  bool wide;                         // every row starts at a multiple of 16 bytes
};

template <int NT> __device__ __forceinline__ uint32_t unit_max(uint32_t v, uint32_t* shared) {
  v = __reduce_max_sync(0xffffffffu, v);
  if (NT == 32) return v;
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  return __reduce_max_sync(0xffffffffu, shared[threadIdx.x & 7]);
}

template <typename T, int TYPE, int NT>
__global__ void __launch_bounds__(256) kv_write_kernel(Cache c, Batch p, Source src, int pieces) {
  using Q = Quant<TYPE>;
  constexpr int N = Pack<T>::N;
  __shared__ uint32_t shared[8];
  const int tid = threadIdx.x % NT;
  const int64_t unit = int64_t(blockIdx.x) * (256 / NT) + threadIdx.x / NT;
  const int which = int(unit & 1), bs = 1 << c.block_log2;
  const int head = int((unit >> 1) % c.heads);
  const int64_t piece64 = (unit >> 1) / c.heads;
  if (piece64 >= pieces) return;
  const int piece = int(piece64);
  // Pieces of sequence b are numbered from starts[b] / block + 2 b: it has at most (rows of it) / block + 2 of them, so every number has one owner and
  // the numbers need no sum over the sequences.
  int b = piece, base = piece;
  if (p.starts != nullptr) {
    const int log2 = c.block_log2;
    auto key = [&](int i) { return int64_t(__ldg(p.starts + i) >> log2) + 2 * i; };
    b = last_at_most(p.sequences, piece, key);
    base = int(key(b));
  }
  const Rows rows = rows_of(p, b);
  const int length = __ldg(p.lengths + b);
  const int first = length - rows.count;                       // position of the first new token
  const int block = (max(first, 0) >> c.block_log2) + (piece - base);
  const int low = max(max(first, 0), block << c.block_log2), high = int(min(int64_t(length), (int64_t(block) + 1) << c.block_log2));
  if (piece < base || low >= high) return;
  const int id = block_at(p, c.blocks, b, block);
  if (id < 0) return;

  const T* x = static_cast<const T*>(src.x[which]) + head * src.head_stride[which] + int64_t(rows.first + low - first) * src.row_stride[which];
  const int64_t stride = src.row_stride[which];
  const int per_row = c.dim / N, total = (high - low) * per_row;
  uint32_t largest = 0;                                        // as bits: an infinity or a NaN is larger than every number
  for (int i = tid; i < total; i += NT) {
    Pack<T> v;
    v.load(x + (i / per_row) * stride + (i % per_row) * N, src.wide);
#pragma unroll
    for (int j = 0; j < N; ++j) largest = max(largest, __float_as_uint(to_float<T>(v.v[j])) & 0x7fffffffu);
  }
  largest = unit_max<NT>(largest, shared);
  float* scale = c.scale[which] + int64_t(id) * c.heads + head;
  const int kept = low - (block << c.block_log2);              // tokens that were in the block before
  const float before = kept > 0 ? *scale : 0.f;
  const float wanted = largest < 0x7f800000u ? Q::wanted(__uint_as_float(largest)) : __uint_as_float(0x7fc00000u);
  const float after = before != before || wanted != wanted ? __uint_as_float(0x7fc00000u) : fmaxf(before, wanted);
  uint8_t* dst = c.data[which] + ((int64_t(id) * c.heads + head) << c.block_log2) * c.dim;
  if (NT > 32) __syncthreads(); else __syncwarp();             // everyone has read the scale
  if (tid == 0) *scale = after;
  if (kept > 0 && after != before && after == after) {
    const float ratio = __fdiv_rn(before, after);
    for (int i = tid; i < kept * c.dim / 4; i += NT) {
      const uint32_t q = reinterpret_cast<const uint32_t*>(dst)[i];
      uint32_t r = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) r |= Q::nearest(__fmul_rn(Q::up((q >> (8 * j)) & 0xffu), ratio)) << (8 * j);
      reinterpret_cast<uint32_t*>(dst)[i] = r;
    }
  }
  dst += int64_t(kept) * c.dim;
  const typename Q::Down down(after);                          // a NaN scale: zeros
  for (int i = tid; i < total; i += NT) {
    Pack<T> v;
    v.load(x + (i / per_row) * stride + (i % per_row) * N, src.wide);
    uint32_t w[N / 4];
#pragma unroll
    for (int j = 0; j < N; j += 4) w[j / 4] = down(to_float<T>(v.v[j])) | down(to_float<T>(v.v[j + 1])) << 8 | down(to_float<T>(v.v[j + 2])) << 16 | down(to_float<T>(v.v[j + 3])) << 24;
#pragma unroll
    for (int j = 0; j < N / 4; ++j) reinterpret_cast<uint32_t*>(dst)[i * (N / 4) + j] = w[j];
  }
}

int cache_write(const DinoB200KvCache* cache, const DinoB200KvBatch* batch, const void* k, const void* v, int dtype, int64_t k_row_stride,
                int64_t k_head_stride, int64_t v_row_stride, int64_t v_head_stride, cudaStream_t s) {
  Cache c;
  Batch p;
  if (int rc = cache_view(cache, &c)) return rc;
  if (k == nullptr || v == nullptr) return RC_NULL;
  if (int rc = batch_view(batch, true, &p)) return rc;
  return with_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    if (((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & (sizeof(T) - 1)) != 0) return RC_ALIGN;
    const uint64_t every = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                           uint64_t(k_row_stride | k_head_stride | v_row_stride | v_head_stride) * sizeof(T);
    const Source src{{k, v}, {k_row_stride, v_row_stride}, {k_head_stride, v_head_stride}, (every & 15) == 0};
    const int64_t pieces = p.starts == nullptr ? p.rows : int64_t(p.rows >> c.block_log2) + 2 * int64_t(p.sequences);
    const int64_t units = 2 * pieces * c.heads;
    const bool few = p.rows < 8 * int64_t(p.sequences);
    const int64_t ctas = few ? (units + 7) / 8 : units;
    if (pieces > INT32_MAX || ctas > INT32_MAX) return RC_RANGE;
    auto launch = [&](auto kern) {
      kern<<<unsigned(ctas), 256, 0, s>>>(c, p, src, int(pieces));
      return cudaGetLastError() == cudaSuccess ? RC_OK : RC_LAUNCH;
    };
    if (cache->type == DINOML_B200_KV_INT8) return few ? launch(kv_write_kernel<T, DINOML_B200_KV_INT8, 32>) : launch(kv_write_kernel<T, DINOML_B200_KV_INT8, 256>);
    return few ? launch(kv_write_kernel<T, DINOML_B200_KV_E4M3, 32>) : launch(kv_write_kernel<T, DINOML_B200_KV_E4M3, 256>);
  });
}

// ---- read -------------------------------------------------------------------------------------------------------------------
constexpr int kReadRows = 8;         // rows of a CTA

template <typename T, int TYPE>
__global__ void __launch_bounds__(256) kv_read_kernel(Cache c, Batch p, const int* begins, T* k_out, T* v_out) {
  using Q = Quant<TYPE>;
  __shared__ int ids[kReadRows], slots[kReadRows];
  const int row0 = blockIdx.x * kReadRows, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (row0 + warp < p.rows) {                                  // one warp finds one row's block
    const int row = row0 + warp;
    int b = row;
    if (p.starts != nullptr) b = last_at_most(p.sequences, row, [&](int i) { return int64_t(__ldg(p.starts + i)); });
    const Rows rows = rows_of(p, b);
    const int64_t position = int64_t(row) - rows.first + (begins != nullptr ? __ldg(begins + b) : 0);
    int id = -1;
    if (row >= rows.first && row < rows.first + rows.count && position >= 0 && position <= INT32_MAX) id = block_at(p, c.blocks, b, int(position >> c.block_log2));
    if (lane == 0) { ids[warp] = id; slots[warp] = int(position) & ((1 << c.block_log2) - 1); }
  }
  __syncthreads();
  const int per_row = c.heads * c.dim / 16, rows = min(kReadRows, p.rows - row0);
  for (int i = threadIdx.x; i < rows * per_row; i += 256) {
    const int r = i / per_row, at = i % per_row, head = at * 16 / c.dim, column = at * 16 % c.dim;
    const int id = ids[r];
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      uint4 raw = make_uint4(0, 0, 0, 0);
      float scale = 0.f;
      if (id >= 0) {
        const int64_t block = int64_t(id) * c.heads + head;
        raw = *reinterpret_cast<const uint4*>(c.data[which] + ((block << c.block_log2) + slots[r]) * c.dim + column);
        scale = c.scale[which][block];
      }
      const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
      constexpr int N = Pack<T>::N;
      uint4* out = reinterpret_cast<uint4*>((which == 0 ? k_out : v_out) + (int64_t(row0) + r) * c.heads * c.dim + at * 16);
#pragma unroll
      for (int o = 0; o < 16 / N; ++o) {
        Pack<T> v;
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const int e = o * N + j;
          v.v[j] = from_float<T>(__fmul_rn(Q::up((words[e / 4] >> (8 * (e % 4))) & 0xffu), scale));
        }
        out[o] = v.raw;
      }
    }
  }
}

int cache_read(const DinoB200KvCache* cache, const DinoB200KvBatch* batch, const int* begins, void* k_out, void* v_out, int dtype, cudaStream_t s) {
  Cache c;
  Batch p;
  if (int rc = cache_view(cache, &c)) return rc;
  if (k_out == nullptr || v_out == nullptr) return RC_NULL;
  if (((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15) != 0) return RC_ALIGN;
  if (int rc = batch_view(batch, false, &p)) return rc;
  return with_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    const unsigned ctas = unsigned((int64_t(p.rows) + kReadRows - 1) / kReadRows);
    if (cache->type == DINOML_B200_KV_INT8) kv_read_kernel<T, DINOML_B200_KV_INT8><<<ctas, 256, 0, s>>>(c, p, begins, static_cast<T*>(k_out), static_cast<T*>(v_out));
    else kv_read_kernel<T, DINOML_B200_KV_E4M3><<<ctas, 256, 0, s>>>(c, p, begins, static_cast<T*>(k_out), static_cast<T*>(v_out));
    return cudaGetLastError() == cudaSuccess ? RC_OK : RC_LAUNCH;
  });
}

}  // namespace kv

// Status word of the cache's kernels on the current device (read once).
int kv_device_status() {
  int value = 0;
  int* p = kv::status_ptr();
  if (p == nullptr || cudaMemcpy(&value, p, sizeof(int), cudaMemcpyDeviceToHost) != cudaSuccess) return 0;
  if (value != 0) cudaMemset(p, 0, sizeof(int));
  if (value == kv::ST_KV_TIMEOUT) kv::attention_reset();
  return value;
}

}  // namespace b200gguf

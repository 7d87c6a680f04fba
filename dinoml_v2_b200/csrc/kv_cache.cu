// Write and read of the 8-bit cache of keys and values (layout: kv_cache.cuh).
#include <algorithm>
#include <mutex>
#include <type_traits>

#include "kv_attention.cuh"

namespace b200gguf {
namespace kv {

static __device__ int g_kv_status[kStatusWords];

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

// Both kernels are bound by bytes, and a short call by its chain of dependent reads (starts, length, table, data): every thread has all of its
// reads of a step under way before it uses the first, and a launch starts while the one before it ends.

// A launch that starts while the one before it in the stream ends; the kernel waits for that itself.
template <typename... P, typename... A> static int start(void (*kernel)(P...), unsigned ctas, cudaStream_t s, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess ? RC_OK : RC_LAUNCH;
}
__device__ __forceinline__ void wait_for_launch_before() {
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
}

// ---- write ------------------------------------------------------------------------------------------------------------------
// A unit is the new tokens of one sequence in one block, for one head of K or of V: the only writer of that block and head, so the scale and the
// tokens that are there already need no atomics.  NT threads work on a unit, a warp or a CTA (cache_write).  A thread keeps the first kHeld pieces of 16 bytes that
// it has between the maximum and the rounding and reads the others again.  8 heads of 128, launches one after the other: 64 single tokens 3.6 us, 2671 tokens in five prompts 8.0,
// 12006 in six 24.9 (74 MB, 3.0 TB/s).
constexpr int kHeld = 4;
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
  wait_for_launch_before();
  const int tid = threadIdx.x % NT;
  const int64_t unit = int64_t(blockIdx.x) * (256 / NT) + threadIdx.x / NT;
  auto pick = [&](const auto& of) { return (unit & 1) == 0 ? of[0] : of[1]; };      // of K or V
  const int head = int((unit >> 1) % c.heads);
  const int64_t piece64 = (unit >> 1) / c.heads;
  if (piece64 >= pieces) return;
  const int piece = int(piece64);
  // Pieces of sequence b are numbered from starts[b] / block + 2 b: it has at most (rows of it) / block + 2 of them, so every number has one owner and
  // the numbers need no sum over the sequences.
  int b = piece, base = piece;
  if (p.starts != nullptr) {
    const int log2 = c.block_log2;
    auto key = [&](int i) { return int64_t(fetch(p.starts + i) >> log2) + 2 * i; };
    b = last_at_most(p.sequences, piece, key);
    base = int(key(b));
  }
  const Rows rows = rows_of(p, b);
  const int length = fetch(p.lengths + b);
  const int first = length - rows.count;                       // position of the first new token
  const int block = (max(first, 0) >> c.block_log2) + (piece - base);
  const int low = max(max(first, 0), block << c.block_log2), high = int(min(int64_t(length), (int64_t(block) + 1) << c.block_log2));
  if (piece < base || low >= high) return;

  const T* x = static_cast<const T*>(pick(src.x)) + head * pick(src.head_stride) + int64_t(rows.first + low - first) * pick(src.row_stride);
  const int64_t stride = pick(src.row_stride);
  const int log2 = __ffs(c.dim / N) - 1, total = (high - low) << log2;
  auto load = [&](int i, Pack<T>& v) { v.load(x + (i >> log2) * stride + (i & ((1 << log2) - 1)) * N, src.wide); };
  Pack<T> held[kHeld];
#pragma unroll
  for (int k = 0; k < kHeld; ++k)
    if (tid + k * NT < total) load(tid + k * NT, held[k]);
  const int id = block_at(p, c.blocks, b, block);
  if (id < 0) return;
  float* scale = pick(c.scale) + int64_t(id) * c.heads + head;
  const int kept = low - (block << c.block_log2);              // tokens that were in the block before
  const float before = kept > 0 ? *scale : 0.f;
  uint32_t largest = 0;                                        // as bits: an infinity or a NaN is larger than every number
  auto meet = [&](const Pack<T>& v) {
#pragma unroll
    for (int j = 0; j < N; ++j) largest = max(largest, __float_as_uint(to_float<T>(v.v[j])) & 0x7fffffffu);
  };
#pragma unroll
  for (int k = 0; k < kHeld; ++k)
    if (tid + k * NT < total) meet(held[k]);
  for (int i = tid + kHeld * NT; i < total; i += NT) {
    Pack<T> v;
    load(i, v);
    meet(v);
  }
  largest = unit_max<NT>(largest, shared);
  const float wanted = largest < 0x7f800000u ? Q::wanted(__uint_as_float(largest)) : __uint_as_float(0x7fc00000u);
  const float after = before != before || wanted != wanted ? __uint_as_float(0x7fc00000u) : fmaxf(before, wanted);
  uint8_t* dst = pick(c.data) + ((int64_t(id) * c.heads + head) << c.block_log2) * c.dim;
  if (NT > 32) __syncthreads(); else __syncwarp();             // everyone has read the scale
  if (tid == 0) *scale = after;
  if (kept > 0 && after != before && after == after) {
    const float ratio = __fdiv_rn(before, after);
    uint4* old = reinterpret_cast<uint4*>(dst);
    const int count = kept * c.dim / 16;
    for (int i = tid; i < count; i += kHeld * NT) {
      uint4 q[kHeld];
#pragma unroll
      for (int k = 0; k < kHeld; ++k)
        if (i + k * NT < count) q[k] = old[i + k * NT];
#pragma unroll
      for (int k = 0; k < kHeld; ++k) {
        if (i + k * NT >= count) break;
        uint32_t* w = &q[k].x;
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          uint32_t r = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) r |= Q::nearest(__fmul_rn(Q::up((w[m] >> (8 * j)) & 0xffu), ratio)) << (8 * j);
          w[m] = r;
        }
        old[i + k * NT] = q[k];
      }
    }
  }
  dst += int64_t(kept) * c.dim;
  const typename Q::Down down(after);                          // a NaN scale: zeros
  auto store = [&](int i, const Pack<T>& v) {
    uint32_t w[N / 4];
#pragma unroll
    for (int j = 0; j < N; j += 4) w[j / 4] = down(to_float<T>(v.v[j])) | down(to_float<T>(v.v[j + 1])) << 8 | down(to_float<T>(v.v[j + 2])) << 16 | down(to_float<T>(v.v[j + 3])) << 24;
    if constexpr (N == 8) reinterpret_cast<uint2*>(dst)[i] = make_uint2(w[0], w[1]);
    else reinterpret_cast<uint32_t*>(dst)[i] = w[0];
  };
#pragma unroll
  for (int k = 0; k < kHeld; ++k)
    if (tid + k * NT < total) store(tid + k * NT, held[k]);
  for (int i = tid + kHeld * NT; i < total; i += NT) {
    Pack<T> v;
    load(i, v);
    store(i, v);
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
    // A CTA is done with a unit sooner, a warp has 4 to 8 times as many of them under way.  So a unit is a warp's where there are more of them than one for every SM and two
    // thirds of one more for every 128 values of a head that a unit brings.  Measured (a warp, a CTA; 8 heads of 128, bfloat16, blocks of 16): 1 sequence of 64 new tokens
    // 8.1 and 3.5 us, 16 of 4 4.1 and 5.7, 64 of 1 3.6 and 6.8, 64 of 8 6.5 and 11.1, 128 of 16 12.8 and 28.6; blocks of 128, 64 new tokens: 16 sequences 29.1 and 6.9,
    // 128 42.6 and 34.1.  Over 120 sizes, head sizes and types the rule's choice takes up to 1.06 times the better one.
    const int sms = stream::sm_count();
    if (sms <= 0) return RC_LAUNCH;
    const int64_t tokens = std::min((int64_t(p.rows) + p.sequences - 1) / p.sequences, int64_t(1) << c.block_log2);
    const bool few = 3 * units > sms * (3 + 2 * tokens * c.dim / 128);
    const int64_t ctas = few ? (units + 7) / 8 : units;
    if (pieces > INT32_MAX || ctas > INT32_MAX) return RC_RANGE;
    auto launch = [&](auto kern) { return start(kern, unsigned(ctas), s, c, p, src, int(pieces)); };
    if (cache->type == DINOML_B200_KV_INT8) return few ? launch(kv_write_kernel<T, DINOML_B200_KV_INT8, 32>) : launch(kv_write_kernel<T, DINOML_B200_KV_INT8, 256>);
    return few ? launch(kv_write_kernel<T, DINOML_B200_KV_E4M3, 32>) : launch(kv_write_kernel<T, DINOML_B200_KV_E4M3, 256>);
  });
}

// ---- read -------------------------------------------------------------------------------------------------------------------
// A warp has one row of K and V: 512 bytes of the result at a time, kReadAhead of them under way.  82062 tokens of 8 heads of 128 (four contexts), int8 to bfloat16: 80.6 us,
// 6.26 TB/s (a CTA for eight rows with one piece of 16 bytes a thread under way: 98.7).
constexpr int kReadWarps = 8, kReadAhead = 4;

template <typename T, int TYPE>
__global__ void __launch_bounds__(32 * kReadWarps) kv_read_kernel(Cache c, Batch p, const int* begins, T* k_out, T* v_out) {
  using Q = Quant<TYPE>;
  constexpr int N = 16 / int(sizeof(T));                       // values of a lane: 4 or 8 bytes of the cache
  using Raw = std::conditional_t<N == 8, uint2, uint32_t>;
  wait_for_launch_before();
  const int lane = threadIdx.x & 31;
  const int64_t row64 = int64_t(blockIdx.x) * kReadWarps + (threadIdx.x >> 5);
  if (row64 >= p.rows) return;
  const int row = int(row64);
  int b = row;
  if (p.starts != nullptr) b = last_at_most(p.sequences, row, [&](int i) { return int64_t(fetch(p.starts + i)); });
  const Rows rows = rows_of(p, b);
  const int64_t position = int64_t(row) - rows.first + (begins != nullptr ? fetch(begins + b) : 0);
  int id = -1;
  if (row >= rows.first && row < rows.first + rows.count) {
    if (position >= 0 && position <= INT32_MAX) id = block_at(p, c.blocks, b, int(position >> c.block_log2));
    else flag_range(p.status);
  }
  const int slot = int(position) & ((1 << c.block_log2) - 1), log2 = __ffs(c.dim) - 1, width = c.heads << log2;
  const int64_t to = row64 * width;
  for (int i = lane * N; i < width; i += 32 * N * kReadAhead) {
    Raw raw[kReadAhead][2];
    float scale[kReadAhead][2];
#pragma unroll
    for (int k = 0; k < kReadAhead; ++k) {
      const int at = i + 32 * N * k;
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        raw[k][which] = Raw{};
        scale[k][which] = 0.f;
        if (at < width && id >= 0) {
          const int64_t block = int64_t(id) * c.heads + (at >> log2);
          raw[k][which] = fetch(reinterpret_cast<const Raw*>(c.data[which] + ((((block << c.block_log2) + slot) << log2) + (at & (c.dim - 1)))));
          scale[k][which] = fetch(c.scale[which] + block);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < kReadAhead; ++k) {
      const int at = i + 32 * N * k;
      if (at >= width) break;
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        uint32_t words[2];
        if constexpr (N == 8) { words[0] = raw[k][which].x; words[1] = raw[k][which].y; } else { words[0] = raw[k][which]; }
        Pack<T> v;
#pragma unroll
        for (int j = 0; j < N; ++j) v.v[j] = from_float<T>(__fmul_rn(Q::up((words[j / 4] >> (8 * (j % 4))) & 0xffu), scale[k][which]));
        *reinterpret_cast<uint4*>((which == 0 ? k_out : v_out) + to + at) = v.raw;
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
    const unsigned ctas = unsigned((int64_t(p.rows) + kReadWarps - 1) / kReadWarps);
    auto launch = [&](auto kern) { return start(kern, ctas, s, c, p, begins, static_cast<T*>(k_out), static_cast<T*>(v_out)); };
    return cache->type == DINOML_B200_KV_INT8 ? launch(kv_read_kernel<T, DINOML_B200_KV_INT8>) : launch(kv_read_kernel<T, DINOML_B200_KV_E4M3>);
  });
}

}  // namespace kv

// Status of the cache's kernels on the current device (read once).
int kv_device_status() { return kv::take_status(kv::status_ptr(), kv::attention_reset); }

}  // namespace b200gguf

// The paged cache of keys and values in 8 bits: what its kernels share.  Layout and batch description: include/dinoml_b200_decoder.h.
//
// A block of one head is block_size x head_dim bytes in one piece, so it is what a kernel copies at once, and it has one float32 scale for K and
// one for V.  Everything that only the device sees is checked here: a table entry outside of the cache is no block.
#pragma once
#include <cuda_fp8.h>

#include "../../include/dinoml_b200_decoder.h"
#include "gguf_common.cuh"
#include "kv_status.h"

namespace b200gguf {
namespace kv {

struct Cache {
  uint8_t* data[2];                  // keys, values
  float* scale[2];
  int blocks, heads, dim, block_log2;
};
struct Batch {
  const int *table, *lengths, *starts;
  int64_t table_stride;
  int table_blocks, sequences, rows;
  int* status;                       // the words of kv_status.h
};

// Host: checks and the device's view of the two structs; a return code.
int cache_view(const DinoB200KvCache* cache, Cache* out);
int batch_view(const DinoB200KvBatch* batch, bool needs_lengths, Batch* out);

#ifdef __CUDACC__
// A plain read.  (A read as of constant data may be moved ahead of a kernel's wait for the launch before it.)
template <typename T> __device__ __forceinline__ T fetch(const T* p) { return *p; }

__device__ __forceinline__ void flag_range(int* status) { atomicExch(status, ST_KV_RANGE); }
__device__ __forceinline__ void flag_timeout(int* status) { atomicExch(status + 1, ST_KV_TIMEOUT); }

// Block j of sequence b, -1 if there is none.
__device__ __forceinline__ int block_at(const Batch& p, int blocks, int b, int j) {
  int id = -1;
  if (unsigned(j) < unsigned(p.table_blocks)) id = fetch(p.table + int64_t(b) * p.table_stride + j);
  if (unsigned(id) < unsigned(blocks)) return id;
  flag_range(p.status);
  return -1;
}

struct Rows {
  int first, count;
};
// Packed rows of sequence b.
__device__ __forceinline__ Rows rows_of(const Batch& p, int b) {
  if (p.starts == nullptr) return {b, b < p.rows ? 1 : 0};
  const int s0 = fetch(p.starts + b), s1 = fetch(p.starts + b + 1);
  if (s0 < 0 || s1 < s0 || s1 > p.rows) {
    flag_range(p.status);
    return {0, 0};
  }
  return {s0, s1 - s0};
}

// The last b in [0, count) with key(b) <= u, for keys that do not fall and key(0) <= u: 32 places at a time, by a converged warp (a sequence is
// found in two or three dependent loads, where halving takes eight).
template <typename Key>
__device__ __forceinline__ int last_at_most(int count, int64_t u, Key key) {
  const int lane = threadIdx.x & 31;
  int low = 0;
  for (int span = count; span > 1;) {
    const int step = (span + 31) >> 5;
    const int at = low + lane * step;
    const bool in = lane * step < span && (lane == 0 || key(at) <= u);
    const int hits = __popc(__ballot_sync(0xffffffffu, in));
    low += (hits - 1) * step;
    span = min(step, span - (hits - 1) * step);
  }
  return low;
}

// 8-bit values as float32 and back.
template <int TYPE> struct Quant;
template <> struct Quant<DINOML_B200_KV_INT8> {
  static __device__ __forceinline__ float up(uint32_t byte) { return float(int(int8_t(byte))); }
  // the scale that brings values of this size into the type's range
  static __device__ __forceinline__ float wanted(float largest) { return __fmul_rn(largest, 1.0f / 127.0f); }
  struct Down {                      // x / scale, rounded to the type
    float scale;
    __device__ __forceinline__ explicit Down(float s) : scale(s) {}
    __device__ __forceinline__ uint32_t operator()(float x) const { return scale > 0.f ? nearest(__fdiv_rn(x, scale)) : 0u; }
  };
  static __device__ __forceinline__ uint32_t nearest(float v) { return uint32_t(__float2int_rn(fminf(fmaxf(v, -127.f), 127.f))) & 0xffu; }
};
template <> struct Quant<DINOML_B200_KV_E4M3> {
  static __device__ __forceinline__ float up(uint32_t byte) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(__nv_fp8_storage_t(byte), __NV_E4M3)));
  }
  static __device__ __forceinline__ float wanted(float largest) {      // 448 = 1.75 * 2^8
    if (largest == 0.f) return 0.f;
    const uint32_t bits = __float_as_uint(largest);
    int e = int(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);      // biased exponent (a denormal's is 0: the scale is 2^-126)
    e = max(e, 1);
    return __uint_as_float(uint32_t(e) << 23);
  }
  struct Down {                      // by the exact inverse of a power of two (what this library writes), by division otherwise
    float scale, inverse;
    __device__ __forceinline__ explicit Down(float s) : scale(s) {
      const uint32_t bits = __float_as_uint(s);
      inverse = (bits & 0x7fffffu) == 0 && bits - 1u < (254u << 23) - 1u ? __uint_as_float((254u << 23) - bits) : 0.f;
    }
    __device__ __forceinline__ uint32_t operator()(float x) const {
      return inverse > 0.f ? nearest(__fmul_rn(x, inverse)) : scale > 0.f ? nearest(__fdiv_rn(x, scale)) : 0u;
    }
  };
  static __device__ __forceinline__ uint32_t nearest(float v) { return __nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3); }
};

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Sixteen bytes of a row as N = 16 / sizeof(T) values; `wide`: the address is a multiple of 16.
template <typename T> struct Pack {
  static constexpr int N = 16 / int(sizeof(T));
  union {
    uint4 raw;
    T v[N];
  };
  __device__ __forceinline__ Pack() {}
  __device__ __forceinline__ void load(const T* p, bool wide) {
    if (wide) {
      raw = fetch(reinterpret_cast<const uint4*>(p));
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = p[i];
    }
  }
};
#endif  // __CUDACC__

// f(T{}) for the activation type; the code of an unknown one.
template <typename F> inline int with_dtype(int dtype, F f) {
  switch (dtype) {
    case DINO_F16: return f(__half{});
    case DINO_BF16: return f(__nv_bfloat16{});
    case DINO_F32: return f(float{});
    default: return RC_DTYPE;
  }
}

}  // namespace kv
}  // namespace b200gguf

// Rows of a GGUF table for the tokens of a step: out[i] = round(dequant(table[tokens[i]]) * scale).
//
// Bound by bytes, most of them the result's (8192 values of Q4_K are 4.6 KB read and 16 KB written, and a text's tokens repeat); a single token by its chain of reads (token, block,
// result) and the launch.  A CTA has a token's row or a part of it, a thread eight values at a time: they are one store of 16 or 32 bytes, and neighbours read neighbouring bytes.
#include <algorithm>

#include "dependent_launch.cuh"
#include "kv_cache.cuh"

namespace b200gguf {
namespace stream { int sm_count(); }             // gemv_stream.cu
namespace embed {

constexpr int kThreads = 256;

template <int QT, typename T, typename I>
__global__ void __launch_bounds__(kThreads) embedding_kernel(const I* tokens, const uint8_t* table, int64_t vocabulary, T* out, int64_t items, int parts, int units,
                                                            int per_item, float scale, int* status) {
  constexpr int kOf = QTraits<QT>::kBlock / 8, kBytes = QTraits<QT>::kBytes;      // units of a block
  const int64_t row_bytes = int64_t(units / kOf) * kBytes;
  wait_for_launch_before();
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t i = parts == 1 ? item : item / parts;
    const int begin = int(item - i * parts) * per_item, end = min(begin + per_item, units);
    const int64_t token = int64_t(tokens[i]);
    const bool in = token >= 0 && token < vocabulary;
    if (!in && token != -1 && threadIdx.x == 0) kv::flag_range(status);
    const uint8_t* row = table + (in ? token : 0) * row_bytes;
    T* to = out + i * int64_t(units) * 8;
#pragma unroll 4
    for (int u = begin + int(threadIdx.x); u < end; u += kThreads) {
      float w[8];
      if (in) {
        decode8<QT>(row + int64_t(u / kOf) * kBytes, u % kOf * 8, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = __fmul_rn(w[j], scale);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = 0.f;
      }
      constexpr int N = 16 / int(sizeof(T));
#pragma unroll
      for (int j = 0; j < 8; j += N) {
        kv::Pack<T> v;
#pragma unroll
        for (int m = 0; m < N; ++m) v.v[m] = kv::from_float<T>(w[j + m]);
        *reinterpret_cast<uint4*>(to + int64_t(u) * 8 + j) = v.raw;
      }
    }
  }
}

template <int QT, typename T, typename I>
static int launch(const void* tokens, const void* table, int64_t vocabulary, void* out, int64_t count, int64_t width, float scale, int* status, cudaStream_t s) {
  const int sms = stream::sm_count();
  if (sms <= 0) return RC_LAUNCH;
  const int units = int(width / 8);
  // A row in parts of one unit a thread where that leaves SMs without work, else in one.
  const int parts = count < 4 * sms ? (units + kThreads - 1) / kThreads : 1;
  const int per_item = parts == 1 ? units : kThreads;
  const int64_t items = count * parts;
  const unsigned ctas = unsigned(std::min<int64_t>(items, 8 * int64_t(sms)));
  return launch_dependent(embedding_kernel<QT, T, I>, dim3(ctas), kThreads, 0, 1, s, static_cast<const I*>(tokens), static_cast<const uint8_t*>(table), vocabulary,
                          static_cast<T*>(out), items, parts, units, per_item, scale, status);
}

}  // namespace embed

int embedding(const void* tokens, int token_bytes, const void* table, int64_t vocabulary, void* out, int qtype, int dtype, int64_t count, int64_t width, float scale,
              cudaStream_t s) {
  if (tokens == nullptr || table == nullptr || out == nullptr) return RC_NULL;
  if (vocabulary <= 0 || count <= 0 || width <= 0) return RC_DIMS;
  const int of = qtype_block_size(qtype);
  if (of == 0) return RC_QTYPE;
  if (width % of != 0) return RC_KBLOCK;
  if (token_bytes != 4 && token_bytes != 8) return RC_DTYPE;
  if (width > INT32_MAX || count > INT64_MAX / width / 4 || vocabulary > INT64_MAX / width) return RC_RANGE;
  if ((reinterpret_cast<uintptr_t>(tokens) & (token_bytes - 1)) != 0 || (reinterpret_cast<uintptr_t>(out) & 15) != 0 ||
      (reinterpret_cast<uintptr_t>(table) & (qtype_alignment(qtype) - 1)) != 0)
    return RC_ALIGN;
  if (dtype != DINO_F16 && dtype != DINO_BF16 && dtype != DINO_F32) return RC_DTYPE;
  int* status = kv::status_words();
  if (status == nullptr) return RC_LAUNCH;
  return kv::with_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    auto of_type = [&](auto qt) -> int {
      constexpr int QT = decltype(qt)::value;
      return token_bytes == 4 ? embed::launch<QT, T, int32_t>(tokens, table, vocabulary, out, count, width, scale, status, s)
                              : embed::launch<QT, T, int64_t>(tokens, table, vocabulary, out, count, width, scale, status, s);
    };
    switch (qtype) {
      case QTYPE_Q4_0: return of_type(std::integral_constant<int, QTYPE_Q4_0>{});
      case QTYPE_Q8_0: return of_type(std::integral_constant<int, QTYPE_Q8_0>{});
      case QTYPE_Q2_K: return of_type(std::integral_constant<int, QTYPE_Q2_K>{});
      case QTYPE_Q3_K: return of_type(std::integral_constant<int, QTYPE_Q3_K>{});
      case QTYPE_Q4_K: return of_type(std::integral_constant<int, QTYPE_Q4_K>{});
      case QTYPE_Q5_K: return of_type(std::integral_constant<int, QTYPE_Q5_K>{});
      case QTYPE_Q6_K: return of_type(std::integral_constant<int, QTYPE_Q6_K>{});
      case QTYPE_MXFP4: return of_type(std::integral_constant<int, QTYPE_MXFP4>{});
      case QTYPE_NVFP4: return of_type(std::integral_constant<int, QTYPE_NVFP4>{});
      default: return RC_QTYPE;
    }
  });
}

}  // namespace b200gguf

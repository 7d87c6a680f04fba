// Root-mean-square norm with the residual's addition: t = x + residual, y = t / sqrt(mean(t^2) + eps) * weight, one CTA per row, in float32 with one
// rounding at the end; y in the activation type or as Q8_0 blocks.
#include "kv_cache.cuh"

namespace b200gguf {
namespace norm {

using kv::from_float;
using kv::to_float;

template <typename T, typename W>
__global__ void __launch_bounds__(256) rms_norm_kernel(const T* x, const T* residual, const W* weight, void* y, T* total, int width, float eps, bool q8_0) {
  __shared__ float sums[8];
  const int64_t row = blockIdx.x;
  x += row * width;
  auto value = [&](int i) { return to_float<T>(x[i]) + (residual != nullptr ? to_float<T>(residual[row * width + i]) : 0.f); };
  float sum = 0.f;
  for (int i = threadIdx.x; i < width; i += 256) {
    const float t = value(i);
    sum += t * t;
  }
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = sum;
  __syncthreads();
  sum = 0.f;
  for (int i = 0; i < 8; ++i) sum += sums[i];
  const float r = rsqrtf(sum / float(width) + eps);
  for (int i = threadIdx.x; i < width; i += 256) {                // total may be x or residual: a value is read and written by one thread
    const float t = value(i), v = t * r * to_float<W>(weight[i]);
    if (total != nullptr) total[row * width + i] = from_float<T>(t);
    if (!q8_0) {
      static_cast<T*>(y)[row * width + i] = from_float<T>(v);
    } else {                                                     // whole warps: width is a multiple of 32
      const float largest = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v) & 0x7fffffffu));
      const __half d = __float2half_rn(__fmul_rn(largest, 1.0f / 127.0f));
      const float scale = __half2float(d);
      uint8_t* block = static_cast<uint8_t*>(y) + (row * width + i) / 32 * 34;
      const int lane = threadIdx.x & 31;
      block[2 + lane] = scale > 0.f ? uint8_t(__float2int_rn(fminf(fmaxf(__fdiv_rn(v, scale), -127.f), 127.f))) : 0;
      if (lane == 0) *reinterpret_cast<__half*>(block) = d;
    }
  }
}

int rms_norm(const void* x, const void* residual, const void* weight, void* y, void* total, int dtype, int weight_dtype, int rows, int width, float eps, int q8_0,
             cudaStream_t s) {
  if (x == nullptr || weight == nullptr || y == nullptr) return RC_NULL;
  if (rows <= 0 || width <= 0) return RC_DIMS;
  if (q8_0 != 0 && width % 32 != 0) return RC_KBLOCK;
  if (weight_dtype != DINO_F32 && weight_dtype != dtype) return RC_DTYPE;
  return kv::with_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    const uintptr_t all = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual) | reinterpret_cast<uintptr_t>(total);
    if ((all & (sizeof(T) - 1)) != 0 || (reinterpret_cast<uintptr_t>(y) & (q8_0 ? 1 : sizeof(T) - 1)) != 0) return RC_ALIGN;
    if ((reinterpret_cast<uintptr_t>(weight) & (weight_dtype == DINO_F32 ? 3 : sizeof(T) - 1)) != 0) return RC_ALIGN;
    if (weight_dtype == DINO_F32)
      rms_norm_kernel<T, float><<<unsigned(rows), 256, 0, s>>>(static_cast<const T*>(x), static_cast<const T*>(residual), static_cast<const float*>(weight), y,
                                                               static_cast<T*>(total), width, eps, q8_0 != 0);
    else
      rms_norm_kernel<T, T><<<unsigned(rows), 256, 0, s>>>(static_cast<const T*>(x), static_cast<const T*>(residual), static_cast<const T*>(weight), y,
                                                           static_cast<T*>(total), width, eps, q8_0 != 0);
    return cudaGetLastError() == cudaSuccess ? RC_OK : RC_LAUNCH;
  });
}

}  // namespace norm
}  // namespace b200gguf

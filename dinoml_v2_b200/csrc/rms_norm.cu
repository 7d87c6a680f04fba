// Root-mean-square norm with the residual's addition: t = x + residual, y = t / sqrt(mean(t^2) + eps) * weight, in float32 with one rounding at the
// end; y in the activation type or as Q8_0 blocks.
//
// Bound by bytes: x and the residual in, t and y out; to Q8_0 by instructions beside them.  A CTA has a row and a thread keeps its values of t in registers between the sum
// of squares and the products, so each is read once; rows that registers do not hold are read a second time (from L2).  NT threads of V values, R rounds: as few threads
// as hold a row in 16 bytes each, since a CTA of few warps starts and meets sooner (a row of 4096: 6.2 us with 1024 threads of 4 values, 5.7 so, both with the call from Python).
// 2048 rows of 8192 float16 with residual to Q8_0, and decoded again: 67.6 us with a CTA a row and 1024 threads, 47.4 with 512, 39.4 with the next row copied ahead, 37.2 with one
// reciprocal a block instead of divisions.  The norm alone, launches one after the other: 30.0 us of these (119 MB, 3.9 TB/s); bfloat16 to bfloat16 with residual 23.1 us (134 MB, 5.8 TB/s),
// 2048 rows of 4096 13.4 us, 8192 of 4096 48.5 us (5.5 TB/s), 2048 of 8192 float32 61.1 us (4.4 TB/s).
#include <algorithm>

#include "kv_cache.cuh"

namespace b200gguf {
namespace stream { int sm_count(); }             // gemv_stream.cu
namespace norm {

using kv::from_float;
using kv::to_float;

constexpr int kThreads = 1024;       // of an SM: 64 registers each

// V values from or to memory: WIDE: at an address that is a multiple of 16, in accesses of 16 bytes.
template <typename T, int N> struct alignas(sizeof(T) * N) Vec { T v[N]; };
template <typename T, int V> struct Values {
  T v[V];
  template <bool WIDE> __device__ __forceinline__ void load(const T* p) {
    constexpr int N = !WIDE ? 1 : V * int(sizeof(T)) > 16 ? 16 / int(sizeof(T)) : V;
#pragma unroll
    for (int i = 0; i < V; i += N) {
      const Vec<T, N> a = *reinterpret_cast<const Vec<T, N>*>(p + i);
#pragma unroll
      for (int j = 0; j < N; ++j) v[i + j] = a.v[j];
    }
  }
};
template <bool WIDE, int V, typename T> __device__ __forceinline__ void store_values(T* p, const float (&t)[V]) {
  constexpr int N = WIDE ? V : 1;
#pragma unroll
  for (int i = 0; i < V; i += N) {
    Vec<T, N> a;
#pragma unroll
    for (int j = 0; j < N; ++j) a.v[j] = from_float<T>(t[i + j]);
    *reinterpret_cast<Vec<T, N>*>(p + i) = a;
  }
}

__device__ __forceinline__ void copy16(void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(uint32_t(__cvta_generic_to_shared(to))), "l"(from) : "memory");
}

template <typename T, typename W, int V, bool WIDE, int R, int NT, bool Q8>
__global__ void __launch_bounds__(NT, kThreads / NT) rms_norm_kernel(const T* x, const T* residual, const W* weight, void* y, T* total, int rows, int width, float eps) {
  __shared__ float sums[2][NT / 32];
  const int tid = threadIdx.x, lane = tid & 31;
  const int first = tid * V, step = NT * V;
  bool in[R];
#pragma unroll
  for (int r = 0; r < R; ++r) in[r] = first + r * step < width;
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  // The row after this one, in shared memory: a thread reads what it has copied itself.
  constexpr bool AHEAD = WIDE && R <= 2;
  __shared__ Vec<T, V> ahead[AHEAD ? 2 * R : 1][AHEAD ? NT : 1];
  auto fetch = [&](int64_t row) {
    if constexpr (AHEAD) {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (!in[r]) continue;
        copy16(&ahead[2 * r][tid], x + row * width + first + r * step);
        if (residual != nullptr) copy16(&ahead[2 * r + 1][tid], residual + row * width + first + r * step);
      }
      asm volatile("cp.async.commit_group;\n" ::: "memory");
    }
  };
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    auto load = [&](int i, float (&t)[V]) {
      Values<T, V> v;
      v.template load<WIDE>(x + row * width + i);
#pragma unroll
      for (int j = 0; j < V; ++j) t[j] = to_float<T>(v.v[j]);
      if (residual == nullptr) return;
      v.template load<WIDE>(residual + row * width + i);
#pragma unroll
      for (int j = 0; j < V; ++j) t[j] += to_float<T>(v.v[j]);
    };
    float t[R][V], sum = 0.f;
    if (AHEAD && row != blockIdx.x) {
      asm volatile("cp.async.wait_all;\n" ::: "memory");
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const Vec<T, V> a = ahead[AHEAD ? 2 * r : 0][AHEAD ? tid : 0], b = ahead[AHEAD ? 2 * r + 1 : 0][AHEAD ? tid : 0];
#pragma unroll
        for (int j = 0; j < V; ++j) {
          t[r][j] = in[r] ? to_float<T>(a.v[j]) : 0.f;
          if (residual != nullptr && in[r]) t[r][j] += to_float<T>(b.v[j]);
        }
      }
    } else {
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (in[r]) {
          load(first + r * step, t[r]);
        } else {
#pragma unroll
          for (int j = 0; j < V; ++j) t[r][j] = 0.f;
        }
      }
    }
    if (row + gridDim.x < rows) fetch(row + gridDim.x);                    // (rows do not overlap: total may be x or the residual)
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < V; ++j) s = fmaf(t[r][j], t[r][j], s);
      sum += s;
    }
    for (int i = first + R * step; i < width; i += step) {
      float u[V], s = 0.f;
      load(i, u);
#pragma unroll
      for (int j = 0; j < V; ++j) s = fmaf(u[j], u[j], s);
      sum += s;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    float* met = sums[(row / gridDim.x) & 1];                              // (two places: one barrier a row)
    if (lane == 0) met[tid >> 5] = sum;
    __syncthreads();
    sum = lane < NT / 32 ? met[lane] : 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float scale = rsqrtf(sum / float(width) + eps);
    auto finish = [&](int i, const float (&u)[V], bool here) {             // (called by whole warps where there are blocks)
      float v[V];
      if (here) {
        Values<W, V> w;
        w.template load<WIDE>(weight + i);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = u[j] * scale * to_float<W>(w.v[j]);
        if (total != nullptr) store_values<WIDE, V>(total + row * width + i, u);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = 0.f;
      }
      if (!Q8) {
        if (here) store_values<WIDE, V>(static_cast<T*>(y) + row * width + i, v);
      } else {                                                             // 32 / V lanes have a block (a width of blocks: all of them or none)
        uint32_t largest = 0;
#pragma unroll
        for (int j = 0; j < V; ++j) largest = max(largest, __float_as_uint(v[j]) & 0x7fffffffu);
#pragma unroll
        for (int o = 16 / V; o > 0; o >>= 1) largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, o));
        if (!here) return;
        const __half d = __float2half_rn(__fmul_rn(__uint_as_float(largest), 1.0f / 127.0f));
        const float step8 = __half2float(d);
        // blocks are multiples of two bytes
        uint16_t* block = reinterpret_cast<uint16_t*>(static_cast<uint8_t*>(y) + (row * width + i) / 32 * 34);
        if ((i & 31) == 0) block[0] = __half_as_ushort(d);
        // The integer nearest to v / step, in the last bits of v * (1 / step) + 1.5 2^23.  With a reciprocal within 2 units of its last place v / step is at
        // most 127.1 * 2^-22 < 2^-14 away: where that is further from half way between two integers than 1e-4 both have the same nearest one, elsewhere,
        // and where the step is no normal float16 (so that values may be beyond 127 of it, or none is finite), the division decides.
        constexpr float kRound = 12582912.f;
        const float up = __fdividef(1.f, step8);
        uint32_t q[V];
        float worst = 0.f;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float t = fmaf(v[j], up, kRound);
          q[j] = __float_as_uint(t) & 0xffu;
          worst = fmaxf(worst, fabsf(fmaf(v[j], up, kRound - t)));
        }
        if (!(worst < 0.4999f && step8 >= 0x1p-14f && step8 <= 65504.f)) {
#pragma unroll
          for (int j = 0; j < V; ++j) q[j] = step8 > 0.f ? uint32_t(__float2int_rn(fminf(fmaxf(__fdiv_rn(v[j], step8), -127.f), 127.f))) & 0xffu : 0u;
        }
#pragma unroll
        for (int j = 0; j + 1 < V; j += 2) block[1 + ((i & 31) + j) / 2] = uint16_t(q[j] | (q[j + 1] << 8));
      }
    };
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (!Q8 || first - lane * V + r * step < width) finish(first + r * step, t[r], in[r]);
    for (int i = first + R * step; i - lane * V < width; i += step) {      // (a value of total is read and written by one thread)
      float u[V];
      if (i < width) load(i, u);
      finish(i, u, i < width);
    }
  }
}

template <typename T, typename W, int V, bool WIDE, int R, int NT, bool Q8>
static int launch(const void* x, const void* residual, const void* weight, void* y, void* total, int rows, int width, float eps, cudaStream_t s) {
  // Where an SM has more rows than it holds CTAs, a CTA takes several and fetches one while it has the one before.
  const int sms = stream::sm_count();
  if (sms <= 0) return RC_LAUNCH;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(std::min(rows, sms * (kThreads / NT))));
  cfg.blockDim = dim3(NT);
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, rms_norm_kernel<T, W, V, WIDE, R, NT, Q8>, static_cast<const T*>(x), static_cast<const T*>(residual), static_cast<const W*>(weight), y,
                            static_cast<T*>(total), rows, width, eps) == cudaSuccess
             ? RC_OK
             : RC_LAUNCH;
}

// The same threads have the same values whatever the addresses are, so that results do not depend on those.
template <typename T, typename W, bool Q8, bool WIDE>
static int pick(const void* x, const void* residual, const void* weight, void* y, void* total, int rows, int width, float eps, cudaStream_t s) {
  constexpr int V = 16 / int(sizeof(T));
  if (width % V != 0) return launch<T, W, 1, false, 8, 1024, false>(x, residual, weight, y, total, rows, width, eps, s);
  if (width <= 128 * V) return launch<T, W, V, WIDE, 1, 128, Q8>(x, residual, weight, y, total, rows, width, eps, s);
  if (width <= 256 * V) return launch<T, W, V, WIDE, 1, 256, Q8>(x, residual, weight, y, total, rows, width, eps, s);
  if (width <= 512 * V) return launch<T, W, V, WIDE, 1, 512, Q8>(x, residual, weight, y, total, rows, width, eps, s);
  if (width <= 1024 * V) return launch<T, W, V, WIDE, 2, 512, Q8>(x, residual, weight, y, total, rows, width, eps, s);
  return launch<T, W, V, WIDE, 4, 1024, Q8>(x, residual, weight, y, total, rows, width, eps, s);
}

int rms_norm(const void* x, const void* residual, const void* weight, void* y, void* total, int dtype, int weight_dtype, int rows, int width, float eps, int q8_0,
             cudaStream_t s) {
  if (x == nullptr || weight == nullptr || y == nullptr) return RC_NULL;
  if (rows <= 0 || width <= 0) return RC_DIMS;
  if (q8_0 != 0 && width % 32 != 0) return RC_KBLOCK;
  if (weight_dtype != DINO_F32 && weight_dtype != dtype) return RC_DTYPE;
  return kv::with_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    const uintptr_t all = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(residual) | reinterpret_cast<uintptr_t>(total), out = reinterpret_cast<uintptr_t>(y);
    if ((all & (sizeof(T) - 1)) != 0 || (out & (q8_0 ? 1 : sizeof(T) - 1)) != 0) return RC_ALIGN;
    if ((reinterpret_cast<uintptr_t>(weight) & (weight_dtype == DINO_F32 ? 3 : sizeof(T) - 1)) != 0) return RC_ALIGN;
    const bool wide = ((all | reinterpret_cast<uintptr_t>(weight) | (q8_0 ? 0 : out) | uint64_t(width) * sizeof(T)) & 15) == 0;
    auto go = [&](auto w) -> int {
      using W = decltype(w);
      if (q8_0) return wide ? pick<T, W, true, true>(x, residual, weight, y, total, rows, width, eps, s) : pick<T, W, true, false>(x, residual, weight, y, total, rows, width, eps, s);
      return wide ? pick<T, W, false, true>(x, residual, weight, y, total, rows, width, eps, s) : pick<T, W, false, false>(x, residual, weight, y, total, rows, width, eps, s);
    };
    return weight_dtype == DINO_F32 ? go(float{}) : go(T{});
  });
}

}  // namespace norm
}  // namespace b200gguf

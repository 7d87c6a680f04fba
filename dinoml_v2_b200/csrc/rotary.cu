// Rotation of queries and keys by position, with the norm of each head in the same pass.
//
// t = x / sqrt(mean(x^2) + eps) * w over a head, then pairs (a, b) -> m (a cos - b sin, b cos + a sin), the angle position * frequency.  A value is read and written once: bound by
// bytes, a single token by its chain of reads (position, angle, result).  A lane has P pairs of a head, the two halves of a pair in one register file: 16 bytes of a from the first
// half and 16 of b from the second (or 32 bytes in one piece where neighbours are pairs), so that neither the norm (a sum over the lanes of a head) nor the rotation needs shared memory.
// The angles are a row's, not a head's: each is reduced once a CTA, in float64 (131072 radians in float32 are 0.008 off), to turns in [-1/2, 1/2], whose sine and cosine
// in float32 all heads of the row share.
#include <algorithm>

#include "dependent_launch.cuh"
#include "kv_cache.cuh"

namespace b200gguf {
namespace rope {

constexpr int kWarps = 8, kMaxDim = 512;

struct Side {
  const void* x;
  void* out;
  const void* weight;
  int64_t row_stride, head_stride, out_row_stride, out_head_stride;
  int heads;
  bool in_place;
};

// N values from or to p; WIDE: in one access.
template <typename T, int N> struct alignas(sizeof(T) * N) Piece { T v[N]; };

// P: pairs of a unit (a lane's share of a head); N: units of a lane; a head has `lanes` lanes, a power of two.
template <typename T, int P, int N>
__global__ void __launch_bounds__(32 * kWarps) rotary_kernel(Side q, Side k, const int* positions, const double* frequencies, int pairs, bool weight_f32, int head_dim,
                                                             int lanes_log2, int units, int turned, float eps, float magnitude, bool interleaved) {
  __shared__ float2 turn[kMaxDim / 2];                     // (cos, sin) of the row's angles, times the magnitude
  using Two = Piece<T, P>;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = blockIdx.x;
  wait_for_launch_before();
  const int position = positions[row];
  const int lanes = 1 << lanes_log2, heads = q.heads + k.heads, per_pass = 32 >> lanes_log2;
  const int at = lane & (lanes - 1);
  const int passes = (heads + per_pass - 1) / per_pass;
  const int first = blockIdx.y * kWarps + warp, step = gridDim.y * kWarps;

  // Channels of unit u: P at `a` and P at `b` (units behind the turned ones: 2 P in one piece, which stay).
  auto channels = [&](int u, int& a, int& b) {
    if (u < turned && !interleaved) {
      a = u * P;
      b = pairs + u * P;
    } else {
      a = u < turned ? 2 * u * P : 2 * pairs + 2 * (u - turned) * P;
      b = a + P;
    }
  };
  struct Held { Two a, b; };
  Held held[N];
  auto load = [&](int pass) {
    const int h = pass * per_pass + (lane >> lanes_log2);
    if (pass >= passes || h >= heads) return;
    const Side& s = h < q.heads ? q : k;
    const T* x = static_cast<const T*>(s.x) + row * s.row_stride + (h < q.heads ? h : h - q.heads) * s.head_stride;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int u = at + n * lanes;
      int a, b;
      channels(u, a, b);
      if (u < units) {
        held[n].a = *reinterpret_cast<const Two*>(x + a);
        held[n].b = *reinterpret_cast<const Two*>(x + b);
      }
    }
  };
  if (position >= 0) {
    load(first);
    for (int i = threadIdx.x; i < pairs; i += 32 * kWarps) {
      // half turns in [-1, 1], in two floats: the second is a rounding's rest, by which sine and cosine are moved to first order
      const double turns = double(position) * frequencies[i] * 0.15915494309189533577, part = 2. * (turns - rint(turns));
      const float high = float(part), low = float(part - double(high)) * 3.14159265358979f;
      float sin, cos;
      sincospif(high, &sin, &cos);
      turn[i] = make_float2(magnitude * fmaf(-sin, low, cos), magnitude * fmaf(cos, low, sin));
    }
  }
  __syncthreads();
  for (int pass = first; pass < passes; pass += step) {
    const int h = pass * per_pass + (lane >> lanes_log2);
    const bool here = h < heads;
    const Side& s = h < q.heads ? q : k;
    T* out = static_cast<T*>(s.out) + row * s.out_row_stride + (h < q.heads ? h : h - q.heads) * s.out_head_stride;
    if (position < 0) {
      if (!here || s.in_place) continue;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int u = at + n * lanes;
        int a, b;
        channels(u, a, b);
        if (u >= units) continue;
        Two zero;
#pragma unroll
        for (int j = 0; j < P; ++j) zero.v[j] = kv::from_float<T>(0.f);
        *reinterpret_cast<Two*>(out + a) = zero;
        *reinterpret_cast<Two*>(out + b) = zero;
      }
      continue;
    }
    float va[N][P], vb[N][P], sum = 0.f;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const bool in = here && at + n * lanes < units;
#pragma unroll
      for (int j = 0; j < P; ++j) {
        va[n][j] = in ? kv::to_float<T>(held[n].a.v[j]) : 0.f;
        vb[n][j] = in ? kv::to_float<T>(held[n].b.v[j]) : 0.f;
        sum = fmaf(va[n][j], va[n][j], sum);
        sum = fmaf(vb[n][j], vb[n][j], sum);
      }
    }
    load(pass + step);
    if (q.weight != nullptr || k.weight != nullptr) {
      for (int o = lanes >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (here && s.weight != nullptr) {
        const float scale = rsqrtf(sum / float(head_dim) + eps);
#pragma unroll
        for (int n = 0; n < N; ++n) {
          const int u = at + n * lanes;
          int a, b;
          channels(u, a, b);
          if (u >= units) continue;
          if (weight_f32) {
            const Piece<float, P> wa = *reinterpret_cast<const Piece<float, P>*>(static_cast<const float*>(s.weight) + a);
            const Piece<float, P> wb = *reinterpret_cast<const Piece<float, P>*>(static_cast<const float*>(s.weight) + b);
#pragma unroll
            for (int j = 0; j < P; ++j) {
              va[n][j] *= scale * wa.v[j];
              vb[n][j] *= scale * wb.v[j];
            }
          } else {
            const Two wa = *reinterpret_cast<const Two*>(static_cast<const T*>(s.weight) + a), wb = *reinterpret_cast<const Two*>(static_cast<const T*>(s.weight) + b);
#pragma unroll
            for (int j = 0; j < P; ++j) {
              va[n][j] *= scale * kv::to_float<T>(wa.v[j]);
              vb[n][j] *= scale * kv::to_float<T>(wb.v[j]);
            }
          }
        }
      }
    }
    if (!here) continue;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int u = at + n * lanes;
      int a, b;
      channels(u, a, b);
      if (u >= units) continue;
      Two oa, ob;
      if (u < turned) {
        float ra[P], rb[P];
#pragma unroll
        for (int j = 0; j < P; ++j) {
          // pair j of a lane: (a_j, b_j), or neighbours in the 2 P values of a and b
          const float x = interleaved ? (2 * j < P ? va[n][2 * j < P ? 2 * j : 0] : vb[n][2 * j < P ? 0 : 2 * j - P]) : va[n][j];
          const float y = interleaved ? (2 * j + 1 < P ? va[n][2 * j + 1 < P ? 2 * j + 1 : 0] : vb[n][2 * j + 1 < P ? 0 : 2 * j + 1 - P]) : vb[n][j];
          const float2 t = turn[u * P + j];
          ra[j] = x * t.x - y * t.y;
          rb[j] = y * t.x + x * t.y;
        }
#pragma unroll
        for (int j = 0; j < P; ++j) {
          // back to where they were: value i of the 2 P is side i % 2 of pair i / 2
          const float x = interleaved ? (j % 2 == 0 ? ra[j / 2] : rb[j / 2]) : ra[j];
          const float y = interleaved ? ((P + j) % 2 == 0 ? ra[(P + j) / 2] : rb[(P + j) / 2]) : rb[j];
          oa.v[j] = kv::from_float<T>(x);
          ob.v[j] = kv::from_float<T>(y);
        }
      } else {
#pragma unroll
        for (int j = 0; j < P; ++j) {
          oa.v[j] = kv::from_float<T>(va[n][j]);
          ob.v[j] = kv::from_float<T>(vb[n][j]);
        }
      }
      *reinterpret_cast<Two*>(out + a) = oa;
      *reinterpret_cast<Two*>(out + b) = ob;
    }
  }
}

template <typename T, int P, int N>
static int launch(const Side& q, const Side& k, const int* positions, const double* frequencies, int pairs, bool weight_f32, int rows, int head_dim, float eps, float magnitude,
                  bool interleaved, cudaStream_t s) {
  const int units = head_dim / (2 * P), turned = pairs / P;
  int log2 = 0;
  while (log2 < 5 && (1 << log2) * N < units) ++log2;
  const int passes = (q.heads + k.heads + (32 >> log2) - 1) / (32 >> log2);
  const unsigned y = unsigned(std::min((passes + 2 * kWarps - 1) / (2 * kWarps), 65535));
  return launch_dependent(rotary_kernel<T, P, N>, dim3(unsigned(rows), y), 32 * kWarps, 0, 1, s, q, k, positions, frequencies, pairs, weight_f32, head_dim, log2, units, turned,
                          eps, magnitude, interleaved);
}

}  // namespace rope

int rotary(const DinoB200Heads* q, const DinoB200Heads* k, const int* positions, const double* frequencies, int pairs, int dtype, int weight_dtype, int rows, int head_dim,
           float eps, float magnitude, int interleaved, cudaStream_t s) {
  using namespace rope;
  if (q == nullptr || positions == nullptr || q->x == nullptr || q->out == nullptr || (k != nullptr && (k->x == nullptr || k->out == nullptr))) return RC_NULL;
  if (pairs > 0 && frequencies == nullptr) return RC_NULL;
  if (rows <= 0 || head_dim <= 0 || q->heads <= 0 || (k != nullptr && k->heads <= 0)) return RC_DIMS;
  if (head_dim % 2 != 0 || head_dim > kMaxDim || pairs < 0 || 2 * pairs > head_dim || int64_t(q->heads) + (k != nullptr ? k->heads : 0) > (1 << 20)) return RC_RANGE;
  if (weight_dtype != DINO_F32 && weight_dtype != dtype) return RC_DTYPE;
  return kv::with_dtype(dtype, [&](auto t) -> int {
    using T = decltype(t);
    Side sides[2] = {};
    // Addresses that every piece of P values starts at a multiple of.
    uint64_t every = 0, weights = 0;
    for (int i = 0; i < (k != nullptr ? 2 : 1); ++i) {
      const DinoB200Heads& h = i == 0 ? *q : *k;
      sides[i] = {h.x, h.out, h.weight, h.row_stride, h.head_stride, h.out_row_stride, h.out_head_stride, h.heads,
                  h.x == h.out && h.row_stride == h.out_row_stride && h.head_stride == h.out_head_stride};
      const uint64_t row = rows > 1 ? uint64_t(h.row_stride | h.out_row_stride) : 0, head = h.heads > 1 ? uint64_t(h.head_stride | h.out_head_stride) : 0;
      every |= reinterpret_cast<uintptr_t>(h.x) | reinterpret_cast<uintptr_t>(h.out) | (row | head) * sizeof(T);
      weights |= reinterpret_cast<uintptr_t>(h.weight);
    }
    if ((every & (sizeof(T) - 1)) != 0 || (weights & ((weight_dtype == DINO_F32 ? 4 : sizeof(T)) - 1)) != 0) return RC_ALIGN;
    if ((reinterpret_cast<uintptr_t>(positions) & 3) != 0 || (reinterpret_cast<uintptr_t>(frequencies) & 7) != 0) return RC_ALIGN;
    const bool f32 = weight_dtype == DINO_F32;
    auto fits = [&](int p) {      // whole units of p pairs, at their alignment
      return (every & (p * sizeof(T) - 1)) == 0 && (weights & (p * (f32 ? 4 : sizeof(T)) - 1)) == 0 && pairs % p == 0 && (head_dim - 2 * pairs) % (2 * p) == 0;
    };
    auto go = [&](auto kern) { return kern(sides[0], sides[1], positions, frequencies, pairs, f32, rows, head_dim, eps, magnitude, interleaved != 0, s); };
    if constexpr (sizeof(T) == 2) {
      if (fits(8)) return go(launch<T, 8, 1>);
    }
    if (fits(4)) return head_dim <= 256 ? go(launch<T, 4, 1>) : go(launch<T, 4, 2>);
    return go(launch<T, 1, 8>);
  });
}

}  // namespace b200gguf

// Rotation of queries and keys by position, with the norm of each head in the same pass.
//
// t = x / sqrt(mean(x^2) + eps) * w over a head, then pairs (a, b) -> m (a cos - b sin, b cos + a sin), the angle position * frequency.  A value is read and written once: bound by
// bytes, a single token by its chain of reads (position, angle, result).  A warp has a row, or some of its heads where there are few rows; a lane has P pairs of a head, the two halves of
// a pair in one register file: 16 bytes of a from the first half and 16 of b from the second (or 32 bytes in one piece where neighbours are pairs), so that neither the norm (a
// sum over the lanes of a head) nor the rotation needs shared memory, and warps never wait for one another.  Several heads' reads are under way while one is computed.  The angles are a
// row's, not a head's: a warp reduces each once, in float64 (131072 radians in float32 are 0.008 off), to half turns in [-1, 1], whose sine and cosine in float32 all of its heads share.
#include <algorithm>

#include "dependent_launch.cuh"
#include "kv_cache.cuh"

namespace b200gguf {
namespace stream { int sm_count(); }             // gemv_stream.cu
namespace rope {

constexpr int kWarps = 4, kMaxDim = 512;

struct Side {
  const void* x;
  void* out;
  const void* weight;
  int64_t row_stride, head_stride, out_row_stride, out_head_stride;
  int heads;
  bool in_place;
};
struct Args {
  Side q, k;
  const int* positions;
  const double* frequencies;
  int64_t items;                 // rows x slices: a warp has one
  int slices, pairs, head_dim, lanes_log2, units, turned;
  float eps, magnitude;
  bool weight_f32;
};

// N values from or to p; WIDE: in one access.  (The same lanes have the same values whatever the addresses are, so that results do not depend on those.)
template <typename T, int N> struct alignas(sizeof(T) * N) Piece { T v[N]; };
template <bool WIDE, typename T, int N> __device__ __forceinline__ void get(Piece<T, N>& to, const T* p) {
  if constexpr (WIDE) {
    to = *reinterpret_cast<const Piece<T, N>*>(p);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) to.v[i] = p[i];
  }
}
template <bool WIDE, typename T, int N> __device__ __forceinline__ void put(T* p, const Piece<T, N>& from) {
  if constexpr (WIDE) {
    *reinterpret_cast<Piece<T, N>*>(p) = from;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = from.v[i];
  }
}

// P: pairs of a unit (a lane's share of a head); N: units of a lane; a head has 2^lanes_log2 lanes; U: passes over heads whose reads are under way.
template <typename T, int P, int N, int U, bool WIDE, bool NEXT>
__global__ void __launch_bounds__(32 * kWarps, N == 1 && WIDE ? 4 : 3) rotary_kernel(Args g) {
  __shared__ float2 turns[kWarps][kMaxDim / 2];            // (cos, sin) of the row's angles, times the magnitude
  using Two = Piece<T, P>;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t item = int64_t(blockIdx.x) * kWarps + warp;
  wait_for_launch_before();
  if (item >= g.items) return;
  const int64_t row = g.slices == 1 ? item : item / g.slices;
  const int slice = int(item - row * g.slices);
  const int position = g.positions[row];
  const int lanes = 1 << g.lanes_log2, heads = g.q.heads + g.k.heads, per_pass = 32 >> g.lanes_log2;
  const int at = lane & (lanes - 1), sub = lane >> g.lanes_log2;
  const int passes = (heads + per_pass - 1) / per_pass;

  // Channels of unit n: P at a and P at b (units behind the turned ones: 2 P in one piece, which stay).
  int a[N], b[N];
  bool in[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int u = at + n * lanes;
    in[n] = u < g.units;
    if (u < g.turned && !NEXT) {
      a[n] = u * P;
      b[n] = g.pairs + u * P;
    } else {
      a[n] = u < g.turned ? 2 * u * P : 2 * g.pairs + 2 * (u - g.turned) * P;
      b[n] = a[n] + P;
    }
  }
  struct Held { Two a[N], b[N]; };
  Held held[U];
  auto side_of = [&](int h) -> const Side& { return h < g.q.heads ? g.q : g.k; };
  auto load = [&](int pass, Held& to) {
    const int h = pass * per_pass + sub;
    if (pass >= passes || h >= heads) return;
    const Side& s = side_of(h);
    const T* x = static_cast<const T*>(s.x) + row * s.row_stride + (h < g.q.heads ? h : h - g.q.heads) * s.head_stride;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if (!in[n]) continue;
      get<WIDE>(to.a[n], x + a[n]);
      get<WIDE>(to.b[n], x + b[n]);
    }
  };
  auto out_of = [&](int h, const Side& s) { return static_cast<T*>(s.out) + row * s.out_row_stride + (h < g.q.heads ? h : h - g.q.heads) * s.out_head_stride; };
  if (position < 0) {                                      // nobody's
    Two zero;
#pragma unroll
    for (int j = 0; j < P; ++j) zero.v[j] = kv::from_float<T>(0.f);
    for (int pass = slice; pass < passes; pass += g.slices) {
      const int h = pass * per_pass + sub;
      if (h >= heads || side_of(h).in_place) continue;
      T* out = out_of(h, side_of(h));
#pragma unroll
      for (int n = 0; n < N; ++n) {
        if (!in[n]) continue;
        put<WIDE>(out + a[n], zero);
        put<WIDE>(out + b[n], zero);
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < U; ++i) load(slice + i * g.slices, held[i]);
  for (int i = lane; i < g.pairs; i += 32) {
    // half turns in [-1, 1], in two floats: the second is a rounding's rest, by which sine and cosine are moved to first order
    const double all = double(position) * g.frequencies[i] * 0.15915494309189533577, part = 2. * (all - rint(all));
    const float high = float(part), low = float(part - double(high)) * 3.14159265358979f;
    float sin, cos;
    sincospif(high, &sin, &cos);
    turns[warp][i] = make_float2(g.magnitude * fmaf(-sin, low, cos), g.magnitude * fmaf(cos, low, sin));
  }
  __syncwarp();
  float2 turn[N][P];
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int j = 0; j < P; ++j) turn[n][j] = at + n * lanes < g.turned ? turns[warp][(at + n * lanes) * P + j] : make_float2(1.f, 0.f);

  auto pass_of = [&](int pass, Held& x) {
    const int h = pass * per_pass + sub;
    const bool here = h < heads;
    const Side& s = side_of(h);
    float va[N][P], vb[N][P], sum = 0.f;
#pragma unroll
    for (int n = 0; n < N; ++n) {
#pragma unroll
      for (int j = 0; j < P; ++j) {
        va[n][j] = here && in[n] ? kv::to_float<T>(x.a[n].v[j]) : 0.f;
        vb[n][j] = here && in[n] ? kv::to_float<T>(x.b[n].v[j]) : 0.f;
        sum = fmaf(va[n][j], va[n][j], sum);
        sum = fmaf(vb[n][j], vb[n][j], sum);
      }
    }
    load(pass + U * g.slices, x);
    if (g.q.weight != nullptr || g.k.weight != nullptr) {
      for (int o = lanes >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (here && s.weight != nullptr) {
        const float scale = rsqrtf(sum / float(g.head_dim) + g.eps);
#pragma unroll
        for (int n = 0; n < N; ++n) {
          if (!in[n]) continue;
          auto times = [&](auto w) {                       // (weights stay in L1)
            using W = decltype(w);
            Piece<W, P> wa, wb;
            get<WIDE>(wa, static_cast<const W*>(s.weight) + a[n]);
            get<WIDE>(wb, static_cast<const W*>(s.weight) + b[n]);
#pragma unroll
            for (int j = 0; j < P; ++j) {
              va[n][j] *= scale * kv::to_float<W>(wa.v[j]);
              vb[n][j] *= scale * kv::to_float<W>(wb.v[j]);
            }
          };
          if (g.weight_f32) times(float{}); else times(T{});
        }
      }
    }
    if (!here) return;
    T* out = out_of(h, s);
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if (!in[n]) continue;
      Two oa, ob;
      if (at + n * lanes < g.turned) {
        float ra[P], rb[P];
#pragma unroll
        for (int j = 0; j < P; ++j) {
          // pair j of a lane: (a_j, b_j), or neighbours in the 2 P values of a and b
          const float x0 = NEXT ? (2 * j < P ? va[n][2 * j < P ? 2 * j : 0] : vb[n][2 * j < P ? 0 : 2 * j - P]) : va[n][j];
          const float x1 = NEXT ? (2 * j + 1 < P ? va[n][2 * j + 1 < P ? 2 * j + 1 : 0] : vb[n][2 * j + 1 < P ? 0 : 2 * j + 1 - P]) : vb[n][j];
          ra[j] = x0 * turn[n][j].x - x1 * turn[n][j].y;
          rb[j] = x1 * turn[n][j].x + x0 * turn[n][j].y;
        }
#pragma unroll
        for (int j = 0; j < P; ++j) {
          // back to where they were: value i of the 2 P is side i % 2 of pair i / 2
          oa.v[j] = kv::from_float<T>(NEXT ? (j % 2 == 0 ? ra[j / 2] : rb[j / 2]) : ra[j]);
          ob.v[j] = kv::from_float<T>(NEXT ? ((P + j) % 2 == 0 ? ra[(P + j) / 2] : rb[(P + j) / 2]) : rb[j]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < P; ++j) {
          oa.v[j] = kv::from_float<T>(va[n][j]);
          ob.v[j] = kv::from_float<T>(vb[n][j]);
        }
      }
      put<WIDE>(out + a[n], oa);
      put<WIDE>(out + b[n], ob);
    }
  };
  for (int pass = slice; pass < passes; pass += U * g.slices) {
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (pass + i * g.slices < passes) pass_of(pass + i * g.slices, held[i]);
  }
}

template <typename T, int P, int N, int U, bool WIDE, bool NEXT> static int launch(Args g, int rows, cudaStream_t s) {
  const int sms = stream::sm_count();
  if (sms <= 0) return RC_LAUNCH;
  g.units = g.head_dim / (2 * P);
  g.turned = g.pairs / P;
  g.lanes_log2 = 0;
  while (g.lanes_log2 < 5 && (1 << g.lanes_log2) * N < g.units) ++g.lanes_log2;
  // A row's heads are shared by several warps where there are fewer rows than an SM has room for warps.
  const int passes = (g.q.heads + g.k.heads + (32 >> g.lanes_log2) - 1) / (32 >> g.lanes_log2);
  g.slices = int(std::min<int64_t>(passes, std::max<int64_t>(1, int64_t(sms) * 16 / rows)));
  g.items = int64_t(rows) * g.slices;
  return launch_dependent(rotary_kernel<T, P, N, U, WIDE, NEXT>, dim3(unsigned((g.items + kWarps - 1) / kWarps)), 32 * kWarps, 0, 1, s, g);
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
    Args g = {};
    // Addresses that every piece of P values starts at a multiple of.
    uint64_t every = 0, weights = 0;
    for (int i = 0; i < (k != nullptr ? 2 : 1); ++i) {
      const DinoB200Heads& h = i == 0 ? *q : *k;
      (i == 0 ? g.q : g.k) = {h.x, h.out, h.weight, h.row_stride, h.head_stride, h.out_row_stride, h.out_head_stride, h.heads,
                              h.x == h.out && h.row_stride == h.out_row_stride && h.head_stride == h.out_head_stride};
      const uint64_t row = rows > 1 ? uint64_t(h.row_stride | h.out_row_stride) : 0, head = h.heads > 1 ? uint64_t(h.head_stride | h.out_head_stride) : 0;
      every |= reinterpret_cast<uintptr_t>(h.x) | reinterpret_cast<uintptr_t>(h.out) | (row | head) * sizeof(T);
      weights |= reinterpret_cast<uintptr_t>(h.weight);
    }
    if ((every & (sizeof(T) - 1)) != 0 || (weights & ((weight_dtype == DINO_F32 ? 4 : sizeof(T)) - 1)) != 0) return RC_ALIGN;
    if ((reinterpret_cast<uintptr_t>(positions) & 3) != 0 || (reinterpret_cast<uintptr_t>(frequencies) & 7) != 0) return RC_ALIGN;
    g.positions = positions;
    g.frequencies = frequencies;
    g.pairs = pairs;
    g.head_dim = head_dim;
    g.eps = eps;
    g.magnitude = magnitude;
    g.weight_f32 = weight_dtype == DINO_F32;
    auto whole = [&](int p) { return pairs % p == 0 && (head_dim - 2 * pairs) % (2 * p) == 0; };      // units of p pairs
    auto wide = [&](int p) { return (every & (p * sizeof(T) - 1)) == 0 && (weights & (p * (g.weight_f32 ? 4 : sizeof(T)) - 1)) == 0; };
    auto go = [&](auto p, auto n, auto u) {
      constexpr int P = decltype(p)::value, N = decltype(n)::value, U = decltype(u)::value;
      if (interleaved) return P > 1 && wide(P) ? launch<T, P, N, U, true, true>(g, rows, s) : launch<T, P, N, U, P == 1, true>(g, rows, s);
      return P > 1 && wide(P) ? launch<T, P, N, U, true, false>(g, rows, s) : launch<T, P, N, U, P == 1, false>(g, rows, s);
    };
    using std::integral_constant;
    if constexpr (sizeof(T) == 2) {
      if (whole(8)) return go(integral_constant<int, 8>{}, integral_constant<int, 1>{}, integral_constant<int, 4>{});
    }
    if (whole(4) && head_dim <= 256) return go(integral_constant<int, 4>{}, integral_constant<int, 1>{}, integral_constant<int, 4>{});
    if (whole(4)) return go(integral_constant<int, 4>{}, integral_constant<int, 2>{}, integral_constant<int, 2>{});
    return go(integral_constant<int, 1>{}, integral_constant<int, 8>{}, integral_constant<int, 1>{});
  });
}

}  // namespace b200gguf

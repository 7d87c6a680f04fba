// Rotation of queries and keys by position, with the norm of each head in the same pass.
//
// t = x / sqrt(mean(x^2) + eps) * w over a head, then pairs (a, b) -> m (a cos - b sin, b cos + a sin), the angle position * frequency.  A value is read and written once: bound by
// bytes, a single token by its chain of reads (position, angle, result).  A lane has P pairs of a head, the two halves of a pair in one register file: 16 bytes of a from the first half
// and 16 of b from the second (or 32 bytes in one piece where neighbours are pairs), so that neither the norm (a sum over the lanes of a head) nor the rotation needs shared memory.
// The angles are a row's, not a head's: a CTA has some rows and reduces each of their angles once, the float64 product without a further loss (131072 radians in float32 are 0.008 off), to half turns in [-1, 1], whose sine
// and cosine in float32 all heads share; a warp then has the same heads of all of these rows, their weights in registers and the next rows' values under way.
// 2048 rows of 32 and 8 heads of 128, bfloat16 with norms: 8.7 us one after the other (42 MB, 4.8 TB/s), a row 2.5 us (launch and chain); a warp for a row and its angles 17, a CTA for a row 22.
// What is left is latency: twenty warps an SM (96 registers a thread), each with a chain of 265 instructions for four heads of a row, a third of them conversions and pairs of registers, keep
// the issue slots half busy.
#include <algorithm>

#include "dependent_launch.cuh"
#include "kv_cache.cuh"

namespace b200gguf {
namespace stream { int sm_count(); }             // gemv_stream.cu
namespace rope {

constexpr int kWarps = 10, kMaxDim = 512, kTile = 8;      // rows whose angles are in shared memory

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
  int rows, pairs, head_dim, lanes_log2, units, turned;
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

// Two float32 values that one instruction works on.
using Duo = unsigned long long;
__device__ __forceinline__ Duo duo(float x, float y) {
  Duo d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(x), "f"(y));
  return d;
}
__device__ __forceinline__ float2 of_duo(Duo d) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(d));
  return f;
}
__device__ __forceinline__ Duo mul(Duo a, Duo b) {
  Duo d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ Duo fma(Duo a, Duo b, Duo c) {
  Duo d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
template <typename T> __device__ __forceinline__ Duo two_of(const T* p) { return duo(kv::to_float<T>(p[0]), kv::to_float<T>(p[1])); }
template <typename T> __device__ __forceinline__ void put_two(T* to, Duo d);
template <> __device__ __forceinline__ void put_two<float>(float* to, Duo d) {
  const float2 f = of_duo(d);
  to[0] = f.x;
  to[1] = f.y;
}
template <> __device__ __forceinline__ void put_two<__half>(__half* to, Duo d) {
  const __half2 t = __float22half2_rn(of_duo(d));
  to[0] = t.x;
  to[1] = t.y;
}
template <> __device__ __forceinline__ void put_two<__nv_bfloat16>(__nv_bfloat16* to, Duo d) {
  const __nv_bfloat162 t = __float22bfloat162_rn(of_duo(d));
  to[0] = t.x;
  to[1] = t.y;
}

// Rows whose reads are under way: of wide accesses as many as cover the memory's latency (44 KB an SM at the measured bandwidth), else the one at hand.
template <typename T, int P, int N, bool WIDE> constexpr int ahead() { return WIDE && P * int(sizeof(T)) >= 8 ? (N == 1 ? 4 : 2) : 0; }
template <typename T, int P> __device__ __forceinline__ void copy_async(Piece<T, P>* to, const T* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;\n" ::"r"(uint32_t(__cvta_generic_to_shared(to))), "l"(from), "n"(P * sizeof(T)) : "memory");
}

// P: pairs of a unit (a lane's share of a head); N: units of a lane; a head has 2^lanes_log2 lanes.  A pass is 32 / lanes heads of q or of k.
template <typename T, int P, int N, bool WIDE, bool NEXT, bool PART>
__global__ void __launch_bounds__(32 * kWarps, N == 1 && WIDE ? 2 : 1) rotary_kernel(const __grid_constant__ Args g) {
  // Cosine and sine of the rows' angles, times the magnitude, as the twos that they are multiplied with lie: neighbours of a half beside each other, or each pair's (cos, cos, -sin, sin).
  // (These by their place in a unit, then by units: neighbouring lanes read neighbouring ones; a unit's beside one another were 24.9 us for 2048 rows, not 9.)
  constexpr bool PAIRS = NEXT || P == 1;
  constexpr int kUnits = kMaxDim / 2 / P;
  __shared__ __align__(16) float turns[kTile][(PAIRS ? 4 : 2) * (kMaxDim / 2)];
  __shared__ int place[kTile];
  // A lane's own values of the next rows: it copies and reads them itself, so that nobody waits for it.
  constexpr int AHEAD = ahead<T, P, N, WIDE>();
  extern __shared__ __align__(16) uint8_t raw[];
  Piece<T, P>* const ring = reinterpret_cast<Piece<T, P>*>(raw) + (threadIdx.x >> 5) * (AHEAD * 2 * N * 32) + (threadIdx.x & 31);      // [row][2 N][32 lanes] of the warp
  using Two = Piece<T, P>;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  const int begin = int(int64_t(g.rows) * blockIdx.x / gridDim.x), end = int(int64_t(g.rows) * (blockIdx.x + 1) / gridDim.x);
  const int lanes = 1 << g.lanes_log2, per_pass = 32 >> g.lanes_log2;
  const int at = lane & (lanes - 1), sub = lane >> g.lanes_log2;
  const int q_passes = (g.q.heads + per_pass - 1) / per_pass, passes = q_passes + (g.k.heads + per_pass - 1) / per_pass;
  const float inverse = 1.f / float(g.head_dim);

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
  // A unit's 2 P values are P twos: neighbours of a, then of b, or where neighbours are pairs (and with P = 1) a pair each.
  wait_for_launch_before();

  for (int tile = begin; tile < end; tile += kTile) {
    const int rows = min(kTile, end - tile);
    for (int pass = warp; pass < passes; pass += warps) {  // (there are no more warps than passes)
      const bool k = pass >= q_passes;
      const Side& s = k ? g.k : g.q;
      const int head = (k ? pass - q_passes : pass) * per_pass + sub;
      bool live[N];
#pragma unroll
      for (int n = 0; n < N; ++n) live[n] = in[n] && head < s.heads;
      const T* from = static_cast<const T*>(s.x) + tile * s.row_stride + head * s.head_stride;
      T* to = static_cast<T*>(s.out) + tile * s.out_row_stride + head * s.out_head_stride;
      // turns of the lane's first unit
      const Duo* turn[N];
#pragma unroll
      for (int n = 0; n < N; ++n) turn[n] = reinterpret_cast<const Duo*>(&turns[0][0]) + (PAIRS ? 2 : P / 2) * (in[n] && at + n * lanes < g.turned ? at + n * lanes : 0);
      const int64_t row_stride = s.row_stride, out_row_stride = s.out_row_stride;
      int asked = 0;                                       // rows whose reads are under way or done
      auto ask = [&] {
        if (asked < rows) {
#pragma unroll
          for (int n = 0; n < N; ++n) {
            if (!live[n]) continue;
            copy_async(ring + (asked % AHEAD * 2 * N + 2 * n) * 32, from + a[n]);
            copy_async(ring + (asked % AHEAD * 2 * N + 2 * n + 1) * 32, from + b[n]);
          }
          from += row_stride;
        }
        asm volatile("cp.async.commit_group;\n" ::: "memory");
        ++asked;
      };
      Two xa[N], xb[N];
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int j = 0; j < P; ++j) xa[n].v[j] = xb[n].v[j] = kv::from_float<T>(0.f);      // lanes without a unit add nothing to a sum
      if constexpr (AHEAD > 0) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) ask();
      }
      const bool normed = s.weight != nullptr;
      Duo w[N][P];                                         // weights, as the values lie
#pragma unroll
      for (int n = 0; n < N; ++n) {
        auto read = [&](auto type) {
          using W = decltype(type);
          Piece<W, P> pa, pb;
          get<WIDE>(pa, static_cast<const W*>(s.weight) + a[n]);
          get<WIDE>(pb, static_cast<const W*>(s.weight) + b[n]);
          if constexpr (P == 1) {
            w[n][0] = duo(kv::to_float<W>(pa.v[0]), kv::to_float<W>(pb.v[0]));
          } else {
#pragma unroll
            for (int j = 0; j < P; ++j) w[n][j] = two_of(j < P / 2 ? pa.v + 2 * j : pb.v + 2 * j - P);
          }
        };
        if (normed && in[n]) {
          if (g.weight_f32) read(float{}); else read(T{});
        }
      }
      if (pass == warp) {                                  // (every warp comes here once a tile)
        if (tile != begin) __syncthreads();                // (the angles before are used)
        const int pieces = (g.pairs + 31) >> 5;
        for (int i = warp; i < rows * pieces; i += warps) {
          const int r = i / pieces, p = (i - r * pieces) * 32 + lane;
          const int position = g.positions[tile + r];
          if (p == 0) place[r] = position;
          if (p >= g.pairs) continue;
          // Turns by 1 / (2 pi) in two parts and the product's rounding: of an angle of 2^31 the turns alone would be 2^-22 off.  Then half turns in [-1, 1], in two floats: the second is a
          // rounding's rest, by which sine and cosine are moved to first order.  (A product that is not fused into the difference: its rounding is what `rest` has.)
          const double angle = double(position) * g.frequencies[p], all = __dmul_rn(angle, 0.15915494309189533577), rest = ::fma(angle, -9.839338337591243e-18, ::fma(angle, 0.15915494309189533577, -all));
          const double part = 2. * (all - rint(all) + rest);
          const float high = float(part), low = float(part - double(high)) * 3.14159265358979f;
          float sin, cos;
          sincospif(high, &sin, &cos);
          const float c = g.magnitude * fmaf(-sin, low, cos), d = g.magnitude * fmaf(cos, low, sin);
          if constexpr (PAIRS) {
            *reinterpret_cast<float4*>(&turns[r][4 * (p % P * kUnits + p / P)]) = make_float4(c, c, -d, d);
          } else {
            turns[r][p] = c;
            turns[r][kMaxDim / 2 + p] = d;
          }
        }
        if (g.pairs == 0 && int(threadIdx.x) < rows) place[threadIdx.x] = g.positions[tile + threadIdx.x];
        __syncthreads();
      }
#pragma unroll 1
      for (int r = 0; r < rows; ++r, to += out_row_stride) {
        if constexpr (AHEAD > 0) {
          asm volatile("cp.async.wait_group %0;\n" ::"n"(AHEAD - 1) : "memory");
#pragma unroll
          for (int n = 0; n < N; ++n) {
            if (!live[n]) continue;
            xa[n] = ring[(r % AHEAD * 2 * N + 2 * n) * 32];
            xb[n] = ring[(r % AHEAD * 2 * N + 2 * n + 1) * 32];
          }
        } else {
#pragma unroll
          for (int n = 0; n < N; ++n) {
            if (!live[n]) continue;
            get<WIDE>(xa[n], from + a[n]);
            get<WIDE>(xb[n], from + b[n]);
          }
          from += row_stride;
        }
        Duo v[N][P];
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
          for (int j = 0; j < P; ++j) {
            if constexpr (P == 1) v[n][j] = duo(kv::to_float<T>(xa[n].v[0]), kv::to_float<T>(xb[n].v[0]));
            else v[n][j] = two_of(j < P / 2 ? xa[n].v + 2 * j : xb[n].v + 2 * j - P);
          }
        if constexpr (AHEAD > 0) ask();                    // (into the place that has just been read)
        if (place[r] < 0) {                                // nobody's
          if (s.in_place) continue;
          Two zero;
#pragma unroll
          for (int j = 0; j < P; ++j) zero.v[j] = kv::from_float<T>(0.f);
#pragma unroll
          for (int n = 0; n < N; ++n) {
            if (!live[n]) continue;
            put<WIDE>(to + a[n], zero);
            put<WIDE>(to + b[n], zero);
          }
          continue;
        }
        if (normed) {
          Duo two = 0;
#pragma unroll
          for (int n = 0; n < N; ++n)
#pragma unroll
            for (int j = 0; j < P; ++j) two = fma(v[n][j], v[n][j], two);
          float sum = of_duo(two).x + of_duo(two).y;
#pragma unroll
          for (int o = 16; o > 0; o >>= 1)
            if (o < lanes) sum += __shfl_xor_sync(0xffffffffu, sum, o);
          const float scale = rsqrtf(fmaf(sum, inverse, g.eps));
          const Duo by = duo(scale, scale);
#pragma unroll
          for (int n = 0; n < N; ++n)
#pragma unroll
            for (int j = 0; j < P; ++j) v[n][j] = mul(v[n][j], mul(w[n][j], by));
        }
#pragma unroll
        for (int n = 0; n < N; ++n) {
          Two oa, ob;
          const int u = at + n * lanes;
          const bool stays = PART && u >= g.turned;
          const Duo* t = turn[n] + r * ((PAIRS ? 2 : 1) * (kMaxDim / 2));
#pragma unroll
          for (int j = 0; j < P; ++j) {
            Duo z;
            if constexpr (PAIRS) {                         // (x cos - y sin, y cos + x sin)
              const float2 f = of_duo(v[n][j]);
              z = fma(v[n][j], t[2 * j * kUnits], mul(duo(f.y, f.x), t[2 * j * kUnits + 1]));
            } else {
              const int p = j % (P / 2);
              const Duo sine = t[kMaxDim / 4 + p];
              z = fma(v[n][j], t[p], j < P / 2 ? mul(v[n][j + P / 2], sine ^ 0x8000000080000000ull) : mul(v[n][j - P / 2], sine));
            }
            if (stays) z = v[n][j];                        // (an infinity beside it does not reach a value that stays)
            if constexpr (P == 1) {
              oa.v[0] = kv::from_float<T>(of_duo(z).x);
              ob.v[0] = kv::from_float<T>(of_duo(z).y);
            } else {
              put_two<T>(j < P / 2 ? oa.v + 2 * j : ob.v + 2 * j - P, z);
            }
          }
          if (live[n]) {
            put<WIDE>(to + a[n], oa);
            put<WIDE>(to + b[n], ob);
          }
        }
      }
    }
  }
}

template <typename T, int P, int N, bool WIDE, bool NEXT, bool PART> static int launch(Args g, cudaStream_t s) {
  const int sms = stream::sm_count();
  if (sms <= 0) return RC_LAUNCH;
  g.units = g.head_dim / (2 * P);
  g.turned = g.pairs / P;
  g.lanes_log2 = 0;
  while (g.lanes_log2 < 5 && (1 << g.lanes_log2) * N < g.units) ++g.lanes_log2;
  const int per_pass = 32 >> g.lanes_log2, passes = (g.q.heads + per_pass - 1) / per_pass + (g.k.heads + per_pass - 1) / per_pass;
  const int warps = (passes + (passes + kWarps - 1) / kWarps - 1) / ((passes + kWarps - 1) / kWarps);      // as few as take the passes in the same number of turns
  const size_t shared = size_t(ahead<T, P, N, WIDE>()) * 2 * N * warps * 32 * P * sizeof(T);
  auto kernel = rotary_kernel<T, P, N, WIDE, NEXT, PART>;
  static std::atomic<uint64_t> done{0};
  if (int rc = allow_shared(kernel, size_t(ahead<T, P, N, WIDE>()) * 2 * N * kWarps * 32 * P * sizeof(T), done)) return rc;
  return launch_dependent(kernel, dim3(unsigned(std::min(g.rows, 2 * sms * std::max(1, kWarps / warps)))), 32 * warps, shared, 1, s, g);
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
    g.rows = rows;
    g.pairs = pairs;
    g.head_dim = head_dim;
    g.eps = eps;
    g.magnitude = magnitude;
    g.weight_f32 = weight_dtype == DINO_F32;
    auto whole = [&](int p) { return pairs % p == 0 && (head_dim - 2 * pairs) % (2 * p) == 0; };      // units of p pairs
    auto wide = [&](int p) { return (every & (p * sizeof(T) - 1)) == 0 && (weights & (p * (g.weight_f32 ? 4 : sizeof(T)) - 1)) == 0; };
    auto go = [&](auto p, auto n) {
      constexpr int P = decltype(p)::value, N = decltype(n)::value;
      auto next = [&](auto w, auto x) {
        constexpr bool W = decltype(w)::value, X = decltype(x)::value;
        return 2 * pairs < head_dim ? launch<T, P, N, W, X, true>(g, s) : launch<T, P, N, W, X, false>(g, s);
      };
      using std::bool_constant;
      if (P > 1 && !wide(P)) return interleaved ? next(bool_constant<P == 1>{}, bool_constant<true>{}) : next(bool_constant<P == 1>{}, bool_constant<false>{});
      return interleaved ? next(bool_constant<true>{}, bool_constant<true>{}) : next(bool_constant<true>{}, bool_constant<false>{});
    };
    using std::integral_constant;
    // As many pairs a lane as 16 bytes hold of each side, where the head and its turned part are whole units of them.  2048 rows of 40 heads of 128 in 16 bits: eight pairs 8.8 us, four 11.0, one 13.2;
    // eight pairs at addresses that are no multiples of 16 bytes 19.8.
    if constexpr (sizeof(T) == 2) {
      if (whole(8)) return go(integral_constant<int, 8>{}, integral_constant<int, 1>{});
    }
    if (whole(4) && head_dim <= 256) return go(integral_constant<int, 4>{}, integral_constant<int, 1>{});
    if (whole(4)) return go(integral_constant<int, 4>{}, integral_constant<int, 2>{});
    return go(integral_constant<int, 1>{}, integral_constant<int, 8>{});
  });
}

}  // namespace b200gguf

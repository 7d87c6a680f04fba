// The next token of every row of logits from one given random number: temperature, top-k, top-p, min-p (include/dinoml_b200_decoder.h has the definition).
//
// Every filter keeps a beginning of one order - by value, the lowest index first among equals - and the choice is where the running sum of the weights in that order passes u times
// the sum of the kept.  So a row is never sorted: what is wanted is a few places of the order, each found from sums over ranges of values.
//
// 16-bit logits have 65536 values, so that how often each is there says everything but the indices: a row is read once, into counts (a CTA's part of the row into 128 KB of its
// shared memory, two 16-bit counts a word).  The weight of a value is computed once, in float64, and only where its count is not zero: a row of 128256 has some thousand different
// values.  Sums over groups of 32 values, their running sums, and then each place by one warp: the group, the value in it, how many of its equals.  At the end the part of the row
// that has the chosen one among its equals is searched for it.
// float32 logits: ranges of values instead of values.  2048 ranges of equal width in (largest - x) / temperature, whose counts and sums of weights (whole numbers of a unit of the
// range) all CTAs add up; running sums over the ranges are float64, in one order; each place is then narrowed down by the bits of the values in its range until one value is left, by the
// first CTA alone where these are few.
//
// A row is a cluster's, of up to eight CTAs while there are fewer rows than SMs: its CTAs have parts of it, the first one finds the places.  Bound by latency there: one row of 128256 bfloat16
// with top-k and top-p 14.0 us, 12 of them behind the launch: counting 1.4, bitmaps and the first meeting 1.8, reads of one another's counts 2.0, powers and sums 0.7, the second meeting, which
// waits for the slowest CTA, 2.0, running sums 0.9, places 2.6, the last meeting 0.5, the rest the search.  Seven rows of 50001 float32 16.2 us; 64 rows of
// 128256 with settings of their own 21.7 us.  256 rows of 128256 float16 51 us (66 MB, 1.3 TB/s), two rows a CTA: of 25 us a row counting takes 12 (its atomics meet on random banks, 3.5
// wavefronts for 32), the sums 5, the places 2, the search 4.
#include <cooperative_groups.h>

#include <algorithm>

#include "dependent_launch.cuh"
#include "kv_cache.cuh"
#include "sample_clusters.h"

namespace b200gguf {
namespace stream { int sm_count(); }             // gemv_stream.cu
namespace choice {
namespace cg = cooperative_groups;

constexpr int kThreads = 512, kWarps = kThreads / 32, kGroups = 2048, kMaxVocabulary = 262144;
constexpr int kPart32 = 32768;                   // of a row, at most

struct Args {
  const void* logits;
  int64_t row_stride, rows;
  int vocabulary;
  const float* uniforms;
  DinoB200SampleSettings set;
  int* tokens;
  float* probabilities;
  int* status;
};

struct Row {
  float temperature, top_p, min_p, u;
  int top_k;
  bool valid, first;                             // settings are numbers; the first of the order is the answer
};
__device__ __forceinline__ Row row_of(const Args& a, int64_t row) {
  Row r;
  r.temperature = a.set.temperature != nullptr ? a.set.temperature[row] : a.set.temperature_all;
  r.top_k = a.set.top_k != nullptr ? a.set.top_k[row] : a.set.top_k_all;
  r.top_p = a.set.top_p != nullptr ? a.set.top_p[row] : a.set.top_p_all;
  r.min_p = a.set.min_p != nullptr ? a.set.min_p[row] : a.set.min_p_all;
  r.u = a.uniforms[row];
  r.valid = r.temperature >= 0.f && r.top_p == r.top_p && r.min_p == r.min_p && r.u == r.u;
  r.u = fminf(fmaxf(r.u, 0.f), 0x1.fffffep-1f);
  r.first = r.temperature == 0.f || r.top_k == 1 || r.top_p <= 0.f || r.min_p > 1.f;
  return r;
}

// Order of values as unsigned numbers, the largest value first; NaN before inf and behind -inf.
template <typename T> struct Code;
template <> struct Code<__nv_bfloat16> {
  static constexpr uint32_t kInf = 0x007f, kMinusInf = 0xff80;
  static constexpr int kMantissa = 7;
  static __device__ __forceinline__ float spacing(int binade) { return ldexpf(1.f, max(binade, 1) - 134); }
  static __device__ __forceinline__ float value(uint32_t d) { return __uint_as_float(((d & 0x8000u) ? d : d ^ 0x7fffu) << 16); }
};
template <> struct Code<__half> {
  static constexpr uint32_t kInf = 0x03ff, kMinusInf = 0xfc00;
  static constexpr int kMantissa = 10;
  static __device__ __forceinline__ float spacing(int binade) { return ldexpf(1.f, max(binade, 1) - 25); }
  static __device__ __forceinline__ float value(uint32_t d) { return __half2float(__ushort_as_half(uint16_t((d & 0x8000u) ? d : d ^ 0x7fffu))); }
};
template <> struct Code<float> {
  static constexpr uint32_t kInf = 0x007fffff, kMinusInf = 0xff800000;
  static __device__ __forceinline__ float value(uint32_t d) { return __uint_as_float((d & 0x80000000u) ? d : d ^ 0x7fffffffu); }
  static __device__ __forceinline__ uint32_t of(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);           // (-0 becomes 0)
    return (b & 0x80000000u) ? b : b ^ 0x7fffffffu;
  }
};
// Two values at once.  -0, code 0x8000, comes right behind 0.
constexpr uint32_t kZero = 0x7fff, kMinusZero = 0x8000;
__device__ __forceinline__ uint32_t codes_of(uint32_t w) { return w ^ (((~w >> 15) & 0x00010001u) * 0x7fffu); }

template <typename T> struct Weight {
  uint32_t first;                                // the largest value's code
  double largest, inverse;
  bool infinite;
  __device__ __forceinline__ Weight(uint32_t first, float temperature)
      : first(first), largest(double(Code<T>::value(first))), inverse(1. / double(temperature)), infinite(first == Code<T>::kInf) {}
  __device__ __forceinline__ double operator()(uint32_t d) const {
    return d == first ? 1. : infinite ? 0. : exp((double(Code<T>::value(d)) - largest) * inverse);
  }
};

// The last code in [low, high] with holds(code), which holds for low and up to some code: by a converged warp.
template <typename F> __device__ __forceinline__ uint32_t last_that(uint32_t low, uint32_t high, F holds) {
  const uint32_t lane = threadIdx.x & 31;
  uint64_t span = uint64_t(high) - low + 1;
  while (span > 1) {
    const uint64_t step = (span + 31) >> 5, at = lane * step;
    const bool in = at < span && (lane == 0 || holds(uint32_t(low + at)));
    const int hits = __popc(__ballot_sync(0xffffffffu, in));
    low += uint32_t((hits - 1) * step);
    span = min(step, span - (hits - 1) * step);
  }
  return low;
}

// The first of 2048 running sums that passes: by a converged warp; the last one if none does.
template <typename F> __device__ __forceinline__ int first_of(F passes) {
  const int lane = threadIdx.x & 31;
  uint32_t hit = __ballot_sync(0xffffffffu, passes(lane * 64 + 63));
  if (hit == 0) return kGroups - 1;
  const int at = (__ffs(hit) - 1) * 64;
  hit = __ballot_sync(0xffffffffu, passes(at + 2 * lane + 1));
  const int pair = at + 2 * (__ffs(hit) - 1);
  return passes(pair) ? pair : pair + 1;
}

template <typename V> __device__ __forceinline__ V warp_running(V v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  return v;
}

// Running sums of 2048 counts and masses in place, by all threads.
template <int NT, typename M> __device__ __forceinline__ void running_sums(uint32_t* count, M* mass, uint32_t* warp_count, M* warp_mass) {
  constexpr int N = kGroups / NT;
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  uint32_t c[N];
  M m[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    c[i] = count[N * t + i];
    m[i] = mass[N * t + i];
    if (i > 0) {
      c[i] += c[i - 1];
      m[i] += m[i - 1];
    }
  }
  const uint32_t all_c = warp_running(c[N - 1]);
  const M all_m = warp_running(m[N - 1]);
  if (lane == 31) {
    warp_count[warp] = all_c;
    warp_mass[warp] = all_m;
  }
  __syncthreads();
  const uint32_t wc = warp_running(lane < NT / 32 ? warp_count[lane] : 0u);
  const M wm = warp_running(lane < NT / 32 ? warp_mass[lane] : M(0));
  uint32_t base_c = __shfl_sync(0xffffffffu, wc, (warp + 31) & 31);
  M base_m = __shfl_sync(0xffffffffu, wm, (warp + 31) & 31);
  if (warp == 0) {
    base_c = 0;
    base_m = M(0);
  }
  // (as a difference the own part would lose what a small group adds to a large sum)
  const uint32_t up_c = __shfl_up_sync(0xffffffffu, all_c, 1);
  const M up_m = __shfl_up_sync(0xffffffffu, all_m, 1);
  base_c += lane > 0 ? up_c : 0u;
  base_m += lane > 0 ? up_m : M(0);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    count[N * t + i] = base_c + c[i];
    mass[N * t + i] = base_m + m[i];
  }
  __syncthreads();
}

__device__ __forceinline__ void answer(const Args& a, int64_t row, int token, float probability) {
  a.tokens[row] = token;
  if (a.probabilities != nullptr) a.probabilities[row] = probability;
}

// ---- 16-bit logits ------------------------------------------------------------------------------------------------------------------------------------
// A row that is one CTA's is counted in turns of kTurn vectors of eight, behind which the counts that could pass 65535 in the next turn are set aside; parts of a row have no more values.
constexpr int kPart16 = 65528, kTurn = 6144, kAside = 65535 - 8 * kTurn - 16, kMostAside = kMaxVocabulary / (kAside + 1) + 2;

struct Decision {
  int owner, place;
  uint32_t code;
};
struct Shared16 {
  uint32_t counts[32768];                        // word d & 0x7fff: of code d in its upper half if d >= 0x8000, else in its lower half
  double mass[kGroups];                          // of groups of 32 codes, then running; the first CTA's
  uint32_t count[kGroups];
  double power[32][32];                      // of a binade: the weights of a group's values relative to its first one's
  double warp_mass[32];
  uint32_t warp_count[32];
  uint32_t least, most;                          // codes of this part
  uint32_t all_least[8], all_most[8];            // of all parts
  uint32_t some[8][2][kGroups / 64];             // of all parts: which groups have anything
  uint32_t aside, aside_code[kMostAside], aside_count[kMostAside];
  Decision decision;
};

// What was set aside, added to its groups by all threads: few, and in the order of codes and counts, whoever came first.
template <typename T> __device__ __forceinline__ void add_aside(Shared16& sh, const Weight<T>& weight) {
  const int tid = threadIdx.x, aside = int(sh.aside);
  uint32_t code = 0, count = 0, before = 0;
  if (tid < aside) {
    code = sh.aside_code[tid];
    count = sh.aside_count[tid];
    for (int i = 0; i < aside; ++i) {
      const uint32_t c = sh.aside_code[i], n = sh.aside_count[i];
      before += c < code || (c == code && (n < count || (n == count && i < tid))) ? 1u : 0u;
    }
  }
  __syncthreads();
  if (tid < aside) {
    sh.aside_code[before] = code;
    sh.aside_count[before] = count;
  }
  __syncthreads();
  if (tid == 0) {
    for (int i = 0; i < aside; ++i) {
      const uint32_t d = sh.aside_code[i];
      if (d < weight.first || d >= Code<T>::kMinusInf) continue;
      sh.count[d >> 5] += sh.aside_count[i];
      sh.mass[d >> 5] += double(sh.aside_count[i]) * weight(d);
    }
  }
  __syncthreads();
}

template <typename T, int ctas, int kThreads>
__global__ void __launch_bounds__(kThreads, 1) sample16_kernel(Args a) {
  constexpr int kWarps = kThreads / 32;
  extern __shared__ __align__(16) uint8_t raw[];
  Shared16& sh = *reinterpret_cast<Shared16*>(raw);
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = ctas > 1 ? int(cluster.block_rank()) : 0;
  auto meet = [&] {
    if (ctas > 1) cluster.sync(); else __syncthreads();
  };
  auto of_rank = [&](auto* p, int r) {           // p of another CTA
    if constexpr (ctas > 1) return cluster.map_shared_rank(p, r); else return p;
  };
  const int part = ((a.vocabulary + ctas - 1) / ctas + 7) & ~7;
  const int begin = min(rank * part, a.vocabulary), length = min(part, a.vocabulary - begin);
  bool waited = false;
  for (int64_t row = blockIdx.x / ctas, step = gridDim.x / ctas; row < a.rows; row += step) {
    for (int i = tid; i < 32768 / 4; i += kThreads) reinterpret_cast<uint4*>(sh.counts)[i] = make_uint4(0, 0, 0, 0);
    if (rank == 0) {
      for (int i = tid; i < kGroups; i += kThreads) {
        sh.mass[i] = 0.;
        sh.count[i] = 0;
      }
    }
    if (tid == 0) {
      sh.least = 0xffffu;
      sh.most = 0;
      sh.aside = 0;
    }
    if (!waited) wait_for_launch_before();
    waited = true;
    __syncthreads();
    const Row set = row_of(a, row);

    // This part of the row: values up to an address that is a multiple of 16, vectors of eight, the rest.
    const uint16_t* x = static_cast<const uint16_t*>(a.logits) + row * a.row_stride + begin;
    const int head = min(int((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / 2, length);
    const int vectors = (length - head) / 8, rest = length - head - 8 * vectors;
    const uint4* wide = reinterpret_cast<const uint4*>(x + head);
    uint32_t least = 0xffffffffu, most = 0;
    auto add = [&](uint32_t two) {
      uint32_t minus;                            // ffff where a half is negative
      asm("prmt.b32 %0, %1, 0, 0xbb99;" : "=r"(minus) : "r"(two));
      const uint32_t d = two ^ (~minus & 0x7fff7fffu);
      if (ctas > 1) {
        least = __vminu2(least, d);
        most = __vmaxu2(most, d);
      }
      // 1 in the lower half of a positive value's word, in the upper one of a negative's
      atomicAdd(&sh.counts[d & 0x7fffu], (minus & 0xffffu) + 1u);
      atomicAdd(&sh.counts[d >> 16 & 0x7fffu], (minus >> 16) + 1u);
    };
    auto add_one = [&](uint32_t v) {
      const uint32_t d = codes_of(v) & 0xffffu;
      if (ctas > 1) {
        least = __vminu2(least, d | d << 16);
        most = __vmaxu2(most, d | d << 16);
      }
      atomicAdd(&sh.counts[d & 0x7fffu], (d & 0x8000u) ? 0x10000u : 1u);
    };
    // A step is a vector of every thread; a thread has kAhead of them on their way, those of the next turn too while the counts are looked through.
    constexpr int kSteps = kTurn / kThreads, kAhead = kThreads == 1024 ? 2 : 6;
    static_assert(kSteps % kAhead == 0, "");
    const int turns = ctas > 1 ? 1 : max(1, (vectors + kTurn - 1) / kTurn);
    const uint4* next = wide + tid;
    uint4 q[kAhead];
    auto use = [&](const uint4& v) {
      add(v.x);
      add(v.y);
      add(v.z);
      add(v.w);
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (tid + i * kThreads < vectors) q[i] = kv::fetch(next + i * kThreads);
    int turn_left = kSteps, left = vectors - tid;      // steps of this turn; vectors at and behind the thread's next one
    for (int all = vectors; all > 0; all -= kAhead * kThreads) {
      next += kAhead * kThreads;
      if (all >= 2 * kAhead * kThreads) {        // (everyone has all of these and of the next ones)
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          use(q[i]);
          q[i] = kv::fetch(next + i * kThreads);
        }
      } else {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
          if (left > i * kThreads) use(q[i]);
          if (left > (i + kAhead) * kThreads) q[i] = kv::fetch(next + i * kThreads);
        }
      }
      left -= kAhead * kThreads;
      turn_left -= kAhead;
      if (ctas == 1 && turn_left == 0 && all > kAhead * kThreads) {
        turn_left = kSteps;
        __syncthreads();
        for (int i = tid; i < 32768 / 4; i += kThreads) {
          const uint4 q = reinterpret_cast<const uint4*>(sh.counts)[i];
          const uint32_t top = __vmaxu2(__vmaxu2(q.x, q.y), __vmaxu2(q.z, q.w));
          if (max(top & 0xffffu, top >> 16) <= uint32_t(kAside)) continue;
          for (int j = 0; j < 8; ++j) {
            const uint32_t w = sh.counts[4 * i + j / 2], n = j & 1 ? w >> 16 : w & 0xffffu, d = uint32_t(4 * i + j / 2) + (j & 1) * 0x8000u;
            if (n <= uint32_t(kAside)) continue;
            const uint32_t at = atomicAdd(&sh.aside, 1u);
            sh.aside_code[at] = d == kMinusZero ? kZero : d;
            sh.aside_count[at] = n;
            sh.counts[4 * i + j / 2] = w - (j & 1 ? n << 16 : n);
          }
        }
        __syncthreads();
      }
    }
    if (tid < head) add_one(x[tid]);
    if (tid < rest) add_one(x[head + 8 * vectors + tid]);
    if (tid == 0 && row + step < a.rows) {       // the next row's part, while this one is worked on
      const uint16_t* ahead = x + step * a.row_stride;
      const int skip = min(int((16 - (reinterpret_cast<uintptr_t>(ahead) & 15)) & 15) / 2, length), bytes = (length - skip) / 8 * 16;
      if (bytes > 0) asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;\n" ::"l"(ahead + skip), "r"(bytes) : "memory");
    }
    least = __reduce_min_sync(0xffffffffu, min(least & 0xffffu, least >> 16));
    most = __reduce_max_sync(0xffffffffu, max(most & 0xffffu, most >> 16));
    if (ctas > 1 && lane == 0) {
      atomicMin(&sh.least, least == kMinusZero ? kZero : least);
      atomicMax(&sh.most, most);
    }
    __syncthreads();
    if (tid == 0) {                              // -0 is 0
      const uint32_t minus = sh.counts[kMinusZero & 0x7fffu] >> 16;
      if (minus > 0) {
        sh.counts[kMinusZero & 0x7fffu] -= minus << 16;
        if (turns == 1) {
          sh.counts[kZero] += minus;
        } else {
          sh.aside_code[sh.aside] = kZero;
          sh.aside_count[sh.aside++] = minus;
        }
      }
    }
    __syncthreads();
    // Which groups have anything here, told to all: the others read no more of this part than that.
    for (int block = warp; block < 32; block += kWarps) {
      uint32_t any = 0;                          // a lane has a group of 32 words
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint4 q = reinterpret_cast<const uint4*>(sh.counts)[(block * 32 + lane) * 8 + ((i + lane) & 7)];
        any |= q.x | q.y | q.z | q.w;
      }
      const uint32_t low = __ballot_sync(0xffffffffu, (any & 0xffffu) != 0), high = __ballot_sync(0xffffffffu, (any >> 16) != 0);
      if (lane < ctas) {
        Shared16* other = of_rank(&sh, lane);
        other->some[rank][0][block] = low;
        other->some[rank][1][block] = high;
      }
    }
    if constexpr (ctas > 1) {
      if (tid < ctas) {
        Shared16* other = of_rank(&sh, tid);
        other->all_least[rank] = sh.least;
        other->all_most[rank] = sh.most;
      }
      cluster.sync();
      least = __reduce_min_sync(0xffffffffu, lane < ctas ? sh.all_least[lane] : 0xffffu);
      most = __reduce_max_sync(0xffffffffu, lane < ctas ? sh.all_most[lane] : 0u);
    } else {
      __syncthreads();
      // The first and the last code that is there, what was set aside among them.
      least = 0xffffu;
      most = 0;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t word = sh.some[0][half][lane], there = __ballot_sync(0xffffffffu, word != 0);
        if (there == 0) continue;
        const uint32_t from = __shfl_sync(0xffffffffu, uint32_t(__ffs(word) - 1), __ffs(there) - 1) + 32 * (__ffs(there) - 1);
        const uint32_t to = __shfl_sync(0xffffffffu, uint32_t(31 - __clz(word)), 31 - __clz(there)) + 32 * (31 - __clz(there));
        const uint32_t in_from = __ballot_sync(0xffffffffu, (sh.counts[from * 32 + lane] >> (16 * half) & 0xffffu) != 0);
        const uint32_t in_to = __ballot_sync(0xffffffffu, (sh.counts[to * 32 + lane] >> (16 * half) & 0xffffu) != 0);
        least = min(least, half * 0x8000u + from * 32 + __ffs(in_from) - 1);
        most = max(most, half * 0x8000u + to * 32 + 31 - __clz(in_to));
      }
      for (uint32_t i = 0; i < sh.aside; ++i) {
        least = min(least, sh.aside_code[i]);
        most = max(most, sh.aside_code[i]);
      }
    }

    const uint32_t first = least;
    if (!set.valid || first < Code<T>::kInf || most > Code<T>::kMinusInf || first >= Code<T>::kMinusInf) {
      if (rank == 0 && tid == 0) {
        if (!set.valid) kv::flag_range(a.status);
        answer(a, row, -1, 0.f);
      }
      meet();                                    // (others may be reading what the next row begins with)
      continue;
    }
    const Weight<T> weight(first, set.temperature);
    if (!set.first) {
      Shared16* lead = of_rank(&sh, 0);
      // Blocks of 32 groups are a CTA's each, in turn: it adds the other parts' counts to its own.  What passes 65535 is set aside.
      if constexpr (ctas > 1) {
        static_assert(ctas == 1 || kWarps == 16, "groups w and w + 16 of a block are warp w's");
        for (int block = rank; block < 32; block += ctas) {
          uint32_t from[2] = {0, 0}, w[2][ctas];
#pragma unroll
          for (int r = 0; r < ctas; ++r) {
            const uint32_t there = (sh.some[r][0][block] | sh.some[r][1][block]) >> warp;
            from[0] |= (there & 1) << r;
            from[1] |= (there >> 16 & 1) << r;
          }
          if (((from[0] | from[1]) & ~(1u << rank)) == 0) continue;
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < ctas; ++r) {     // (all on their way before the first is used)
              w[i][r] = 0;
              if (from[i] >> r & 1) w[i][r] = of_rank(sh.counts, r)[(block * 32 + warp + 16 * i) * 32 + lane];
            }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int at = (block * 32 + warp + 16 * i) * 32 + lane;
            uint32_t low = 0, high = 0;
#pragma unroll
            for (int r = 0; r < ctas; ++r) {
              low += w[i][r] & 0xffffu;
              high += w[i][r] >> 16;
            }
            if ((from[i] & ~(1u << rank)) != 0) sh.counts[at] = min(low, 65535u) | min(high, 65535u) << 16;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const uint32_t n = half ? high : low;
              if (n <= 65535u) continue;
              const uint32_t place = atomicAdd(&lead->aside, 1u);
              lead->aside_code[place] = uint32_t(at) + half * 0x8000u;
              lead->aside_count[place] = n - 65535u;
            }
          }
        }
      }
      // Sums of groups of 32 values, a lane a group.  The values of a binade are equally far apart, so that the weights of a group are powers, w0 q^j, and q^j is the same for all groups of
      // a binade: a lane adds up its counts times these, from a place on where no other lane has its bank, and multiplies by w0 at the end.  So exponentials are few: 32 of powers, one
      // for a group.  The largest value's group is summed value by value, so that its weight is one.
      constexpr int kMantissa = Code<T>::kMantissa;
      // Powers of 32 binades: all of float16's; of bfloat16 those from the largest value's down 24 and up 7, where it is negative up 31.
      const int lowest = kMantissa == 10 ? 0 : max(0, first < 0x8000u ? int((0x7fffu - first) >> kMantissa) - 24 : int((first & 0x7fffu) >> kMantissa));
      auto group_weight = [&](uint32_t code0, double powers) {    // (before the largest value there is nothing)
        return powers > 0. && !weight.infinite ? powers * exp((double(Code<T>::value(code0)) - weight.largest) * weight.inverse) : 0.;
      };
      auto step_of = [&](int binade) { return -double(Code<T>::spacing(binade)) * weight.inverse; };
      for (int i = warp; i < 32; i += kWarps) sh.power[i][lane] = exp(step_of(lowest + i) * double(lane));
      __syncthreads();
      for (int task = warp; task < 64 / ctas; task += kWarps) {
        const uint32_t half = task & 1, block = uint32_t((task >> 1) * ctas + rank), group0 = block * 32, task0 = group0 * 32 + half * 0x8000u;
        uint32_t any = 0;
#pragma unroll
        for (int r = 0; r < ctas; ++r) any |= sh.some[r][half][block];
        if (any == 0 || task0 >= Code<T>::kMinusInf) continue;
        const uint32_t code0 = task0 + lane * 32;
        const int binade = int((half ? code0 & 0x7fffu : 0x7fffu - code0) >> kMantissa);
        const bool known = unsigned(binade - lowest) < 32u;
        const double* power = sh.power[known ? binade - lowest : 0];
        const uint32_t* counts = sh.counts + (group0 + lane) * 32;
        const uint32_t shift = half * 16;
        uint32_t n = 0;
        double mass = 0.;
        if (__any_sync(0xffffffffu, !known)) {             // (far from where the largest value is: bfloat16)
          for (int i = 0; i < 32; ++i) {
            const int j = (i + lane) & 31;
            const uint32_t c = counts[j] >> shift & 0xffffu;
            n += c;
            if (c != 0) mass = ::fma(double(c), exp(step_of(binade) * double(j)), mass);
          }
        } else {
#pragma unroll 8
          for (int i = 0; i < 32; ++i) {
            const int j = (i + lane) & 31;
            const uint32_t c = counts[j] >> shift & 0xffffu;
            n += c;
            mass = ::fma(__hiloint2double(0x43300000, int(c)) - 4503599627370496., power[j], mass);      // (2^52 + c: a conversion takes four times as long)
          }
        }
        if (code0 < Code<T>::kMinusInf && n != 0 && code0 >> 5 != first >> 5) {
          lead->count[code0 >> 5] = n;
          lead->mass[code0 >> 5] = group_weight(code0, mass);
        }
        if (first >= task0 && first < task0 + 1024) {      // (the whole warp)
          const uint32_t d = (first & ~31u) + lane, c = sh.counts[d & 0x7fffu] >> shift & 0xffffu;
          double m = c != 0 ? double(c) * weight(d) : 0.;
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
          const uint32_t all = __reduce_add_sync(0xffffffffu, c);
          if (lane == 0) {
            lead->count[first >> 5] = all;
            lead->mass[first >> 5] = m;
          }
        }
      }
    }
    meet();
    if (rank == 0) {
      if (!set.first) {
        if (sh.aside > 0) add_aside<T>(sh, weight);
        running_sums<kThreads>(sh.count, sh.mass, sh.warp_count, sh.warp_mass);
      }
      if (warp == 0) {
        uint32_t code = first;
        int place = 0;
        double share = 1.;
        if (!set.first) {
          // One group: how often each of its values is there, its weight, running sums before and with it.
          uint32_t n, n_with;
          double w, m_before, m_with;
          auto open = [&](int g) {
            const int word = (g & (kGroups / 2 - 1)) * 32 + lane;
            const uint32_t d = uint32_t(g * 32 + lane);
            const uint32_t v = of_rank(sh.counts, (word >> 10) % ctas)[word];
            n = g < kGroups / 2 ? v & 0xffffu : v >> 16;
            for (uint32_t i = 0; i < sh.aside; ++i)
              if (sh.aside_code[i] == d) n += sh.aside_count[i];
            if (d >= Code<T>::kMinusInf) n = 0;  // (and what stands for NaN is not there)
            w = n != 0 ? weight(d) : 0.;
            n_with = (g > 0 ? sh.count[g - 1] : 0u) + warp_running(n);
            const double own = warp_running(double(n) * w), base = g > 0 ? sh.mass[g - 1] : 0.;
            const double up = __shfl_up_sync(0xffffffffu, own, 1);
            m_before = base + (lane > 0 ? up : 0.);
            m_with = base + own;
          };
          auto pick = [&](bool passes) {         // the first lane that passes, or the last that has anything
            const uint32_t hit = __ballot_sync(0xffffffffu, passes && n != 0), any = __ballot_sync(0xffffffffu, n != 0);
            return hit != 0 ? __ffs(hit) - 1 : any != 0 ? 31 - __clz(any) : 0;
          };
          auto from = [&](auto v, int l) { return __shfl_sync(0xffffffffu, v, l); };
          uint32_t end = 0xffffu, take = 0xffffffffu;      // kept: what comes before code `end`, and `take` of it
          double kept = sh.mass[kGroups - 1];              // the sum of the kept
          if (set.top_k > 0 && uint32_t(set.top_k) < sh.count[kGroups - 1]) {
            const uint32_t k = uint32_t(set.top_k);
            const int g = first_of([&](int i) { return sh.count[i] >= k; });
            open(g);
            const int l = pick(n_with >= k);
            end = uint32_t(g * 32 + l);
            take = k - from(n_with - n, l);
            kept = from(m_before, l) + double(take) * from(w, l);
          }
          if (set.top_p < 1.f) {
            const double wanted = double(set.top_p) * kept;
            const int g = first_of([&](int i) { return sh.mass[i] >= wanted; });
            open(g);
            const int l = pick(m_with >= wanted);
            const uint32_t e = uint32_t(g * 32 + l), c = from(n, l);
            const double we = from(w, l), before = from(m_before, l), some = we > 0. ? ceil((wanted - before) / we) : 1.;
            const uint32_t t = uint32_t(fmin(fmax(some, 1.), double(c)));
            if (e < end || (e == end && t < take)) {
              end = e;
              take = t;
              kept = before + double(t) * we;
            }
          }
          if (set.min_p > 0.f) {
            const uint32_t e = last_that(first, Code<T>::kMinusInf - 1, [&](uint32_t d) { return weight(d) >= double(set.min_p); });
            if (e < end) {
              open(int(e >> 5));
              end = e;
              take = 0xffffffffu;
              kept = from(m_with, int(e & 31));
            }
          }
          const double target = double(set.u) * kept;
          const int g = first_of([&](int i) { return sh.mass[i] > target; });
          open(g);
          const int l = pick(m_with > target);
          code = uint32_t(g * 32 + l);
          const double wc = from(w, l), there = wc > 0. ? floor((target - from(m_before, l)) / wc) : 0.;
          uint32_t most_place = from(n, l) - 1;
          if (code == end && take <= most_place) most_place = take - 1;
          place = int(fmin(fmax(there, 0.), double(most_place)));
          share = wc / kept;
        }
        // Whose part has it: the equals of the parts before come first.
        int owner = 0, before = 0;
        if (ctas > 1) {
          uint32_t mine = 0;
          const int adder = int(code >> 10 & 31u) % ctas;          // which has all parts' there, unless nobody added
          if (lane < ctas) {
            const uint32_t v = of_rank(sh.counts, lane)[code & 0x7fffu];
            mine = (code & 0x8000u) ? v >> 16 : v & 0xffffu;
          }
          if (!set.first) {
            for (uint32_t i = 0; i < sh.aside; ++i)
              if (sh.aside_code[i] == code && lane == adder) mine += sh.aside_count[i];
            const uint32_t all = __shfl_sync(0xffffffffu, mine, adder), theirs = __reduce_add_sync(0xffffffffu, lane != adder ? mine : 0u);
            if (lane == adder) mine = all - theirs;
          }
          const uint32_t with = warp_running(mine), hit = __ballot_sync(0xffffffffu, int(with) > place);
          owner = __ffs(hit) - 1;
          before = int(__shfl_sync(0xffffffffu, with - mine, owner & 31));
        }
        if (lane < ctas) *of_rank(&sh.decision, lane) = Decision{owner, place - before, code};
        if (lane == 0 && a.probabilities != nullptr) a.probabilities[row] = float(share);
      }
    }
    meet();
    const Decision what = sh.decision;
    if (what.owner != rank) continue;

    // The place-th of its equals in this part: among the values before the vectors, the vectors, the rest.  A warp has a piece of the vectors.
    // As they are in memory: one pattern, of zero two.
    const uint32_t bits = (what.code & 0x8000u) ? what.code : what.code ^ 0x7fffu, here = bits * 0x10001u, also = bits == 0 ? 0x80008000u : here;
    auto is_it = [&](uint32_t v) { return v == bits || v == (also & 0xffffu); };
    auto may_hit = [&](const uint4& q) {         // a half that is zero takes a borrow
      auto zeros = [](uint32_t t) { return (t - 0x00010001u) & ~t; };
      uint32_t any = zeros(q.x ^ here) | zeros(q.y ^ here) | zeros(q.z ^ here) | zeros(q.w ^ here);
      if (bits == 0) any |= zeros(q.x ^ also) | zeros(q.y ^ also) | zeros(q.z ^ also) | zeros(q.w ^ also);
      return (any & 0x80008000u) != 0;
    };
    auto hits_of = [&](const uint4& q) -> uint32_t {       // bit i: value i is one
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
      uint32_t hits = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) hits |= (is_it(w[i] & 0xffffu) ? 1u << (2 * i) : 0u) | (is_it(w[i] >> 16) ? 2u << (2 * i) : 0u);
      return hits;
    };
    const int each = (vectors + kWarps - 1) / kWarps, from_v = min(warp * each, vectors), to_v = min(from_v + each, vectors);
    uint32_t found = 0;
    uint64_t seen = 0;                           // bit i: there was something in turn i
    constexpr int kLook = 4;
    for (int v = from_v, turn = 0; v < to_v; v += 32 * kLook, turn += kLook) {
      uint4 p[kLook];
      if (v + 32 * kLook <= to_v) {
#pragma unroll
        for (int i = 0; i < kLook; ++i) p[i] = kv::fetch(wide + v + 32 * i + lane);
      } else {
#pragma unroll
        for (int i = 0; i < kLook; ++i) {
          p[i] = make_uint4(~here, ~here, ~here, ~here);   // (none)
          if (v + 32 * i + lane < to_v) p[i] = kv::fetch(wide + v + 32 * i + lane);
        }
      }
      uint32_t may = 0;
#pragma unroll
      for (int i = 0; i < kLook; ++i) may |= may_hit(p[i]) ? 1u << i : 0u;
      if (may == 0) continue;
#pragma unroll
      for (int i = 0; i < kLook; ++i) {
        const uint32_t n = (may >> i & 1) && v + 32 * i + lane < to_v ? __popc(hits_of(p[i])) : 0u;
        found += n;
        seen |= uint64_t(n != 0) << (turn + i);
      }
    }
    found = __reduce_add_sync(0xffffffffu, found);
    seen = __reduce_or_sync(0xffffffffu, uint32_t(seen)) | uint64_t(__reduce_or_sync(0xffffffffu, uint32_t(seen >> 32))) << 32;
    if (lane == 0) sh.warp_count[warp] = found;
    __syncthreads();
    const uint32_t with = warp_running(lane < kWarps ? sh.warp_count[lane] : 0u);
    const uint32_t begin_hits = __ballot_sync(0xffffffffu, lane < head && is_it(x[min(lane, length - 1)])), early = __popc(begin_hits);
    uint32_t place = uint32_t(what.place);
    if (place < early) {
      if (tid == 0) {
        uint32_t hits = begin_hits;
        for (; place > 0; --place) hits &= hits - 1;
        a.tokens[row] = begin + __ffs(hits) - 1;
      }
      continue;
    }
    place -= early;
    const uint32_t hit = __ballot_sync(0xffffffffu, with > place);
    if (hit == 0) {                              // behind the vectors
      place -= __shfl_sync(0xffffffffu, with, 31);
      uint32_t hits = __ballot_sync(0xffffffffu, lane < rest && is_it(x[min(head + 8 * vectors + lane, length - 1)]));
      if (tid == 0) {
        for (; place > 0; --place) hits &= hits - 1;
        a.tokens[row] = begin + head + 8 * vectors + __ffs(hits) - 1;
      }
    } else if (__ffs(hit) - 1 == warp) {
      place -= warp > 0 ? __shfl_sync(0xffffffffu, with, warp > 0 ? warp - 1 : 0) : 0u;
      for (; seen != 0; seen &= seen - 1) {
        const int v = from_v + (__ffsll(int64_t(seen)) - 1) * 32 + lane;
        uint32_t hits = v < to_v ? hits_of(kv::fetch(wide + v)) : 0u;
        const uint32_t c = __popc(hits), run = warp_running(c), all = __shfl_sync(0xffffffffu, run, 31);
        if (place < all) {
          if (run > place && run - c <= place) {
            for (uint32_t skip = place - (run - c); skip > 0; --skip) hits &= hits - 1;
            a.tokens[row] = begin + head + 8 * v + __ffs(hits) - 1;
          }
          break;
        }
        place -= all;
      }
    }
  }
}
static_assert(kMaxVocabulary / 8 <= 64 * 32 * kWarps, "turns of a search in 64 bits");

// ---- float32 logits -----------------------------------------------------------------------------------------------------------------------------------
// A weight as the whole numbers that are added up, so that atomics in any order give the same: round(2^(45 + s) e^x), with an s for each range that puts its weights between 0.49 and 1.008
// times 2^45.  That is 44 bits of every weight, however small, and 2^18 of them do not pass 64.  (Multiples of 2^-45 for all ranges left a weight of 2^-40 with 6 bits.)  Behind x = -32 there is one
// range for all, in multiples of 2^-91: less than 2^-28 of the whole together, so that no number u and no float32 top_p below one has its border there.
constexpr double kPer = kGroups / 32.;           // ranges of one in x
__device__ __forceinline__ int scale_of(int range) { return range * 1477 >> 16; }        // (log2(e) / kPer from below)
__device__ __forceinline__ double unit_of(int range) { return __hiloint2double((1023 - 45 - scale_of(range)) << 20, 0); }
static_assert(kGroups == 2048, "scale_of");

struct Weighed {
  int range;
  unsigned long long weight;                     // times unit_of(range)
};
// From x <= 0.  e^x by 2^n e^r with |r| <= ln(2) / 2 and Taylor's sum for e^r to r^12 (the next term is 2^-52), n ln(2) in two parts of which the first is exact, n from the last bits of
// x / ln(2) + 1.5 2^52; the range in the same way.
__device__ __forceinline__ int range_of(double x) { return min(__double2loint(::fma(x, -kPer, 6755399441055744.)), kGroups - 1); }
__device__ __forceinline__ Weighed weighed_of(double x) {
  const double t = ::fma(x, 1.4426950408889634074, 6755399441055744.), n = t - 6755399441055744., r = ::fma(-n, -1.904654299957768e-9, ::fma(-n, double(0.693147182464599609375f), x));
  double p = 1. / 479001600.;
  p = ::fma(p, r, 1. / 39916800.);
  p = ::fma(p, r, 1. / 3628800.);
  p = ::fma(p, r, 1. / 362880.);
  p = ::fma(p, r, 1. / 40320.);
  p = ::fma(p, r, 1. / 5040.);
  p = ::fma(p, r, 1. / 720.);
  p = ::fma(p, r, 1. / 120.);
  p = ::fma(p, r, 1. / 24.);
  p = ::fma(p, r, 1. / 6.);
  p = ::fma(p, r, 0.5);
  p = ::fma(p, r, 1.);
  p = ::fma(p, r, 1.);
  const int range = range_of(x);
  const double scale = __hiloint2double((1023 + 45 + scale_of(range) + __double2loint(t)) << 20, 0);
  return {range, (unsigned long long)__double_as_longlong(::fma(p, scale, 4503599627370496.)) & 0xfffffffffffffull};      // 2^52 + a whole number
}

struct Place {                                   // a range of codes, what comes before it, what is in it
  uint32_t low, high;
  uint32_t count_before, count;
  double mass_before, unit;
  unsigned long long mass;                       // times unit
  __device__ __forceinline__ bool open() const { return count > 1 && low < high && mass > 0; }      // (without weight it does not matter which of them)
  __device__ __forceinline__ unsigned long long one() const { return mass / max(count, 1u); }       // of a place of equals
};
constexpr int kList = 2048;                      // values that the first CTA narrows down by itself
struct Shared32 {
  uint32_t codes[kPart32];
  double mass[kGroups];                          // sums of the 2048 ranges (the first CTA's: of all, running)
  unsigned long long range_mass[kGroups];        // of a range that is narrowed down, times its unit
  uint32_t count[kGroups], range_count[kGroups];
  uint32_t own_mass[3][kGroups], own_count[kGroups];      // this part's; the mass as sums of 15, 15 and 16 bits of each weight, whose 32768 do not pass 32 (a sum of 64 bits is no single atomic);
                                                 // the first CTA's after that: 32 and 32 bits of every range's sum of all parts
  uint32_t list_code[kList], list_index[kList];  // the values of a range, the first CTA's
  unsigned long long warp_mass[kWarps];
  double warp_sum[kWarps];
  uint32_t warp_count[kWarps];
  uint32_t least, most, list;
  uint32_t all_least[8], all_most[8];
  Place place[2], own;                           // written in turn: a slow CTA may be reading the one before
  unsigned long long sum_mass;
  uint32_t sum_count;
  uint32_t found[8];
};

__global__ void __launch_bounds__(kThreads, 1) sample32_kernel(Args a) {
  extern __shared__ __align__(16) uint8_t raw[];
  Shared32& sh = *reinterpret_cast<Shared32*>(raw);
  using C = Code<float>;
  cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int ctas = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  const int64_t row = blockIdx.x / ctas;
  for (int i = tid; i < kGroups; i += kThreads) {
    sh.own_mass[0][i] = sh.own_mass[1][i] = sh.own_mass[2][i] = 0;
    sh.range_mass[i] = 0;
    sh.own_count[i] = sh.range_count[i] = 0;
  }
  if (tid == 0) {
    sh.least = 0xffffffffu;
    sh.most = 0;
    sh.list = 0;
    sh.sum_mass = 0;
    sh.sum_count = 0;
  }
  wait_for_launch_before();
  __syncthreads();
  const Row set = row_of(a, row);
  const int part = (a.vocabulary + ctas - 1) / ctas;
  const int begin = min(rank * part, a.vocabulary), length = min(part, a.vocabulary - begin);
  const float* x = static_cast<const float*>(a.logits) + row * a.row_stride + begin;
  uint32_t least = 0xffffffffu, most = 0;
#pragma unroll 8
  for (int i = tid; i < length; i += kThreads) {
    const uint32_t d = C::of(kv::fetch(x + i));
    sh.codes[i] = d;
    least = min(least, d);
    most = max(most, d);
  }
  least = __reduce_min_sync(0xffffffffu, least);
  most = __reduce_max_sync(0xffffffffu, most);
  if (lane == 0) {
    atomicMin(&sh.least, least);
    atomicMax(&sh.most, most);
  }
  __syncthreads();
  if (tid < ctas) {
    Shared32* other = cluster.map_shared_rank(&sh, tid);
    other->all_least[rank] = sh.least;
    other->all_most[rank] = sh.most;
  }
  cluster.sync();
  const uint32_t first = __reduce_min_sync(0xffffffffu, lane < ctas ? sh.all_least[lane] : 0xffffffffu);
  most = __reduce_max_sync(0xffffffffu, lane < ctas ? sh.all_most[lane] : 0u);
  if (!set.valid || first < C::kInf || most > C::kMinusInf || first >= C::kMinusInf) {
    if (rank == 0 && tid == 0) {
      if (!set.valid) kv::flag_range(a.status);
      answer(a, row, -1, 0.f);
    }
    return;
  }
  const Weight<float> weight(first, set.temperature);
  Shared32* lead = cluster.map_shared_rank(&sh, 0);
  Place found{first, first, 0, 1, 0., 1., 1};    // where the chosen one is
  uint32_t place = 0;                            // and which of the equals there (the first CTA's)
  bool listed = false;
  if (!set.first) {
    // (largest - logit) / temperature of every value, which its range and its weight go by.  A NaN (inf - inf, 0 inf) is the largest value's or has no weight.
    auto x_of = [&](uint32_t d) {
      const double x = (double(C::value(d)) - weight.largest) * weight.inverse;
      return d == first ? 0. : x > -64. ? x : -64.;        // (e^-64 2^91 is less than a half)
    };
    auto range = [&](uint32_t d) { return range_of(x_of(d)); };
    auto weighed = [&](uint32_t d) { return weighed_of(x_of(d)); };
    constexpr int kTogether = 4;                 // values whose chains of instructions go side by side
    for (int i = tid; i < length; i += kTogether * kThreads) {
      uint32_t d[kTogether];
      Weighed m[kTogether];
#pragma unroll
      for (int j = 0; j < kTogether; ++j) d[j] = i + j * kThreads < length ? sh.codes[i + j * kThreads] : C::kMinusInf;
#pragma unroll
      for (int j = 0; j < kTogether; ++j) m[j] = weighed(d[j]);
#pragma unroll
      for (int j = 0; j < kTogether; ++j) {
        if (d[j] == C::kMinusInf) continue;
        const int r = m[j].range;
        const uint32_t low = uint32_t(m[j].weight) & 0x7fffu, middle = uint32_t(m[j].weight >> 15) & 0x7fffu, high = uint32_t(m[j].weight >> 30);
        atomicAdd(&sh.own_count[r], 1u);
        if (low != 0) atomicAdd(&sh.own_mass[0][r], low);
        if (middle != 0) atomicAdd(&sh.own_mass[1][r], middle);
        if (high != 0) atomicAdd(&sh.own_mass[2][r], high);
      }
    }
    cluster.sync();
    for (int i = rank * kThreads + tid; i < kGroups; i += ctas * kThreads) {
      uint32_t c = 0;
      unsigned long long m = 0;
#pragma unroll 8
      for (int r = 0; r < ctas; ++r) {
        const Shared32* other = cluster.map_shared_rank(&sh, r);
        c += other->own_count[i];
        m += other->own_mass[0][i] + ((unsigned long long)(other->own_mass[1][i]) << 15) + ((unsigned long long)(other->own_mass[2][i]) << 30);
      }
      lead->count[i] = c;
      lead->mass[i] = double(m) * unit_of(i);
      lead->own_mass[0][i] = uint32_t(m);        // (range i is this thread's alone, and all parts' are read)
      lead->own_mass[1][i] = uint32_t(m >> 32);
    }
    cluster.sync();
    if (rank == 0) running_sums<kThreads>(sh.count, sh.mass, sh.warp_count, sh.warp_sum);
    // What is kept: how many, their weights.  The first CTA's; the others follow the places that it gives.
    uint32_t keep = 0;
    double sum = 0.;
    if (rank == 0) {
      keep = sh.count[kGroups - 1];
      sum = sh.mass[kGroups - 1];
    }
    int turn = 0;
    auto tell = [&](const Place& p) {            // the first CTA's first warp
      if (lane < ctas) *cluster.map_shared_rank(&sh.place[turn], lane) = p;
    };
    auto told = [&] {
      cluster.sync();
      const Place p = sh.place[turn];
      turn ^= 1;
      return p;
    };
    // The part of place p that the running sums of its 2048 parts (range_count, range_mass) say; by the first CTA, which gives the sums back as zeros.
    auto narrow = [&](const Place& p, int shift, auto passes) {
      running_sums<kThreads>(sh.range_count, sh.range_mass, sh.warp_count, sh.warp_mass);
      Place q = p;
      if (warp == 0) {
        // (or the last that has anything: the sums of the ranges and of a range's parts have roundings of their own)
        const int g = first_of([&](int i) { return sh.range_count[i] >= p.count || passes(p.count_before + sh.range_count[i], p.mass_before + double(sh.range_mass[i]) * p.unit); });
        const uint32_t c = g > 0 ? sh.range_count[g - 1] : 0u;
        const unsigned long long m = g > 0 ? sh.range_mass[g - 1] : 0ull;
        q.low = p.low + (uint32_t(g) << shift);
        q.high = min(p.high, q.low + ((1u << shift) - 1));
        q.count_before = p.count_before + c;
        q.mass_before = p.mass_before + double(m) * p.unit;
        q.count = sh.range_count[g] - c;
        q.mass = sh.range_mass[g] - m;
      }
      __syncthreads();
      for (int i = tid; i < kGroups; i += kThreads) {
        sh.range_mass[i] = 0;
        sh.range_count[i] = 0;
      }
      return q;                                  // (of the first warp)
    };
    auto shift_of = [](const Place& p) { return max(0, 32 - __clz(int(p.high - p.low)) - 11); };
    // The place where the running count reaches `count` (by_count) or the running sum reaches, or with `above` passes, `mass`; nowhere if `none`.  All that the first CTA says is the first's.
    auto descend = [&](bool none, bool by_count, uint32_t count, double mass, bool above) -> Place {
      auto passes = [&](uint32_t c, double m) { return by_count ? c >= count : above ? m > mass : m >= mass; };
      if (rank == 0 && warp == 0) {
        const int g = first_of([&](int i) { return sh.count[i] == sh.count[kGroups - 1] || passes(sh.count[i], sh.mass[i]); });
        Place p{first, first, 0, 0, 0., 0., 0};
        if (!none) {
          p.low = g == 0 ? first : last_that(first, C::kMinusInf - 1, [&](uint32_t d) { return range(d) < g; }) + 1;
          p.high = last_that(first, C::kMinusInf - 1, [&](uint32_t d) { return range(d) <= g; });
          p.count_before = g > 0 ? sh.count[g - 1] : 0u;
          p.mass_before = g > 0 ? sh.mass[g - 1] : 0.;
          p.count = sh.count[g] - p.count_before;
          p.mass = sh.own_mass[0][g] | (unsigned long long)(sh.own_mass[1][g]) << 32;
          p.unit = unit_of(g);
        }
        if (lane == 0) sh.list = 0;
        tell(p);
      }
      Place p = told();
      listed = p.open() && p.count <= uint32_t(kList);
      if (listed) {                              // few: the first CTA takes them all and goes on by itself
        for (int i = tid; i < length; i += kThreads) {
          const uint32_t d = sh.codes[i];
          if (d < p.low || d > p.high) continue;
          const uint32_t at = atomicAdd(&lead->list, 1u);
          lead->list_code[at] = d;
          lead->list_index[at] = uint32_t(begin + i);
        }
        cluster.sync();
        if (rank != 0) return p;
        const int n = int(sh.list);
        while (p.open()) {
          const int shift = shift_of(p);
          for (int i = tid; i < n; i += kThreads) {
            const uint32_t d = sh.list_code[i];
            if (d < p.low || d > p.high) continue;
            atomicAdd(&sh.range_count[(d - p.low) >> shift], 1u);
            atomicAdd(&sh.range_mass[(d - p.low) >> shift], weighed(d).weight);
          }
          __syncthreads();
          const Place q = narrow(p, shift, passes);
          if (tid == 0) sh.own = q;
          __syncthreads();
          p = sh.own;
        }
        return p;
      }
      while (p.open()) {
        const int shift = shift_of(p);
        for (int i = tid; i < length; i += kThreads) {
          const uint32_t d = sh.codes[i];
          if (d < p.low || d > p.high) continue;
          atomicAdd(&lead->range_count[(d - p.low) >> shift], 1u);
          atomicAdd(&lead->range_mass[(d - p.low) >> shift], weighed(d).weight);
        }
        cluster.sync();
        if (rank == 0) {
          const Place q = narrow(p, shift, passes);
          if (warp == 0) tell(q);
        }
        p = told();
      }
      return p;
    };
    if (set.top_k > 0) {
      const uint32_t k = uint32_t(set.top_k);
      const Place p = descend(rank == 0 && k >= keep, true, k, 0., false);
      if (k < keep) {
        keep = k;
        sum = p.mass_before + double(p.one() * (k - p.count_before)) * p.unit;
      }
    }
    if (set.top_p < 1.f) {
      const double wanted = double(set.top_p) * sum;
      const Place p = descend(false, false, 0, wanted, false);
      const double w = double(p.one()) * p.unit, some = w > 0. ? ceil((wanted - p.mass_before) / w) : 1.;
      const uint32_t t = uint32_t(fmin(fmax(some, 1.), double(max(p.count, 1u))));
      if (p.count_before + t < keep) {
        keep = p.count_before + t;
        sum = p.mass_before + w * double(t);
      }
    }
    if (set.min_p > 0.f) {
      // the last one with that weight: what is kept are the ranges before its own and of that one what comes up to it
      const uint32_t e = last_that(first, C::kMinusInf - 1, [&](uint32_t d) { return weight(d) >= double(set.min_p); });
      const int g = range(e);
      unsigned long long m = 0;
      uint32_t c = 0;
      for (int i = tid; i < length; i += kThreads) {
        const uint32_t d = sh.codes[i];
        if (d > e) continue;
        const Weighed q = weighed(d);
        if (q.range != g) continue;
        ++c;
        m += q.weight;
      }
      c = __reduce_add_sync(0xffffffffu, c);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
      if (lane == 0 && c > 0) {
        atomicAdd(&lead->sum_count, c);
        atomicAdd(&lead->sum_mass, m);
      }
      cluster.sync();
      const uint32_t some = rank == 0 ? (g > 0 ? sh.count[g - 1] : 0u) + sh.sum_count : 0u;
      if (rank == 0 && some < keep) {
        keep = some;
        sum = (g > 0 ? sh.mass[g - 1] : 0.) + double(sh.sum_mass) * unit_of(g);
      }
    }
    const double target = double(set.u) * sum;
    found = descend(false, false, 0, target, true);
    if (rank == 0) {
      const double w = double(found.one()) * found.unit, there = w > 0. ? floor((target - found.mass_before) / w) : 0.;
      uint32_t most_place = max(found.count, 1u) - 1;
      if (found.count_before + most_place >= keep) most_place = keep > found.count_before ? keep - found.count_before - 1 : 0u;
      place = uint32_t(fmin(fmax(there, 0.), double(most_place)));
      if (tid == 0 && a.probabilities != nullptr) a.probabilities[row] = float(w / sum);
    }
  } else if (rank == 0 && tid == 0 && a.probabilities != nullptr) {
    a.probabilities[row] = 1.f;
  }

  if (listed) {                                  // the first CTA has all that it may be: the one with `place` of its equals before it
    if (rank != 0) return;
    const int n = int(sh.list);
    for (int i = tid; i < n; i += kThreads) {
      const uint32_t d = sh.list_code[i], index = sh.list_index[i];
      if (d < found.low || d > found.high) continue;
      uint32_t before = 0;
      if (found.count > 1)
        for (int j = 0; j < n; ++j) before += sh.list_code[j] >= found.low && sh.list_code[j] <= found.high && sh.list_index[j] < index ? 1u : 0u;
      if (before == place) a.tokens[row] = int(index);
    }
    return;
  }
  // The place-th of its equals: a warp has a piece of the part.
  if (rank == 0 && tid == 0) sh.sum_count = place;
  const int each = (length + kWarps - 1) / kWarps, from_i = min(warp * each, length), to_i = min(from_i + each, length);
  auto is_one = [&](int i) { return i < to_i && sh.codes[i] >= found.low && sh.codes[i] <= found.high; };
  uint32_t hits = 0;
  for (int i = from_i; i < to_i; i += 32) hits += __popc(__ballot_sync(0xffffffffu, is_one(i + lane)));
  __syncthreads();
  if (lane == 0) sh.warp_count[warp] = hits;
  __syncthreads();
  const uint32_t with = warp_running(lane < kWarps ? sh.warp_count[lane] : 0u), own = __shfl_sync(0xffffffffu, with, 31);
  if (warp == 0 && lane < ctas) cluster.map_shared_rank(sh.found, lane)[rank] = own;
  cluster.sync();
  place = lead->sum_count;
  uint32_t before = 0;
  for (int r = 0; r < rank; ++r) before += sh.found[r];
  cluster.sync();                                // (all have read what the first CTA says)
  if (place < before) return;
  place -= before;
  const uint32_t hit = __ballot_sync(0xffffffffu, with > place);
  if (hit == 0 || __ffs(hit) - 1 != warp) return;
  uint32_t left = place - (warp > 0 ? __shfl_sync(0xffffffffu, with, warp > 0 ? warp - 1 : 0) : 0u);
  for (int i = from_i; i < to_i; i += 32) {
    uint32_t here = __ballot_sync(0xffffffffu, is_one(i + lane));
    const uint32_t c = __popc(here);
    if (left < c) {
      for (; left > 0; --left) here &= here - 1;
      if (lane == 0) a.tokens[row] = begin + i + __ffs(here) - 1;
      return;
    }
    left -= c;
  }
}

// Clusters of `ctas` CTAs that run at once on the current device (the SMs of a part of it may not be a multiple of that), looked up once (known: one more); negative: that failed.
template <typename K> static int clusters_of(K kernel, int ctas, int threads, size_t shared, std::atomic<int> (&known)[64]) {
  int dev = -1, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -1;
  if ((n = known[dev].load(std::memory_order_acquire)) > 0) return n - 1;
  if (ctas == 1) {
    if ((n = stream::sm_count()) <= 0) return -1;
  } else {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(unsigned(ctas) * 64);
    cfg.blockDim = dim3(unsigned(threads));
    cfg.dynamicSmemBytes = shared;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = unsigned(ctas);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 0) return -1;
  }
  known[dev].store(n + 1, std::memory_order_release);
  return n;
}

// One CTA a row has 1024 threads (256 rows of 128256 51 us, 53.5 with 512).
template <int C> constexpr int threads16() { return C == 1 ? 1024 : kThreads; }
template <typename T, int C> static int fits16() {
  static std::atomic<uint64_t> done{0};
  static std::atomic<int> known[64];
  if (allow_shared(sample16_kernel<T, C, threads16<C>()>, sizeof(Shared16), done)) return -1;
  return clusters_of(sample16_kernel<T, C, threads16<C>()>, C, threads16<C>(), sizeof(Shared16), known);
}
template <typename T> static int launch16(const Args& a, cudaStream_t s) {
  const SampleClusters c = sample_clusters_16(a.vocabulary, a.rows, kPart16, [](int ctas) { return ctas == 8 ? fits16<T, 8>() : ctas == 4 ? fits16<T, 4>() : ctas == 2 ? fits16<T, 2>() : fits16<T, 1>(); });
  auto go = [&](auto of) {                       // as many clusters as run at once; each takes rows in turn
    constexpr int C = decltype(of)::value;
    return launch_dependent(sample16_kernel<T, C, threads16<C>()>, dim3(unsigned(std::min<int64_t>(a.rows, c.at_once) * C)), threads16<C>(), sizeof(Shared16), C, s, a);
  };
  switch (c.ctas) {
    case 8: return go(std::integral_constant<int, 8>{});
    case 4: return go(std::integral_constant<int, 4>{});
    case 2: return go(std::integral_constant<int, 2>{});
    case 1: return go(std::integral_constant<int, 1>{});
    default: return RC_LAUNCH;
  }
}

static int launch32(const Args& a, cudaStream_t s) {
  static std::atomic<uint64_t> done{0};
  static std::atomic<int> known[9][64];
  if (int rc = allow_shared(sample32_kernel, sizeof(Shared32), done)) return rc;
  const SampleClusters c = sample_clusters_32(a.vocabulary, a.rows, kPart32, [](int ctas) { return clusters_of(sample32_kernel, ctas, kThreads, sizeof(Shared32), known[ctas]); });
  if (c.ctas == 0) return RC_LAUNCH;
  return launch_dependent(sample32_kernel, dim3(unsigned(a.rows * c.ctas)), kThreads, sizeof(Shared32), unsigned(c.ctas), s, a);
}

}  // namespace choice

int sample(const void* logits, int64_t row_stride, int dtype, int rows, int vocabulary, const float* uniforms, const DinoB200SampleSettings* settings, int* tokens,
           float* probabilities, cudaStream_t s) {
  using namespace choice;
  if (logits == nullptr || uniforms == nullptr || settings == nullptr || tokens == nullptr) return RC_NULL;
  if (rows <= 0 || vocabulary <= 0) return RC_DIMS;
  if (vocabulary > kMaxVocabulary || rows > INT32_MAX / 8 || (rows > 1 && row_stride < vocabulary)) return RC_RANGE;
  if (dtype != DINO_F16 && dtype != DINO_BF16 && dtype != DINO_F32) return RC_DTYPE;
  if ((reinterpret_cast<uintptr_t>(logits) & (dtype == DINO_F32 ? 3 : 1)) != 0) return RC_ALIGN;
  int* status = kv::status_words();
  if (status == nullptr) return RC_LAUNCH;
  const Args a{logits, row_stride, rows, vocabulary, uniforms, *settings, tokens, probabilities, status};
  switch (dtype) {
    case DINO_F16: return launch16<__half>(a, s);
    case DINO_BF16: return launch16<__nv_bfloat16>(a, s);
    default: return launch32(a, s);
  }
}

}  // namespace b200gguf

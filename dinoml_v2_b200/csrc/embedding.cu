// Rows of a GGUF table for the tokens of a step: out[i] = round(dequant(table[tokens[i]]) * scale).
//
// Bound by bytes, most of them the result's (8192 values of Q4_K are 4.6 KB read and 16 KB written, and a text's tokens repeat); a single token by its chain of reads (token, block,
// result) and the launch.  A thread has an item of a row (dequant_items.cuh: 32 weights of Q4_K in 16 bits), a CTA one row, or several short ones, at a time; it reads the next row's
// item before it writes this one's.  8192 tokens of a table of 128256 rows, Q4_K of 8192 values to bfloat16: 29.2 us (134 MB written, 18 read: 5.2 TB/s; eight values a thread with scales of their
// own 58); 301 tokens of 2880 Q8_0 to float32 2.8 us, one of 4096 Q6_K 2.0.
#include <algorithm>

#include "dependent_launch.cuh"
#include "dequant_items.cuh"
#include "kv_cache.cuh"

namespace b200gguf {
namespace stream { int sm_count(); }             // gemv_stream.cu
namespace embed {

constexpr int kThreads = 256;

template <typename I> struct Args {
  const I* tokens;
  const uint8_t* table;
  void* out;
  int64_t vocabulary, count, groups;             // groups: of tokens that a CTA has at once
  int64_t first_edge, last_edge;                 // blocks of the table whose first or last aligned word holds bytes outside of it
  int blocks, items, each, chunks;               // of a row: blocks, items; tokens of a group; turns that a CTA needs for a row
  float scale;
  bool wide;
  int* status;
};

// A: alignment of the table that all of its blocks keep.
template <int QT, typename T, typename I, int A>
__global__ void __launch_bounds__(kThreads) embedding_kernel(Args<I> a) {
  using G = ItemGeom<QT, run_of<QT, T>()>;
  const int sub = a.each > 1 ? int(threadIdx.x) / a.items : 0, own = int(threadIdx.x) - sub * a.items;
  const int64_t units = a.groups * a.chunks;
  struct Job {
    int64_t row;                                 // of the result; -1: nothing
    int item;
    bool in;                                     // the token is in the table
    Item<QT, T, A> what;
  };
  auto load = [&](int64_t unit, Job& job) {
    job.row = -1;
    job.in = false;
    if (unit >= units || sub >= a.each) return;
    const int64_t group = a.chunks == 1 ? unit : unit / a.chunks;
    const int at = own + int(unit - group * a.chunks) * kThreads;
    const int64_t row = group * a.each + sub;
    if (at >= a.items || row >= a.count) return;
    const int64_t token = int64_t(a.tokens[row]);
    job.row = row;
    job.item = at;
    job.in = token >= 0 && token < a.vocabulary;
    if (job.in) {
      const int64_t block = token * a.blocks + at / G::kItems;
      job.what.load(a.table + block * QTraits<QT>::kBytes, at % G::kItems, block == a.first_edge || block == a.last_edge);
    } else if (token != -1 && at == 0) {
      kv::flag_range(a.status);
    }
  };
  auto store = [&](const Job& job) {
    if (job.row < 0) return;
    const int block = job.item / G::kItems, item = job.item % G::kItems;
    T* to = static_cast<T*>(a.out) + (job.row * a.blocks + block) * QTraits<QT>::kBlock;
    if (job.in) {
      if (a.scale == 1.f) job.what.emit(to, item, a.wide); else job.what.template emit<true>(to, item, a.wide, a.scale);
      return;
    }
    constexpr int R = run_of<QT, T>();
#pragma unroll
    for (int j = 0; j < G::kRuns; ++j)
#pragma unroll
      for (int i = 0; i < R * int(sizeof(T)); i += 16) *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(to + job.what.first(item, j)) + i) = make_uint4(0, 0, 0, 0);
  };
  wait_for_launch_before();
  Job now, next;
  int64_t unit = blockIdx.x;
  load(unit, now);
  while (true) {
    unit += gridDim.x;
    if (unit >= units) break;
    load(unit, next);
    store(now);
    now = next;
  }
  store(now);
}

template <int QT, typename T, typename I, int A>
static int launch(Args<I> a, int64_t width, cudaStream_t s) {
  using G = ItemGeom<QT, run_of<QT, T>()>;
  const int sms = stream::sm_count();
  if (sms <= 0) return RC_LAUNCH;
  a.blocks = int(width / QTraits<QT>::kBlock);
  if (int64_t(a.blocks) * G::kItems > INT32_MAX) return RC_RANGE;
  a.items = a.blocks * G::kItems;
  a.each = std::max(1, kThreads / a.items);
  a.chunks = (a.items + kThreads - 1) / kThreads;
  a.groups = (a.count + a.each - 1) / a.each;
  const uintptr_t begin = reinterpret_cast<uintptr_t>(a.table);
  const int64_t blocks = a.vocabulary * a.blocks;
  a.first_edge = begin & 3 ? 0 : -1;
  a.last_edge = (begin + uintptr_t(blocks) * QTraits<QT>::kBytes) & 3 ? blocks - 1 : -1;
  a.wide = (reinterpret_cast<uintptr_t>(a.out) & 31) == 0;
  return launch_dependent(embedding_kernel<QT, T, I, A>, dim3(unsigned(std::min<int64_t>(a.groups * a.chunks, 5 * int64_t(sms)))), kThreads, 0, 1, s, a);
}

template <int QT, typename T, typename I>
static int aligned(const Args<I>& a, int64_t width, cudaStream_t s) {
  constexpr int kAlign = ItemGeom<QT, run_of<QT, T>()>::kAlign;
  const uintptr_t at = reinterpret_cast<uintptr_t>(a.table);
  if constexpr (kAlign == 16)
    if ((at & 15) == 0) return launch<QT, T, I, 16>(a, width, s);
  if constexpr (kAlign >= 4)
    if ((at & 3) == 0) return launch<QT, T, I, 4>(a, width, s);
  if constexpr (QT == QTYPE_Q4_K) return RC_ALIGN;         // the entry has refused these
  else return launch<QT, T, I, 1>(a, width, s);
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
      auto with = [&](auto i) {
        using I = decltype(i);
        embed::Args<I> a = {};
        a.tokens = static_cast<const I*>(tokens);
        a.table = static_cast<const uint8_t*>(table);
        a.out = out;
        a.vocabulary = vocabulary;
        a.count = count;
        a.scale = scale;
        a.status = status;
        return embed::aligned<QT, T, I>(a, width, s);
      };
      return token_bytes == 4 ? with(int32_t{}) : with(int64_t{});
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

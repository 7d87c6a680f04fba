// What the attention kernels over the 8-bit cache share: whose rows a piece of work has and what they see, the line of units that CTAs cut
// between them, 8-bit pairs as float16.
#pragma once
#include "kv_cache.cuh"
#include "umma_frame.cuh"

namespace b200gguf {
namespace stream { int sm_count(); }             // gemv_stream.cu
namespace kv {

constexpr float kLog2e = 1.4426950408889634f;
constexpr uint32_t kPolls = 1u << 18;       // of a barrier before a wait gives up, a second or two: waits are within a CTA

// n / d for 0 <= n < 2^31: the quotient is (mulhi(n, m) + n) >> s with s = ceil(log2 d), m = floor(2^32 (2^s - d) / d) + 1 (Granlund and Montgomery).
struct Divisor {
  uint32_t m, s;
  void set(uint32_t d) {
    s = 0;
    while ((uint64_t(1) << s) < d) ++s;
    m = uint32_t((((uint64_t(1) << s) - d) << 32) / d) + 1u;
  }
#ifdef __CUDACC__
  __device__ __forceinline__ int operator()(int n) const { return int((__umulhi(uint32_t(n), m) + uint32_t(n)) >> s); }
#endif
};

struct AttnParams {
  Cache c;
  Batch p;
  const void* q;
  void* out;
  int64_t row_stride, head_stride;           // of q, in elements
  float scale;                               // of the scores, times log2(e)
  int window, heads, group, dtype;
  Divisor by_group;
  int row_tile, row_tile_log2;               // rows (token x head of the group) of an item
  int ends;                                  // what an item costs beside its tiles, in tiles
  int min_rows, max_rows;                    // sequences with fewer or more rows (tokens x group) are another launch's
  float* partial;                            // two cut pieces per CTA
  int* arrived;                              // a counter per CTA, zero between launches
};

// A sequence's part of the call.
struct Sequence {
  int row, count;                            // packed rows
  int first;                                 // position of the first of them
  int end;                                   // positions that exist: its tokens, as far as the table reaches
};
__device__ __forceinline__ Sequence sequence_at(const AttnParams& a, int b) {
  const Rows rows = rows_of(a.p, b);
  const int length = fetch(a.p.lengths + b);
  const int reach = int(min(int64_t(a.p.table_blocks) << a.c.block_log2, int64_t(INT32_MAX)));
  if (length > reach) flag_range(a.p.status);
  const int64_t total = int64_t(rows.count) * a.group;
  const bool mine = total >= a.min_rows && total <= a.max_rows;
  return {rows.first, mine ? rows.count : 0, length - rows.count, max(0, min(length, reach))};
}

// Rows [r0, r1) of a sequence (row r: token r / group, head r % group of it) against cached positions [low, high).
struct Item {
  int r0, r1, low, high;
};
__device__ __forceinline__ Item item_at(const AttnParams& a, const Sequence& s, int row_tile) {
  Item it;
  it.r0 = row_tile * a.row_tile;
  it.r1 = min(it.r0 + a.row_tile, s.count * a.group);
  const int first = s.first + a.by_group(it.r0), last = s.first + a.by_group(it.r1 - 1);
  it.high = max(0, min(last + 1, s.end));
  it.low = a.window > 0 ? max(0, first - a.window + 1) : 0;
  if (it.low > it.high) it.low = it.high;
  return it;
}
__device__ __forceinline__ int row_tiles(const AttnParams& a, const Sequence& s) { return (s.count * a.group + a.row_tile - 1) >> a.row_tile_log2; }
// Tiles of `size` positions (a power of two) that an item covers; one that sees nothing still has its rows to write.
__device__ __forceinline__ int tiles_of(const Item& it, int log2) { return it.high > it.low ? ((it.high - 1) >> log2) - (it.low >> log2) + 1 : 1; }

// The units of the launch are one line: sequences, their row tiles, the cached heads, and for each of these items `ends` units for its beginning and its end, in
// which there is nothing to do, and its tiles of cached positions.  Worker c of G (a CTA; those beyond G have nothing to do) takes units
// [c W / G, (c + 1) W / G): the same work for every CTA whatever the lengths are, at the price that an item that is cut is finished by whoever of its CTAs
// comes last.
struct Walk {
  int b, row_tile, head, tile;               // the next tile
  int workers, per, more;                    // units of a worker, and how many of `workers` parts of one more unit
  int64_t units, start;                      // of the launch; the first one of this CTA's range
  int64_t unit, stop;                        // number of the next unit, and the end of the range
  int64_t item_unit;                         // number of the item's first unit
  Sequence s;
  Item item;
  int tiles, ends;                           // of the item

  __device__ __forceinline__ bool done() const { return unit >= stop; }
  __device__ __forceinline__ int64_t first_tile() const { return item_unit + ends; }
  __device__ __forceinline__ int end_tile() const { return int(min(int64_t(tiles), stop - first_tile())); }
  // Numbers of the partial sums of this CTA's part of the item, and of the item's first part: a CTA has two at most, one of the item that its range begins in.
  __device__ __forceinline__ int piece() const { return 2 * int(blockIdx.x) + (start >= item_unit ? 0 : 1); }
  __device__ __forceinline__ int first_piece(int owner_of_it) const { return 2 * owner_of_it + (start_of(owner_of_it) >= item_unit ? 0 : 1); }
  __device__ __forceinline__ void open(const AttnParams& a, int log2) {
    item = item_at(a, s, row_tile);
    tiles = tiles_of(item, log2);
  }
  __device__ __forceinline__ void next_item(const AttnParams& a, int log2) {
    unit = item_unit = first_tile() + tiles;
    tile = 0;
    if (done()) return;
    unit += ends;
    if (done() || ++head < a.c.heads) return;
    head = 0;
    if (++row_tile >= row_tiles(a, s)) {
      row_tile = 0;
      do s = sequence_at(a, ++b);
      while (s.count == 0 && b + 1 < a.p.sequences);      // (a unit is left, so there is one with rows)
    }
    open(a, log2);
  }
  __device__ __forceinline__ int64_t start_of(int worker) const { return int64_t(worker) * per + worker * more / workers; }      // worker * units / workers
  __device__ __forceinline__ int owner(int64_t u) const {
    if (units < int64_t(1) << 21) return int((uint32_t(u + 1) * uint32_t(workers) - 1u) / uint32_t(units));      // (at most 1024 workers)
    return int(((u + 1) * workers - 1) / units);
  }
};

// Block-wide: the range of this CTA and where it begins; at least `least` units for every worker.  NT threads; `shared`: 2 + NT / 32 words of 8 bytes.
template <int NT>
__device__ __forceinline__ Walk walk_of(const AttnParams& a, int log2, int least, int64_t* shared) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (a.p.sequences + NT - 1) / NT;
  auto units_of = [&](const Sequence& s) {
    int64_t n = 0;
    for (int t = row_tiles(a, s) - 1; t >= 0; --t) n += a.ends + tiles_of(item_at(a, s, t), log2);
    return n * a.c.heads;
  };
  int64_t mine = 0;
  for (int b = tid * per; b < min((tid + 1) * per, a.p.sequences); ++b) mine += units_of(sequence_at(a, b));
  int64_t sum = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t up = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += up;
  }
  if (lane == 31) shared[2 + warp] = sum;
  __syncthreads();
  int64_t before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < NT / 32; ++w) {
    if (w < warp) before += shared[2 + w];
    total += shared[2 + w];
  }
  Walk k;
  k.ends = a.ends;
  k.units = total;
  const bool small = total < int64_t(1) << 31;                      // 64-bit divisions are slow
  k.workers = int(max(int64_t(1), min(int64_t(gridDim.x), small ? int64_t(uint32_t(total) / uint32_t(least)) : total / least)));
  k.per = small ? int(uint32_t(total) / uint32_t(k.workers)) : int(total / k.workers);
  k.more = int(total - int64_t(k.per) * k.workers);
  k.start = k.unit = k.start_of(min(int(blockIdx.x), k.workers));
  k.stop = k.start_of(min(int(blockIdx.x) + 1, k.workers));
  int64_t at = before + sum - mine;
  if (k.unit >= at && k.unit < at + mine) {  // one thread, where there is a unit
    int b = tid * per;
    for (;; ++b) {
      const int64_t n = units_of(sequence_at(a, b));
      if (k.unit < at + n) break;
      at += n;
    }
    shared[0] = at;
    shared[1] = b;
  }
  __syncthreads();
  if (k.done()) return k;
  k.b = int(shared[1]);
  k.item_unit = shared[0];
  k.row_tile = 0;
  k.s = sequence_at(a, k.b);
  k.open(a, log2);
  while (k.unit >= k.item_unit + int64_t(k.ends + k.tiles) * a.c.heads) {
    k.item_unit += int64_t(k.ends + k.tiles) * a.c.heads;
    ++k.row_tile;
    k.open(a, log2);
  }
  const int each = k.ends + k.tiles;
  k.head = k.unit - k.item_unit < int64_t(1) << 31 ? int(uint32_t(k.unit - k.item_unit) / uint32_t(each)) : int((k.unit - k.item_unit) / each);
  k.item_unit += int64_t(k.head) * each;
  k.unit = max(k.unit, k.first_tile());
  k.tile = int(k.unit - k.first_tile());
  return k;
}

// Two bytes of a cached word as two float16, exactly.
template <int TYPE> struct Half2Of;
template <> struct Half2Of<DINOML_B200_KV_INT8> {
  // 1024 + value + 128 has the value + 128 in its last byte; 1152 is taken off again before any product: as part of the keys it would be in the scores' sums, whose
  // rounding then goes with 1152 times the sum of q instead of with the score.
  template <int LO, int HI> static __device__ __forceinline__ uint32_t pair(uint32_t w) {
    const uint32_t m = __byte_perm(w, 0x64646464u, 0x4040 | LO | (HI << 8));
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&m), __half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  // bytes 0, 1 and 2, 3; bytes 0, 2 and 1, 3
  static __device__ __forceinline__ void along(uint32_t w, uint32_t& a, uint32_t& b) {
    w ^= 0x80808080u;
    a = pair<0, 1>(w);
    b = pair<2, 3>(w);
  }
  static __device__ __forceinline__ void across(uint32_t w, uint32_t& a, uint32_t& b) {
    w ^= 0x80808080u;
    a = pair<0, 2>(w);
    b = pair<1, 3>(w);
  }
};
template <> struct Half2Of<DINOML_B200_KV_E4M3> {
  static __device__ __forceinline__ void along(uint32_t w, uint32_t& a, uint32_t& b) {
    asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}\n" : "=r"(a), "=r"(b) : "r"(w));
  }
  static __device__ __forceinline__ void across(uint32_t w, uint32_t& a, uint32_t& b) { along(__byte_perm(w, w, 0x3120), a, b); }
};

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

int attention_many(AttnParams& a, int type, cudaStream_t s);
int attention_few_int8(AttnParams& a, int tiles, cudaStream_t s);
int attention_few_e4m3(AttnParams& a, int tiles, cudaStream_t s);
void attention_reset();                      // counters of the current device, after a launch that gave up
float* attention_scratch(size_t floats, int ctas, cudaStream_t s, int** arrived);

}  // namespace kv
}  // namespace b200gguf

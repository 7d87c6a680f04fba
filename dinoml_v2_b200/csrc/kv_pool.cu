// Who has which blocks of the 8-bit cache: one step of all sequences, on the device, so that a captured step can begin a block, take tokens back and give a request up.
//
// kept = max(0, length - drop), blocks behind ceil(kept / size) go onto the stack of free ones, sequences whose new tokens fit take theirs from its top; starts are the running sum of
// the new tokens, and every packed row gets its position and slot.  All of it is a few reads a sequence, three running sums and 8 bytes a row: bound by latency.  One cluster:
// every CTA of it makes the sums over all sequences (a few hundred numbers, from L2), so that they need not meet for them, and has a part of the blocks and rows to write.
// They meet once: blocks that go back are on the stack before any is taken, and nobody writes lengths or the count before all have read them.
// 64 sequences with a token each 5.4 us, 256 5.7, 256 with 33,000 rows 9.7 (a row at a time 13.0; CTAs of 512 threads 11.5).  One CTA of 256 threads is as fast for 64 rows (5.2 us; 16 sequences
// with 60 rows each 6.1 and 6.7) and slower for more (256 sequences with one each 11.9, 64 with 16 each 11.3 and 7.4), so that there is none.
#include <algorithm>

#include "dependent_launch.cuh"
#include "kv_cache.cuh"

namespace b200gguf {
namespace kv {

constexpr int kPoolMaxSequences = 8192, kPoolCluster = 8, kPoolThreads = 1024;

struct PoolArgs {
  int *table, *lengths, *free_blocks, *free_count;
  const int *new_tokens, *drop;
  int *out_lengths, *starts, *positions, *slots, *status;
  int64_t table_stride;
  int table_blocks, sequences, blocks, block_log2, rows;
};

// Sums of S numbers over all threads of the CTA before this one (in v), and over all (in all).
template <int S, int NT> __device__ __forceinline__ void scan(int64_t (&v)[S], int64_t (&all)[S], int64_t (*shared)[NT / 32]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t own[S];
#pragma unroll
  for (int i = 0; i < S; ++i) {
    own[i] = v[i];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t u = __shfl_up_sync(0xffffffffu, v[i], o);
      if (lane >= o) v[i] += u;
    }
    if (lane == 31) shared[i][warp] = v[i];
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < S; ++i) {
    int64_t w = lane < NT / 32 ? shared[i][lane] : 0;
#pragma unroll
    for (int o = 1; o < NT / 32; o <<= 1) {
      const int64_t u = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += u;
    }
    const int64_t before = __shfl_sync(0xffffffffu, w, (warp + 31) & 31);
    v[i] += (warp > 0 ? before : 0) - own[i];
    all[i] = __shfl_sync(0xffffffffu, w, NT / 32 - 1);
  }
  __syncthreads();
}

// What one sequence asks for.
struct Wish {
  int64_t kept, fresh;      // tokens that stay, tokens that it would get
  int held, left, need;     // blocks before, with the kept tokens, for the new ones beside these
  bool bad;                 // a length or a count that is none
};
__device__ __forceinline__ Wish wish_of(const PoolArgs& a, int b) {
  Wish w;
  const int64_t most = int64_t(a.table_blocks) << a.block_log2;
  const int64_t length = a.lengths[b], fresh = a.new_tokens[b], drop = a.drop != nullptr ? a.drop[b] : 0;
  w.bad = length < 0 || length > most || fresh < 0 || drop < 0 || (a.starts == nullptr && fresh > 1);
  const int64_t old = min(max(length, int64_t(0)), most);
  w.kept = max(old - max(drop, int64_t(0)), int64_t(0));
  const int round = (1 << a.block_log2) - 1;
  w.held = int((old + round) >> a.block_log2);
  w.left = int((w.kept + round) >> a.block_log2);
  const bool fits = fresh > 0 && (a.starts != nullptr || fresh == 1) && w.kept + fresh <= most;
  w.fresh = fits ? fresh : 0;
  w.need = fits ? int((w.kept + fresh + round) >> a.block_log2) - w.left : 0;
  return w;
}

__device__ __forceinline__ void cluster_meet() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}

__global__ void __launch_bounds__(kPoolThreads) kv_pool_kernel(PoolArgs a) {
  constexpr int NT = kPoolThreads;
  extern __shared__ int of[];                              // of each sequence: first row, tokens kept, blocks taken and given back before its own
  __shared__ int64_t sums[3][NT / 32];
  int *first_row = of, *kept = of + a.sequences + 1, *taken = kept + a.sequences, *gone = taken + a.sequences;
  uint32_t rank, ctas;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
  wait_for_launch_before();
  const int tid = threadIdx.x, lane = tid & 31;
  const int each = (a.sequences + NT - 1) / NT, low = min(tid * each, a.sequences), high = min(low + each, a.sequences);
  const int count = min(max(a.free_count[0], 0), a.blocks);
  bool bad = count != a.free_count[0];

  int64_t v[3] = {0, 0, 0}, all[3];
  for (int b = low; b < high; ++b) {
    const Wish w = wish_of(a, b);
    bad |= w.bad;
    v[0] += w.held - w.left;
    v[1] += w.need;
    v[2] += w.fresh;
  }
  scan<3, NT>(v, all, sums);
  const int64_t back = all[0], available = min(count + back, int64_t(a.blocks));
  bad |= count + back > a.blocks;
  // which sequences get theirs, and the running sums of what is really taken
  int64_t u[2] = {0, 0}, got[2];
  int64_t blocks_before = v[1], rows_before = v[2], gone_before = v[0];
  for (int b = low; b < high; ++b) {
    const Wish w = wish_of(a, b);
    blocks_before += w.need;
    rows_before += w.fresh;
    const bool granted = w.fresh > 0 && (w.need == 0 || blocks_before <= available) && rows_before <= a.rows;
    if (granted) {
      u[0] += w.need;
      u[1] += w.fresh;
    }
    gone[b] = int(gone_before);
    gone_before += w.held - w.left;
    kept[b] = int(w.kept);
    first_row[b] = granted ? int(w.fresh) : 0;
    taken[b] = granted ? w.need : 0;
  }
  scan<2, NT>(u, got, sums);
  for (int b = low; b < high; ++b) {
    const int rows = first_row[b], need = taken[b];
    first_row[b] = int(u[1]);
    taken[b] = int(u[0]);
    u[0] += need;
    u[1] += rows;
  }
  if (tid == 0) first_row[a.sequences] = int(got[1]);
  __syncthreads();

  // Blocks that go back, by a warp a sequence.  The last sequence's last block is the lowest of them.
  const int warp = int(rank) * (NT / 32) + (tid >> 5), warps = int(ctas) * (NT / 32);
  const int round = (1 << a.block_log2) - 1;
  for (int b = warp; b < a.sequences; b += warps) {
    const Wish w = wish_of(a, b);
    const int64_t top = count + (back - gone[b]) - 1;      // where its first one comes
    int* row = a.table + int64_t(b) * a.table_stride;
    for (int j = w.left + lane; j < w.held; j += 32) {
      const int64_t at = top - (j - w.left);
      const int id = row[j];
      bad |= unsigned(id) >= unsigned(a.blocks);
      if (at >= 0 && at < a.blocks) a.free_blocks[at] = id;
      row[j] = -1;
    }
  }
  if (__syncthreads_or(bad) && tid == 0) flag_range(a.status);
  cluster_meet();

  // Blocks that are taken, by a warp a sequence.
  for (int b = warp; b < a.sequences; b += warps) {
    const int rows = first_row[b + 1] - first_row[b];
    if (lane == 0) {
      a.lengths[b] = kept[b] + rows;
      a.out_lengths[b] = rows > 0 ? kept[b] + rows : 0;
      if (a.starts != nullptr) a.starts[b] = first_row[b];
    }
    const int left = (kept[b] + round) >> a.block_log2, last = (kept[b] + rows + round) >> a.block_log2;
    int* row = a.table + int64_t(b) * a.table_stride;
    for (int j = left + lane; j < last; j += 32) {
      const int id = __ldcg(a.free_blocks + (available - 1 - (taken[b] + j - left)));
      if (unsigned(id) >= unsigned(a.blocks)) flag_range(a.status);
      row[j] = id;
    }
  }
  if (rank == 0 && tid == 0) {
    a.free_count[0] = int(available - got[0]);
    if (a.starts != nullptr) a.starts[a.sequences] = int(got[1]);
  }
  // Positions and slots of the rows; the block of one comes from the stack where it was taken in this step.
  // Some rows at once, whose searches and reads go side by side.
  constexpr int kRows = 4;
  const int64_t step = int64_t(ctas) * NT;
  for (int64_t row = int64_t(rank) * NT + tid; row < a.rows; row += kRows * step) {
    int b[kRows], position[kRows], id[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int64_t r = row + i * step;
      b[i] = -1;
      position[i] = -1;
      if (r >= a.rows) continue;
      if (a.starts == nullptr) {
        if (first_row[r + 1] > first_row[r]) b[i] = int(r);
      } else if (r < got[1]) {
        b[i] = 0;
      }
    }
    if (a.starts != nullptr) {                             // the last sequence whose first row is not behind it (one without rows has the next one's)
      for (int span = a.sequences; span > 1;) {
        const int half = span >> 1;
#pragma unroll
        for (int i = 0; i < kRows; ++i)
          if (b[i] >= 0 && first_row[b[i] + half] <= int(row + i * step)) b[i] += half;
        span -= half;
      }
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      id[i] = -1;
      if (b[i] < 0) continue;
      position[i] = kept[b[i]] + (a.starts != nullptr ? int(row + i * step) - first_row[b[i]] : 0);
      const int j = position[i] >> a.block_log2, left = (kept[b[i]] + round) >> a.block_log2;
      id[i] = j < left ? a.table[int64_t(b[i]) * a.table_stride + j] : __ldcg(a.free_blocks + (available - 1 - (taken[b[i]] + j - left)));
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int64_t r = row + i * step;
      if (r >= a.rows) break;
      a.positions[r] = position[i];
      a.slots[r] = unsigned(id[i]) < unsigned(a.blocks) ? (id[i] << a.block_log2) + (position[i] & round) : -1;
    }
  }
}

int pool_step(const DinoB200KvPool* pool, const int* new_tokens, const int* drop, int rows, int* lengths, int* starts, int* positions, int* slots, cudaStream_t s) {
  if (pool == nullptr || pool->block_table == nullptr || pool->lengths == nullptr || pool->free_blocks == nullptr || pool->free_count == nullptr || new_tokens == nullptr ||
      lengths == nullptr || positions == nullptr || slots == nullptr)
    return RC_NULL;
  if (pool->sequences <= 0 || pool->blocks <= 0 || pool->table_blocks <= 0 || rows < 0) return RC_DIMS;
  int log2 = 4;
  while (log2 < 7 && (1 << log2) != pool->block_size) ++log2;
  if ((1 << log2) != pool->block_size || pool->sequences > kPoolMaxSequences) return RC_RANGE;
  if ((pool->table_stride < pool->table_blocks && pool->sequences > 1) || (starts == nullptr && rows != pool->sequences)) return RC_RANGE;
  if ((int64_t(pool->blocks) << log2) > INT32_MAX || (int64_t(pool->table_blocks) << log2) > INT32_MAX) return RC_RANGE;
  int* status = status_words();
  if (status == nullptr) return RC_LAUNCH;
  const PoolArgs a{pool->block_table, pool->lengths, pool->free_blocks, pool->free_count, new_tokens, drop, lengths, starts, positions, slots, status, pool->table_stride,
                   pool->table_blocks, pool->sequences, pool->blocks, log2, rows};
  const size_t shared = (4 * size_t(pool->sequences) + 1) * sizeof(int);
  static std::atomic<uint64_t> done{0};
  if (int rc = allow_shared(kv_pool_kernel, (4 * size_t(kPoolMaxSequences) + 1) * sizeof(int), done)) return rc;
  return launch_dependent(kv_pool_kernel, dim3(kPoolCluster), kPoolThreads, shared, kPoolCluster, s, a);
}

}  // namespace kv
}  // namespace b200gguf

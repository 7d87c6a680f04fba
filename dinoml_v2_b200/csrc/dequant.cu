// Standalone GGUF dequantize kernel: packed blocks -> dense f32 / f16 / bf16, bit-exact.
//
// Replaces the un-vendored libgguf device entry the reference's generated module declares at
// src/dinoml/templates/gpu_module.cu.j2:35-42 and calls from src/dinoml/lowering/ops/gemm.py:745,
// keeping its name and argument list so the generated launch text links unchanged.
//
// HBM-bound and write-dominated (Q4_K -> f32 writes 7.1 bytes per byte read).  One kernel for the nine types and three outputs: an item
// is R consecutive packed bytes and every run of R weights that they hold, so each packed byte is loaded once and each run is one
// streaming store of whole 32-byte sectors.  What was measured, [11008 x 4096] in a graph, buffers of more than the L2 in turn, before
// (one 8-weight unit per thread, or items with 8-weight runs, two per thread) -> now, us:
//                f16                          f32
//   Q4_K    20.5 -> 18.6  (6.2 TB/s)    42.7 -> 33.8  (6.1 TB/s)
//   Q5_K    28.9 -> 19.9                52.1 -> 34.7
//   Q6_K    25.0 -> 22.0                50.4 -> 35.9
//   Q8_0    28.7 -> 23.0                45.2 -> 36.8
//   Q4_0    21.3 -> 19.3                46.9 -> 33.2
//   Q2_K    18.9 -> 17.6                38.5 -> 32.2
//   Q3_K    23.5 -> 19.3                48.9 -> 33.3
//   MXFP4   24.7 -> 19.2                46.2 -> 32.9
//   NVFP4   24.8 -> 20.5                47.0 -> 32.9
// and [512 x 2048], where the launch counts: 2.1 - 2.9 -> 1.5 - 1.9 (f16), 2.8 - 4.7 -> 2.0 - 2.5 (f32).  Where it came from:
//   * a 256-bit store per run: as two 128-bit stores, each half fills its sectors (f32: 43 -> 34);
//   * four quants decoded at a time: masks and shifts for four bytes at once, then one byte permute (0x4B0000qq is 2^23 + q) and one exact
//     subtraction per weight instead of shift, mask and conversion (Q5_K 28.9 -> 20.7);
//   * words for blocks that start at any address, shifted into place, instead of bytes or halves (MXFP4 24.7 -> 19.9);
//   * programmatic dependent launch, 0.3 - 0.4 us per call: the next kernel's CTAs are let in once a CTA holds its packed bytes.  From the first
//     instruction on they would fill the SMs that happen to be free, and a small grid ends up uneven (Q2_K [2048 x 4096] 4.7 -> 5.2).
// Decoding uses explicitly rounded fp32 operations, those of decode8<QT> in its order (bit-exact).
#include "dequant_items.cuh"

namespace b200gguf {

constexpr int kDequantThreads = 256;

// Items per thread.  Two for 16-bit NVFP4, whose item is a single store of few instructions: [28672 x 8192] 96 us, 105 with one ([2048 x 4096]
// 5.1 / 5.0).  One elsewhere: Q8_0 [2048 x 4096] 5.8 -> 5.7 (f16), 8.8 -> 8.2 (f32), Q4_K 4.6 -> 5.2 with two.
template <int QT, typename T> constexpr int items_per_thread() { return QT == QTYPE_NVFP4 && sizeof(T) == 2 ? 2 : 1; }

// A: alignment of the packed buffer where all its blocks keep it (16: Q4_K and Q5_K; 4: also Q2_K and NVFP4), 1: any start and block size,
// 0: Q6_K from a 16-byte boundary, through shared memory.  An item of Q6_K is 3 misaligned pieces of its block; a CTA's 32 or 16 blocks
// in 16-byte loads first cost a barrier and save the rest: [11008 x 4096] f16 25.0 -> 22.0 us, f32 37.0 -> 35.9, [512 x 2048] f32 3.1 -> 2.4.
// The other types with odd blocks have shorter pieces and lose by it: Q8_0 f16 23.4 -> 24.5, Q3_K 19.3 -> 20.7, MXFP4 19.2 -> 20.9, Q4_0 equal.
template <int QT, typename T, int A>
__global__ void __launch_bounds__(kDequantThreads)
dequant_kernel(const uint8_t* in, T* __restrict__ out, int64_t total_items, int64_t first_edge, int64_t last_edge, bool wide) {
  using G = ItemGeom<QT, run_of<QT, T>()>;
  constexpr int kPer = items_per_thread<QT, T>();
  asm volatile("griddepcontrol.wait;\n" ::: "memory");          // the packed bytes may be the preceding kernel's output
  if constexpr (A == 0) {
    constexpr int kBlocks = kDequantThreads / G::kItems, kBytes = kBlocks * QTraits<QT>::kBytes, kVec = kBytes / 16;
    static_assert(kPer == 1 && kBytes % 16 == 0, "");
    __shared__ __align__(16) uint8_t stage[kBytes + 16];
    const int64_t blk0 = int64_t(blockIdx.x) * kBlocks, blocks = total_items / G::kItems;
    const uint8_t* src = in + blk0 * QTraits<QT>::kBytes;
    const int bytes = blocks - blk0 >= kBlocks ? kBytes : int(blocks - blk0) * QTraits<QT>::kBytes, vecs = bytes / 16;
#pragma unroll
    for (int i = 0; i < (kVec + kDequantThreads - 1) / kDequantThreads; ++i) {
      const int at = i * kDequantThreads + threadIdx.x;
      if (at < vecs) *reinterpret_cast<uint4*>(stage + 16 * at) = reinterpret_cast<const uint4*>(src)[at];
    }
    for (int at = 16 * vecs + threadIdx.x; at < bytes; at += kDequantThreads) stage[at] = src[at];
    __syncthreads();
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    const int blk = threadIdx.x / G::kItems, item = threadIdx.x % G::kItems;
    if (blk0 + blk < blocks) {
      Item<QT, T, A> one;
      one.load(stage + blk * QTraits<QT>::kBytes, item, false);
      one.emit(out + (blk0 + blk) * QTraits<QT>::kBlock, item, wide);
    }
  } else {
    const int64_t base = int64_t(blockIdx.x) * (kPer * kDequantThreads) + threadIdx.x;
    Item<QT, T, A> it[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int64_t at = base + i * kDequantThreads, blk = at / G::kItems;
      if (at < total_items) it[i].load(in + blk * QTraits<QT>::kBytes, int(at % G::kItems), blk == first_edge || blk == last_edge);
    }
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int64_t at = base + i * kDequantThreads, blk = at / G::kItems;
      if (at < total_items) it[i].emit(out + blk * QTraits<QT>::kBlock, int(at % G::kItems), wide);
    }
  }
}

template <int QT, typename T, int A>
static int launch_items(const void* in, void* out, int64_t weights, cudaStream_t stream) {
  using G = ItemGeom<QT, run_of<QT, T>()>;
  constexpr int kPer = items_per_thread<QT, T>();
  const int64_t items = weights / QTraits<QT>::kBlock * G::kItems, per_cta = int64_t(kDequantThreads) * kPer;
  const int64_t grid = (items + per_cta - 1) / per_cta;
  if (grid > 0x7fffffffLL) return RC_RANGE;
  // blocks whose first or last aligned word holds bytes outside the buffer (only A == 1 looks)
  const uintptr_t begin = reinterpret_cast<uintptr_t>(in);
  const int64_t blocks = weights / QTraits<QT>::kBlock, first_edge = begin & 3 ? 0 : -1;
  const int64_t last_edge = (begin + uintptr_t(blocks) * QTraits<QT>::kBytes) & 3 ? blocks - 1 : -1;
  const bool wide = (reinterpret_cast<uintptr_t>(out) & 31) == 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(grid));
  cfg.blockDim = dim3(kDequantThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, dequant_kernel<QT, T, A>, static_cast<const uint8_t*>(in), static_cast<T*>(out), items, first_edge,
                                           last_edge, wide);
  return e == cudaSuccess && cudaGetLastError() == cudaSuccess ? RC_OK : RC_LAUNCH;
}

template <int QT, typename T>
static int launch_dequant(const void* in, void* out, int64_t rows, int64_t n_per_row, cudaStream_t stream) {
  using G = ItemGeom<QT, run_of<QT, T>()>;
  const uintptr_t at = reinterpret_cast<uintptr_t>(in);
  if constexpr (G::kAlign == 16)
    if ((at & 15) == 0) return launch_items<QT, T, 16>(in, out, rows * n_per_row, stream);
  if constexpr (G::kAlign >= 4)
    if ((at & 3) == 0) return launch_items<QT, T, 4>(in, out, rows * n_per_row, stream);
  if constexpr (QT == QTYPE_Q6_K)
    if ((at & 15) == 0) return launch_items<QT, T, 0>(in, out, rows * n_per_row, stream);
  if constexpr (QT == QTYPE_Q4_K) return RC_ALIGN;                  // the entry has refused these
  else return launch_items<QT, T, 1>(in, out, rows * n_per_row, stream);
}

template <int QT>
static int launch_dequant_dtype(const void* in, void* out, int64_t rows, int64_t n_per_row, int out_dtype,
                                cudaStream_t stream) {
  switch (out_dtype) {
    case OUT_F32: return launch_dequant<QT, float>(in, out, rows, n_per_row, stream);
    case OUT_F16: return launch_dequant<QT, __half>(in, out, rows, n_per_row, stream);
    case OUT_BF16: return launch_dequant<QT, __nv_bfloat16>(in, out, rows, n_per_row, stream);
    default: return RC_DTYPE;
  }
}

int dequantize_rows(const void* dev_in, int64_t qtype, int64_t rows, int64_t n_per_row, int output_dtype,
                    void* dev_out, cudaStream_t stream) {
  if (dev_in == nullptr || dev_out == nullptr) return RC_NULL;
  if (rows <= 0 || n_per_row <= 0) return RC_DIMS;
  const int bs = qtype_block_size(qtype);
  if (bs == 0) return RC_QTYPE;
  if (n_per_row % bs) return RC_KBLOCK;
  const uintptr_t in_a = reinterpret_cast<uintptr_t>(dev_in), out_a = reinterpret_cast<uintptr_t>(dev_out);
  if ((in_a & uintptr_t(qtype_alignment(qtype) - 1)) || (out_a & 15)) return RC_ALIGN;
  switch (qtype) {
    case QTYPE_Q8_0: return launch_dequant_dtype<QTYPE_Q8_0>(dev_in, dev_out, rows, n_per_row, output_dtype, stream);
    case QTYPE_Q4_K: return launch_dequant_dtype<QTYPE_Q4_K>(dev_in, dev_out, rows, n_per_row, output_dtype, stream);
    case QTYPE_Q6_K: return launch_dequant_dtype<QTYPE_Q6_K>(dev_in, dev_out, rows, n_per_row, output_dtype, stream);
    case QTYPE_Q4_0: return launch_dequant_dtype<QTYPE_Q4_0>(dev_in, dev_out, rows, n_per_row, output_dtype, stream);
    case QTYPE_Q5_K: return launch_dequant_dtype<QTYPE_Q5_K>(dev_in, dev_out, rows, n_per_row, output_dtype, stream);
    case QTYPE_Q2_K: return launch_dequant_dtype<QTYPE_Q2_K>(dev_in, dev_out, rows, n_per_row, output_dtype, stream);
    case QTYPE_Q3_K: return launch_dequant_dtype<QTYPE_Q3_K>(dev_in, dev_out, rows, n_per_row, output_dtype, stream);
    case QTYPE_MXFP4: return launch_dequant_dtype<QTYPE_MXFP4>(dev_in, dev_out, rows, n_per_row, output_dtype, stream);
    case QTYPE_NVFP4: return launch_dequant_dtype<QTYPE_NVFP4>(dev_in, dev_out, rows, n_per_row, output_dtype, stream);
    default: return RC_QTYPE;
  }
}

}  // namespace b200gguf

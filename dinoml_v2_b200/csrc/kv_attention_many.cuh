// Attention of many rows per cached head (prompts, chunks of them) over the 8-bit cache, on tcgen05: bound by the products and by the exponentials, which
// take the same time (256 rows against 128 tokens, heads of 128: four MMAs of 512 cycles, 32768 exponentials at 16 a cycle).
//
// A CTA has 256 rows (token x head of the group, so a cached tile is read once for all heads that share it) as two tiles of 128, whose softmax and
// MMAs alternate: while one tile's warps take exponentials, the other one's products run.
//   * warps 0..3 and 4..7: softmax, a row of scores per thread, S_i from tensor memory, P_i back into the same columns;
//   * warps 8..11: K and V of the next tiles, 8 bits in global memory to float16 in shared memory (swizzled as the MMA reads them);
//   * warp 12: issues the MMAs, S_i = Q_i K^T from shared memory and O_i += P_i V with P_i from tensor memory; V stays [token][channel], an MN-major operand;
//   * warp 13: walks the CTA's items.
// 8-bit values are exact in float16, q is brought to [2^12, 2^13) by a power of two per row, so products and their float32 sums are those of the stored
// values.  The scale of a block's K multiplies the scores; that of its V goes into the exponent: with y = s + log2(vs), P = 2^(y - ref + 7) is
// what V is multiplied by, and the softmax's sum takes P / vs in float32.  ref is the row's largest y when it was last set; O is rescaled only when y
// outgrows it by 2^8, so that P stays below 2^15 and loses bits (as a float16 denormal) only below 2^-21 of that.
#pragma once
#include "kv_attention.cuh"

namespace b200gguf {
namespace kv {
namespace many {

constexpr int kRows = 128, kItemRows = 2 * kRows, kTile = 128, kLog2 = 7;      // rows of an MMA, of an item; cached tokens of a tile
constexpr int kThreads = 512, kSegments = 4, kScales = 4;
constexpr uint32_t kTmem = 512, kS = 0, kO = 256;                             // columns: S_i at 128 i, O_i at 256 + D i
constexpr float kGrow = 8.f, kUp = 7.f;

template <int D_> struct Shape {
  static constexpr int D = D_;
  static constexpr int kBlock = kRows * 128;                  // bytes of 128 rows of 64 float16
  static constexpr int kOperand = kBlock * (D / 64);          // of a tile of Q, K or V
  static constexpr size_t kSmem = 1024 + 6 * size_t(kOperand);
};

struct Segment {
  Sequence s;
  Item item;
  int b, head, tiles, tile0, tile1;
  int piece, c0, c1, piece0;                  // as in the kernel of few rows
};

struct Shared {
  uint64_t described[kSegments], closed[kSegments], q_ready;
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_ready[2], o_full[2], together, drain;
  Segment segments[kSegments];
  float4 scales[kScales][kTile / 16];         // of 16 tokens: K's scale, log2 of V's, 1 / V's, whether there is a block
  int64_t walk[2 + kThreads / 32];
  uint32_t tmem;
  int last, lost;
};

__device__ __forceinline__ bool wait(const AttnParams& a, Shared& sh, uint64_t* bar, uint32_t parity) {      // bounded; by a converged warp
  const uint32_t at = umma::smem_u32(bar);
  volatile int* lost = &sh.lost;
  bool ok = umma::mbar_test_wait(at, parity);
  for (uint32_t i = 0; i < kPolls && !ok; ++i) {
    ok = umma::mbar_try_wait(at, parity);
    if (!ok && (i & 255u) == 255u && *lost) break;
  }
  ok = __all_sync(0xffffffffu, ok) != 0;
  if (!ok && !*lost) {
    *lost = 1;
    atomicCAS(a.p.status, 0, ST_KV_TIMEOUT);
  }
  return ok;
}

__device__ __forceinline__ void tmem_ld32(uint32_t at, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
        "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
        "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(at)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t at, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};\n" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
      "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]),
      "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void umma_f16_ss(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(tmem_d), "l"(desc_a),
               "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}
// V as it lies: rows of tokens (K of the product), 64 channels (N) of 128 bytes, blocks of 64 channels one after the other.
__device__ __forceinline__ uint64_t smem_desc_mn(uint32_t addr, int block_bytes) {
  return uint64_t((addr & 0x3ffffu) >> 4) | (uint64_t(uint32_t(block_bytes) >> 4) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ void st_shared16(uint32_t at, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};\n" ::"r"(at), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }
// Address of 16 bytes (8 float16) of an operand tile: K-major rows of 64 values with the 128-byte swizzle, blocks of 64 columns one after the other.
__device__ __forceinline__ uint32_t operand_at(int row, int chunk) {
  return uint32_t((chunk >> 3) * (kRows * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
}

// ---- warp 13
__device__ __forceinline__ void walk_items(const AttnParams& a, Shared& sh, Walk w) {
  for (int segment = 0;; ++segment, w.next_item(a, kLog2)) {
    const int slot = segment % kSegments;
    if (!wait(a, sh, &sh.closed[slot], uint32_t(segment / kSegments + 1) & 1u)) return;
    const bool done = w.done();
    if ((threadIdx.x & 31) == 0) {
      Segment g;
      g.s = w.s; g.item = w.item;
      g.b = w.b; g.head = w.head; g.tiles = w.tiles;
      g.tile0 = done ? 0 : w.tile;
      g.tile1 = done ? 0 : int(min(int64_t(w.tiles), w.stop - w.item_unit));
      g.piece = -1; g.c0 = g.c1 = g.piece0 = 0;
      if (!done && (g.tile0 != 0 || g.tile1 != w.tiles)) {
        g.piece = 2 * int(blockIdx.x) + (w.item_unit + g.tile0 == w.start ? 0 : 1);
        g.c0 = w.owner(w.item_unit);
        g.c1 = w.owner(w.item_unit + w.tiles - 1);
        g.piece0 = 2 * g.c0 + (w.start_of(g.c0) >= w.item_unit ? 0 : 1);
      }
      sh.segments[slot] = g;
      umma::mbar_arrive(umma::smem_u32(&sh.described[slot]));
    }
    if (done) return;
  }
}

// A lane's values of a tile, to[0] and to[1] being the places of its first 16.  BIASED: K of int8 stays 1152 too large (Half2Of), which the rows' scores take
// off again.
template <int TYPE, class S, bool BIASED, int COPIES> __device__ __forceinline__ void store_operand(const uint4 (&x)[COPIES], uint32_t smem, const uint32_t (&to)[2]) {
  using H = Half2Of<TYPE>;
  constexpr int kStep = 32 / COPIES;
#pragma unroll
  for (int i = 0; i < COPIES; ++i) {
    uint32_t h[8];
    H::template along<BIASED>(x[i].x, h[0], h[1]);
    H::template along<BIASED>(x[i].y, h[2], h[3]);
    H::template along<BIASED>(x[i].z, h[4], h[5]);
    H::template along<BIASED>(x[i].w, h[6], h[7]);
    const uint32_t turn = kStep == 4 && (i & 1) != 0 ? 64u : 0u;         // rows 4..7 of eight
    const uint32_t at = smem + uint32_t(i * kStep * 128);
    st_shared16((at + to[0]) ^ turn, h[0], h[1], h[2], h[3]);
    st_shared16((at + to[1]) ^ turn, h[4], h[5], h[6], h[7]);
  }
  fence_async_smem();
  __syncwarp();
}

// ---- warps 8..11.  A warp has 32 tokens of every tile, in kCopies steps of kStep tokens, 16 values a lane.
template <int TYPE, class S>
__device__ __forceinline__ void convert_tiles(const AttnParams& a, Shared& sh, uint32_t k_smem, uint32_t v_smem) {
  constexpr int kChunks = S::D / 16, kStep = 32 / kChunks, kCopies = 32 / kStep;
  const int warp = (threadIdx.x >> 5) & 3, lane = threadIdx.x & 31, chunk = lane % kChunks;
  // Where eight lanes have one row of 128 values, those of its second half take the neighbouring row instead: their stores go to the other banks.
  const int row = lane / kChunks ^ (kChunks == 8 ? (lane >> 2) & 1 : 0);
  const int log2 = a.c.block_log2, mask = (1 << log2) - 1;
  uint32_t to[2];                                                       // of a lane's two times 8 float16 in the first step
#pragma unroll
  for (int h = 0; h < 2; ++h) to[h] = operand_at(32 * warp + row, 2 * chunk + h);
  int n = 0;
  for (int segment = 0;; ++segment) {
    const int slot = segment % kSegments;
    if (!wait(a, sh, &sh.described[slot], uint32_t(segment / kSegments) & 1u)) return;
    const Segment& sg = sh.segments[slot];
    const int tile0 = sg.tile0, tile1 = sg.tile1, low = sg.item.low, high = sg.item.high, base = (low >> kLog2) << kLog2, b = sg.b, head = sg.head;
    if (tile0 == tile1) return;
    // The block of this lane's half of the warp's tokens (lane / 16: the first or the last 16), as block x head, -1 if there is none.
    auto look_up = [&](int tile) {
      const int token = base + tile * kTile + 32 * warp + (lane & 16);
      if (tile >= tile1 || token >= high || token + 16 <= low) return -1;
      const int id = block_at(a.p, a.c.blocks, b, token >> log2);
      return id < 0 ? -1 : id * a.c.heads + head;
    };
    uint4 raw[2][kCopies];
    auto load = [&](uint4 (&x)[kCopies], int which, int tile, int first_bh, int second_bh) {
      const int token = base + tile * kTile + 32 * warp + row;           // (16 tokens from a multiple of 16 are in one block)
      const uint8_t* const data = a.c.data[which] + chunk * 16;
      const uint8_t *p0 = data + ((int64_t(first_bh) << log2) + (token & mask)) * S::D, *p1 = data + ((int64_t(second_bh) << log2) + ((token + 16) & mask)) * S::D - 16 * S::D;
#pragma unroll
      for (int i = 0; i < kCopies; ++i) {
        const bool first = i * kStep < 16;
        x[i] = make_uint4(0u, 0u, 0u, 0u);                              // (what nobody sees has to be finite: zeros)
        if ((first ? first_bh : second_bh) >= 0 && token + i * kStep >= low && token + i * kStep < high)
          x[i] = __ldg(reinterpret_cast<const uint4*>((first ? p0 : p1) + i * kStep * S::D));
      }
    };
    int now = look_up(tile0);
    load(raw[0], 0, tile0, __shfl_sync(0xffffffffu, now, 0), __shfl_sync(0xffffffffu, now, 16));
    for (int tile = tile0; tile < tile1; ++tile, ++n) {
      const int first_bh = __shfl_sync(0xffffffffu, now, 0), second_bh = __shfl_sync(0xffffffffu, now, 16);
      const int next = look_up(tile + 1);
      load(raw[1], 1, tile, first_bh, second_bh);
      float ks = 0.f, vs = 0.f;
      if (now >= 0) {
        ks = __ldg(a.c.scale[0] + now);
        vs = __ldg(a.c.scale[1] + now);
      }
      const uint32_t lap = uint32_t(n >> 1) & 1u;
      if (!wait(a, sh, &sh.k_empty[n & 1], lap ^ 1u)) return;
      if ((lane & 15) == 0) {
        const float v = vs < 0x1p-100f ? 0x1p-100f : vs;                // (a NaN stays)
        sh.scales[n % kScales][2 * warp + (lane >> 4)] = make_float4(ks, log2f(v), 1.f / v, now >= 0 ? 1.f : 0.f);
      }
      store_operand<TYPE, S, true>(raw[0], k_smem + uint32_t((n & 1) * S::kOperand), to);
      if (lane == 0) umma::mbar_arrive(umma::smem_u32(&sh.k_full[n & 1]));
      load(raw[0], 0, tile + 1, __shfl_sync(0xffffffffu, next, 0), __shfl_sync(0xffffffffu, next, 16));
      if (!wait(a, sh, &sh.v_empty[n & 1], lap ^ 1u)) return;
      store_operand<TYPE, S, false>(raw[1], v_smem + uint32_t((n & 1) * S::kOperand), to);
      if (lane == 0) umma::mbar_arrive(umma::smem_u32(&sh.v_full[n & 1]));
      now = next;
    }
    if (lane == 0) umma::mbar_arrive(umma::smem_u32(&sh.closed[slot]));
  }
}

// ---- warp 12
template <class S>
__device__ __forceinline__ void issue_mmas(const AttnParams& a, Shared& sh, uint32_t q_smem, uint32_t k_smem, uint32_t v_smem) {
  const uint32_t tmem = sh.tmem;
  const uint32_t idesc_s = (1u << 4) | (uint32_t(kTile >> 3) << 17) | (uint32_t(kRows >> 4) << 24);                    // float16, float32 sums
  const uint32_t idesc_o = (1u << 4) | (1u << 16) | (uint32_t(S::D >> 3) << 17) | (uint32_t(kRows >> 4) << 24);        // B is MN-major
  int n = 0;
  auto scores = [&](int i, int stage) {
    if (umma::elect_one()) {
      const uint64_t q = umma::smem_desc_sw128(q_smem + uint32_t(i * S::kOperand)), k = umma::smem_desc_sw128(k_smem + uint32_t(stage * S::kOperand));
#pragma unroll
      for (int s = 0; s < S::D / 16; ++s) {
        const uint64_t off = uint64_t(((s >> 2) * S::kBlock + (s & 3) * 32) >> 4);
        umma_f16_ss(tmem + kS + uint32_t(i * kTile), q + off, k + off, idesc_s, s != 0);
      }
      umma::umma_commit<false>(umma::smem_u32(&sh.s_full[i]), 0);
      if (i == 1) umma::umma_commit<false>(umma::smem_u32(&sh.k_empty[stage]), 0);
    }
    __syncwarp();
  };
  for (int segment = 0;; ++segment) {
    const int slot = segment % kSegments;
    if (!wait(a, sh, &sh.described[slot], uint32_t(segment / kSegments) & 1u)) return;
    const int tiles = sh.segments[slot].tile1 - sh.segments[slot].tile0;
    if (tiles == 0) return;
    if (!wait(a, sh, &sh.q_ready, uint32_t(segment) & 1u) || !wait(a, sh, &sh.k_full[n & 1], uint32_t(n >> 1) & 1u)) return;
    umma::tcgen05_fence_after();
    scores(0, n & 1);
    scores(1, n & 1);
    for (int j = 0; j < tiles; ++j, ++n) {
      const int stage = n & 1;
      if (!wait(a, sh, &sh.v_full[stage], uint32_t(n >> 1) & 1u)) return;
      for (int i = 0; i < 2; ++i) {
        if (!wait(a, sh, &sh.p_ready[i], uint32_t(n) & 1u)) return;
        umma::tcgen05_fence_after();
        if (umma::elect_one()) {
          const uint64_t v = smem_desc_mn(v_smem + uint32_t(stage * S::kOperand), S::kBlock);
#pragma unroll
          for (int s = 0; s < kTile / 16; ++s)
            umma::umma_f16_ts<false>(tmem + kO + uint32_t(i * S::D), tmem + kS + uint32_t(i * kTile + 8 * s), v + uint64_t((16 * 128 * s) >> 4), idesc_o,
                                     (j != 0 || s != 0) ? 1u : 0u);
          if (i == 1) umma::umma_commit<false>(umma::smem_u32(&sh.v_empty[stage]), 0);
          if (j + 1 == tiles) umma::umma_commit<false>(umma::smem_u32(&sh.o_full[i]), 0);
        }
        __syncwarp();
        if (j + 1 < tiles) {
          if (i == 0 && !wait(a, sh, &sh.k_full[stage ^ 1], uint32_t((n + 1) >> 1) & 1u)) return;
          umma::tcgen05_fence_after();
          scores(i, stage ^ 1);
        }
      }
    }
    if (umma::elect_one()) umma::mbar_arrive(umma::smem_u32(&sh.closed[slot]));
    __syncwarp();
  }
}

// Columns [32 c, 32 c + 32) of a tile's scores, in turn: f(c, registers), the next ones on their way meanwhile.
template <typename F> __device__ __forceinline__ void for_columns(uint32_t tmem_s, F f) {
  uint32_t r[2][32];
  tmem_ld32(tmem_s, r[0]);
  umma::tmem_ld_wait();
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    if (c < 3) tmem_ld32(tmem_s + uint32_t(32 * (c + 1)), r[(c + 1) & 1]);
    f(c, r[c & 1]);
    umma::tmem_ld_wait();
  }
}

// A row's tile: the largest score, the sums so far brought to it if it has outgrown them, weights into the scores' place.  EVERY: the row sees
// all of its columns, else those in [low, high) of blocks that are there.
template <class S, bool EVERY>
__device__ __forceinline__ void tile_weights(uint32_t tmem_s, uint32_t tmem_o, const float4* scales, float factor, float unbias, int low, int high, bool more,
                                             float& ref, float& l) {
  float top = -INFINITY;
  for_columns(tmem_s, [&](int c, const uint32_t (&r)[32]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float4 x = scales[2 * c + h];
      float m[4];
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        float s = __uint_as_float(r[16 * h + k]);
        if (!EVERY) s = x.w != 0.f && 32 * c + 16 * h + k >= low && 32 * c + 16 * h + k < high ? s : -INFINITY;
        m[k & 3] = k < 4 ? s : fmaxf(m[k & 3], s);
      }
      const float best = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])), f = x.x * factor;
      if (EVERY || best != -INFINITY) top = fmaxf(top, fmaf(best - unbias, f, x.y));
    }
  });
  const bool grow = top > ref + kGrow || (ref == -INFINITY && top != -INFINITY);
  if (__any_sync(0xffffffffu, grow)) {
    const float old = ref;
    if (grow) ref = top;
    if (more) {
      const float keep = grow ? exp2_approx(old - ref) : 1.f;           // (nothing so far: 2^-inf)
      l *= keep;
#pragma unroll 1
      for (int c = 0; c < S::D / 32; ++c) {
        uint32_t o[32];
        tmem_ld32(tmem_o + uint32_t(32 * c), o);
        umma::tmem_ld_wait();
#pragma unroll
        for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * keep);
        tmem_st32(tmem_o + uint32_t(32 * c), o);
      }
    }
  }
  const float bias = (ref == -INFINITY ? 0.f : -ref) + kUp;
  for_columns(tmem_s, [&](int c, const uint32_t (&r)[32]) {
    uint32_t p[16];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float4 x = scales[2 * c + h];
      const float f = x.x * factor, add = fmaf(-unbias, f, x.y + bias);
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int k = 0; k < 16; k += 2) {
        float w[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          w[j] = exp2_approx(fmaf(__uint_as_float(r[16 * h + k + j]), f, add));
          // what is not seen has no weight, whatever the block's scales are
          if (!EVERY) w[j] = x.w != 0.f && 32 * c + 16 * h + k + j >= low && 32 * c + 16 * h + k + j < high ? w[j] : 0.f;
          sum[j] += w[j];
        }
        p[8 * h + k / 2] = pack_half(w[0], w[1]);
      }
      const float both = sum[0] + sum[1];
      if (EVERY || both != 0.f) l = fmaf(both, x.z, l);
    }
    umma::tmem_st16(tmem_s + uint32_t(16 * c), p);                           // (behind the columns that are still to be read)
  });
}

// ---- warps 0..7: tile i of the item, a row per thread
template <int TYPE, class S>
__device__ __forceinline__ void softmax_rows(const AttnParams& a, Shared& sh, uint32_t q_smem) {
  constexpr int D = S::D, kPiece = kItemRows * (D + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, i = warp >> 2, my_row = 32 * (warp & 3) + lane;
  const uint32_t lanes = sh.tmem + (uint32_t(32 * (warp & 3)) << 16), tmem_s = lanes + kS + uint32_t(i * kTile), tmem_o = lanes + kO + uint32_t(i * D);
  int n = 0, meetings = 0;
  auto meet = [&] {
    __syncwarp();
    if (lane == 0) umma::mbar_arrive(umma::smem_u32(&sh.together));
    return wait(a, sh, &sh.together, uint32_t(meetings++) & 1u);
  };
  for (int segment = 0;; ++segment) {
    const int slot = segment % kSegments;
    if (!wait(a, sh, &sh.described[slot], uint32_t(segment / kSegments) & 1u)) return;
    const Segment& sg = sh.segments[slot];
    const int tile0 = sg.tile0, tile1 = sg.tile1;
    if (tile0 == tile1) return;
    const int r = sg.item.r0 + i * kRows + my_row;
    const bool mine = r < sg.item.r1;
    const int token = a.by_group(mine ? r : sg.item.r0), head = sg.head * a.group + (mine ? r : sg.item.r0) - token * a.group;
    const int64_t out_at = (int64_t(sg.s.row + token) * a.heads + head) * D;
    float factor, unbias = 0.f;
    {                                                                   // q of this row
      const int64_t at = int64_t(sg.s.row + token) * a.row_stride + int64_t(head) * a.head_stride;
      const bool wide = ((reinterpret_cast<uintptr_t>(a.q) | uint64_t(a.row_stride * 2) | uint64_t(a.head_stride * 2)) & 15) == 0;
      const uint16_t* src = static_cast<const uint16_t*>(a.q) + at;
      uint32_t x[D / 2];
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (mine) {
          if (wide) {
            v = __ldg(reinterpret_cast<const uint4*>(src + 8 * c));
          } else {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = uint32_t(src[8 * c + 2 * k]) | (uint32_t(src[8 * c + 2 * k + 1]) << 16);
            v = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
        x[4 * c] = v.x; x[4 * c + 1] = v.y; x[4 * c + 2] = v.z; x[4 * c + 3] = v.w;
      }
      uint32_t largest = 0;                                             // of the 16-bit magnitudes: their order is that of the values
#pragma unroll
      for (int k = 0; k < D / 2; ++k) largest = __vmaxu2(largest, x[k] & 0x7fff7fffu);
      largest = max(largest & 0xffffu, largest >> 16);
      const bool f16 = a.dtype == DINO_F16;
      const float top = f16 ? __half2float(__ushort_as_half(uint16_t(largest))) : __uint_as_float(largest << 16);
      const uint32_t e = __float_as_uint(top) >> 23;
      const bool plain = e == 0 || e == 255;
      const int shift = plain ? 0 : min(max(127 + 12 - int(e), -126), 126);
      const float up = __uint_as_float(uint32_t(127 + shift) << 23);
      const float sign = a.scale < 0.f ? -up : up;                      // scores' factors are not negative
      factor = fabsf(a.scale) * __uint_as_float(uint32_t(127 - shift) << 23);
      const uint32_t q = q_smem + uint32_t(i * S::kOperand);
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        uint32_t h[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t w = x[4 * c + k];
          float2 v;
          if (f16) v = __half22float2(*reinterpret_cast<const __half2*>(&w));
          else v = make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
          h[k] = pack_half(v.x * sign, v.y * sign);
          const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&h[k]));
          unbias += back.x + back.y;
        }
        st_shared16(q + operand_at(my_row, c), h[0], h[1], h[2], h[3]);
      }
      unbias *= Half2Of<TYPE>::kBias;                                   // K's of int8 are that much too large
      fence_async_smem();
      __syncwarp();
      if (lane == 0) umma::mbar_arrive(umma::smem_u32(&sh.q_ready));
    }
    const int position = sg.s.first + token;
    const int high = mine ? min(position + 1, sg.s.end) : 0, low = a.window > 0 ? max(0, position - a.window + 1) : 0;
    const int all_high = __reduce_min_sync(0xffffffffu, mine ? high : INT32_MAX), all_low = __reduce_max_sync(0xffffffffu, mine ? low : 0);
    const int base = (sg.item.low >> kLog2) << kLog2;
    float ref = -INFINITY, l = 0.f;
    bool lost = false;
    for (int tile = tile0; tile < tile1; ++tile, ++n) {
      if (!wait(a, sh, &sh.s_full[i], uint32_t(n) & 1u)) { lost = true; break; }
      umma::tcgen05_fence_after();
      const float4* const scales = sh.scales[n % kScales];
      const int token0 = base + tile * kTile;
      bool every = token0 >= all_low && token0 + kTile <= all_high;
#pragma unroll
      for (int g = 0; g < kTile / 16; ++g) every = every && scales[g].w != 0.f;
      if (every) tile_weights<S, true>(tmem_s, tmem_o, scales, factor, unbias, 0, 0, tile > tile0, ref, l);
      else tile_weights<S, false>(tmem_s, tmem_o, scales, factor, unbias, low - token0, high - token0, tile > tile0, ref, l);
      umma::tmem_st_wait();
      umma::tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) umma::mbar_arrive(umma::smem_u32(&sh.p_ready[i]));
    }
    if (lost) return;
    if (!wait(a, sh, &sh.o_full[i], uint32_t(segment) & 1u)) return;
    umma::tcgen05_fence_after();
    const float f = l == 0.f ? 0.f : 1.f / l;
    float* const part = a.partial + size_t(max(sg.piece, 0)) * kPiece + size_t(i * kRows + my_row) * D;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      uint32_t o[32];
      tmem_ld32(tmem_o + uint32_t(32 * c), o);
      umma::tmem_ld_wait();
      if (mine && sg.piece >= 0) {
#pragma unroll
        for (int k = 0; k < 32; k += 4)
          __stcg(reinterpret_cast<uint4*>(part + 32 * c + k), make_uint4(o[k], o[k + 1], o[k + 2], o[k + 3]));
      } else if (mine) {
        uint32_t h[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const float u = __uint_as_float(o[2 * k]) * f, v = __uint_as_float(o[2 * k + 1]) * f;
          if (a.dtype == DINO_F16) {
            h[k] = pack_half(u, v);
          } else {
            const __nv_bfloat162 x = __floats2bfloat162_rn(u, v);
            h[k] = *reinterpret_cast<const uint32_t*>(&x);
          }
        }
        uint4* dst = reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + out_at + 32 * c);
#pragma unroll
        for (int k = 0; k < 4; ++k) dst[k] = make_uint4(h[4 * k], h[4 * k + 1], h[4 * k + 2], h[4 * k + 3]);
      }
      __syncwarp();
    }
    umma::tcgen05_fence_before();
    if (sg.piece >= 0) {                                                // cut: the last of its CTAs to arrive adds the pieces up, in order
      if (mine) __stcg(reinterpret_cast<float2*>(a.partial + size_t(sg.piece) * kPiece + kItemRows * D) + (i * kRows + my_row), make_float2(ref, l));
      if (!meet()) return;
      if (threadIdx.x == 0) {
        int before = 0;
        asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;\n" : "=r"(before) : "l"(a.arrived + sg.c0) : "memory");
        sh.last = before == sg.c1 - sg.c0;
        if (sh.last) a.arrived[sg.c0] = 0;
      }
      if (!meet()) return;
      if (sh.last) {
        const int rows = sg.item.r1 - sg.item.r0, count = sg.c1 - sg.c0 + 1;
        constexpr int U = 4;                                            // places under way at a time
        for (int x0 = int(threadIdx.x); x0 < rows * (D / 4); x0 += 256 * U) {
          float high_ref[U], sum[U];
          float4 v[U];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            high_ref[u] = -INFINITY;
            sum[u] = 0.f;
            v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
          }
          for (int c = 0; c < count; ++c) {
            const float* src = a.partial + size_t(c == 0 ? sg.piece0 : 2 * (sg.c0 + c)) * kPiece;
            float2 ml[U];
            float4 y[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
              const int x = min(x0 + 256 * u, rows * (D / 4) - 1);
              ml[u] = __ldcg(reinterpret_cast<const float2*>(src + kItemRows * D) + x / (D / 4));
              y[u] = __ldcg(reinterpret_cast<const float4*>(src) + x);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
              const float next = fmaxf(high_ref[u], ml[u].x);
              const float f0 = high_ref[u] == -INFINITY ? 1.f : exp2_approx(high_ref[u] - next), f1 = ml[u].x == -INFINITY ? 1.f : exp2_approx(ml[u].x - next);
              sum[u] = fmaf(ml[u].y, f1, sum[u] * f0);
              v[u] = make_float4(fmaf(y[u].x, f1, v[u].x * f0), fmaf(y[u].y, f1, v[u].y * f0), fmaf(y[u].z, f1, v[u].z * f0), fmaf(y[u].w, f1, v[u].w * f0));
              high_ref[u] = next;
            }
          }
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int x = x0 + 256 * u, row = x / (D / 4), d = x % (D / 4) * 4;
            if (row >= rows) continue;
            const float inv = sum[u] == 0.f ? 0.f : 1.f / sum[u];
            const int t = a.by_group(sg.item.r0 + row), hd = sg.head * a.group + sg.item.r0 + row - t * a.group;
            const int64_t at = (int64_t(sg.s.row + t) * a.heads + hd) * D + d;
            uint2 h;
            if (a.dtype == DINO_F16) {
              h = make_uint2(pack_half(v[u].x * inv, v[u].y * inv), pack_half(v[u].z * inv, v[u].w * inv));
            } else {
              const __nv_bfloat162 lo = __floats2bfloat162_rn(v[u].x * inv, v[u].y * inv), hi = __floats2bfloat162_rn(v[u].z * inv, v[u].w * inv);
              h = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
            }
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at) = h;
          }
        }
      }
    }
    __syncwarp();
    if (lane == 0) umma::mbar_arrive(umma::smem_u32(&sh.closed[slot]));
  }
}

template <int TYPE, class S>
__global__ void __launch_bounds__(kThreads, 1) attention_many_kernel(const __grid_constant__ AttnParams a) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ Shared sh;
  const uint32_t smem = (umma::smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t q_smem = smem, k_smem = smem + 2 * S::kOperand, v_smem = smem + 4 * S::kOperand;
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kSegments; ++i) {
      umma::mbar_init(umma::smem_u32(&sh.described[i]), 1);
      umma::mbar_init(umma::smem_u32(&sh.closed[i]), 13);              // eight, four and one warps
    }
    umma::mbar_init(umma::smem_u32(&sh.q_ready), 8);
    for (int i = 0; i < 2; ++i) {
      umma::mbar_init(umma::smem_u32(&sh.k_full[i]), 4);
      umma::mbar_init(umma::smem_u32(&sh.v_full[i]), 4);
      umma::mbar_init(umma::smem_u32(&sh.k_empty[i]), 1);
      umma::mbar_init(umma::smem_u32(&sh.v_empty[i]), 1);
      umma::mbar_init(umma::smem_u32(&sh.s_full[i]), 1);
      umma::mbar_init(umma::smem_u32(&sh.p_ready[i]), 4);
      umma::mbar_init(umma::smem_u32(&sh.o_full[i]), 1);
    }
    umma::mbar_init(umma::smem_u32(&sh.together), 8);
    umma::mbar_init(umma::smem_u32(&sh.drain), 1);
    sh.lost = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  __syncwarp();
  if (warp == 12) umma::tmem_alloc<false>(umma::smem_u32(&sh.tmem), kTmem);
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  asm volatile("griddepcontrol.wait;\n" ::: "memory");                // nothing of the launches before is read before this
  umma::tcgen05_fence_before();
  const Walk first = walk_of<kThreads>(a, kLog2, 1, sh.walk);         // (its barriers: the inits and the allocation are visible)
  __syncthreads();
  umma::tcgen05_fence_after();
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 176;\n");            // 2 x 176 + 96 + 64 = 4 x 128
    softmax_rows<TYPE, S>(a, sh, q_smem);
  } else if (warp < 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;\n");
    convert_tiles<TYPE, S>(a, sh, k_smem, v_smem);
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;\n");
    if (warp == 12) {
      issue_mmas<S>(a, sh, q_smem, k_smem, v_smem);
      if (*static_cast<volatile int*>(&sh.lost)) {                     // given up: what has been issued finishes before tensor memory is freed
        if (umma::elect_one()) {
          umma::umma_commit<false>(umma::smem_u32(&sh.drain), 0);
          umma::mbar_wait_plain(umma::smem_u32(&sh.drain), 0);
        }
      }
      __syncwarp();
    } else if (warp == 13) {
      walk_items(a, sh, first);
    }
  }
  umma::tcgen05_fence_before();
  __syncthreads();
  if (warp == 12) {
    umma::tcgen05_fence_after();
    umma::tmem_dealloc<false>(sh.tmem, kTmem);
  }
}

template <int TYPE, int D> int launch(AttnParams& a, cudaStream_t s) {
  using S = Shape<D>;
  a.row_tile = kItemRows;
  a.row_tile_log2 = 8;
  const int ctas = stream::sm_count();
  a.partial = attention_scratch(size_t(ctas) * 2 * kItemRows * (D + 2), ctas, s, &a.arrived);
  if (a.partial == nullptr) return RC_LAUNCH;
  static SmemOptIn opt;
  auto kern = attention_many_kernel<TYPE, S>;
  if (!smem_opt_in(kern, S::kSmem, opt)) return RC_LAUNCH;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, a) == cudaSuccess ? RC_OK : RC_LAUNCH;
}

}  // namespace many
}  // namespace kv
}  // namespace b200gguf

// Attention of many rows per cached head (prompts, chunks of them) over the 8-bit cache, on tcgen05: bound by the products and by the exponentials, which
// take the same time (256 rows against 64 tokens, heads of 128: four MMAs of 256 cycles, 16384 exponentials at 16 a cycle).
//
// A CTA has 256 rows (token x head of the group, so a cached tile is read once for all heads that share it) as two tiles of 128.  The scores of a tile
// have two places in tensor memory: the next ones are there when the softmax of a tile is done, which so never waits for products.
//   * warps 0..3 and 4..7: softmax, a row of scores per thread, S_i from tensor memory, P_i back into the same columns;
//   * warps 8..11: K and V of the next tiles, 8 bits in global memory to float16 in shared memory (swizzled as the MMA reads them);
//   * heads of 256 and float32 (q and P in two float16 terms, the second one's MMAs behind the first's into the same sums): one tile of 128 rows, warps 4..7 convert too;
//   * warp 12: issues the MMAs, S_i = Q_i K^T from shared memory and O_i += P_i V with P_i from tensor memory; V stays [token][channel], an MN-major operand;
//   * warp 13: walks the CTA's items.
// 8-bit values are exact in float16, q is brought to [2^12, 2^13) by a power of two per row, so products and their float32 sums are those of the stored
// values.  The scale of a block's K multiplies the scores; that of its V goes into the exponent: with y = s + log2(vs), P = 2^(y - ref + 7) is
// what V is multiplied by, and the softmax's sum takes P / vs in float32.  ref is the row's largest y when it was last set; O is rescaled only when y
// outgrows it by 2^8, so that P stays below 2^15 and loses bits (as a float16 denormal) only below 2^-21 of that: a channel in which all larger weights meet zeros is what
// shows it.  (Twelve binades above ref and three of growth would keep weights down to 2^-26; 2048 tokens after 6144 took 329 us so instead of 310 on one GPU, chunks of up to 300
// tokens 106 instead of 94, since O is rescaled more often.)  A scale of V below 2^-100 counts as 2^-100, so that its logarithm leaves the exponent room: values are then 4e-28 off at most.
//
// Measured, int8, blocks of 64, 2048 tokens after 6144, 32 heads on 8 cached ones, launches one after the other on three sets of inputs: heads of 128 292 us (822 TFLOP/s), of 256
// 577 to 591 us (820), of 64 240 us (501), float32 of 128 512 to 530 us, of 64 393 us.  A tile of 64 tokens takes 2015 cycles: MMAs 1415 of them (scores 940, 64 columns being bound by shared memory; P V 516), the softmax warps 1100 and the wait for scores.
#pragma once
#include <type_traits>

#include "kv_attention.cuh"

namespace b200gguf {
namespace kv {
namespace many {

constexpr int kRows = 128, kTile = 64, kLog2 = 6;                             // rows of an MMA; cached tokens of a tile
constexpr int kThreads = 512, kSegments = 4;
// A stage is V of a tile and K of the tile two behind it, which the MMAs read one after the other: one barrier for both.  Items begin at stage 0 (the
// last ones of an item may be empty): addresses of the MMAs are constants, and S of a tile is in the place that its stage's number says.
constexpr int kAhead = 2, kMostStages = 4, kScales = 8;                       // stages in shared memory; tiles whose scales are kept
constexpr uint32_t kTmem = 512, kO = 256;                                     // columns: S_i of even and odd tiles at 128 i and 128 i + 64, O_i at 256 + D i
// An item's q, its results and, where it is cut, the pieces' way through memory take as long as some tiles do: counted as none a CTA with ends of many items was
// the last one by far (chunks of up to 300 tokens in 8 sequences 126 us, with 4 to 12 tiles 113, 100, 104, 100; 2048 tokens after 6144 317, 308, 306, 306, 306).
constexpr int kEnds = 8, kLeast = 12;          // in tiles; units that a CTA takes at least
constexpr float kGrow = 8.f, kUp = 7.f;
constexpr unsigned kPolynomial = 0x11;      // of eight pairs of exponentials, those that the FMA units take: the special function units are the bound
                                             // (none 380 us, these two 342, four 347, all 429 for the prompt above at an earlier state of the rest)

// PARTS: float16 terms of a q and of a weight, 2 for float32 activations.  Shared memory has room for two tiles of rows where q takes 256 bytes a row, for
// one tile beyond; the warps that had the other one are converters then.
template <int D_, int PARTS_> struct Shape {
  static constexpr int D = D_, PARTS = PARTS_;
  static constexpr int kTiles = PARTS == 1 && D <= 128 ? 2 : 1, kStages = D <= 128 ? kMostStages : 2, kConverters = kTiles == 2 ? 4 : 8;
  static constexpr int kItemRows = kTiles * kRows, kPiece = kItemRows * (D + 2);      // rows of an item; floats of a piece
  static constexpr int kQ = kRows * D * PARTS * 2, kKv = kTile * D * 2;               // bytes of a tile of Q, of K or V
  static constexpr size_t kSmem = 1024 + size_t(kTiles) * kQ + 2 * kStages * size_t(kKv);
};

struct Segment {
  Sequence s;
  Item item;
  int b, head, tiles, tile0, tile1;
  int piece, c0, c1, piece0;                  // as in the kernel of few rows
};

struct Shared {
  uint64_t described[kSegments], closed[kSegments], q_ready;
  uint64_t full[kMostStages], empty[kMostStages];
  uint64_t s_full[2][2], p_ready[2][2], together, drain;    // of row tile i, even and odd stages: its MMAs are done, its weights are there
  Segment segments[kSegments];
  float4 scales[kScales][kTile / 16];         // of 16 tokens: K's scale, log2 of V's, 1 / V's, whether there is a block
  int4 whole[kScales];                        // of 16 tokens each: whether there is a block
  int64_t walk[2 + kThreads / 32];
  uint32_t tmem;
  int last, lost;
};

template <class S> __device__ __forceinline__ int stages_of(int tiles) { return (tiles + kAhead + S::kStages - 1) / S::kStages * S::kStages; }

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
    flag_timeout(a.p.status);
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
// MMAs whose operands lie A_OFF, B_OFF (in 16 bytes) behind a descriptor's address.  The sums are made beside each MMA: as constants of an unrolled loop
// they become hundreds of registers, and the issuing warp, which everything waits for, spills.
template <int A_OFF, int B_OFF> __device__ __forceinline__ void umma_f16_ss(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\tadd.s64 a, %1, %5;\n\tadd.s64 b, %2, %6;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}\n" ::"r"(tmem_d),
               "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "n"(A_OFF), "n"(B_OFF) : "memory");
}
template <int A_OFF, int B_OFF> __device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t.reg .b32 a;\n\tadd.s32 a, %1, %5;\n\tadd.s64 b, %2, %6;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [a], b, %3, p;\n\t}\n" ::"r"(tmem_d),
               "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "n"(A_OFF), "n"(B_OFF) : "memory");
}
// O += P V and S = Q K^T of a stage, step by step of sixteen.  Terms: those of the weights lie one after the other, those of q step by step.
template <class S, int I> __device__ __forceinline__ void issue_weights(uint32_t tmem_o, uint32_t tmem_p, uint64_t v, uint32_t idesc, bool more) {
  umma_f16_ts<8 * I, (16 * 128 * (I % (kTile / 16))) / 16>(tmem_o, tmem_p, v, idesc, more || I != 0 ? 1u : 0u);
  if constexpr (I + 1 < S::PARTS * kTile / 16) issue_weights<S, I + 1>(tmem_o, tmem_p, v, idesc, more);
}
template <class S, int I> __device__ __forceinline__ void issue_scores(uint32_t tmem_s, uint64_t q, uint64_t k, uint32_t idesc) {
  constexpr int J = I / S::PARTS;
  umma_f16_ss<((I >> 2) * kRows * 128 + (I & 3) * 32) / 16, ((J >> 2) * kTile * 128 + (J & 3) * 32) / 16>(tmem_s, q, k, idesc, I != 0);
  if constexpr (I + 1 < S::PARTS * S::D / 16) issue_scores<S, I + 1>(tmem_s, q, k, idesc);
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
__device__ __forceinline__ uint4 lds128(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }
// Address of 16 bytes (8 float16) of an operand tile of ROWS rows: rows of 64 values with the 128-byte swizzle, blocks of 64 columns one after the other.
template <int ROWS> __device__ __forceinline__ uint32_t operand_at(int row, int chunk) {
  return uint32_t((chunk >> 3) * (ROWS * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
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
      g.tile1 = done ? 0 : w.end_tile();
      g.piece = -1; g.c0 = g.c1 = g.piece0 = 0;
      if (!done && (g.tile0 != 0 || g.tile1 != w.tiles)) {
        g.piece = w.piece();
        g.c0 = w.owner(w.first_tile());
        g.c1 = w.owner(w.first_tile() + w.tiles - 1);
        g.piece0 = w.first_piece(g.c0);
      }
      sh.segments[slot] = g;
      umma::mbar_arrive(umma::smem_u32(&sh.described[slot]));
    }
    if (done) return;
  }
}

// A lane's values of a tile, to[0] and to[1] being the places of its first 16.
template <int TYPE, int COPIES> __device__ __forceinline__ void store_operand(const uint4 (&x)[COPIES], uint32_t smem, const uint32_t (&to)[2]) {
  using H = Half2Of<TYPE>;
  constexpr int kStep = 16 / COPIES;
#pragma unroll
  for (int i = 0; i < COPIES; ++i) {
    uint32_t h[8];
    H::along(x[i].x, h[0], h[1]);
    H::along(x[i].y, h[2], h[3]);
    H::along(x[i].z, h[4], h[5]);
    H::along(x[i].w, h[6], h[7]);
    const uint32_t turn = kStep == 4 && (i & 1) != 0 ? 64u : 0u;         // rows 4..7 of eight
    const uint32_t at = smem + uint32_t(i * kStep * 128);
    st_shared16((at + to[0]) ^ turn, h[0], h[1], h[2], h[3]);
    st_shared16((at + to[1]) ^ turn, h[4], h[5], h[6], h[7]);
  }
}

// ---- the converters, up to warp 11.  A warp has 16 tokens of every tile, which are of one block, and kChannels of their channels, in kCopies steps of kStep
// tokens, 16 values a lane.
template <int TYPE, class S>
__device__ __forceinline__ void convert_tiles(const AttnParams& a, Shared& sh, uint32_t k_smem, uint32_t v_smem) {
  constexpr int kStages = S::kStages, kChannels = 4 * S::D / S::kConverters, kChunks = kChannels / 16, kStep = 32 / kChunks, kCopies = 16 / kStep;
  const int warp = (threadIdx.x >> 5) & 3, part = (threadIdx.x >> 5) - (12 - S::kConverters) >= 4, lane = threadIdx.x & 31, chunk = lane % kChunks;
  // Where eight lanes have one row of 128 values, those of its second half take the neighbouring row instead: their stores go to the other banks.
  const int row = lane / kChunks ^ (kChunks == 8 ? (lane >> 2) & 1 : 0);
  const int log2 = a.c.block_log2, mask = (1 << log2) - 1;
  uint32_t to[2];                                                       // of a lane's two times 8 float16 in the first step
#pragma unroll
  for (int h = 0; h < 2; ++h) to[h] = operand_at<kTile>(16 * warp + row, part * (kChannels / 8) + 2 * chunk + h);
  int n = 0, first = 0;                                                 // stages so far; tiles before this item's
  for (int segment = 0;; ++segment) {
    const int slot = segment % kSegments;
    if (!wait(a, sh, &sh.described[slot], uint32_t(segment / kSegments) & 1u)) return;
    const Segment& sg = sh.segments[slot];
    const int tile0 = sg.tile0, tile1 = sg.tile1, low = sg.item.low, high = sg.item.high, base = (low >> kLog2) << kLog2, b = sg.b, head = sg.head;
    if (tile0 == tile1) return;
    auto look_up = [&](int tile) {                                      // the warp's block, as block x head, -1 if there is none
      const int token = base + tile * kTile + 16 * warp;
      if (tile >= tile1 || token >= high || token + 16 <= low) return -1;
      const int id = block_at(a.p, a.c.blocks, b, token >> log2);
      return id < 0 ? -1 : id * a.c.heads + head;
    };
    uint4 raw[2][kCopies];
    auto load = [&](uint4 (&x)[kCopies], int which, int tile, int bh) {
      const int token = base + tile * kTile + 16 * warp + row;
      const uint8_t* const from = a.c.data[which] + part * kChannels + chunk * 16 + ((int64_t(bh) << log2) + (token & mask)) * S::D;
#pragma unroll
      for (int i = 0; i < kCopies; ++i) {
        x[i] = make_uint4(0u, 0u, 0u, 0u);                              // (what nobody sees has to be finite: zeros)
        if (bh >= 0 && token + i * kStep >= low && token + i * kStep < high) x[i] = fetch(reinterpret_cast<const uint4*>(from + i * kStep * S::D));
      }
    };
    // Stage u of an item has K of tile u and V of tile u - kAhead.  All that it is made of was asked for while the one before was stored.
    const int tiles = tile1 - tile0;
    int bh[kAhead + 2];                                                 // of tiles u - kAhead .. u + 1
#pragma unroll
    for (int i = 0; i < kAhead; ++i) bh[i] = -1;
    bh[kAhead] = look_up(tile0);
    bh[kAhead + 1] = look_up(tile0 + 1);
    float ks = 0.f, vs = 0.f;                                           // of tile u
    auto load_k = [&](int tile, int at) {
      load(raw[0], 0, tile, at);
      ks = vs = 0.f;
      if (at >= 0) {
        ks = fetch(a.c.scale[0] + at);
        vs = fetch(a.c.scale[1] + at);
      }
    };
    load_k(tile0, bh[kAhead]);
    for (int u = 0; u < stages_of<S>(tiles); ++u, ++n) {
      const int after = look_up(tile0 + u + 2), stage = n % kStages;
      if (!wait(a, sh, &sh.empty[stage], (uint32_t(n / kStages) & 1u) ^ 1u)) return;
      if (u < tiles) {
        const int at = (first + u) % kScales;
        if (lane == 0 && part == 0) {
          const float v = vs < 0x1p-100f ? 0x1p-100f : vs;              // (a NaN stays)
          sh.scales[at][warp] = make_float4(ks, __log2f(v), __fdividef(1.f, v), bh[kAhead] >= 0 ? 1.f : 0.f);
          reinterpret_cast<int*>(&sh.whole[at])[warp] = bh[kAhead] >= 0;
        }
        store_operand<TYPE>(raw[0], k_smem + uint32_t(stage * S::kKv), to);
      }
      load_k(tile0 + u + 1, bh[kAhead + 1]);
      if (u >= kAhead && u < tiles + kAhead) store_operand<TYPE>(raw[1], v_smem + uint32_t(stage * S::kKv), to);
      if (u + 1 >= kAhead) load(raw[1], 1, tile0 + u + 1 - kAhead, bh[1]);
      fence_async_smem();
      __syncwarp();
      if (lane == 0) umma::mbar_arrive(umma::smem_u32(&sh.full[stage]));
#pragma unroll
      for (int i = 0; i <= kAhead; ++i) bh[i] = bh[i + 1];
      bh[kAhead + 1] = after;
    }
    first += tiles;
    if (lane == 0) umma::mbar_arrive(umma::smem_u32(&sh.closed[slot]));
  }
}

// ---- warp 12
template <class S>
__device__ __forceinline__ void issue_mmas(const AttnParams& a, Shared& sh, uint32_t q_smem, uint32_t k_smem, uint32_t v_smem) {
  const uint32_t tmem = sh.tmem;
  const uint32_t idesc_s = (1u << 4) | (uint32_t(kTile >> 3) << 17) | (uint32_t(kRows >> 4) << 24);                    // float16, float32 sums
  const uint32_t idesc_o = (1u << 4) | (1u << 16) | (uint32_t(S::D >> 3) << 17) | (uint32_t(kRows >> 4) << 24);        // B is MN-major
  const uint64_t q0 = umma::smem_desc_sw128(q_smem), k0 = umma::smem_desc_sw128(k_smem), v0 = smem_desc_mn(v_smem, kTile * 128);
  int n = 0;                                                            // stages so far, a multiple of kStages
  uint32_t weights = 0;                                                 // phases of p_ready, a bit for even and one for odd stages
  for (int segment = 0;; ++segment) {
    const int slot = segment % kSegments;
    if (!wait(a, sh, &sh.described[slot], uint32_t(segment / kSegments) & 1u)) return;
    const int tiles = sh.segments[slot].tile1 - sh.segments[slot].tile0;
    if (tiles == 0) return;
    if (!wait(a, sh, &sh.q_ready, uint32_t(segment) & 1u)) return;
    for (int u = 0; u < stages_of<S>(tiles); ++u, ++n) {
      const int stage = u % S::kStages, j = u - kAhead;                 // K of tile u, V of tile j
      const uint64_t k = k0 + uint64_t(uint32_t(stage * S::kKv) >> 4), v = v0 + uint64_t(uint32_t(stage * S::kKv) >> 4);
      if (!wait(a, sh, &sh.full[stage], uint32_t(n / S::kStages) & 1u)) return;
#pragma unroll
      for (int i = 0; i < S::kTiles; ++i) {
        if (j >= 0 && j < tiles && !wait(a, sh, &sh.p_ready[i][u & 1], (weights >> (u & 1)) & 1u)) return;
        umma::tcgen05_fence_after();
        if (umma::elect_one()) {
          const uint32_t scores = tmem + uint32_t(i * 128 + (u & 1) * 64);
          if (j >= 0 && j < tiles) issue_weights<S, 0>(tmem + kO + uint32_t(i * S::D), scores, v, idesc_o, j != 0);
          if (u < tiles) issue_scores<S, 0>(scores, q0 + uint64_t((i * S::kQ) >> 4), k, idesc_s);      // into the place of the weights just read
          // (Not at the empty stages behind an item's last products: nothing there waits for the softmax, so that a phase of the barrier could pass it by.)
          if (j < tiles) umma::umma_commit<false>(umma::smem_u32(&sh.s_full[i][u & 1]), 0);
          if (i == S::kTiles - 1) umma::umma_commit<false>(umma::smem_u32(&sh.empty[stage]), 0);
        }
        __syncwarp();
      }
      if (j >= 0 && j < tiles) weights ^= 1u << (u & 1);
    }
    if (umma::elect_one()) umma::mbar_arrive(umma::smem_u32(&sh.closed[slot]));
    __syncwarp();
  }
}

// Two float32 in a register pair.
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(v) : "f"(lo), "f"(hi));
  return v;
}
__device__ __forceinline__ float2 halves_of(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;\n" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t v;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(v) : "l"(a), "l"(b), "l"(c));
  return v;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t v;
  asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(v) : "l"(a), "l"(b));
  return v;
}
__device__ __forceinline__ float max3_or_nan(float a, float b, float c) {
  float v;
  asm("max.NaN.f32 %0, %1, %2, %3;\n" : "=f"(v) : "f"(a), "f"(b), "f"(c));
  return v;
}

// 2^x of two numbers below 2^7 without the special function unit: x = n + f with n the nearest integer (its bits are the last ones of x + 1.5 2^23), a
// polynomial of degree four for 2^f on [-1/2, 1/2] (Remez exchange, relative error 2.6e-6), n added to its exponent.  Below 2^-126: 2^-126, and so is a NaN, which
// the caller has to look for.
__device__ __forceinline__ float2 exp2_pair(uint64_t x) {
  const float2 raw = halves_of(x);
  x = pair_of(fmaxf(raw.x, -126.f), fmaxf(raw.y, -126.f));
  constexpr float kRound = 12582912.f;
  const uint64_t t = add2(x, pair_of(kRound, kRound)), n = add2(t, pair_of(-kRound, -kRound)), f = fma2(n, pair_of(-1.f, -1.f), x);
  uint64_t p = fma2(f, pair_of(0.009570102207362652f, 0.009570102207362652f), pair_of(0.05591785907745361f, 0.05591785907745361f));
  p = fma2(p, f, pair_of(0.240247443318367f, 0.240247443318367f));
  p = fma2(p, f, pair_of(0.6931217908859253f, 0.6931217908859253f));
  p = fma2(p, f, pair_of(0.9999992847442627f, 0.9999992847442627f));
  const float2 q = halves_of(p), e = halves_of(t);
  return make_float2(__uint_as_float(__float_as_uint(q.x) + (__float_as_uint(e.x) << 23)), __uint_as_float(__float_as_uint(q.y) + (__float_as_uint(e.y) << 23)));
}

// Weights of 32 columns (two blocks' scales), their sum over each block's V scale; the largest y = s + log2(vs) of them.
// EVERY: the row sees all of its columns, else those in [low, high) of blocks that are there.
// PARTS: terms of a weight, the second one behind the first.  With two the FMA units' exponentials would be what limits the result.
template <bool EVERY, int PARTS>
__device__ __forceinline__ void weights_of(const uint32_t (&r)[32], const float4 (&x)[2], float factor, int low, int high, float bias,
                                           uint32_t (&p)[PARTS][16], float& l, float& top) {
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    const float f = x[g].x * factor, add = x[g].y + bias;
    const uint64_t ff = pair_of(f, f), aa = pair_of(add, add);
    uint64_t sum[2] = {0u, 0u};
    float best = -INFINITY;
#pragma unroll
    for (int k = 0; k < 16; k += 2) {
      const float s[2] = {__uint_as_float(r[16 * g + k]), __uint_as_float(r[16 * g + k + 1])};
      const uint64_t y = fma2(pair_of(s[0], s[1]), ff, aa);
      float w[2];
      if (EVERY && PARTS == 1 && (kPolynomial >> (k / 2) & 1) != 0) {
        const float2 e = exp2_pair(y);
        w[0] = e.x;
        w[1] = e.y;
      } else {
        w[0] = exp2_approx(halves_of(y).x);
        w[1] = exp2_approx(halves_of(y).y);
      }
      if (EVERY) {
        best = max3_or_nan(best, s[0], s[1]);
      } else {                                                          // what is not seen has no weight, whatever the block's scales are
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const bool seen = x[g].w != 0.f && 16 * g + k + j >= low && 16 * g + k + j < high;
          w[j] = seen ? w[j] : 0.f;
          best = fmaxf(best, seen ? s[j] : -INFINITY);
        }
      }
      sum[(k >> 1) & 1] = add2(sum[(k >> 1) & 1], pair_of(w[0], w[1]));
      p[0][8 * g + k / 2] = pack_half(w[0], w[1]);
      if (PARTS == 2) {
        const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&p[0][8 * g + k / 2]));
        p[PARTS - 1][8 * g + k / 2] = pack_half(w[0] - back.x, w[1] - back.y);
      }
    }
    const float2 both = halves_of(add2(sum[0], sum[1]));
    if (EVERY || both.x + both.y != 0.f) l = fmaf(both.x + both.y, x[g].z, l);
    // Scores are finite but for a key's NaN, which the polynomial loses.  (2^n as a product, which keeps it: a prompt takes 2.9 % longer.)
    if (EVERY && PARTS == 1) l = fmaf(best, 0.f, l);
    if (EVERY || best != -INFINITY) top = fmaxf(top, fmaf(best, f, x[g].y));
  }
}

// A row's tile: weights into the scores' place, their sum to l.  They are taken relative to what was the largest so far, at once, and again where the tile has
// outgrown that (O is brought along then, once products_done() says that the tile before is in it; false where that gives up): the first tiles do.
template <class S, bool EVERY, typename Wait>
__device__ __forceinline__ bool tile_weights(uint32_t tmem_s, uint32_t tmem_o, const float4* scales, float factor, int low, int high, bool more,
                                             float& ref, float& l, Wait products_done) {
  uint32_t r[2][32], p[2][S::PARTS][16];                                // p: of the first and the last 32 columns
  tmem_ld32(tmem_s, r[0]);
  float4 x[2][2];
#pragma unroll
  for (int g = 0; g < 4; ++g) x[g >> 1][g & 1] = scales[g];
  umma::tmem_ld_wait();
  tmem_ld32(tmem_s + 32u, r[1]);
  float bias = (ref == -INFINITY ? 0.f : -ref) + kUp, sum = 0.f, top = -INFINITY;
  weights_of<EVERY, S::PARTS>(r[0], x[0], factor, low, high, bias, p[0], sum, top);
  umma::tmem_ld_wait();
  weights_of<EVERY, S::PARTS>(r[1], x[1], factor, low - 32, high - 32, bias, p[1], sum, top);
  const bool grow = top > ref + kGrow || (ref == -INFINITY && top != -INFINITY);
  if (__any_sync(0xffffffffu, grow)) {
    const float old = ref;
    if (grow) ref = top;
    if (more) {
      if (!products_done()) return false;
      umma::tcgen05_fence_after();
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
    bias = (ref == -INFINITY ? 0.f : -ref) + kUp;
    sum = 0.f;
    float again = -INFINITY;
#pragma unroll 1
    for (int c = 0; c < 2; ++c) {
      uint32_t s[32], w[S::PARTS][16];
      tmem_ld32(tmem_s + uint32_t(32 * c), s);
      float4 y[2] = {scales[2 * c], scales[2 * c + 1]};
      umma::tmem_ld_wait();
      weights_of<false, S::PARTS>(s, y, factor, EVERY ? 0 : low - 32 * c, EVERY ? 32 : high - 32 * c, bias, w, sum, again);
#pragma unroll
      for (int k = 0; k < 16 * S::PARTS; ++k) {
        if (c == 0) p[0][k / 16][k % 16] = w[k / 16][k % 16]; else p[1][k / 16][k % 16] = w[k / 16][k % 16];
      }
    }
  }
  l += sum;
#pragma unroll
  for (int t = 0; t < S::PARTS; ++t) {
    umma::tmem_st16(tmem_s + 32u * t, p[0][t]);
    umma::tmem_st16(tmem_s + 32u * t + 16u, p[1][t]);
  }
  return true;
}

// What the ends of an item need to know of it, in registers: every access to shared memory in between would have them read again.
struct Ends {
  int row, r0, r1, head, piece;               // packed row of the sequence's first token; rows [r0, r1); first head of the group; as in Segment
  // Where row r of the item stands among packed rows and heads, times head_dim.
  __device__ __forceinline__ int64_t place(const AttnParams& a, int r) const {
    const int token = a.by_group(r0 + r);
    return (int64_t(row + token) * a.heads + head + r0 + r - token * a.group) * a.c.dim;
  }
};

// q of a warp's 32 rows, from row r0 of the sequence, into its place in shared memory; factor: of the row of this lane.  It is copied there as it is
// (16 bytes a lane) and worked on in place by a thread a row: eight lanes' chunks lie in different banks by the swizzle, and nothing is shuffled (4000
// to 5700 cycles an item went into shuffles).  What happens once an item is short loops: unrolled code is fetched more slowly than it runs.
template <class S>
__device__ __forceinline__ void open_rows(const AttnParams& a, const Ends e, uint32_t q_smem, int r0, float& factor) {
  using T = std::conditional_t<S::PARTS == 2, uint32_t, uint16_t>;
  constexpr int kChunks = S::D * S::PARTS / 8, kEach = 16 / int(sizeof(T));      // of a row, of 16 bytes; values of one
  const int lane = threadIdx.x & 31, row0 = 32 * ((threadIdx.x >> 5) & 3);
  const bool wide = ((reinterpret_cast<uintptr_t>(a.q) | uint64_t(a.row_stride * sizeof(T)) | uint64_t(a.head_stride * sizeof(T))) & 15) == 0, f16 = a.dtype == DINO_F16;
#pragma unroll 4
  for (int k = 0; k < kChunks; ++k) {
    const int at = 32 * k + lane, row = at / kChunks, chunk = at % kChunks;
    const int r = r0 + row, token = a.by_group(min(r, e.r1 - 1)), head = e.head + r - token * a.group;
    const T* src = static_cast<const T*>(a.q) + int64_t(e.row + token) * a.row_stride + int64_t(head) * a.head_stride + kEach * chunk;
    const uint32_t to = q_smem + operand_at<kRows>(row0 + row, chunk);
    if (r >= e.r1) {
      st_shared16(to, 0u, 0u, 0u, 0u);
    } else if (wide) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(to), "l"(src) : "memory");
    } else {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (S::PARTS == 2) w[j] = src[j];
        else w[j] = uint32_t(src[2 * j]) | (uint32_t(src[2 * j + 1]) << 16);
      }
      st_shared16(to, w[0], w[1], w[2], w[3]);
    }
  }
  asm volatile("cp.async.wait_all;\n" ::: "memory");
  __syncwarp();
  uint32_t largest = 0;                                                 // of the magnitudes, as bits: their order is that of the values
#pragma unroll 4
  for (int c = 0; c < kChunks; ++c) {
    const uint4 x = lds128(q_smem + operand_at<kRows>(row0 + lane, c));
    if (S::PARTS == 2) largest = max(max(largest, max(x.x & 0x7fffffffu, x.y & 0x7fffffffu)), max(x.z & 0x7fffffffu, x.w & 0x7fffffffu));
    else largest = __vmaxu2(largest, __vmaxu2(__vmaxu2(x.x & 0x7fff7fffu, x.y & 0x7fff7fffu), __vmaxu2(x.z & 0x7fff7fffu, x.w & 0x7fff7fffu)));
  }
  if (S::PARTS == 1) {
    largest = max(largest & 0xffffu, largest >> 16);
    largest = f16 ? __float_as_uint(__half2float(__ushort_as_half(uint16_t(largest)))) : largest << 16;
  }
  const uint32_t exponent = largest >> 23;
  const bool plain = exponent == 0 || exponent == 255;
  const int shift = plain ? 0 : min(max(127 + 12 - int(exponent), -126), 126);
  const float up = __uint_as_float(uint32_t(127 + shift) << 23), sign = a.scale < 0.f ? -up : up;      // scores' factors are not negative
  if constexpr (S::PARTS == 2) {                                        // 16 values: the float16 nearest to them, and what is left
#pragma unroll 1
    for (int c = 0; c < kChunks; c += 4) {
      uint32_t h[8], rest[8];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint4 x = lds128(q_smem + operand_at<kRows>(row0 + lane, c + k));
        const float v[4] = {__uint_as_float(x.x) * sign, __uint_as_float(x.y) * sign, __uint_as_float(x.z) * sign, __uint_as_float(x.w) * sign};
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          h[2 * k + j] = pack_half(v[2 * j], v[2 * j + 1]);
          const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&h[2 * k + j]));
          rest[2 * k + j] = pack_half(v[2 * j] - back.x, v[2 * j + 1] - back.y);
        }
      }
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        st_shared16(q_smem + operand_at<kRows>(row0 + lane, c + k), h[4 * k], h[4 * k + 1], h[4 * k + 2], h[4 * k + 3]);
        st_shared16(q_smem + operand_at<kRows>(row0 + lane, c + 2 + k), rest[4 * k], rest[4 * k + 1], rest[4 * k + 2], rest[4 * k + 3]);
      }
    }
  } else {
#pragma unroll 2
    for (int c = 0; c < kChunks; ++c) {
      const uint32_t at = q_smem + operand_at<kRows>(row0 + lane, c);
      const uint4 x = lds128(at);
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
      uint32_t h[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 v = f16 ? __half22float2(*reinterpret_cast<const __half2*>(&w[j])) : make_float2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u));
        h[j] = pack_half(v.x * sign, v.y * sign);
      }
      st_shared16(at, h[0], h[1], h[2], h[3]);
    }
  }
  // (an infinite or NaN q: NaN, also where all of its scores are -inf and would look like those of a row that sees nothing)
  factor = exponent == 255 ? __uint_as_float(0x7fc00000u) : fabsf(a.scale) * __uint_as_float(uint32_t(127 - shift) << 23);
  fence_async_smem();
  __syncwarp();
}

// O of a warp's 32 rows (row0: the first one's number in the item): results, or float32 sums of a piece.  Through the place of these rows' q, which nobody
// reads any more (that of other rows may be the next item's already): 2 D bytes a row, so that rows leave in whole lines.
template <class S>
__device__ __forceinline__ void close_rows(const AttnParams& a, const Ends e, uint32_t q_smem, uint32_t tmem_o, int row0, float inverse) {
  constexpr int D = S::D, kLanes = D / 8, kStep = 32 / kLanes;          // of a row; rows at once
  const int lane = threadIdx.x & 31, rows = e.r1 - e.r0 - row0;         // of this warp's
  const int first = 32 * ((threadIdx.x >> 5) & 3);
  auto at = [&](int row, int chunk) { return q_smem + operand_at<kRows>(first + row, chunk); };
  if (S::PARTS == 1 && e.piece < 0) {
#pragma unroll 1
    for (int c = 0; c < D / 32; ++c) {
      uint32_t o[32], h[16];
      tmem_ld32(tmem_o + uint32_t(32 * c), o);
      umma::tmem_ld_wait();
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const float u = __uint_as_float(o[2 * k]) * inverse, v = __uint_as_float(o[2 * k + 1]) * inverse;
        if (a.dtype == DINO_F16) {
          h[k] = pack_half(u, v);
        } else {
          const __nv_bfloat162 x = __floats2bfloat162_rn(u, v);
          h[k] = *reinterpret_cast<const uint32_t*>(&x);
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) st_shared16(at(lane, 4 * c + k), h[4 * k], h[4 * k + 1], h[4 * k + 2], h[4 * k + 3]);
    }
    __syncwarp();
#pragma unroll 4
    for (int k = 0; k < 32; k += kStep) {
      const int row = k + lane / kLanes, chunk = lane % kLanes;
      if (row < rows) *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + e.place(a, row0 + row) + 8 * chunk) = lds128(at(row, chunk));
    }
    __syncwarp();
    return;
  }
  float* const part = a.partial + size_t(e.piece) * S::kPiece + size_t(row0) * D;
#pragma unroll 1
  for (int half = 0; half < 2; ++half) {                                // D / 2 columns at a time
#pragma unroll 1
    for (int c = 0; c < D / 64; ++c) {
      uint32_t o[32];
      tmem_ld32(tmem_o + uint32_t(half * (D / 2) + 32 * c), o);
      umma::tmem_ld_wait();
      if (S::PARTS == 2 && e.piece < 0) {
#pragma unroll
        for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * inverse);
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) st_shared16(at(lane, 8 * c + k), o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
    }
    __syncwarp();
#pragma unroll 4
    for (int k = 0; k < 32; k += kStep) {
      const int row = k + lane / kLanes, chunk = lane % kLanes;
      if (row >= rows) continue;
      float* const to = S::PARTS == 2 && e.piece < 0 ? static_cast<float*>(a.out) + e.place(a, row0 + row) : part + size_t(row) * D;
      __stcg(reinterpret_cast<uint4*>(to + half * (D / 2) + 4 * chunk), lds128(at(row, chunk)));
    }
    __syncwarp();
  }
}

// The results of a cut item from its pieces, by a thread for each row of an item.  First a row's largest y and its sum by a thread each (kept in the place of q), then the sums of
// all columns, kPlaces of four columns and kPieces pieces under way at a time.
template <class S, typename Meet> __device__ __forceinline__ bool join_rows(const AttnParams& a, const Ends e, int c0, int c1, int piece0, uint32_t q_smem, Meet meet) {
  constexpr int D = S::D, kPlaces = 8, kPieces = 2;
  const int rows = e.r1 - e.r0, count = c1 - c0 + 1, tid = int(threadIdx.x);
  auto piece = [&](int c) { return a.partial + size_t(c == 0 ? piece0 : 2 * (c0 + c)) * S::kPiece; };
  auto weight = [](float ref, float top) { return ref == -INFINITY ? 0.f : exp2_approx(ref - top); };
  if (tid < rows) {
    float top = -INFINITY, sum = 0.f;
#pragma unroll 1
    for (int c = 0; c < count; c += 4) {
      float2 ml[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) ml[k] = c + k < count ? __ldcg(reinterpret_cast<const float2*>(piece(c + k) + S::kItemRows * D) + tid) : make_float2(-INFINITY, 0.f);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float next = fmaxf(top, ml[k].x);
        sum = fmaf(ml[k].y, weight(ml[k].x, next), sum * weight(top, next));
        top = next;
      }
    }
    const float inverse = sum == 0.f ? 0.f : 1.f / sum;
    asm volatile("st.shared.v2.f32 [%0], {%1,%2};\n" ::"r"(q_smem + 8u * uint32_t(tid)), "f"(top), "f"(inverse) : "memory");
  }
  if (!meet()) return false;
  auto stats = [&](int row) {
    float2 v;
    asm volatile("ld.shared.v2.f32 {%0,%1}, [%2];\n" : "=f"(v.x), "=f"(v.y) : "r"(q_smem + 8u * uint32_t(row)) : "memory");
    return v;
  };
  const int last = rows * (D / 4) - 1;
#pragma unroll 1
  for (int x0 = tid; x0 <= last; x0 += S::kItemRows * kPlaces) {
    float4 v[kPlaces];
    float top[kPlaces];
#pragma unroll
    for (int u = 0; u < kPlaces; ++u) {
      v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      top[u] = stats(min(x0 + S::kItemRows * u, last) / (D / 4)).x;
    }
#pragma unroll 1
    for (int c = 0; c < count; c += kPieces) {
      float ref[kPieces][kPlaces];
      float4 y[kPieces][kPlaces];
#pragma unroll
      for (int k = 0; k < kPieces; ++k) {
        const float* const src = piece(min(c + k, count - 1));
#pragma unroll
        for (int u = 0; u < kPlaces; ++u) {
          const int x = min(x0 + S::kItemRows * u, last);
          y[k][u] = __ldcg(reinterpret_cast<const float4*>(src) + x);
          ref[k][u] = __ldcg(src + S::kItemRows * D + 2 * (x / (D / 4)));
        }
      }
#pragma unroll
      for (int k = 0; k < kPieces; ++k) {
        if (c + k >= count) break;
#pragma unroll
        for (int u = 0; u < kPlaces; ++u) {
          const float f = weight(ref[k][u], top[u]);
          v[u] = make_float4(fmaf(y[k][u].x, f, v[u].x), fmaf(y[k][u].y, f, v[u].y), fmaf(y[k][u].z, f, v[u].z), fmaf(y[k][u].w, f, v[u].w));
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kPlaces; ++u) {
      const int x = x0 + S::kItemRows * u;
      if (x > last) break;
      const float inv = stats(x / (D / 4)).y;
      if constexpr (S::PARTS == 2) {
        __stcg(reinterpret_cast<float4*>(static_cast<float*>(a.out) + e.place(a, x / (D / 4)) + x % (D / 4) * 4), make_float4(v[u].x * inv, v[u].y * inv, v[u].z * inv, v[u].w * inv));
        continue;
      }
      uint2 h;
      if (a.dtype == DINO_F16) {
        h = make_uint2(pack_half(v[u].x * inv, v[u].y * inv), pack_half(v[u].z * inv, v[u].w * inv));
      } else {
        const __nv_bfloat162 lo = __floats2bfloat162_rn(v[u].x * inv, v[u].y * inv), hi = __floats2bfloat162_rn(v[u].z * inv, v[u].w * inv);
        h = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
      }
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + e.place(a, x / (D / 4)) + x % (D / 4) * 4) = h;
    }
  }
  return meet();                                                        // (the next item's q goes where the rows' sums are)
}

// ---- warps 0..3 and, where there are two tiles of rows, 4..7: tile i of the item, a row per thread
template <class S>
__device__ __forceinline__ void softmax_rows(const AttnParams& a, Shared& sh, uint32_t q_smem) {
  constexpr int D = S::D;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, i = warp >> 2, my_row = 32 * (warp & 3) + lane;
  const uint32_t lanes = sh.tmem + (uint32_t(32 * (warp & 3)) << 16), tmem_s = lanes + uint32_t(i * 128), tmem_o = lanes + kO + uint32_t(i * D);
  int first = 0, meetings = 0;                                          // tiles so far
  uint32_t scores = 0;                                                  // phases of s_full, a bit for even and one for odd stages
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
    const Ends e = {sg.s.row, sg.item.r0, sg.item.r1, sg.head * a.group, sg.piece};
    const int r = e.r0 + i * kRows + my_row;
    const bool mine = r < e.r1;
    const int token = a.by_group(mine ? r : e.r0);
    float factor = 0.f;
    open_rows<S>(a, e, q_smem + uint32_t(i * S::kQ), e.r0 + i * kRows + 32 * (warp & 3), factor);
    if (lane == 0) umma::mbar_arrive(umma::smem_u32(&sh.q_ready));
    const int position = sg.s.first + token;
    const int high = mine ? min(position + 1, sg.s.end) : 0, low = a.window > 0 ? max(0, position - a.window + 1) : 0;
    const int all_high = __reduce_min_sync(0xffffffffu, mine ? high : INT32_MAX), all_low = __reduce_max_sync(0xffffffffu, mine ? low : 0);
    const int base = (sg.item.low >> kLog2) << kLog2;
    float ref = -INFINITY, l = 0.f;
    bool lost = false;
    const int tiles = tile1 - tile0;
    for (int u = 0; u < tiles; ++u) {
      const int tile = tile0 + u;
      if (!wait(a, sh, &sh.s_full[i][u & 1], (scores >> (u & 1)) & 1u)) { lost = true; break; }
      scores ^= 1u << (u & 1);
      umma::tcgen05_fence_after();
      const float4* const scales = sh.scales[(first + u) % kScales];
      const int token0 = base + tile * kTile;
      const int4 whole = sh.whole[(first + u) % kScales];
      const bool every = token0 >= all_low && token0 + kTile <= all_high && (whole.x & whole.y & whole.z & whole.w) != 0;
      const uint32_t at = tmem_s + uint32_t((u & 1) * 64);
      auto products_done = [&] { return wait(a, sh, &sh.s_full[i][(u + 1) & 1], (scores >> ((u + 1) & 1)) & 1u); };      // the MMAs of the stage after this one
      if (!(every ? tile_weights<S, true>(at, tmem_o, scales, factor, 0, 0, u > 0, ref, l, products_done)
                  : tile_weights<S, false>(at, tmem_o, scales, factor, low - token0, high - token0, u > 0, ref, l, products_done))) {
        lost = true;
        break;
      }
      umma::tmem_st_wait();
      umma::tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) umma::mbar_arrive(umma::smem_u32(&sh.p_ready[i][u & 1]));
    }
    if (lost) return;
    for (int u = tiles; u < tiles + kAhead; ++u) {                       // the last products
      if (!wait(a, sh, &sh.s_full[i][u & 1], (scores >> (u & 1)) & 1u)) return;
      scores ^= 1u << (u & 1);
    }
    first += tiles;
    umma::tcgen05_fence_after();
    close_rows<S>(a, e, q_smem + uint32_t(i * S::kQ), tmem_o, i * kRows + 32 * (warp & 3), l == 0.f ? 0.f : 1.f / l);
    umma::tcgen05_fence_before();
    if (e.piece >= 0) {                                                 // cut: the last of its CTAs to arrive adds the pieces up, in order
      if (mine) __stcg(reinterpret_cast<float2*>(a.partial + size_t(e.piece) * S::kPiece + S::kItemRows * D) + (i * kRows + my_row), make_float2(ref, l));
      if (!meet()) return;
      if (threadIdx.x == 0) {
        int before = 0;
        asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;\n" : "=r"(before) : "l"(a.arrived + sg.c0) : "memory");
        sh.last = before == sg.c1 - sg.c0;
        if (sh.last) a.arrived[sg.c0] = 0;
      }
      if (!meet()) return;
      if (sh.last) {
        if (!join_rows<S>(a, e, sg.c0, sg.c1, sg.piece0, q_smem, meet)) return;
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
  const uint32_t q_smem = smem, k_smem = smem + S::kTiles * S::kQ, v_smem = k_smem + S::kStages * S::kKv;
  const int warp = threadIdx.x >> 5;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kSegments; ++i) {
      umma::mbar_init(umma::smem_u32(&sh.described[i]), 1);
      umma::mbar_init(umma::smem_u32(&sh.closed[i]), 4 * S::kTiles + S::kConverters + 1);
    }
    umma::mbar_init(umma::smem_u32(&sh.q_ready), 4 * S::kTiles);
    for (int i = 0; i < S::kStages; ++i) {
      umma::mbar_init(umma::smem_u32(&sh.full[i]), S::kConverters);
      umma::mbar_init(umma::smem_u32(&sh.empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      for (int k = 0; k < 2; ++k) {
        umma::mbar_init(umma::smem_u32(&sh.s_full[i][k]), 1);
        umma::mbar_init(umma::smem_u32(&sh.p_ready[i][k]), 4);
      }
    }
    umma::mbar_init(umma::smem_u32(&sh.together), 4 * S::kTiles);
    umma::mbar_init(umma::smem_u32(&sh.drain), 1);
    sh.lost = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  __syncwarp();
  if (warp == 12) umma::tmem_alloc<false>(umma::smem_u32(&sh.tmem), kTmem);
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  asm volatile("griddepcontrol.wait;\n" ::: "memory");                // nothing of the launches before is read before this
  umma::tcgen05_fence_before();
  const Walk first = walk_of<kThreads>(a, kLog2, kLeast, sh.walk);         // (its barriers: the inits and the allocation are visible)
  __syncthreads();
  umma::tcgen05_fence_after();
  // Two tiles of rows: 2 x 176 + 96 + 64 = 4 x 128 registers; one: 192 + 2 x 96 + 64 of them.
  if (warp < 4 * S::kTiles) {
    if constexpr (S::kTiles == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 176;\n");
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 192;\n");
    softmax_rows<S>(a, sh, q_smem);
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

template <int TYPE, int D, int PARTS> int launch(AttnParams& a, cudaStream_t s) {
  using S = Shape<D, PARTS>;
  a.row_tile = S::kItemRows;
  a.row_tile_log2 = S::kTiles == 2 ? 8 : 7;
  a.ends = kEnds;
  const int ctas = stream::sm_count();
  a.partial = attention_scratch(size_t(ctas) * 2 * S::kPiece, ctas, s, &a.arrived);
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

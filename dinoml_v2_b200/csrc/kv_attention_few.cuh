// Attention of few rows per cached head (decode, short chunks) over the 8-bit cache: the call is bound by the bytes of the cache, so they are
// streamed once and the products follow on mma.sync at a fraction of its rate.
//
// S^T = K Q^T and O^T = V^T P^T, the cached tile as the 16-row operand: with one to eight heads per cached head the 8-column operand is filled
// best by the heads.  Two warps take a tile of one head, half of its tokens each.  Two more keep them at it:
//   * the copying warp walks the CTA's items, looks blocks up 32 at a time and copies tiles into a ring (TMA with the 128-byte swizzle, a box is one
//     block's share of the tile), across the ends of items.  A tile costs it about 500 cycles whatever its size is;
//   * the opening warp makes q of the next item ready and joins the pieces of items that several CTAs share: what waits for memory between
//     items is not in the way of the others.
//   * K rows are read 16 bytes at a time; the four bytes of word i of lane (g, t) are k = 16 t + 4 i .. + 3 of a 64-byte group, for K and for Q alike.
//     Token tok(g) stands in row g so that eight lanes touch all banks.
//   * V comes by ldmatrix.trans on pairs of bytes: one register holds channels 2g, 2g + 1 of two tokens, a byte permutation makes a
//     float16 pair along the tokens of each channel - the transposition is the conversion.  Rows g and g + 8 are channels 16c + 2g, 16c + 2g + 1.
//   * 8-bit values are exact in float16.  q is brought to [2^12, 2^13) by a power of two for each row, which keeps every bit of it that matters
//     (bfloat16: all but values 2^-37 of the row's largest); float32 rows are two float16 terms (PARTS = 2).
//   * The products of a tile start from zero, with weights relative to the tile's own maxima: p = 2^(s - top) (vs / vt), vs the scale of a block's V and vt
//     the largest in the tile, is rounded to float16 as 2^14 p, and the result joins O in float32: the sums of a long cache are float32 additions.
//     Below 2^-28 such a weight is a float16 denormal; a tile that has one adds what the rounding left, 2^11 times as large, in a second
//     pass over V (float32, PARTS = 2: every tile), so that bits are lost only below 2^-40.  The sum l takes p before any rounding.
// Cut items leave (m, l, O) in the workspace; the last CTA to arrive adds them up in order, so results do not depend on who that is.
#pragma once
#include "kv_attention.cuh"

namespace b200gguf {
namespace kv {
namespace few {

constexpr int kCtasPerSm = 2, kSegments = 4;
// What an item costs beside its tiles (q, the join of its pieces), in tiles.  64 ragged sequences of up to 8192 tokens: 108.5 us with 0, 99.4 with 2, 96.2 with 6,
// 98.4 with 11; three of 131072, 35361 and 26873 tokens: 95.6, 86.3, 78.6, 78.8.
constexpr int kEnds = 6;

template <int D_, int NT_, int PARTS_> struct Shape {
  static constexpr int D = D_, NT = NT_, PARTS = PARTS_;
  static constexpr int R = 8 * NT;                                        // rows of an item
  static constexpr int TK = D == 256 ? 16 : 32;                           // tokens of a warp's half of a tile
  static constexpr int kTile = 2 * TK, kLog2 = D == 256 ? 5 : 6;
  static constexpr int MT = TK / 16, KS = D / 16, DC = D / 16;             // 16-token rows, 16-value steps, 16-channel rows
  // Warps that compute, by the registers of their sums (D NT / 4): with the two others and two CTAs per SM a quarter of an SM has four or three
  // warps, of 128 or 168 registers.
  static constexpr int W = D * NT <= 128 ? 6 : 4;
  static_assert(D * NT <= 256);
  static constexpr int kThreads = (W + 2) * 32;
  static constexpr int kRow = D == 64 ? 64 : 128;                          // bytes of a row; heads of 256 are two such halves, one after the other
  static constexpr int kHalf = kTile * D;                                  // bytes of a tile's K, and of its V
  static constexpr int kQ = KS * NT * PARTS * 32 * 8;                      // q as operand fragments
  static constexpr int kMergeCh = D < 128 ? D : 128, kPitch = kMergeCh + 4;
  static constexpr int kMerge = W * 8 * kPitch * 4;                        // sums of 8 rows and kMergeCh channels of every warp
  static constexpr int kFixed = 1024 + kMerge + 2 * kQ, kStatic = 2000 + W * R * 8 + 40 * R;
  static constexpr int kRoom = (113 * 1024 - kFixed - kStatic) / (2 * kHalf);
  static constexpr int kStages = kRoom < 10 ? kRoom : 10;
  static constexpr int kRing = kStages * 2 * kHalf;
  static constexpr size_t kSmem = kFixed + kRing;
  static_assert(kStages > W / 2, "tiles under way beside those that are read");
};

// token of row g (of 8): with rows of 128 bytes two lanes of a quad of eight differ in bit 2 of the row, which the swizzle puts into the other half
template <int ROW> __device__ __forceinline__ int tok(int g) { return ROW == 128 ? (g >> 1) | ((g & 1) << 2) : g; }
template <int ROW> __device__ __forceinline__ uint32_t swizzled(int row, int chunk) {
  return ROW == 128 ? uint32_t(row * 128 + ((chunk ^ (row & 7)) << 4)) : uint32_t(row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4));
}

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint4 lds128(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}
__device__ __forceinline__ void ldmatrix4t(uint32_t at, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
__device__ __forceinline__ void ldmatrix2t(uint32_t at, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0,%1}, [%2];\n" : "=r"(r[0]), "=r"(r[1]) : "r"(at));
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float load_q(const AttnParams& a, int64_t at) {
  if (a.dtype == DINO_F32) return fetch(static_cast<const float*>(a.q) + at);
  if (a.dtype == DINO_F16) return __half2float(static_cast<const __half*>(a.q)[at]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(a.q)[at]);
}
// Four values of a row of q; `wide`: at a multiple of their size.
__device__ __forceinline__ void load_q4(const AttnParams& a, int64_t at, bool wide, float (&v)[4]) {
  if (!wide) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = load_q(a, at + i);
  } else if (a.dtype == DINO_F32) {
    const float4 x = fetch(reinterpret_cast<const float4*>(static_cast<const float*>(a.q) + at));
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
  } else {
    const uint2 x = fetch(reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.q) + at));
    if (a.dtype == DINO_F16) {
      const float2 lo = __half22float2(*reinterpret_cast<const __half2*>(&x.x)), hi = __half22float2(*reinterpret_cast<const __half2*>(&x.y));
      v[0] = lo.x; v[1] = lo.y; v[2] = hi.x; v[3] = hi.y;
    } else {
      v[0] = __uint_as_float(x.x << 16); v[1] = __uint_as_float(x.x & 0xffff0000u); v[2] = __uint_as_float(x.y << 16); v[3] = __uint_as_float(x.y & 0xffff0000u);
    }
  }
}
__device__ __forceinline__ void store4(const AttnParams& a, int64_t at, float4 v) {      // at: a multiple of 4; out is at a multiple of 16 bytes
  if (a.dtype == DINO_F32) {
    *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = v;
  } else if (a.dtype == DINO_F16) {
    *reinterpret_cast<uint2*>(static_cast<__half*>(a.out) + at) = make_uint2(pack_half(v.x, v.y), pack_half(v.z, v.w));
  } else {
    const __nv_bfloat162 lo = __floats2bfloat162_rn(v.x, v.y), hi = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + at) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
  }
}

// A piece of work as the copying warp hands it to the others: tiles [tile0, tile1) of an item.
struct Segment {
  Sequence s;
  Item item;
  int head, tiles, tile0, tile1;
  int number;                                  // of the first tile in the CTA's sequence of tiles
  int piece;                                   // -1: the whole item; else the place of this piece in the workspace
  int c0, c1, piece0;                          // workers that share the item, the place of c0's piece (the others' is 2 c)
};

// Rows of a warp's half of a tile's V that nobody sees become zeros.
template <class S> __device__ __forceinline__ void clear_unseen(uint32_t vtile, int token0, int low, int high, const float4* boxes) {
  const int lane = threadIdx.x & 31;
  for (int row = 0; row < S::TK; ++row) {
    if (boxes[row >> 4].z != 0.f && token0 + row >= low && token0 + row < high) continue;
    if (lane < S::D / 16)
      asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};\n" ::"r"(vtile + uint32_t((lane / (S::kRow / 16)) * S::kTile * S::kRow + row * S::kRow + (lane % (S::kRow / 16)) * 16)), "r"(0) : "memory");
  }
  asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");       // before the next copy into the tile
  __syncwarp();
}

// An item's rows as the computing warps need them, for two items in turn.
template <class S> struct Rows8 {
  float factor[S::R];                          // of a row's scores: what q was divided by, the softmax scale, log2(e)
  int low[S::R], high[S::R];                   // positions that a row sees
};

template <class S> struct Shared {
  uint64_t full[S::kStages], empty[S::kStages];                   // of a tile: it has landed, it has been read
  uint64_t described[kSegments], closed[kSegments];               // of a segment: the copying warp's account of it is there, is no longer needed
  uint64_t opened[2], written[2];                                 // of a segment: q is there, its results are written
  uint64_t together, merged;                                      // of the computing warps: their sums are there, have been read
  uint64_t ended;                                                 // it is known which items this CTA joins
  float4 boxes[S::kStages][S::kTile / 16];     // of every 16 tokens: their block's scales of K and V, whether there is one
  Segment segments[kSegments], to_join[2];
  Rows8<S> rows[2];
  int64_t walk[4 + S::W];
  int joins, lost;                             // items to join; a wait gave up
  float2 ml[S::W][S::R];                       // every warp's maxima and sums
};

// Waits are bounded: where one gives up every role of the CTA falls through to the end, the results are lost and the status word says so.
template <class S> __device__ __forceinline__ bool wait(const AttnParams& a, Shared<S>& sh, uint64_t* bar, uint32_t parity) {
  const uint32_t at = umma::smem_u32(bar);
  volatile int* lost = &sh.lost;
  if (umma::mbar_test_wait(at, parity)) return true;
  for (uint32_t i = 0; i < kPolls; ++i) {
    if (umma::mbar_try_wait(at, parity)) return true;
    if ((i & 255u) == 255u && *lost) return false;
  }
  *lost = 1;
  flag_timeout(a.p.status);
  return false;
}
template <class S> __device__ __forceinline__ bool warp_wait(const AttnParams& a, Shared<S>& sh, uint64_t* bar, uint32_t parity) {
  return __all_sync(0xffffffffu, wait(a, sh, bar, parity)) != 0;
}

// ---- the copying warp: walks the CTA's units, looks up blocks 32 boxes at a time, copies tiles into the ring.
template <class S>
__device__ __forceinline__ void copy_tiles(const AttnParams& a, Shared<S>& sh, const CUtensorMap* k_map, const CUtensorMap* v_map, uint32_t ring, Walk w) {
  const int lane = threadIdx.x & 31;
  const int boxes = max(1, S::kTile >> a.c.block_log2), box_tokens = S::kTile / boxes, per_look = 32 / boxes;      // blocks of a tile, tiles of a look-up
  int stage = 0, number = 0, segment = 0;
  uint32_t phase = 1;                                                 // of `empty`: true at once on the first lap
  for (;; w.next_item(a, S::kLog2), ++segment) {
    const int slot = segment & (kSegments - 1);
    if (!warp_wait(a, sh, &sh.closed[slot], uint32_t(segment / kSegments + 1) & 1u)) return;
    const bool done = w.done();
    const int tile0 = done ? 0 : w.tile, tile1 = done ? 0 : w.end_tile();
    if (lane == 0) {
      Segment g;
      g.s = w.s; g.item = w.item;
      g.head = w.head; g.tiles = w.tiles; g.tile0 = tile0; g.tile1 = tile1; g.number = number;
      g.piece = -1; g.c0 = g.c1 = g.piece0 = 0;
      if (!done && (tile0 != 0 || tile1 != w.tiles)) {                // the CTA's first piece of work, or its last: others are whole
        g.piece = w.piece();
        g.c0 = w.owner(w.first_tile());
        g.c1 = w.owner(w.first_tile() + w.tiles - 1);
        g.piece0 = w.first_piece(g.c0);
      }
      sh.segments[slot] = g;
      umma::mbar_arrive(umma::smem_u32(&sh.described[slot]));
    }
    if (done) return;
    const int token_base = (w.item.low >> S::kLog2) * S::kTile;
    // Box lane % boxes of tile + lane / boxes: its first row in the maps, -1 where there is none, and its scales.  One warp issues every copy of
    // the CTA, a few hundred cycles each: what can be done for 32 boxes at once is done here.
    struct Box { int row; float k_scale, v_scale; };
    auto look_up = [&](int tile) {
      const int t = tile + lane / boxes, token = token_base + t * S::kTile + lane % boxes * box_tokens;
      Box x{-1, 0.f, 0.f};
      if (t >= tile1 || token >= w.item.high || token + box_tokens <= w.item.low) return x;
      const int id = block_at(a.p, a.c.blocks, w.b, token >> a.c.block_log2);
      if (id < 0) return x;
      const int bh = id * a.c.heads + w.head;                           // (rows of the cache are an int)
      x.row = (bh << a.c.block_log2) + (token & ((1 << a.c.block_log2) - 1));
      x.k_scale = fetch(a.c.scale[0] + bh);
      x.v_scale = fetch(a.c.scale[1] + bh);
      return x;
    };
    Box now = look_up(tile0), ahead = look_up(tile0 + per_look);
    for (int tile = tile0, place = 0; tile < tile1; ++tile, ++number, ++place) {
      if (place == per_look) {
        place = 0;
        now = ahead;
        ahead = look_up(tile + per_look);
      }
      int row[4], tokens = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        row[i] = __shfl_sync(0xffffffffu, now.row, (place * boxes + i) & 31);
        if (i >= boxes) row[i] = -1;
        if (row[i] >= 0) tokens += box_tokens;
      }
      if (!warp_wait(a, sh, &sh.empty[stage], phase)) return;
      // One elected lane of the converged warp: descriptors, coordinates and barriers stay in uniform registers.
      if (umma::elect_one()) {
        const uint32_t bar = umma::smem_u32(&sh.full[stage]);
        uint32_t dst = ring + uint32_t(stage * 2 * S::kHalf);
        umma::mbar_arrive_expect_tx(bar, uint32_t(2 * S::D * tokens));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (row[i] >= 0) {
#pragma unroll
            for (int h = 0; h < S::D / S::kRow; ++h) {
              tma_load_2d(dst + uint32_t(h * S::kTile * S::kRow), k_map, bar, h * 128, row[i]);
              tma_load_2d(dst + uint32_t(S::kHalf + h * S::kTile * S::kRow), v_map, bar, h * 128, row[i]);
            }
          }
          dst += uint32_t(box_tokens * S::kRow);
        }
      }
      __syncwarp();
      if (lane / boxes == place) {                                      // who looked the box up
        const float4 box = make_float4(now.k_scale, now.v_scale, now.row >= 0 ? 1.f : 0.f, 0.f);
        for (int i = 0; i < box_tokens / 16; ++i) sh.boxes[stage][lane % boxes * (box_tokens / 16) + i] = box;
        umma::mbar_arrive(umma::smem_u32(&sh.full[stage]));
      }
      if (++stage == S::kStages) { stage = 0; phase ^= 1u; }
    }
  }
}

// Rows of the call that no sequence has - before the first one, behind the last one (a padded batch), those of starts that point outside - become zeros, by a
// warp of every CTA.
__device__ __forceinline__ void clear_rows_of_nobody(const AttnParams& a) {
  if (a.p.starts == nullptr) return;
  const int lane = threadIdx.x & 31, count = a.p.sequences, rows = a.p.rows;
  const int per_row = a.heads * a.c.dim * (a.dtype == DINO_F32 ? 4 : 2) / 16;      // in 16 bytes
  auto clear = [&](int low, int high, int first, int step) {
    for (int64_t r = int64_t(low) + first; r < high; r += step)
      for (int i = lane; i < per_row; i += 32) static_cast<uint4*>(a.out)[r * per_row + i] = make_uint4(0u, 0u, 0u, 0u);
  };
  clear(0, min(rows, min(fetch(a.p.starts), fetch(a.p.starts + 1))), int(blockIdx.x), int(gridDim.x));
  clear(max(0, max(fetch(a.p.starts + count - 1), fetch(a.p.starts + count))), rows, int(blockIdx.x), int(gridDim.x));
  for (int b0 = 32 * int(blockIdx.x); b0 < count; b0 += 32 * int(gridDim.x)) {
    int s0 = 0, s1 = 0;
    if (b0 + lane < count) {
      s0 = fetch(a.p.starts + b0 + lane);
      s1 = fetch(a.p.starts + b0 + lane + 1);
    }
    for (uint32_t bad = __ballot_sync(0xffffffffu, s0 < 0 || s1 < s0 || s1 > rows); bad != 0; bad &= bad - 1)      // (as in rows_of)
      clear(max(0, __shfl_sync(0xffffffffu, s0, __ffs(bad) - 1)), min(rows, __shfl_sync(0xffffffffu, s1, __ffs(bad) - 1)), 0, 1);
  }
}

// ---- the opening warp.  Rows of an item: q as operand fragments, what their scores are multiplied by, what they see.  Lane (g, t) has the fragments of
// row g, 16 t .. 16 t + 15 of every 64 values, so it reads them, and eight rows are made at once.
template <class S> __device__ __forceinline__ void open_rows(const AttnParams& a, Rows8<S>& out, const Segment& sg, uint2* qfrag) {
  constexpr int D = S::D, NT = S::NT, PARTS = S::PARTS;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, rows = sg.item.r1 - sg.item.r0;
  const int size = a.dtype == DINO_F32 ? 4 : 2;
  const bool wide = ((reinterpret_cast<uintptr_t>(a.q) | uint64_t(a.row_stride * size) | uint64_t(a.head_stride * size)) & uint64_t(4 * size - 1)) == 0;
  for (int n = 0; n < NT; ++n) {
    const int r = 8 * n + g, token = a.by_group(sg.item.r0 + r), head = sg.head * a.group + (sg.item.r0 + r) - token * a.group;
    const int64_t at = int64_t(sg.s.row + token) * a.row_stride + int64_t(head) * a.head_stride + 16 * t;
    float x[D / 16][4];
    uint32_t largest = 0;
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      if (r < rows) load_q4(a, at + 64 * (i / 4) + 4 * (i % 4), wide, x[i]);
      else x[i][0] = x[i][1] = x[i][2] = x[i][3] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) largest = max(largest, __float_as_uint(x[i][j]) & 0x7fffffffu);
    largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
    largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
    // 2^12 <= |largest| up < 2^13; zeros, denormals, infinities and NaN as they are
    const uint32_t e = largest >> 23;
    const bool plain = e == 0 || e == 255;
    const int shift = plain ? 0 : min(max(127 + 12 - int(e), -126), 126);
    const float up = __uint_as_float(uint32_t(127 + shift) << 23), down = __uint_as_float(uint32_t(127 - shift) << 23);
#pragma unroll
    for (int i = 0; i < D / 16; ++i) {
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = x[i][j] * up;
#pragma unroll
      for (int part = 0; part < PARTS; ++part) {
        const uint32_t lo = pack_half(v[0], v[1]), hi = pack_half(v[2], v[3]);
        qfrag[((i * NT + n) * PARTS + part) * 32 + lane] = make_uint2(lo, hi);
        const float2 l = __half22float2(*reinterpret_cast<const __half2*>(&lo)), h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
        v[0] -= l.x; v[1] -= l.y; v[2] -= h.x; v[3] -= h.y;
      }
    }
    if (t == 0) {
      const int position = sg.s.first + token;
      // (an infinite or NaN q has no softmax, also where all of its scores are -inf and would look like those of a row that sees nothing)
      out.factor[r] = e == 255 ? __uint_as_float(0x7fc00000u) : a.scale * down;
      out.high[r] = r < rows ? min(position + 1, sg.s.end) : 0;
      out.low[r] = a.window > 0 ? max(0, position - a.window + 1) : 0;
    }
  }
}

// Channels d .. d + 3 of row r.
__device__ __forceinline__ void finish(const AttnParams& a, const Segment& sg, int dim, int r, int d, float4 v, float sum) {
  const float f = sum == 0.f ? 0.f : 1.f / sum;
  const int token = a.by_group(sg.item.r0 + r), head = sg.head * a.group + (sg.item.r0 + r) - token * a.group;
  store4(a, (int64_t(sg.s.row + token) * a.heads + head) * dim + d, make_float4(v.x * f, v.y * f, v.z * f, v.w * f));
}

// A cut item, whose piece of this CTA is written: pieces are those of workers c0 .. c1, and the one that arrives last adds them up, in order.  The counter is
// that of c0, whose range is the only one that this item leaves at its end.
__device__ __forceinline__ bool arrives_last(const AttnParams& a, const Segment& sg) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  if (lane == 0) asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;\n" : "=r"(before) : "l"(a.arrived + sg.c0) : "memory");
  const bool last = __shfl_sync(0xffffffffu, before, 0) == sg.c1 - sg.c0;
  if (last && lane == 0) a.arrived[sg.c0] = 0;
  __syncwarp();                                                         // all lanes behind the first one's acquire
  return last;
}
// By threads `from`, `from + step` and so on.
template <class S> __device__ __forceinline__ void join_pieces(const AttnParams& a, const Segment& sg, int from, int step) {
  constexpr int D = S::D, kPiece = S::R * (D + 2);
  const int count = sg.c1 - sg.c0 + 1, rows = sg.item.r1 - sg.item.r0;
  constexpr int U = 2, P = 8;                                           // places and pieces under way at a time
  for (int i0 = from; i0 < rows * (D / 4); i0 += step * U) {
    float top[U], sum[U];
    float4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      top[u] = -INFINITY;
      sum[u] = 0.f;
      v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int c = 0; c < count; c += P) {
      float2 ml[U][P];
      float4 y[U][P];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + step * u, r = i / (D / 4), d = i % (D / 4) * 4;
#pragma unroll
        for (int x = 0; x < P; ++x)
          if (r < rows && c + x < count) {
            const float* src = a.partial + size_t(c + x == 0 ? sg.piece0 : 2 * (sg.c0 + c + x)) * kPiece;
            ml[u][x] = __ldcg(reinterpret_cast<const float2*>(src + S::R * D + 2 * r));
            y[u][x] = __ldcg(reinterpret_cast<const float4*>(src + r * D + d));
          } else {
            ml[u][x] = make_float2(-INFINITY, 0.f);
            y[u][x] = make_float4(0.f, 0.f, 0.f, 0.f);
          }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float high = top[u];
#pragma unroll
        for (int x = 0; x < P; ++x) high = fmaxf(high, ml[u][x].x);
        const float f0 = top[u] == -INFINITY ? 1.f : exp2_approx(top[u] - high);
        sum[u] *= f0;
        v[u] = make_float4(v[u].x * f0, v[u].y * f0, v[u].z * f0, v[u].w * f0);
#pragma unroll
        for (int x = 0; x < P; ++x) {
          const float f1 = ml[u][x].x == -INFINITY ? 1.f : exp2_approx(ml[u][x].x - high);
          sum[u] = fmaf(ml[u][x].y, f1, sum[u]);
          v[u] = make_float4(fmaf(y[u][x].x, f1, v[u].x), fmaf(y[u][x].y, f1, v[u].y), fmaf(y[u][x].z, f1, v[u].z), fmaf(y[u][x].w, f1, v[u].w));
        }
        top[u] = high;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + step * u, r = i / (D / 4), d = i % (D / 4) * 4;
      if (r < rows) finish(a, sg, D, r, d, v[u], sum[u]);
    }
  }
}

constexpr int kFewPieces = 4;

// The items that a CTA joins are left to its end, where all warps do it, but for those of few pieces, which this warp does beside the others' work.
template <class S> __device__ __forceinline__ void close_segment(const AttnParams& a, Shared<S>& sh, int segment, bool at_end) {
  const int lane = threadIdx.x & 31;
  const Segment& sg = sh.segments[segment & (kSegments - 1)];
  if (sg.piece >= 0 && arrives_last(a, sg)) {
    if (at_end || sg.c1 - sg.c0 >= kFewPieces) {
      if (lane == 0) sh.to_join[sh.joins++] = sg;                       // (a CTA has two cut items at most)
    } else {
      join_pieces<S>(a, sg, lane, 32);
    }
  }
  __syncwarp();
  if (lane == 0) umma::mbar_arrive(umma::smem_u32(&sh.closed[segment & (kSegments - 1)]));
}
template <class S> __device__ __forceinline__ void join_at_end(const AttnParams& a, Shared<S>& sh, int from) {
  for (int i = 0; i < sh.joins; ++i) join_pieces<S>(a, sh.to_join[i], from, (S::W + 1) * 32);
}

template <class S>
__device__ __forceinline__ void open_and_close(const AttnParams& a, Shared<S>& sh, uint2* qfrag) {
  const int lane = threadIdx.x & 31;
  for (int segment = 0;; ++segment) {
    const int slot = segment & (kSegments - 1);
    if (!warp_wait(a, sh, &sh.described[slot], uint32_t(segment / kSegments) & 1u)) return;
    const bool done = sh.segments[slot].tile0 == sh.segments[slot].tile1;
    if (segment >= 2 && !warp_wait(a, sh, &sh.written[segment & 1], uint32_t((segment - 2) >> 1) & 1u)) return;      // its place is free
    if (!done) open_rows<S>(a, sh.rows[segment & 1], sh.segments[slot], qfrag + (segment & 1) * (S::kQ / 8));
    __syncwarp();
    if (lane == 0) umma::mbar_arrive(umma::smem_u32(&sh.opened[segment & 1]));
    if (segment >= 2) close_segment(a, sh, segment - 2, done);
    if (done) {
      if (segment >= 1) {
        if (!warp_wait(a, sh, &sh.written[(segment - 1) & 1], uint32_t((segment - 1) >> 1) & 1u)) return;
        close_segment(a, sh, segment - 1, true);
      }
      __syncwarp();
      if (lane == 0) umma::mbar_arrive(umma::smem_u32(&sh.ended));
      join_at_end(a, sh, S::W * 32 + lane);
      return;
    }
  }
}

template <int TYPE, class S>
__global__ void __launch_bounds__(S::kThreads, kCtasPerSm) attention_few_kernel(const __grid_constant__ AttnParams a, const __grid_constant__ CUtensorMap k_map,
                                                                                const __grid_constant__ CUtensorMap v_map) {
  using H = Half2Of<TYPE>;
  constexpr int D = S::D, NT = S::NT, PARTS = S::PARTS, TK = S::TK, MT = S::MT, W = S::W;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Shared<S> sh;
  static_assert(sizeof(sh) <= S::kStatic, "two CTAs per SM");
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* merge = reinterpret_cast<float*>(smem + S::kRing);
  uint2* qfrag = reinterpret_cast<uint2*>(smem + S::kRing + S::kMerge);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const uint32_t ring = umma::smem_u32(smem);
  const int boxes = max(1, S::kTile >> a.c.block_log2);                // blocks of a tile
  if (tid == 0) {
    for (int i = 0; i < S::kStages; ++i) {
      umma::mbar_init(umma::smem_u32(&sh.full[i]), uint32_t(boxes + 1));      // who looked its blocks up, and who copies them
      umma::mbar_init(umma::smem_u32(&sh.empty[i]), 2);                // the two warps of the tile
    }
    for (int i = 0; i < kSegments; ++i) {
      umma::mbar_init(umma::smem_u32(&sh.described[i]), 1);
      umma::mbar_init(umma::smem_u32(&sh.closed[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      umma::mbar_init(umma::smem_u32(&sh.opened[i]), 1);
      umma::mbar_init(umma::smem_u32(&sh.written[i]), W);
    }
    umma::mbar_init(umma::smem_u32(&sh.together), W);
    umma::mbar_init(umma::smem_u32(&sh.merged), W);
    umma::mbar_init(umma::smem_u32(&sh.ended), 1);
    sh.lost = sh.joins = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  for (int i = tid; i < 2 * S::kQ / 8; i += S::kThreads) qfrag[i] = make_uint2(0u, 0u);
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  asm volatile("griddepcontrol.wait;\n" ::: "memory");              // nothing of the launches before is read before this
  const Walk first = walk_of<S::kThreads>(a, S::kLog2, W / 2, sh.walk);    // (its barriers: the inits are visible)
  if (warp == W) {
    copy_tiles(a, sh, &k_map, &v_map, ring, first);
    clear_rows_of_nobody(a);
    return;
  }
  if (warp == W + 1) {
    open_and_close<S>(a, sh, qfrag);
    return;
  }

  const int kb = int(swizzled<S::kRow>(tok<S::kRow>(g), t));
  const int vrow = (lane & 8) + tok<S::kRow>(lane & 7) + (MT == 2 ? lane & 16 : 0), vb = int(swizzled<S::kRow>(vrow, 0));

  uint32_t merges = 0;
  for (int segment = 0;; ++segment) {
    if (!warp_wait(a, sh, &sh.opened[segment & 1], uint32_t(segment >> 1) & 1u)) break;
    const Segment& sg = sh.segments[segment & (kSegments - 1)];
    const Rows8<S>& of = sh.rows[segment & 1];
    const uint2* const qf = qfrag + (segment & 1) * (S::kQ / 8) + lane;
    const int tile0 = sg.tile0, tile1 = sg.tile1;
    if (tile0 == tile1) {
      if (!warp_wait(a, sh, &sh.ended, 0)) break;
      join_at_end(a, sh, tid);
      return;
    }
    const int rows = sg.item.r1 - sg.item.r0;
    const int token_base = (sg.item.low >> S::kLog2) * S::kTile + (warp & 1) * TK, number = sg.number - tile0;
    // positions that every row sees: the first row ends first, the last one begins last
    const int all_high = min(sg.s.first + a.by_group(sg.item.r0) + 1, sg.s.end);
    const int all_low = a.window > 0 ? max(0, sg.s.first + a.by_group(sg.item.r1 - 1) - a.window + 1) : 0;
    float factor[NT][2], m[NT][2], l[NT][2], o[S::DC][NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        factor[n][j] = of.factor[8 * n + 2 * t + j];
        m[n][j] = -INFINITY;
        l[n][j] = 0.f;
      }
#pragma unroll
    for (int c = 0; c < S::DC; ++c)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[c][n][j] = 0.f;

    bool lost = false;
    for (int tile = tile0 + (warp >> 1); tile < tile1; tile += W / 2) {
      const uint32_t lap = uint32_t(number + tile) / uint32_t(S::kStages), stage = uint32_t(number + tile) - lap * uint32_t(S::kStages);
      // Tiles land in any order and other laps of this stage are other warps': that the lap before has been read comes first, or the parity of
      // `full` could be that of the lap before it.
      if ((lap > 0 && !warp_wait(a, sh, &sh.empty[stage], (lap - 1u) & 1u)) || !warp_wait(a, sh, &sh.full[stage], lap & 1u)) { lost = true; break; }
      const uint32_t ktile = ring + stage * uint32_t(2 * S::kHalf) + uint32_t((warp & 1) * TK * S::kRow);
      const float4* const box_of = sh.boxes[stage] + (warp & 1) * MT;
      float s[MT][NT][4];
#pragma unroll
      for (int kk = 0; kk < D / 64; ++kk) {
        uint4 raw[MT][2];
        const uint32_t src = ktile + uint32_t((kk >> 1) * S::kTile * S::kRow) + uint32_t(kb ^ ((kk & 1) * 64));
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) raw[i][h] = lds128(src + uint32_t((16 * i + 8 * h) * S::kRow));
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
          uint2 b[NT][PARTS];
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int part = 0; part < PARTS; ++part) b[n][part] = qf[(((4 * kk + i4) * NT + n) * PARTS + part) * 32];
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            uint32_t a0, a1, a2, a3;
            H::along(reinterpret_cast<const uint32_t*>(&raw[i][0])[i4], a0, a2);
            H::along(reinterpret_cast<const uint32_t*>(&raw[i][1])[i4], a1, a3);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int part = 0; part < PARTS; ++part) {
                if (kk == 0 && i4 == 0 && part == 0) mma16816_first(s[i][n], a0, a1, a2, a3, b[n][part].x, b[n][part].y);
                else mma16816(s[i][n], a0, a1, a2, a3, b[n][part].x, b[n][part].y);
              }
          }
        }
      }
      // scores, what is seen of them, the maxima of the tile
      const int token0 = token_base + tile * S::kTile;
      float vs[MT], vt = 0x1p-100f;
      bool every = token0 >= all_low && token0 + TK <= all_high;
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const float4 box = box_of[i];
        const float ks = box.x;
        vs[i] = box.y;
        const bool there = box.z != 0.f;
        vt = fmaxf(vt, vs[i]);                                          // (a NaN is not taken; a box that is not there has zeros)
        every = every && there;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[i][n][j] *= ks * factor[n][j & 1];
      }
      if (!every) {
        // Bytes that no row sees may be anything, and zero times e4m3's NaN codes is not zero: they become zeros.
        if (TYPE == DINOML_B200_KV_E4M3) clear_unseen<S>(ktile + S::kHalf, token0, of.low[0], of.high[rows - 1], box_of);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const bool there = box_of[i].z != 0.f;
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int at = token0 + 16 * i + 8 * (j >> 1) + tok<S::kRow>(g), r = 8 * n + 2 * t + (j & 1);
              if (!there || at < of.low[r] || at >= of.high[r]) s[i][n][j] = -INFINITY;
            }
        }
      }
      float keep[NT][2], join[NT][2], at[NT][2];                        // what O and l, and the tile's share of them, are multiplied by
      bool same = true;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float top = -INFINITY;
#pragma unroll
          for (int i = 0; i < MT; ++i) top = fmaxf(top, fmaxf(s[i][n][j], s[i][n][j + 2]));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
          const float next = fmaxf(m[n][j], top), base = next == -INFINITY ? 0.f : next;
          at[n][j] = top == -INFINITY ? 0.f : top;                      // no score: 2^(-inf - 0) = 0
          keep[n][j] = exp2_approx(m[n][j] - base);
          join[n][j] = exp2_approx(top - base);
          same = same && next == m[n][j];
          m[n][j] = next;
        }
      uint32_t pb[MT][NT][2], rest[MT][NT][2];                          // P^T: row 2t, 2t + 1 (+ 8), column g; what its rounding left, times 2^11
      float sum[NT][2];
      bool tiny = PARTS == 2;
#pragma unroll
      for (int n = 0; n < NT; ++n) sum[n][0] = sum[n][1] = 0.f;
      const float up = 0x1p14f * __frcp_rn(vt);                         // (2^14 vs may be past the largest float32)
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const float f = vs[i] * up;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float p[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float e = exp2_approx(s[i][n][j] - at[n][j & 1]);
            sum[n][j & 1] += e;
            p[j] = s[i][n][j] == -INFINITY ? 0.f : e * f;               // what is not seen has no weight, whatever the block's scale is
            if (PARTS == 1) tiny = tiny || (p[j] > 0.f && p[j] < 0x1p-14f);
          }
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            pb[i][n][h] = pack_half(p[2 * h], p[2 * h + 1]);
            const float2 q = __half22float2(*reinterpret_cast<const __half2*>(&pb[i][n][h]));
            rest[i][n][h] = pack_half((p[2 * h] - q.x) * 0x1p11f, (p[2 * h + 1] - q.y) * 0x1p11f);
            pb[i][n][h] = transposed(pb[i][n][h]);
          }
        }
      }
      same = __all_sync(0xffffffffu, same);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          l[n][j] = l[n][j] * keep[n][j] + sum[n][j] * join[n][j];
          join[n][j] *= vt * 0x1p-14f;
        }
      // V^T P^T, twice where there are two terms, the smaller one first
      bool first_of_two = PARTS == 2 || __any_sync(0xffffffffu, tiny);
      if (first_of_two) {
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) rest[i][n][h] = transposed(rest[i][n][h]);
      }
      const uint32_t vsrc = ktile + S::kHalf + uint32_t(vb);
      while (true) {
        float share[NT][2];
        uint32_t b[MT][NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int j = 0; j < 2; ++j) share[n][j] = first_of_two ? join[n][j] * 0x1p-11f : join[n][j];
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) b[i][n][h] = first_of_two ? rest[i][n][h] : pb[i][n][h];
        }
        if (!same) {
#pragma unroll
          for (int c = 0; c < S::DC; ++c)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int j = 0; j < 4; ++j) o[c][n][j] *= keep[n][j & 1];
        }
#pragma unroll
        for (int c = 0; c < S::DC; ++c) {
          uint32_t r[4];
          const uint32_t src = (vsrc + uint32_t((c >> 3) * S::kTile * S::kRow)) ^ uint32_t((c & (S::kRow / 16 - 1)) << 4);
          if constexpr (MT == 2) ldmatrix4t(src, r); else ldmatrix2t(src, r);
          float x[NT][4];
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            uint32_t a0, a1, a2, a3;
            H::across(r[2 * i], a0, a1);
            H::across(r[2 * i + 1], a2, a3);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              if (i == 0) mma16816_first(x[n], a0, a1, a2, a3, b[i][n][0], b[i][n][1]);
              else mma16816(x[n], a0, a1, a2, a3, b[i][n][0], b[i][n][1]);
            }
          }
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[c][n][j] = fmaf(x[n][j], share[n][j & 1], o[c][n][j]);
        }
        if (!first_of_two) break;
        first_of_two = false;
        same = true;
      }
      __syncwarp();
      if (lane == 0) umma::mbar_arrive(umma::smem_u32(&sh.empty[stage]));
    }
    if (lost) break;

    // ---- the warps' sums become one: eight rows and kMergeCh channels at a time
    constexpr int kPiece = S::R * (D + 2), kPitch = S::kPitch;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float v = l[n][j];
        v += __shfl_xor_sync(0xffffffffu, v, 4);
        v += __shfl_xor_sync(0xffffffffu, v, 8);
        v += __shfl_xor_sync(0xffffffffu, v, 16);
        l[n][j] = v;
      }
    float* mine = merge + warp * 8 * kPitch;
    bool gone = false;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int d0 = 0; d0 < D; d0 += S::kMergeCh) {
        if (gone) break;
        if (merges > 0 && !warp_wait(a, sh, &sh.merged, (merges - 1u) & 1u)) { gone = true; break; }      // what was there has been read
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (d0 == 0 && g == 0) sh.ml[warp][8 * n + 2 * t + j] = make_float2(m[n][j], l[n][j]);
#pragma unroll
          for (int c = 0; c < S::kMergeCh / 16; ++c)
            *reinterpret_cast<float2*>(mine + (2 * t + j) * kPitch + 16 * c + 2 * g) = make_float2(o[d0 / 16 + c][n][j], o[d0 / 16 + c][n][j + 2]);
        }
        __syncwarp();
        if (lane == 0) umma::mbar_arrive(umma::smem_u32(&sh.together));
        if (!warp_wait(a, sh, &sh.together, merges & 1u)) { gone = true; break; }
        for (int i = tid; i < 8 * S::kMergeCh / 4; i += W * 32) {
          const int r = 8 * n + i / (S::kMergeCh / 4), d = i % (S::kMergeCh / 4) * 4;
          if (r >= rows) break;
          float2 ml[W];
          float top = -INFINITY, sum = 0.f;
#pragma unroll
          for (int x = 0; x < W; ++x) {
            ml[x] = sh.ml[x][r];
            top = fmaxf(top, ml[x].x);
          }
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int x = 0; x < W; ++x) {
            const float4 y = *reinterpret_cast<const float4*>(merge + (x * 8 + (r & 7)) * kPitch + d);
            const float f = ml[x].x == -INFINITY ? 1.f : exp2_approx(ml[x].x - top);      // (no score: zeros, or NaN)
            sum = fmaf(ml[x].y, f, sum);
            v = make_float4(fmaf(y.x, f, v.x), fmaf(y.y, f, v.y), fmaf(y.z, f, v.z), fmaf(y.w, f, v.w));
          }
          if (sg.piece < 0) {
            finish(a, sg, D, r, d0 + d, v, sum);
          } else {
            float* part = a.partial + size_t(sg.piece) * kPiece;
            __stcg(reinterpret_cast<float4*>(part + r * D + d0 + d), v);
            if (d0 + d == 0) __stcg(reinterpret_cast<float2*>(part + S::R * D + 2 * r), make_float2(top, sum));
          }
        }
        __syncwarp();
        if (lane == 0) umma::mbar_arrive(umma::smem_u32(&sh.merged));
        ++merges;
      }
    }
    if (gone) break;
    if (lane == 0) umma::mbar_arrive(umma::smem_u32(&sh.written[segment & 1]));      // (behind the __syncwarp above)
  }
  // a wait gave up: copies may still be on their way into this CTA's memory
  for (int i = 0; i < 1000; ++i) __nanosleep(1000);
}

// Map of K or V: rows of head_dim bytes, boxes of one block's share of a tile, swizzled by rows of 128 (64) bytes.
inline bool cache_map(CUtensorMap* map, const void* data, const Cache& c, int tokens) {
  EncodeTiledFn encode = encode_tiled();
  if (encode == nullptr) return false;
  const cuuint64_t dims[2] = {cuuint64_t(c.dim), (cuuint64_t(c.blocks) * c.heads) << c.block_log2}, strides[1] = {cuuint64_t(c.dim)};
  const cuuint32_t box[2] = {cuuint32_t(c.dim == 64 ? 64 : 128), cuuint32_t(tokens)}, steps[2] = {1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(data), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                c.dim == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int TYPE, int D, int NT, int PARTS> int launch(AttnParams& a, cudaStream_t s) {
  using S = Shape<D, NT, PARTS>;
  a.row_tile = S::R;
  a.row_tile_log2 = S::NT == 1 ? 3 : 4;
  a.ends = kEnds;
  const int tokens = S::kTile < (1 << a.c.block_log2) ? S::kTile : 1 << a.c.block_log2;
  CUtensorMap k_map, v_map;
  if (!cache_map(&k_map, a.c.data[0], a.c, tokens) || !cache_map(&v_map, a.c.data[1], a.c, tokens)) return RC_LAUNCH;
  const int ctas = stream::sm_count() * kCtasPerSm;
  a.partial = attention_scratch(size_t(ctas) * 2 * S::R * (D + 2), ctas, s, &a.arrived);
  if (a.partial == nullptr) return RC_LAUNCH;
  static SmemOptIn opt;
  auto kern = attention_few_kernel<TYPE, S>;
  if (!smem_opt_in(kern, S::kSmem, opt)) return RC_LAUNCH;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(ctas));
  cfg.blockDim = dim3(S::kThreads);
  cfg.dynamicSmemBytes = S::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, a, k_map, v_map) == cudaSuccess ? RC_OK : RC_LAUNCH;
}

// `tiles` of eight rows: 1 or 2 (heads of 256: 1).
template <int TYPE, int PARTS> int launch_rows(AttnParams& a, int tiles, cudaStream_t s) {
  switch (a.c.dim) {
    case 64: return tiles == 1 ? launch<TYPE, 64, 1, PARTS>(a, s) : launch<TYPE, 64, 2, PARTS>(a, s);
    case 128: return tiles == 1 ? launch<TYPE, 128, 1, PARTS>(a, s) : launch<TYPE, 128, 2, PARTS>(a, s);
    default: return launch<TYPE, 256, 1, PARTS>(a, s);
  }
}
template <int TYPE> int launch_shape(AttnParams& a, int tiles, cudaStream_t s) {
  return a.dtype == DINO_F32 ? launch_rows<TYPE, 2>(a, tiles, s) : launch_rows<TYPE, 1>(a, tiles, s);
}

}  // namespace few
}  // namespace kv
}  // namespace b200gguf

// Attention of few rows per cached head (decode, short chunks) over the 8-bit cache: the call is bound by the bytes of the cache, so they are
// streamed once and the products follow on mma.sync at a fraction of its rate.
//
// S^T = K Q^T and O^T = V^T P^T, the cached tile as the 16-row operand: with one to eight heads per cached head the 8-column operand is filled
// best by the heads.  A warp takes tiles of TK tokens of one head by itself, through a ring of its own: one lane per box issues the copies
// (TMA with the 128-byte swizzle, a box is one block's share of the tile) and the same warp reads them, so the ring needs no "free" barrier
// and warps meet only where an item ends.
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

constexpr int kWarps = 4, kThreads = kWarps * 32, kCtasPerSm = 2;

template <int D_, int NT_, int PARTS_> struct Shape {
  static constexpr int D = D_, NT = NT_, PARTS = PARTS_;
  static constexpr int R = 8 * NT;                                        // rows of an item
  static constexpr int TK = D == 256 ? 16 : 32, kLog2 = D == 256 ? 4 : 5;  // tokens of a tile
  static constexpr int MT = TK / 16, KS = D / 16, DC = D / 16;             // 16-token rows, 16-value steps, 16-channel rows
  static constexpr int kRow = D == 64 ? 64 : 128;                          // bytes of a row of a box
  static constexpr int kBoxes = D == 256 ? 2 : 1;                          // boxes side by side
  static constexpr int kHalf = TK * D;                                     // bytes of a tile's K, and of its V
  static constexpr int kQ = KS * NT * PARTS * 32 * 8;                      // q as operand fragments
  static constexpr int kStages = D == 64 ? 5 : kQ > 4096 ? 2 : 3;
  static constexpr int kMergeCh = 64;
  static constexpr int kMerge = kWarps * 8 * (kMergeCh + 4) * 4;           // sums of 8 rows and 64 channels of every warp
  static constexpr int kRing = kWarps * kStages * 2 * kHalf;
  static constexpr size_t kSmem = 1024 + kRing + kMerge + kQ;
  static_assert(kSmem + 2048 <= 113 * 1024, "two CTAs per SM");
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
  if (a.dtype == DINO_F32) return __ldg(static_cast<const float*>(a.q) + at);
  if (a.dtype == DINO_F16) return __half2float(static_cast<const __half*>(a.q)[at]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(a.q)[at]);
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

template <class S> struct Shared {
  uint64_t bars[kWarps][S::kStages];
  float scales[kWarps][S::kStages][2][2];      // of the tile's blocks (tiles of 32 tokens have two blocks of 16): K, V
  int valid[kWarps][S::kStages][2];
  float ml[kWarps][S::R][2];
  float factor[S::R];                          // of a row's scores: what q was divided by, the softmax scale, log2(e)
  int low[S::R], high[S::R];                   // positions that a row sees
  int64_t walk[2 + kWarps];
  int last, lost;                              // lost: a copy never arrived
};

template <int TYPE, class S>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) attention_few_kernel(const AttnParams a, const __grid_constant__ CUtensorMap k_map,
                                                                             const __grid_constant__ CUtensorMap v_map) {
  using H = Half2Of<TYPE>;
  constexpr int D = S::D, NT = S::NT, PARTS = S::PARTS, TK = S::TK, MT = S::MT, kStages = S::kStages;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Shared<S> sh;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* merge = reinterpret_cast<float*>(smem + S::kRing);
  uint2* qfrag = reinterpret_cast<uint2*>(smem + S::kRing + S::kMerge);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const uint32_t ring = umma::smem_u32(smem) + uint32_t(warp * kStages * 2 * S::kHalf);
  const int box_tokens = min(TK, 1 << a.c.block_log2), boxes = TK / box_tokens;      // of a tile: 1 or 2 blocks
  if (lane < kStages) umma::mbar_init(umma::smem_u32(&sh.bars[warp][lane]), uint32_t(4 * boxes));
  asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  if (tid == 0) sh.lost = 0;
  const Walk first = walk_of<kThreads>(a, S::kLog2, kWarps, sh.walk);      // (its barriers: the inits are visible)

  // ---- copies: a cursor of its own, kStages tiles ahead.  Lane i < 2 * boxes: box i / 2 of the tile, K or V.
  Walk ahead = first;
  int next = ahead.done() ? 0 : ahead.tile + warp;                    // tile of `ahead`'s item that comes next
  auto settle = [&] {                                                 // on to the first item that has a tile left for this warp
    while (!ahead.done()) {
      const int limit = int(min(int64_t(ahead.tiles), ahead.stop - ahead.item_unit));
      if (next < limit) break;
      ahead.next_item(a, S::kLog2);
      next = ahead.tile + warp;
    }
  };
  settle();
  int id = -1;
  auto look_up = [&] {                                                // the block of this lane's box
    id = -1;
    if (ahead.done() || lane >= 2 * boxes) return;
    const int token = ((ahead.item.low >> S::kLog2) + next) * TK + (lane >> 1) * box_tokens;
    if (token < ahead.item.high && token + box_tokens > ahead.item.low) id = block_at(a.p, a.c.blocks, ahead.b, token >> a.c.block_log2);
  };
  look_up();
  auto issue = [&](int stage) {                                       // the tile that was looked up; then the next one is
    if (ahead.done()) return;
    if (lane < 2 * boxes) {
      const int box = lane >> 1, which = lane & 1;
      const uint32_t bar = umma::smem_u32(&sh.bars[warp][stage]);
      const uint32_t dst = ring + uint32_t(stage * 2 * S::kHalf + which * S::kHalf + box * box_tokens * S::kRow);
      if (which == 0) sh.valid[warp][stage][box] = id >= 0;
      if (id >= 0) {
        const int token = ((ahead.item.low >> S::kLog2) + next) * TK + box * box_tokens;
        const int64_t bh = int64_t(id) * a.c.heads + ahead.head;
        const int row = int((bh << a.c.block_log2) + (token & ((1 << a.c.block_log2) - 1)));
        umma::mbar_arrive_expect_tx(bar, uint32_t(box_tokens * D));
        for (int i = 0; i < S::kBoxes; ++i) tma_load_2d(dst + uint32_t(i * TK * S::kRow), which == 0 ? &k_map : &v_map, bar, i * 128, row);
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(umma::smem_u32(&sh.scales[warp][stage][box][which])), "l"(a.c.scale[which] + bh) : "memory");
        asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];\n" ::"r"(bar) : "memory");
      } else {
        umma::mbar_arrive(bar);
        umma::mbar_arrive(bar);
      }
    }
    next += kWarps;
    settle();
    look_up();
  };
  for (int i = 0; i < kStages; ++i) issue(i);

  // ---- items
  int stage = 0;
  uint32_t phase = 0;
  for (Walk w = first; !w.done(); w.next_item(a, S::kLog2)) {
    const int tile0 = w.tile, tile1 = int(min(int64_t(w.tiles), w.stop - w.item_unit));
    const int rows = w.item.r1 - w.item.r0;
    __syncthreads();                                                  // the last item's q, bounds and sums have been read
    for (int r = warp; r < S::R; r += kWarps) {
      const int token = (w.item.r0 + r) / a.group, head = w.head * a.group + (w.item.r0 + r) % a.group;
      const int64_t at = int64_t(w.s.row + token) * a.row_stride + int64_t(head) * a.head_stride;
      float x[D / 32 < 4 ? 4 : D / 32];
      uint32_t largest = 0;
#pragma unroll
      for (int i = 0; i < (D + 127) / 128; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int e = 128 * i + 4 * lane + j;
          const float v = r < rows && e < D ? load_q(a, at + e) : 0.f;
          x[4 * i + j] = v;
          largest = max(largest, __float_as_uint(v) & 0x7fffffffu);
        }
      largest = __reduce_max_sync(0xffffffffu, largest);
      // 2^12 <= |largest| up < 2^13; zeros, denormals, infinities and NaN as they are
      const uint32_t e = largest >> 23;
      const bool plain = e == 0 || e == 255;
      const int shift = plain ? 0 : min(max(127 + 12 - int(e), -126), 126);
      const float up = __uint_as_float(uint32_t(127 + shift) << 23), down = __uint_as_float(uint32_t(127 - shift) << 23);
#pragma unroll
      for (int i = 0; i < (D + 127) / 128; ++i) {
        const int e0 = 128 * i + 4 * lane;
        if (e0 < D) {
          const int ks = (e0 / 64) * 4 + (e0 % 16) / 4, tt = (e0 % 64) / 16;
          float v[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = x[4 * i + j] * up;
#pragma unroll
          for (int part = 0; part < PARTS; ++part) {
            const uint32_t lo = pack_half(v[0], v[1]), hi = pack_half(v[2], v[3]);
            qfrag[((ks * NT + (r >> 3)) * PARTS + part) * 32 + (r & 7) * 4 + tt] = make_uint2(lo, hi);
            if (part + 1 < PARTS) {
              const float2 l = __half22float2(*reinterpret_cast<const __half2*>(&lo)), h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
              v[0] -= l.x; v[1] -= l.y; v[2] -= h.x; v[3] -= h.y;
            }
          }
        }
      }
      if (lane == 0) {
        const int position = w.s.first + token;
        sh.factor[r] = a.scale * down * H::kFactor;
        sh.high[r] = r < rows ? min(position + 1, w.s.end) : 0;
        sh.low[r] = a.window > 0 ? max(0, position - a.window + 1) : 0;
      }
    }
    __syncthreads();
    float factor[NT][2], m[NT][2], l[NT][2], o[S::DC][NT][4];
    int low[NT][2], high[NT][2];
    int all_low = 0, all_high = INT32_MAX;                             // positions that every row sees
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int r = 8 * n + 2 * t + j;
        factor[n][j] = sh.factor[r];
        low[n][j] = sh.low[r];
        high[n][j] = sh.high[r];
        m[n][j] = -INFINITY;
        l[n][j] = 0.f;
        if (r < rows) {
          all_low = max(all_low, low[n][j]);
          all_high = min(all_high, high[n][j]);
        }
      }
#pragma unroll
    for (int c = 0; c < S::DC; ++c)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[c][n][j] = 0.f;
    all_low = __reduce_max_sync(0xffffffffu, all_low);
    all_high = __reduce_min_sync(0xffffffffu, all_high);

    for (int tile = tile0 + warp; tile < tile1; tile += kWarps) {
      const uint32_t bar = umma::smem_u32(&sh.bars[warp][stage]);
      bool landed = false;
      for (uint32_t i = 0; i < umma::kSpinLimit && !landed && !*static_cast<volatile int*>(&sh.lost); ++i) landed = umma::mbar_try_wait(bar, phase);
      if (!__all_sync(0xffffffffu, landed)) {                           // results are lost, nothing hangs
        sh.lost = 1;
        atomicCAS(a.p.status, 0, ST_KV_TIMEOUT);
        break;
      }
      const uint32_t ktile = ring + uint32_t(stage * 2 * S::kHalf), vtile = ktile + S::kHalf;
      float s[MT][NT][4];
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[i][n][j] = 0.f;
#pragma unroll
      for (int kk = 0; kk < D / 64; ++kk) {
        uint4 raw[MT][2];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            raw[i][h] = lds128(ktile + uint32_t((kk >> 1) * TK * S::kRow) + swizzled<S::kRow>(16 * i + 8 * h + tok<S::kRow>(g), 4 * (kk & 1) + t));
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
          uint2 b[NT][PARTS];
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int part = 0; part < PARTS; ++part) b[n][part] = qfrag[(((4 * kk + i4) * NT + n) * PARTS + part) * 32 + lane];
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            const uint32_t u = H::word(reinterpret_cast<const uint32_t*>(&raw[i][0])[i4]), v = H::word(reinterpret_cast<const uint32_t*>(&raw[i][1])[i4]);
            const uint32_t a0 = H::template pair<0, 1>(u), a2 = H::template pair<2, 3>(u), a1 = H::template pair<0, 1>(v), a3 = H::template pair<2, 3>(v);
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int part = 0; part < PARTS; ++part) mma16816(s[i][n], a0, a1, a2, a3, b[n][part].x, b[n][part].y);
          }
        }
      }
      // scores, what is seen of them, the running maximum
      const int token0 = ((w.item.low >> S::kLog2) + tile) * TK;
      float vs[MT], vt = 0x1p-100f;
      bool every = token0 >= all_low && token0 + TK <= all_high;
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int box = boxes == 1 ? 0 : i;
        const float ks = sh.scales[warp][stage][box][0];
        vs[i] = sh.scales[warp][stage][box][1];
        const bool there = sh.valid[warp][stage][box] != 0;
        if (there) vt = fmaxf(vt, vs[i]);                               // (a NaN is not taken)
        every = every && there;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) s[i][n][j] *= ks * factor[n][j & 1];
      }
      if (!every) {
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const bool there = sh.valid[warp][stage][boxes == 1 ? 0 : i] != 0;
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int at = token0 + 16 * i + 8 * (j >> 1) + tok<S::kRow>(g);
              if (!there || at < low[n][j & 1] || at >= high[n][j & 1]) s[i][n][j] = -INFINITY;
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
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const float f = vs[i] * (0x1p14f / vt);
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
          join[n][j] *= vt * (0x1p-14f * H::kFactor);
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
      while (true) {
        const float small = first_of_two ? 0x1p-11f : 1.f;
        uint32_t b[MT][NT][2];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h) b[i][n][h] = first_of_two ? rest[i][n][h] : pb[i][n][h];
#pragma unroll
        for (int c = 0; c < S::DC; ++c) {
          uint32_t r[4];
          const int row = (lane & 8) + tok<S::kRow>(lane & 7) + (MT == 2 ? lane & 16 : 0);
          const uint32_t src = vtile + uint32_t((c >> 3) * TK * S::kRow) + swizzled<S::kRow>(row, c & (S::kRow / 16 - 1));
          if constexpr (MT == 2) ldmatrix4t(src, r); else ldmatrix2t(src, r);
          float x[NT][4];
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) x[n][j] = 0.f;
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            const uint32_t u = H::word(r[2 * i]), v = H::word(r[2 * i + 1]);
            const uint32_t a0 = H::template pair<0, 2>(u), a1 = H::template pair<1, 3>(u), a2 = H::template pair<0, 2>(v), a3 = H::template pair<1, 3>(v);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma16816(x[n], a0, a1, a2, a3, b[i][n][0], b[i][n][1]);
          }
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              o[c][n][j] = fmaf(x[n][j], join[n][j & 1] * small, same ? o[c][n][j] : o[c][n][j] * keep[n][j & 1]);
        }
        if (!first_of_two) break;
        first_of_two = false;
        same = true;
      }
      __syncwarp();
      issue(stage);
      if (++stage == kStages) { stage = 0; phase ^= 1u; }
    }

    // ---- the warps' sums become one
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float v = l[n][j];
        v += __shfl_xor_sync(0xffffffffu, v, 4);
        v += __shfl_xor_sync(0xffffffffu, v, 8);
        v += __shfl_xor_sync(0xffffffffu, v, 16);
        if (g == 0) {
          sh.ml[warp][8 * n + 2 * t + j][0] = m[n][j];
          sh.ml[warp][8 * n + 2 * t + j][1] = v;
        }
      }
    __syncthreads();
    auto joint = [&](int r, float& top, float& sum) {
      top = -INFINITY;
      sum = 0.f;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) top = fmaxf(top, sh.ml[i][r][0]);
      // (a NaN is in the sums)
#pragma unroll
      for (int i = 0; i < kWarps; ++i) sum += sh.ml[i][r][0] == -INFINITY ? sh.ml[i][r][1] : sh.ml[i][r][1] * exp2_approx(sh.ml[i][r][0] - top);
    };
    const bool whole = tile0 == 0 && tile1 == w.tiles;
    constexpr int kPiece = S::R * (D + 2);
    // The CTA's first piece of work, or its last: others are whole.
    float* part = a.partial + (size_t(blockIdx.x) * 2 + (w.item_unit + tile0 == first.start ? 0 : 1)) * kPiece;
    auto finish = [&](int r, int d, float4 v, float sum) {              // channels d .. d + 3 of a row
      const float f = sum == 0.f ? 0.f : 1.f / sum;
      const int64_t row = w.s.row + (w.item.r0 + r) / a.group, head = w.head * a.group + (w.item.r0 + r) % a.group;
      store4(a, (row * a.heads + head) * D + d, make_float4(v.x * f, v.y * f, v.z * f, v.w * f));
    };
    constexpr int kPitch = S::kMergeCh + 4;
    float* mine = merge + warp * 8 * kPitch;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float f[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float top, sum;
        joint(8 * n + 2 * t + j, top, sum);
        f[j] = m[n][j] == -INFINITY ? 1.f : exp2_approx(m[n][j] - top);
      }
#pragma unroll
      for (int d0 = 0; d0 < D; d0 += S::kMergeCh) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int c = 0; c < S::kMergeCh / 16; ++c)
            *reinterpret_cast<float2*>(mine + (2 * t + j) * kPitch + 16 * c + 2 * g) = make_float2(o[d0 / 16 + c][n][j] * f[j], o[d0 / 16 + c][n][j + 2] * f[j]);
        __syncthreads();
        const int r = 8 * n + tid / (S::kMergeCh / 4), d = tid % (S::kMergeCh / 4) * 4;      // (128 threads: eight rows of sixteen float4)
        if (r < rows) {
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int x = 0; x < kWarps; ++x) {
            const float4 y = *reinterpret_cast<const float4*>(merge + (x * 8 + (r & 7)) * kPitch + d);
            v.x += y.x; v.y += y.y; v.z += y.z; v.w += y.w;
          }
          float top, sum;
          joint(r, top, sum);
          if (whole) {
            finish(r, d0 + d, v, sum);
          } else {
            __stcg(reinterpret_cast<float4*>(part + r * D + d0 + d), v);
            if (d0 + d == 0) __stcg(reinterpret_cast<float2*>(part + S::R * D + 2 * r), make_float2(top, sum));
          }
        }
        if (d0 + S::kMergeCh < D || n + 1 < NT) __syncthreads();
      }
    }
    if (!whole) {
      // Cut: pieces are those of CTAs c0 .. c1; the one that arrives last adds them up.  The counter is that of c0, whose range is the only one that
      // a cut item leaves at its end.
      const int c0 = w.owner(w.item_unit), c1 = w.owner(w.item_unit + w.tiles - 1);
      __threadfence();
      __syncthreads();
      if (tid == 0) sh.last = atomicAdd(a.arrived + c0, 1) == c1 - c0;
      __syncthreads();
      if (sh.last) {
        __threadfence();
        if (tid == 0) a.arrived[c0] = 0;
        for (int i = tid; i < rows * (D / 4); i += kThreads) {
          const int r = i / (D / 4), d = i % (D / 4) * 4;
          float top = -INFINITY, sum = 0.f;
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
          for (int c = c0; c <= c1; ++c) {
            const float* src = a.partial + (size_t(c) * 2 + (w.start_of(c) >= w.item_unit ? 0 : 1)) * kPiece;
            const float2 ml = __ldcg(reinterpret_cast<const float2*>(src + S::R * D + 2 * r));
            const float4 y = __ldcg(reinterpret_cast<const float4*>(src + r * D + d));
            const float high = fmaxf(top, ml.x);
            const float f0 = top == -INFINITY ? 1.f : exp2_approx(top - high), f1 = ml.x == -INFINITY ? 1.f : exp2_approx(ml.x - high);
            sum = sum * f0 + ml.y * f1;
            v = make_float4(v.x * f0 + y.x * f1, v.y * f0 + y.y * f1, v.z * f0 + y.z * f1, v.w * f0 + y.w * f1);
            top = high;
          }
          finish(r, d, v, sum);
        }
      }
    }
  }
  if (sh.lost)                                                          // copies may still be on their way into this CTA's memory
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
  const int tokens = S::TK < (1 << a.c.block_log2) ? S::TK : 1 << a.c.block_log2;
  CUtensorMap k_map, v_map;
  if (!cache_map(&k_map, a.c.data[0], a.c, tokens) || !cache_map(&v_map, a.c.data[1], a.c, tokens)) return RC_LAUNCH;
  const int ctas = stream::sm_count() * kCtasPerSm;
  a.partial = attention_scratch(size_t(ctas) * 2 * S::R * (D + 2), ctas, s, &a.arrived);
  if (a.partial == nullptr) return RC_LAUNCH;
  static SmemOptIn opt;
  auto kern = attention_few_kernel<TYPE, S>;
  if (!smem_opt_in(kern, S::kSmem, opt)) return RC_LAUNCH;
  kern<<<ctas, kThreads, S::kSmem, s>>>(a, k_map, v_map);
  return cudaGetLastError() == cudaSuccess ? RC_OK : RC_LAUNCH;
}

// `tiles` of eight rows: 1, 2 or 4 (float32, and heads of 256: at most 2, the sums are registers).
template <int TYPE> int launch_shape(AttnParams& a, int tiles, cudaStream_t s) {
  if (a.dtype == DINO_F32) {
    switch (a.c.dim) {
      case 64: return tiles == 1 ? launch<TYPE, 64, 1, 2>(a, s) : launch<TYPE, 64, 2, 2>(a, s);
      case 128: return tiles == 1 ? launch<TYPE, 128, 1, 2>(a, s) : launch<TYPE, 128, 2, 2>(a, s);
      default: return tiles == 1 ? launch<TYPE, 256, 1, 2>(a, s) : launch<TYPE, 256, 2, 2>(a, s);
    }
  }
  switch (a.c.dim) {
    case 64: return tiles == 1 ? launch<TYPE, 64, 1, 1>(a, s) : tiles == 2 ? launch<TYPE, 64, 2, 1>(a, s) : launch<TYPE, 64, 4, 1>(a, s);
    case 128: return tiles == 1 ? launch<TYPE, 128, 1, 1>(a, s) : tiles == 2 ? launch<TYPE, 128, 2, 1>(a, s) : launch<TYPE, 128, 4, 1>(a, s);
    default: return tiles == 1 ? launch<TYPE, 256, 1, 1>(a, s) : launch<TYPE, 256, 2, 1>(a, s);
  }
}

}  // namespace few
}  // namespace kv
}  // namespace b200gguf

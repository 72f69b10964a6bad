// Products of streamed weights with a few rows of activations (1 to 32 tokens), shared by the
// few-token layer and the few-row 4-bit projection.
//
// At these sizes a product reads every weight once for a handful of multiply-adds, so it is bound by
// HBM, and what matters is that every SM has enough bytes in flight and spends few instructions per
// byte:
//
// * Each warp owns a ring of shared-memory slots and fills it itself with bulk
//   tensor copies of (rows x 128 bytes) boxes; no warp waits for another inside a reduction.  The
//   warps share out the boxes of a unit (a few weight rows over the whole reduction) and add up
//   their accumulators through shared memory once per unit.  A ring has two or three slots beside sums and
//   kept codes, up to six for eight warps with an SM to themselves, and one where MX boxes are 8 KB (gate and
//   up rows of 32 columns) or 4-bit rows fill the memory: then only the other warps' boxes are in
//   flight while a warp computes.
// * The weights are the A operand (16 rows) of mma.sync.m16n8k16, the tokens its eight columns.
//   tcgen05 wants 128 rows on the A side and its operands in shared memory in their final format;
//   here the 8- and 4-bit codes are widened to halves in registers on the way (exact: e4m3, int8
//   and e2m1 x e4m3 all fit a half).  Products are exact and sums fp32, those of int8 codes too: they
//   can round from 2^24 on, which a block-scaled group of 128 never reaches and 1041 of the largest codes do.  Widening
//   is what bounds the 4-bit kinds, and all kinds once several token tiles use the same weights.
// * The K order inside a box is free as long as both operands agree.  A lane takes 32 contiguous
//   bytes of its row (two 16-byte chunks, which the 128-byte swizzle places without bank
//   conflicts), and the same 32 bytes' worth of its token.  MX codes go by 4-byte words instead, so
//   that one instruction pair covers exactly one 32-value block, whose scales multiply the fp32
//   partial sum: two E8M0 scales span more than a half's exponent.
#pragma once

#include "fp4.cuh"
#include "tc_ptx.cuh"

namespace bolt {
namespace few {
using namespace tc;

constexpr int kMaxTokens = 32;

// values of enum bolt_decode_kind
enum Kind { K_BF16, K_F16, K_F8_BLOCK, K_I8_CHANNEL, K_F8_CHANNEL, K_I8_BLOCK, K_NV4, K_MX4 };
constexpr bool is16(int k) { return k == K_BF16 || k == K_F16; }
constexpr bool is4(int k) { return k == K_NV4 || k == K_MX4; }
constexpr bool is8(int k) { return !is16(k) && !is4(k); }
constexpr bool is_i8(int k) { return k == K_I8_CHANNEL || k == K_I8_BLOCK; }
constexpr bool is_block(int k) { return k == K_F8_BLOCK || k == K_I8_BLOCK; }
constexpr bool is_channel(int k) { return k == K_F8_CHANNEL || k == K_I8_CHANNEL; }
constexpr int box_elems(int k) { return is16(k) ? 64 : is4(k) ? 256 : 128; }   // in 128 bytes
// bytes of a row of n values
__host__ __device__ constexpr int64_t row_bytes(int k, int64_t n) {
  return is16(k) ? 2 * n : is4(k) ? n / 2 : n;
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0,
                                            int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, "
      "{%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr));
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}
// The next kernel of the stream may start (it still waits for this one before it reads its results).
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;"); }
// All earlier kernels of the stream are done and their writes can be read.
__device__ __forceinline__ void wait_for_previous() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

template <bool BF>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1) {
  if (BF)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
        "{%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// four 8-bit codes -> two packed pairs of halves, exact
template <bool INT>
__device__ __forceinline__ void halves4(uint32_t w, uint32_t& p0, uint32_t& p1) {
  if (INT) {
    // 0x6400 + u is the half 1024 + u; u = code + 128
    const uint32_t u = w ^ 0x80808080u;
    const uint32_t lo = __byte_perm(u, 0x64646464u, 0x4140), hi = __byte_perm(u, 0x64646464u, 0x4342);
    const uint32_t off = 0x64806480u;      // 1024 + 128
    const __half2 o = *reinterpret_cast<const __half2*>(&off);
    const __half2 a = __hsub2(*reinterpret_cast<const __half2*>(&lo), o);
    const __half2 b = __hsub2(*reinterpret_cast<const __half2*>(&hi), o);
    p0 = *reinterpret_cast<const uint32_t*>(&a);
    p1 = *reinterpret_cast<const uint32_t*>(&b);
  } else {
    asm("{\n.reg .b16 lo, hi;\nmov.b32 {lo, hi}, %2;\ncvt.rn.f16x2.e4m3x2 %0, lo;\n"
        "cvt.rn.f16x2.e4m3x2 %1, hi;\n}\n"
        : "=r"(p0), "=r"(p1)
        : "r"(w));
  }
}
// E4M3 scale byte i of a word, in both halves of a pair
__device__ __forceinline__ uint32_t scale_pair(uint32_t w, int i) {
  uint32_t lo, hi;
  halves4<false>(w, lo, hi);
  return __byte_perm(i < 2 ? lo : hi, 0u, (i & 1) ? 0x3232 : 0x1010);
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// 32 bytes of one token, as the lane (column lane / 4, position lane % 4) multiplies them, with the
// scales of 4-bit codes: NV the lane's own four E4M3 bytes, MX the eight E8M0 bytes of the columns
// 2 (lane % 4) and 2 (lane % 4) + 1.
template <int K>
struct TokenBox {
  uint32_t w[8];
  uint32_t sf[is4(K) ? (K == K_MX4 ? 4 : 1) : 1];
};
// Scales of weight rows g and g + 8 of a tile: the bytes of 4-bit kinds (NV: of the lane's 64 values,
// MX: of the box), the bits of the box's fp32 scale of block-scaled ones.
template <int K>
struct RowScales {
  uint32_t sf[2][K == K_MX4 ? 2 : 1];
};

// d[tile][token tile] += (box of weights) . (tokens).  The box: rows of 128 bytes, swizzled (16-byte
// chunk c of row r at chunk c ^ (r % 8)).  Tile mt holds the box's rows 8 mt + g and second + 8 mt + g
// (UP: gate rows with their up rows) or 16 mt + g and 16 mt + 8 + g; rows that the box does not fill
// give sums that nobody reads.  Only the token tiles of `live` are computed.
template <int K, int MT, int NT, bool UP>
__device__ __forceinline__ void box_mma(uint32_t box, int second, int lane, const TokenBox<K> (&x)[NT],
                                        const RowScales<K> (&ws)[MT], unsigned live,
                                        float (&d)[MT][NT][4]) {
  const int g = lane >> 2, t = lane & 3;
  // (the rows of a thread lie 8 apart, so one place in the swizzle serves them all; up rows have
  // their own)
  const uint32_t row0 = box + (uint32_t)g * 128u;
  const uint32_t row1 = UP ? box + (uint32_t)(second + g) * 128u : row0 + 1024u;
  const int ph0 = g, ph1 = UP ? (second + g) & 7 : g;
  auto row = [&](int mt, int r) { return (r ? row1 : row0) + (UP ? 1024u : 2048u) * mt; };
  if constexpr (K == K_MX4) {
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const uint32_t at[2] = {(uint32_t)((c ^ ph0) << 4) + 4u * t, (uint32_t)((c ^ ph1) << 4) + 4u * t};
      uint32_t a[MT][2][4];
      float sw[MT][2];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          fp4::halves8(lds32(row(mt, r) + at[r]), a[mt][r]);
          sw[mt][r] = fp4::e8m0_to_f32((ws[mt].sf[r][c >> 2] >> (8 * (c & 3))) & 0xFFu);
        }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        if (!((live >> nt) & 1u)) continue;
        uint32_t b[4];
        fp4::halves8(x[nt].w[c], b);
        const float s0 = fp4::e8m0_to_f32((x[nt].sf[c >> 2] >> (8 * (c & 3))) & 0xFFu);
        const float s1 = fp4::e8m0_to_f32((x[nt].sf[2 + (c >> 2)] >> (8 * (c & 3))) & 0xFFu);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          float part[4] = {0.f, 0.f, 0.f, 0.f};
          mma16816<false>(part, a[mt][0][0], a[mt][1][0], a[mt][0][1], a[mt][1][1], b[0], b[1]);
          mma16816<false>(part, a[mt][0][2], a[mt][1][2], a[mt][0][3], a[mt][1][3], b[2], b[3]);
          d[mt][nt][0] = fmaf(part[0], sw[mt][0] * s0, d[mt][nt][0]);
          d[mt][nt][1] = fmaf(part[1], sw[mt][0] * s1, d[mt][nt][1]);
          d[mt][nt][2] = fmaf(part[2], sw[mt][1] * s0, d[mt][nt][2]);
          d[mt][nt][3] = fmaf(part[3], sw[mt][1] * s1, d[mt][nt][3]);
        }
      }
    }
    return;
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t at[2] = {(uint32_t)(((2 * t + h) ^ ph0) << 4), (uint32_t)(((2 * t + h) ^ ph1) << 4)};
      uint32_t a[MT][2][4];
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint4 v = lds128(row(mt, r) + at[r]);
          a[mt][r][0] = v.x;
          a[mt][r][1] = v.y;
          a[mt][r][2] = v.z;
          a[mt][r][3] = v.w;
        }
      if constexpr (is16(K)) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            if (!((live >> nt) & 1u)) continue;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
              mma16816<K == K_BF16>(d[mt][nt], a[mt][0][2 * s], a[mt][1][2 * s], a[mt][0][2 * s + 1],
                                    a[mt][1][2 * s + 1], x[nt].w[4 * h + 2 * s],
                                    x[nt].w[4 * h + 2 * s + 1]);
          }
      } else if constexpr (is8(K)) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t p[MT][2][2];
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int r = 0; r < 2; ++r) halves4<is_i8(K)>(a[mt][r][j], p[mt][r][0], p[mt][r][1]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            if (!((live >> nt) & 1u)) continue;
            uint32_t b0, b1;
            halves4<is_i8(K)>(x[nt].w[4 * h + j], b0, b1);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
              mma16816<false>(d[mt][nt], p[mt][0][0], p[mt][1][0], p[mt][0][1], p[mt][1][1], b0, b1);
          }
        }
      } else {   // NV: codes times their block's scale, exact in a half
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int blk = 2 * h + (j >> 1);
          uint32_t p[MT][2][4];
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              fp4::halves8(a[mt][r][j], p[mt][r]);
              const uint32_t s = scale_pair(ws[mt].sf[r][0], blk);
#pragma unroll
              for (int i = 0; i < 4; ++i) p[mt][r][i] = hmul2(p[mt][r][i], s);
            }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            if (!((live >> nt) & 1u)) continue;
            uint32_t b[4];
            fp4::halves8(x[nt].w[4 * h + j], b);
            const uint32_t s = scale_pair(x[nt].sf[0], blk);
#pragma unroll
            for (int i = 0; i < 4; ++i) b[i] = hmul2(b[i], s);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              mma16816<false>(d[mt][nt], p[mt][0][0], p[mt][1][0], p[mt][0][1], p[mt][1][1], b[0], b[1]);
              mma16816<false>(d[mt][nt], p[mt][0][2], p[mt][1][2], p[mt][0][3], p[mt][1][3], b[2], b[3]);
            }
          }
        }
      }
    }
  }
}

// One token's 32 bytes of box kb out of rows that are stored in the operand's format (16-bit values,
// 4-bit codes): `row` is the token's row or null (zeros), `bytes` its length.
template <int K>
__device__ __forceinline__ void load_token(TokenBox<K>& x, const uint8_t* row, int bytes, int kb, int t) {
  if constexpr (K == K_MX4) {
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const int off = kb * 128 + 16 * c;
      x.w[c] = row != nullptr && off < bytes ? *reinterpret_cast<const uint32_t*>(row + off + 4 * t) : 0u;
    }
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int off = kb * 128 + 32 * t + 16 * h;
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (row != nullptr && off < bytes) v = *reinterpret_cast<const uint4*>(row + off);
      x.w[4 * h] = v.x;
      x.w[4 * h + 1] = v.y;
      x.w[4 * h + 2] = v.z;
      x.w[4 * h + 3] = v.w;
    }
  }
}
// Asynchronous copy of four bytes; `have` false: zeros, nothing is read.
__device__ __forceinline__ void cp_async_4(uint32_t dst, const void* src, bool have) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(have ? 4u : 0u) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All but the newest `pending` groups of this thread have landed; MOST: the deepest ring's slots less one (a
// deeper one would wait for more than it has to).
template <int MOST, int AT = 0>
__device__ __forceinline__ void cp_async_wait(int pending) {
  if constexpr (AT < MOST) {
    if (pending > AT) return cp_async_wait<MOST, AT + 1>(pending);
  }
  asm volatile("cp.async.wait_group %0;" ::"n"(AT) : "memory");
}

// A warp's ring of weight scales, beside its ring of boxes and as far ahead: read when they are needed,
// one box ahead, they came too late (a load takes as long as a box's copy, thousands of cycles while
// HBM is busy; DeepSeek-V3 fp8, one token: a third of the first kernel's time).  kRows rows per lane
// group g.  NV: word [row][lane], the lane's own 64 values.  MX: word [2 row + half][g].  fp32 scales:
// word [row][g].  Words are shared out to the lanes; a slot is kBytes.
template <int K, int ROWS>
struct ScaleRing {
  static constexpr int kWords = K == K_NV4 ? ROWS * 32 : K == K_MX4 ? ROWS * 16 : is8(K) ? ROWS * 8 : 0;
  static constexpr int kBytes = (kWords * 4 + 15) / 16 * 16;
  uint32_t base;
  // src(row, ok): start of the scales of row i (0 .. ROWS - 1) of lane group g: a row's bytes (4-bit) or
  // the scale itself (fp32)
  template <typename Src>
  __device__ __forceinline__ void bring(int slot, int lane, int kb, int row_bytes, Src src) const {
    const int g = lane >> 2, t = lane & 3;
    const uint32_t dst = base + slot * kBytes;
    if constexpr (K == K_NV4) {
      const int off = kb * 16 + 4 * t;
#pragma unroll
      for (int i = 0; i < ROWS; ++i) cp_async_4(dst + (i * 32 + lane) * 4, src(i) + (off < row_bytes ? off : 0), off < row_bytes);
    } else if constexpr (K == K_MX4) {
#pragma unroll
      for (int q = 0; q < ROWS / 2; ++q) {
        const int w = t * (ROWS / 2) + q, off = kb * 8 + 4 * (w & 1);
        cp_async_4(dst + (w * 8 + g) * 4, src(w >> 1) + (off < row_bytes ? off : 0), off < row_bytes);
      }
    } else if constexpr (is8(K)) {
      if (ROWS >= 4 || t < ROWS) {
#pragma unroll
        for (int q = 0; q < (ROWS + 3) / 4; ++q) {
          const int i = t + 4 * q;
          cp_async_4(dst + (i * 8 + g) * 4, src(i), true);
        }
      }
    }
  }
  // after cp_async_wait (and, but for NV, __syncwarp)
  template <int MT>
  __device__ __forceinline__ void read(RowScales<K> (&ws)[MT], int slot, int lane) const {
    const int g = lane >> 2;
    const uint32_t src = base + slot * kBytes;
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      if constexpr (K == K_NV4) {
        ws[i >> 1].sf[i & 1][0] = lds32(src + (i * 32 + lane) * 4);
      } else if constexpr (K == K_MX4) {
        ws[i >> 1].sf[i & 1][0] = lds32(src + ((2 * i) * 8 + g) * 4);
        ws[i >> 1].sf[i & 1][1] = lds32(src + ((2 * i + 1) * 8 + g) * 4);
      } else if constexpr (is8(K)) {
        ws[i >> 1].sf[i & 1][0] = lds32(src + (i * 8 + g) * 4);
      }
    }
  }
};

// Block scales of box kb out of a row of `bytes` scale bytes (a multiple of four): NV the word of
// the lane's own 64 values, MX both words of the box.
template <int K>
__device__ __forceinline__ void load_block_scales(uint32_t* sf, const uint8_t* row, int bytes, int kb,
                                                  int t) {
  if constexpr (K == K_NV4) {
    const int off = kb * 16 + 4 * t;
    sf[0] = row != nullptr && off < bytes ? *reinterpret_cast<const uint32_t*>(row + off) : 0u;
  } else if constexpr (K == K_MX4) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int off = kb * 8 + 4 * i;
      sf[i] = row != nullptr && off < bytes ? *reinterpret_cast<const uint32_t*>(row + off) : 0u;
    }
  }
}

// four values -> four 8-bit codes, the arithmetic of the row quantisers (quant.cu)
template <int K>
__device__ __forceinline__ uint32_t codes4(const float4& v, float inv) {
  if (is_i8(K))
    return ((uint32_t)(uint8_t)f32_to_i8(v.x * inv)) | ((uint32_t)(uint8_t)f32_to_i8(v.y * inv) << 8) |
           ((uint32_t)(uint8_t)f32_to_i8(v.z * inv) << 16) | ((uint32_t)(uint8_t)f32_to_i8(v.w * inv) << 24);
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v.x * inv, v.y * inv), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v.z * inv, v.w * inv), __NV_SATFINITE, __NV_E4M3);
  return lo | (hi << 16);
}
// Scale of a row or group and its reciprocal: amax times the rounded 1 / 448 (1 / 127).  (The row
// quantisers of quant.cu divide; the scales may differ in the last bit.)
template <int K>
__device__ __forceinline__ void scale8(float amax, float& scale, float& inv) {
  scale = fmaxf(amax, 1.0e-10f) * (is_i8(K) ? (float)(1.0 / 127.0) : (float)(1.0 / 448.0));
  inv = __frcp_rn(scale);
}

// four consecutive values of a row as floats; dt BOLT_BF16 / BOLT_F16 / BOLT_F32
__device__ __forceinline__ float4 load_values4(const void* row, int dt, int at) {
  if (dt == BOLT_F32) return *reinterpret_cast<const float4*>(static_cast<const float*>(row) + at);
  const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(row) + at);
  if (dt == BOLT_BF16)
    return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xFFFF0000u),
                       __uint_as_float(u.y << 16), __uint_as_float(u.y & 0xFFFF0000u));
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
  const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
  return make_float4(a.x, a.y, b.x, b.y);
}

// 32 consecutive values of a 16-bit row as floats (the block quantiser of 4-bit rows)
__device__ __forceinline__ void load_values32(float (&v)[32], const uint16_t* row, int dt, int at) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float4 f = load_values4(row, dt, at + 4 * i);
    v[4 * i] = f.x;
    v[4 * i + 1] = f.y;
    v[4 * i + 2] = f.z;
    v[4 * i + 3] = f.w;
  }
}

}  // namespace few
}  // namespace bolt

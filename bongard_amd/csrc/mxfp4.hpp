// MXFP4 blocks: 32 values sharing one power of two (E8M0 byte e), each an e2m1 code
// (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign bit; two codes a byte, the even element in the low
// nibble). The device side of quantizing a tile whose bf16 values a wave holds in registers.
#pragma once

#include "common.hpp"

namespace bf8 {

// Biased exponent e of a block whose max |x| is the bf16 key k (the bits without the sign): 2^(e - 127) is the
// smallest power of two with max |x| <= 6 * 2^(e - 127), 2^-127 at least. 6 = 1.5 * 2^2, so it is
// E - 2, one more where the mantissa passes 1.5 (64 / 128 above 1): ((k + 63) >> 7) - 2.
__device__ __forceinline__ uint32_t mx4_exponent_finite(uint32_t k) {
  const uint32_t t = (k + 63u) >> 7;
  return t > 2u ? t - 2u : 0u;
}
// The same of any block: 0xFE where the largest is infinite, 0xFF (NaN) where a value is NaN.
__device__ __forceinline__ uint32_t mx4_exponent(uint32_t k) {
  if (k > 0x7F80u) return 0xFFu;
  return k == 0x7F80u ? 0xFEu : mx4_exponent_finite(k);
}

// 2^(e - 127) as the conversions take it: they read the exponent field alone, so that e = 0
// stands for 2^-127 too.
__device__ __forceinline__ float mx4_scale(uint32_t e) { return __uint_as_float(e << 23); }

// Round-to-nearest-even onto the e2m1 grid, as the conversions do, for the blocks that hold inf or
// NaN (a block with a NaN has no value: its codes are 0).
__device__ __forceinline__ uint32_t mx4_code_slow(float x, uint32_t e) {
  if (e == 0xFFu) return 0u;
  const float p = x * (e == 0xFEu ? __uint_as_float(0x00400000u) : __uint_as_float((254u - e) << 23));
  const float a = fabsf(p);
  const uint32_t m = (uint32_t)(a > 0.25f) + (uint32_t)(a >= 0.75f) + (uint32_t)(a > 1.25f) +
                     (uint32_t)(a >= 1.75f) + (uint32_t)(a > 2.5f) + (uint32_t)(a >= 3.5f) +
                     (uint32_t)(a > 5.0f);
  return m | ((__float_as_uint(p) >> 31) << 3);
}

// Byte B of c: the codes of a packed bf16 pair (low half in the low nibble).
template <int B, bool FINITE>
__device__ __forceinline__ uint32_t mx4_pack2(uint32_t c, uint32_t pair, uint32_t e) {
  if constexpr (FINITE)
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, pair),
                                                     mx4_scale(e), B);
  else
    return c | ((mx4_code_slow(bf16_lo(pair), e) | (mx4_code_slow(bf16_hi(pair), e) << 4))
                << (8 * B));
}

// Where a quantizer writes: out [rows, cols / 2] with planes [(cols + 127) / 128][rows] (blocks
// along rows, cols % 32 == 0) and / or out_t [cols, rowsp / 2] with planes_t [(rows + 127) / 128]
// [cols] (blocks along columns; rowsp is rows rounded up to 32, the last block filled up with
// zeros). A plane holds one dword per row and group of 128 K-values, absent blocks 127.
struct Mx4Out {
  int64_t rows, cols;
  uint8_t* out;
  uint32_t* planes;
  uint8_t* out_t;
  uint32_t* planes_t;
};

// A tile of 32 W rows x 8 LPR columns, one wave per 32 rows: lane l holds columns 8 (l % LPR) ..
// +7 of RL = LPR / 2 consecutive rows, RL (l / LPR) .. of its wave's 32 (v[k]: row k; zeros past
// the tensor). A row block of 32 is four neighbouring lanes, a column block the lanes of one
// column group, so both maxima are a few lane exchanges, and a lane's column codes are RL / 2
// consecutive bytes of the columnwise copy. LPR = 32 and W = 8 write whole 128-byte lines of both
// copies; a smaller tile gives a small tensor more waves.
template <int LPR, int W>
struct Mx4Tile {
  static constexpr int kRows = 32 * W, kCols = 8 * LPR;
  static constexpr int RL = LPR / 2;
  static constexpr int kPitch = 16 * W + 4;  // bytes of a staged column (16 a wave)
  struct Shared {
    alignas(16) uint8_t rowsc[kRows][kCols / 32 < 4 ? 4 : kCols / 32];  // exponents by row block
    alignas(16) uint8_t colsc[kCols][W < 4 ? 4 : W];                    // and by column block
    alignas(16) uint8_t stage[kCols][kPitch];
  };
};

template <int LPR, int W, bool FINITE>
__device__ __forceinline__ void mx4_tile_body(const Mx4Out& p, int64_t r0, int64_t c0,
                                              const uint4 (&v)[LPR / 2],
                                              const uint32_t (&rk)[LPR / 2],
                                              const uint32_t (&cm)[4],
                                              typename Mx4Tile<LPR, W>::Shared& sh, int wid,
                                              int lane) {
  constexpr int RL = LPR / 2;
  const int cl = lane % LPR, rg = lane / LPR;
  const int64_t c = c0 + 8 * cl;
  const int lrow = 32 * wid + RL * rg;  // the lane's first row in the tile
  if (p.out) {
#pragma unroll
    for (int k = 0; k < RL; ++k) {
      const int64_t r = r0 + lrow + k;
      const uint32_t e = FINITE ? mx4_exponent_finite(rk[k]) : mx4_exponent(rk[k]);
      uint32_t q = 0;
      q = mx4_pack2<0, FINITE>(q, v[k].x, e);
      q = mx4_pack2<1, FINITE>(q, v[k].y, e);
      q = mx4_pack2<2, FINITE>(q, v[k].z, e);
      q = mx4_pack2<3, FINITE>(q, v[k].w, e);
      if (r < p.rows && c < p.cols)
        *reinterpret_cast<uint32_t*>(p.out + ((r * p.cols + c) >> 1)) = q;
      if ((cl & 3) == 0)
        sh.rowsc[lrow + k][cl >> 2] = c < p.cols ? (uint8_t)e : (uint8_t)kMxPadScale;
    }
  }
  if (!p.out_t) return;
  uint32_t e[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    e[2 * i] = FINITE ? mx4_exponent_finite(cm[i] & 0xFFFFu) : mx4_exponent(cm[i] & 0xFFFFu);
    e[2 * i + 1] = FINITE ? mx4_exponent_finite(cm[i] >> 16) : mx4_exponent(cm[i] >> 16);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {  // column pair 2 i, 2 i + 1
    uint32_t lo[RL / 8 < 1 ? 1 : RL / 8] = {}, hi[RL / 8 < 1 ? 1 : RL / 8] = {};
#pragma unroll
    for (int k = 0; k < RL; k += 2) {
      const uint32_t a = i == 0 ? v[k].x : i == 1 ? v[k].y : i == 2 ? v[k].z : v[k].w;
      const uint32_t b = i == 0 ? v[k + 1].x : i == 1 ? v[k + 1].y : i == 2 ? v[k + 1].z : v[k + 1].w;
      const uint32_t p0 = __byte_perm(a, b, 0x5410), p1 = __byte_perm(a, b, 0x7632);
      uint32_t& x = lo[k / 8];
      uint32_t& y = hi[k / 8];
      switch ((k / 2) & 3) {
        case 0: x = mx4_pack2<0, FINITE>(x, p0, e[2 * i]); y = mx4_pack2<0, FINITE>(y, p1, e[2 * i + 1]); break;
        case 1: x = mx4_pack2<1, FINITE>(x, p0, e[2 * i]); y = mx4_pack2<1, FINITE>(y, p1, e[2 * i + 1]); break;
        case 2: x = mx4_pack2<2, FINITE>(x, p0, e[2 * i]); y = mx4_pack2<2, FINITE>(y, p1, e[2 * i + 1]); break;
        default: x = mx4_pack2<3, FINITE>(x, p0, e[2 * i]); y = mx4_pack2<3, FINITE>(y, p1, e[2 * i + 1]); break;
      }
    }
    uint8_t* s0 = &sh.stage[8 * cl + 2 * i][16 * wid + rg * (RL / 2)];
    uint8_t* s1 = &sh.stage[8 * cl + 2 * i + 1][16 * wid + rg * (RL / 2)];
    if constexpr (RL >= 8) {
#pragma unroll
      for (int j = 0; j < RL / 8; ++j) {
        reinterpret_cast<uint32_t*>(s0)[j] = lo[j];
        reinterpret_cast<uint32_t*>(s1)[j] = hi[j];
      }
    } else {
      *reinterpret_cast<uint16_t*>(s0) = (uint16_t)lo[0];
      *reinterpret_cast<uint16_t*>(s1) = (uint16_t)hi[0];
    }
  }
  if (rg == 0) {
    const bool valid = r0 + 32 * wid < p.rows;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      sh.colsc[8 * cl + j][wid] = valid ? (uint8_t)e[j] : (uint8_t)kMxPadScale;
  }
}

// The loaded tile at (r0, c0), by the W waves of a block (wid 0 .. W - 1), each of which calls it
// alike. W < 4: planes_t's dword is written a byte at a time, and the wave of a tensor's last
// block fills the absent ones of its dword.
template <int LPR, int W>
__device__ __forceinline__ void mx4_tile_finish(const Mx4Out& p, int64_t r0, int64_t c0,
                                                const uint4 (&v)[LPR / 2],
                                                typename Mx4Tile<LPR, W>::Shared& sh, int wid,
                                                int lane) {
  using T = Mx4Tile<LPR, W>;
  constexpr int RL = LPR / 2;
  uint32_t rk[RL], cm[4] = {};
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < RL; ++k) {
    const uint32_t a[4] = {v[k].x & 0x7FFF7FFFu, v[k].y & 0x7FFF7FFFu, v[k].z & 0x7FFF7FFFu,
                           v[k].w & 0x7FFF7FFFu};
#pragma unroll
    for (int i = 0; i < 4; ++i) cm[i] = pk_max_u16(cm[i], a[i]);
    uint32_t m = pk_max_u16(pk_max_u16(a[0], a[1]), pk_max_u16(a[2], a[3]));
    m = pk_max_u16(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0xB1, 0xF, 0xF, true));
    m = pk_max_u16(m, (uint32_t)__builtin_amdgcn_mov_dpp((int)m, 0x4E, 0xF, 0xF, true));
    rk[k] = max(m & 0xFFFFu, m >> 16);
    top = max(top, rk[k]);
  }
  if (p.out_t) {
#pragma unroll
    for (int off = LPR; off < 64; off <<= 1)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        cm[i] = pk_max_u16(cm[i], (uint32_t)__shfl_xor((int)cm[i], off, 64));
  }
  if (__builtin_expect(__any(top >= 0x7F80u), 0))
    mx4_tile_body<LPR, W, false>(p, r0, c0, v, rk, cm, sh, wid, lane);
  else
    mx4_tile_body<LPR, W, true>(p, r0, c0, v, rk, cm, sh, wid, lane);
  __syncthreads();
  const int tid = 64 * wid + lane;
  if (p.out) {
    // the rows' scale dwords: consecutive rows of a plane by consecutive lanes
    constexpr int G = T::kCols / 128;  // planes a tile spans (0: part of one)
    if constexpr (G > 0) {
      for (int i = tid; i < T::kRows * G; i += 64 * W) {
        const int row = i % T::kRows, g = i / T::kRows;
        if (r0 + row < p.rows && c0 + 128 * g < p.cols)
          p.planes[((c0 >> 7) + g) * p.rows + r0 + row] =
              *reinterpret_cast<const uint32_t*>(&sh.rowsc[row][4 * g]);
      }
    } else {
      constexpr int B = T::kCols / 32;
      const int64_t nblk = p.cols >> 5;
      for (int i = tid; i < T::kRows * B; i += 64 * W) {
        const int row = i / B, b = i % B;
        const int64_t blk = (c0 >> 5) + b;
        if (r0 + row < p.rows && blk < nblk) {
          uint8_t* d = reinterpret_cast<uint8_t*>(p.planes + (blk >> 2) * p.rows + r0 + row);
          d[blk & 3] = sh.rowsc[row][b];
          if (blk == nblk - 1)  // the row's last block fills up its dword
            for (int64_t x = (blk & 3) + 1; x < 4; ++x) d[x] = (uint8_t)kMxPadScale;
        }
      }
    }
  }
  if (p.out_t) {
    const int64_t rowsp = (p.rows + 31) & ~31LL;
    constexpr int CH = W;  // 16-byte chunks of a staged column
    for (int i = tid; i < T::kCols * CH; i += 64 * W) {
      const int col = i / CH, ch = i % CH;
      if (c0 + col < p.cols && r0 + 32 * ch < p.rows) {
        const uint32_t* s = reinterpret_cast<const uint32_t*>(&sh.stage[col][16 * ch]);
        *reinterpret_cast<uint4*>(p.out_t + (c0 + col) * (rowsp >> 1) + (r0 >> 1) + 16 * ch) =
            make_uint4(s[0], s[1], s[2], s[3]);
      }
    }
    constexpr int G = W / 4;
    if constexpr (G > 0) {
      for (int i = tid; i < T::kCols * G; i += 64 * W) {
        const int col = i % T::kCols, g = i / T::kCols;
        if (c0 + col < p.cols && r0 + 128 * g < p.rows)
          p.planes_t[((r0 >> 7) + g) * p.cols + c0 + col] =
              *reinterpret_cast<const uint32_t*>(&sh.colsc[col][4 * g]);
      }
    } else {
      const int64_t nblk = rowsp >> 5;
      for (int i = tid; i < T::kCols * W; i += 64 * W) {
        const int col = i % T::kCols, b = i / T::kCols;
        const int64_t blk = (r0 >> 5) + b;
        if (c0 + col < p.cols && blk < nblk) {
          uint8_t* d = reinterpret_cast<uint8_t*>(p.planes_t + (blk >> 2) * p.cols + c0 + col);
          d[blk & 3] = sh.colsc[col][b];
          if (blk == nblk - 1)
            for (int64_t x = (blk & 3) + 1; x < 4; ++x) d[x] = (uint8_t)kMxPadScale;
        }
      }
    }
  }
  __syncthreads();
}

}  // namespace bf8

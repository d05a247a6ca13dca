// MXFP4 blocks: 32 values sharing one power of two (E8M0 byte e), each an e2m1 code
// (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign bit; two codes a byte, the even element in the low
// nibble). The device side of quantizing a tile whose bf16 values a wave holds in registers.
#pragma once

#include "common.hpp"

namespace bf8 {

// Biased exponent e of a block whose max |x| is the bf16 key k (the bits without the sign): 2^(e -
// 127) is the smallest power of two with max |x| <= 6 * 2^(e - 127), 2^-127 at least. 6 = 1.5 *
// 2^2, so it is E - 2, one more where the mantissa passes 1.5 (64 / 128 above 1): ((k + 63) >> 7) -
// 2.
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
// stands for 2^-127 too (and 255 for a NaN, whatever the value).
__device__ __forceinline__ float mx4_scale(uint32_t e) { return __uint_as_float(e << 23); }

// Byte B of c: the codes of a packed bf16 pair (low half in the low nibble). The conversion rounds to
// nearest even and takes an inf to 6; a block with a NaN (not FINITE alone) has no values, its codes are 0.
template <int B, bool FINITE>
__device__ __forceinline__ uint32_t mx4_pack2(uint32_t c, uint32_t pair, uint32_t e) {
  if (!FINITE && e == 0xFFu) pair = e = 0u;
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(c, __builtin_bit_cast(bf16x2_t, pair),
                                                   mx4_scale(e), B);
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

typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

// Per-half maxima of packed pairs over the lanes l, l ^ 16, l ^ 32, l ^ 48, in all of them.
__device__ __forceinline__ uint32_t mx4_groups_max(uint32_t m) {
  u32x2_t s = __builtin_amdgcn_permlane32_swap(m, m, false, false);
  m = pk_max_u16(s[0], s[1]);
  s = __builtin_amdgcn_permlane16_swap(m, m, false, false);
  return pk_max_u16(s[0], s[1]);
}

// Transposes 4 x 4 dwords across the lane groups l / 16: register j of group g becomes what
// register g of group j was.
__device__ __forceinline__ void mx4_groups_transpose(uint32_t (&r)[4]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const u32x2_t s = __builtin_amdgcn_permlane32_swap(r[i], r[i + 2], false, false);
    r[i] = s[0];
    r[i + 2] = s[1];
  }
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    const u32x2_t s = __builtin_amdgcn_permlane16_swap(r[i], r[i + 1], false, false);
    r[i] = s[0];
    r[i + 1] = s[1];
  }
}

// A wave's tile of 32 rows x 128 columns at (r0, c0): lane l holds columns 8 (l % 16) .. +7 of the
// rows 8 (l / 16) .. +7 (v[k]: row k; zeros past the tensor). A row block of 32 is four
// neighbouring lanes, a column block of 32 rows the four lanes of a column group, and a lane's column
// codes are 4 consecutive bytes of the columnwise copy: a transpose of dwords across the lane groups
// leaves every lane the 16 bytes of two whole column blocks. W waves of a block take tiles one below
// the other (r0 is wave w's own). W = 1: those bytes go out as they are, no wave waits for another. W > 1:
// they meet in LDS, and a column's leave as 16 W bytes side by side.
constexpr int kMx4Rows = 32, kMx4Cols = 128;
template <int W>
struct Mx4Stage {
  static constexpr int kPitch = W + 1;  // 16-byte chunks of a staged column
  alignas(16) uint4 codes[W > 1 ? kMx4Cols * kPitch : 1];
  alignas(4) uint8_t scales[W > 1 ? kMx4Cols : 1][W < 4 ? 4 : W];
};

template <int W, bool FINITE>
__device__ __forceinline__ void mx4_wave_body(const Mx4Out& p, int64_t r0, int64_t c0,
                                              const uint4 (&v)[8], const uint32_t (&rk)[8],
                                              const uint32_t (&cm)[4], Mx4Stage<W>* sh, int wid,
                                              int lane) {
  const int cl = lane & 15, g = lane >> 4;
  const int64_t c = c0 + 8 * cl, r = r0 + 8 * g;
  if (p.out && r0 < p.rows) {
    // the tile's rows, cols / 2 bytes each
    const uint32_t ld = (uint32_t)(p.cols >> 1), left = (uint32_t)min(p.rows - r0, (int64_t)kMx4Rows);
    const Window w = window(p.out + r0 * (p.cols >> 1), left * ld);
    const uint32_t o = c < p.cols ? 8 * g * ld + (uint32_t)(c >> 1) : kPastEnd;
    uint32_t mine = 0;  // the scale dword of row r + cl, in the lanes cl < 8
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      uint32_t e = FINITE ? mx4_exponent_finite(rk[k]) : mx4_exponent(rk[k]);
      uint32_t q = 0;
      q = mx4_pack2<0, FINITE>(q, v[k].x, e);
      q = mx4_pack2<1, FINITE>(q, v[k].y, e);
      q = mx4_pack2<2, FINITE>(q, v[k].z, e);
      q = mx4_pack2<3, FINITE>(q, v[k].w, e);
      __builtin_amdgcn_raw_buffer_store_b32(q, w, (int)(o + k * ld), 0, 0);
      if (c >= p.cols) e = kMxPadScale;  // blocks past the row pad its last dword of scales
      // the row's four blocks, four lanes apart: rotations by 4 and by 8 within 16 lanes
      e <<= 8 * (cl >> 2);
      e |= (uint32_t)__builtin_amdgcn_mov_dpp((int)e, 0x124, 0xF, 0xF, true);
      e |= (uint32_t)__builtin_amdgcn_mov_dpp((int)e, 0x128, 0xF, 0xF, true);
      if (cl == k) mine = e;
    }
    if (cl < 8 && r + cl < p.rows) p.planes[(c0 >> 7) * p.rows + r + cl] = mine;
  }
  if (!p.out_t) return;
  uint32_t e[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    e[2 * i] = FINITE ? mx4_exponent_finite(cm[i] & 0xFFFFu) : mx4_exponent(cm[i] & 0xFFFFu);
    e[2 * i + 1] = FINITE ? mx4_exponent_finite(cm[i] >> 16) : mx4_exponent(cm[i] >> 16);
  }
  const int64_t ldt = ((p.rows + 31) >> 5) * 16;
  const int64_t blk = r0 >> 5, nblk = (p.rows + 31) >> 5;
#pragma unroll
  for (int h = 0; h < 2; ++h) {  // columns 4 h .. 4 h + 3 of the lane's eight
    uint32_t q[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t w[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        w[k] = h == 0 ? (i == 0 ? v[k].x : v[k].y) : (i == 0 ? v[k].z : v[k].w);
      const uint32_t ea = e[4 * h + 2 * i], eb = e[4 * h + 2 * i + 1];
      uint32_t x = 0, y = 0;
      x = mx4_pack2<0, FINITE>(x, __byte_perm(w[0], w[1], 0x5410), ea);
      y = mx4_pack2<0, FINITE>(y, __byte_perm(w[0], w[1], 0x7632), eb);
      x = mx4_pack2<1, FINITE>(x, __byte_perm(w[2], w[3], 0x5410), ea);
      y = mx4_pack2<1, FINITE>(y, __byte_perm(w[2], w[3], 0x7632), eb);
      x = mx4_pack2<2, FINITE>(x, __byte_perm(w[4], w[5], 0x5410), ea);
      y = mx4_pack2<2, FINITE>(y, __byte_perm(w[4], w[5], 0x7632), eb);
      x = mx4_pack2<3, FINITE>(x, __byte_perm(w[6], w[7], 0x5410), ea);
      y = mx4_pack2<3, FINITE>(y, __byte_perm(w[6], w[7], 0x7632), eb);
      q[2 * i] = x;
      q[2 * i + 1] = y;
    }
    mx4_groups_transpose(q);
    const int64_t col = c + 4 * h + g;  // the lane's own after the transpose
    uint32_t es = (e[4 * h] | (e[4 * h + 1] << 8) | (e[4 * h + 2] << 16) | (e[4 * h + 3] << 24)) >> (8 * g);
    if constexpr (W > 1) {
      const int lc = 8 * cl + 4 * h + g;
      sh->codes[lc * Mx4Stage<W>::kPitch + wid] = make_uint4(q[0], q[1], q[2], q[3]);
      sh->scales[lc][wid] = r0 < p.rows ? (uint8_t)es : (uint8_t)kMxPadScale;
    } else if (c < p.cols) {
      *reinterpret_cast<uint4*>(p.out_t + col * ldt + 16 * blk) = make_uint4(q[0], q[1], q[2], q[3]);
      uint8_t* d = reinterpret_cast<uint8_t*>(p.planes_t + (blk >> 2) * p.cols + col);
      d[blk & 3] = (uint8_t)es;
      if (blk == nblk - 1)  // a column's last block fills up its dword
        for (int b = (int)(blk & 3) + 1; b < 4; ++b) d[b] = (uint8_t)kMxPadScale;
    }
  }
}

// The loaded tile. W > 1: every wave of the W calls it alike (wid: which), also one past the
// tensor, with a stage of their own; before the stage's next use the caller waits for them.
template <int W>
__device__ __forceinline__ void mx4_wave_tile(const Mx4Out& p, int64_t r0, int64_t c0,
                                              const uint4 (&v)[8], Mx4Stage<W>* sh, int wid,
                                              int lane) {
  uint32_t rk[8], cm[4] = {};
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
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
    for (int i = 0; i < 4; ++i) cm[i] = mx4_groups_max(cm[i]);
  }
  if (__builtin_expect(__any(top >= 0x7F80u), 0))
    mx4_wave_body<W, false>(p, r0, c0, v, rk, cm, sh, wid, lane);
  else
    mx4_wave_body<W, true>(p, r0, c0, v, rk, cm, sh, wid, lane);
  if constexpr (W > 1) {
    if (!p.out_t) return;
    __syncthreads();
    const int64_t rb = r0 - kMx4Rows * wid;  // the first wave's
    const int64_t ldt = ((p.rows + 31) >> 5) * 16;
    const int tid = 64 * wid + lane;
    // chunk t % W of columns t / W, ..
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int col = tid / W + 64 * i, ch = tid % W;
      if (c0 + col < p.cols && rb + kMx4Rows * ch < p.rows)
        *reinterpret_cast<uint4*>(p.out_t + (c0 + col) * ldt + (rb >> 1) + 16 * ch) =
            sh->codes[col * Mx4Stage<W>::kPitch + ch];
    }
    static_assert(W % 4 == 0, "whole dwords of scales");
    if (tid < kMx4Cols * (W / 4)) {
      const int col = tid % kMx4Cols, gr = tid / kMx4Cols;
      if (c0 + col < p.cols && rb + 128 * gr < p.rows)
        p.planes_t[((rb >> 7) + gr) * p.cols + c0 + col] =
            *reinterpret_cast<const uint32_t*>(&sh->scales[col][4 * gr]);
    }
  }
}

}  // namespace bf8

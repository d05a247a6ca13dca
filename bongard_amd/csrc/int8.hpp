// Arithmetic of the 8-bit integer formats: codes under one scale a row (the products' operands) and
// blocks of 32 codes under a power of two (OCP MXINT8, the activation checkpoints).
#pragma once

#include "common.hpp"

namespace bf8 {

// 1.5 * 2^23: adding it rounds a number below 2^22 in magnitude to an integer (ties to even) whose two's
// complement is the sum's low bits.
constexpr float kRoundMagic = 12582912.0f;

// The low bytes of four dwords.
__device__ __forceinline__ uint32_t low_bytes(float a, float b, float c, float d) {
  const uint32_t ab = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040);
  const uint32_t cd = __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040);
  return __byte_perm(ab, cd, 0x5410);
}

// ---- one scale a row -----------------------------------------------------------------
// A row of largest magnitude a (at least kInt8Floor) has the scale a / 127, and its codes are
// 127 x / a rounded to nearest, ties to even. `mult` is 127 / a rounded up, and fma(x, mult,
// kRoundMagic) rounds to exactly that code: x and a hold 8 bits (or a is a power of two), so
// 127 x / a is a tie, where 254 x = (2 k + 1) a, or at least 2^-17 of itself away from one, more than the
// 2^-23 of itself by which rounding mult moves the product. Ties: where a is 254 times a power of two mult
// is exact. Else 127 divides 2 k + 1, so x = +-a / 2, which mult takes from 63.5 to 64, the even code, or
// past it. A row that holds inf or NaN: scale NaN, mult 0 and codes 0 (the low byte of a bf16 NaN as fp32).
constexpr float kInt8Floor = 9.094947017729282e-13f;  // 2^-40

struct Int8Scale {
  float scale, mult;
};

// key: the fp32 bits of the row's largest magnitude.
__device__ __forceinline__ Int8Scale int8_scale(uint32_t key) {
  if (key >= 0x7F800000u) return {__uint_as_float(0x7FC00000u), 0.0f};
  const float a = fmaxf(__uint_as_float(key), kInt8Floor);
  float m = __fdiv_rn(127.0f, a);
  if (__builtin_fmaf(m, a, -127.0f) < 0.0f) m = __uint_as_float(__float_as_uint(m) + 1u);
  return {__fdiv_rn(a, 127.0f), m};
}

// Codes of 8 bf16 values under one multiplier, or under eight.
__device__ __forceinline__ uint2 int8_codes8(uint4 v, float m) {
  auto f = [&](float x) { return __builtin_fmaf(x, m, kRoundMagic); };
  return make_uint2(low_bytes(f(bf16_lo(v.x)), f(bf16_hi(v.x)), f(bf16_lo(v.y)), f(bf16_hi(v.y))),
                    low_bytes(f(bf16_lo(v.z)), f(bf16_hi(v.z)), f(bf16_lo(v.w)), f(bf16_hi(v.w))));
}
__device__ __forceinline__ uint2 int8_codes8(uint4 v, const float (&m)[8]) {
  auto f = [](float x, float mm) { return __builtin_fmaf(x, mm, kRoundMagic); };
  return make_uint2(low_bytes(f(bf16_lo(v.x), m[0]), f(bf16_hi(v.x), m[1]), f(bf16_lo(v.y), m[2]),
                              f(bf16_hi(v.y), m[3])),
                    low_bytes(f(bf16_lo(v.z), m[4]), f(bf16_hi(v.z), m[5]), f(bf16_lo(v.w), m[6]),
                              f(bf16_hi(v.w), m[7])));
}

// Code e of a dword of four.
__device__ __forceinline__ float code_f32(uint32_t w, int e) {
  return (float)(int8_t)(w >> (8 * e));
}

// ---- the maxima that a tensor's scales are made from, as its producer or a pass over it leaves them --------
// (bf16 keys of magnitudes.) rowpart: [row_tiles][rows padded to 8], of 512 columns each, colpart: [strips of
// `strip` rows][cols].
struct Int8Maxima {
  int64_t rows, cols;
  int row_tiles, strip, strips;
  uint16_t *rowpart, *colpart;
};

__host__ __device__ inline int64_t int8_col_tiles(int64_t cols) { return (cols + 511) / 512; }
__host__ __device__ inline int64_t int8_row_pad(int64_t rows) { return (rows + 7) / 8 * 8; }
// The layout for [rows, cols], of `halves` parts side by side (2: d_g and d_u) each with row tiles of its own; ws
// may be NULL (for the sizes). Strips: few, as every tile of codes reads its columns' maxima of all of them,
// but blocks for every CU.
inline Int8Maxima int8_maxima(void* ws, int64_t rows, int64_t cols, int halves = 1) {
  const int64_t tiles = int8_col_tiles(cols / halves);
  int s = 256;
  while (s > 32 && (rows + s - 1) / s * tiles < 1024) s /= 2;
  Int8Maxima p{rows, cols, (int)(halves * tiles), s, (int)((rows + s - 1) / s), (uint16_t*)ws, nullptr};
  p.colpart = p.rowpart + ((size_t)p.row_tiles * int8_row_pad(rows) + 127) / 128 * 128;
  return p;
}
inline size_t int8_maxima_bytes(int64_t rows, int64_t cols, int halves = 1) {
  const Int8Maxima p = int8_maxima(nullptr, rows, cols, halves);
  return (size_t)((uint8_t*)p.colpart - (uint8_t*)p.rowpart) + (size_t)p.strips * cols * 2;
}
// The layout that the gated product's 256 x 128 tiles of H leave, by 128 x 128: row tiles of 128 columns.
inline Int8Maxima int8_tile_maxima(void* ws, int64_t rows, int64_t cols) {
  Int8Maxima p{rows, cols, (int)(cols / 128), 128, (int)((rows + 127) / 128), (uint16_t*)ws, nullptr};
  p.colpart = p.rowpart + ((size_t)p.row_tiles * int8_row_pad(rows) + 127) / 128 * 128;
  return p;
}
inline size_t int8_tile_maxima_bytes(int64_t rows, int64_t cols) {
  const Int8Maxima p = int8_tile_maxima(nullptr, rows, cols);
  return (size_t)((uint8_t*)p.colpart - (uint8_t*)p.rowpart) + (size_t)p.strips * cols * 2;
}
// The codes of x from its maxima (bf8_quantize_int8_maxima_bf16 without its checks).
int int8_codes_of_maxima(const uint16_t* x, const Int8Maxima& p, int8_t* out, float* row_scale, int8_t* out_t,
                         float* col_scale, hipStream_t s);

// The maxima of a wave's eight rows r .. r + 7 (zeros past the tensor's) by 512 columns (lane l: columns 8 l ..
// +7 of column tile tc), row by row: into colmax and, the rows', to rowpart. Two rows share a dword; three
// shuffles leave a pair to each lane of a quad, four more its maximum over the quads.
struct Int8Rows {
  uint32_t pair[4];
  __device__ __forceinline__ void add(int i, uint4 v, uint4& colmax) {
    const uint4 a = make_uint4(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu, v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu);
    colmax = make_uint4(pk_max_u16(colmax.x, a.x), pk_max_u16(colmax.y, a.y), pk_max_u16(colmax.z, a.z),
                        pk_max_u16(colmax.w, a.w));
    const uint32_t k = pk_max_u16(pk_max_u16(a.x, a.y), pk_max_u16(a.z, a.w));
    const uint32_t m = max(k & 0xFFFFu, k >> 16);
    if (i & 1)
      pair[i >> 1] |= m << 16;
    else
      pair[i >> 1] = m;
  }
  __device__ __forceinline__ void store(const Int8Maxima& p, int64_t r, int tc, int lane) {
    const bool odd = lane & 1, high = lane & 2;
    const uint32_t a = pk_max_u16(odd ? pair[1] : pair[0],
                                  (uint32_t)__shfl_xor((int)(odd ? pair[0] : pair[1]), 1, 64));
    const uint32_t b = pk_max_u16(odd ? pair[3] : pair[2],
                                  (uint32_t)__shfl_xor((int)(odd ? pair[2] : pair[3]), 1, 64));
    uint32_t m = pk_max_u16(high ? b : a, (uint32_t)__shfl_xor((int)(high ? a : b), 2, 64));
#pragma unroll
    for (int off = 4; off < 64; off <<= 1) m = pk_max_u16(m, (uint32_t)__shfl_xor((int)m, off, 64));
    // lane 0: rows 0 and 1, lane 1: 2 and 3, ...
    if (lane < 4)
      *reinterpret_cast<uint32_t*>(p.rowpart + tc * int8_row_pad(p.rows) + r + 2 * lane) = m;
  }
};

// The block's column maxima of strip ts (each wave's in k) to colpart.
template <int W>
__device__ __forceinline__ void int8_column_maxima(const Int8Maxima& p, uint4 (*red)[64], uint4 k,
                                                   int64_t ts, int64_t c, int wid, int lane) {
  red[wid][lane] = k;
  __syncthreads();
  if (wid != 0 || c >= p.cols) return;
#pragma unroll
  for (int w = 1; w < W; ++w) {
    const uint4 o = red[w][lane];
    k = make_uint4(pk_max_u16(k.x, o.x), pk_max_u16(k.y, o.y), pk_max_u16(k.z, o.z), pk_max_u16(k.w, o.w));
  }
  *reinterpret_cast<uint4*>(p.colpart + ts * p.cols + c) = k;
}

// ---- blocks of 32 under a power of two -------------------------------------------------
// A block of largest magnitude a has the byte E, the least with a <= 127 * 2^(E - 133), 7 at least (so
// that steps are normal numbers), and the codes x / 2^(E - 133) rounded to nearest, ties to even. A
// code has 7 bits, so bf16 holds code * 2^(E - 133) exactly. Of the bf16 bits of a: 64 steps at its power
// of two leave 127 for 1.984375 of it, so E is the exponent, one more where all seven mantissa bits
// are set; 254 for the largest finite values, whose 127.5 steps are taken as 127. inf or NaN in a
// block: E = 255, all of it reads back as NaN whatever its codes.
__device__ __forceinline__ uint32_t mxi8_exponent(uint32_t key16) {
  const uint32_t e = (key16 + 1) >> 7;
  return key16 >= 0x7F80u ? 255u : e < 7u ? 7u : e > 254u ? 254u : e;
}

__device__ __forceinline__ uint2 mxi8_codes8(uint4 v, uint32_t e) {
  const float m = e == 255u ? 0.0f : __uint_as_float((260u - e) << 23);  // 2^(133 - e)
  auto f = [&](float x) {
    return __builtin_amdgcn_fmed3f(__builtin_fmaf(x, m, kRoundMagic), kRoundMagic - 127.0f,
                                   kRoundMagic + 127.0f);
  };
  return make_uint2(low_bytes(f(bf16_lo(v.x)), f(bf16_hi(v.x)), f(bf16_lo(v.y)), f(bf16_hi(v.y))),
                    low_bytes(f(bf16_lo(v.z)), f(bf16_hi(v.z)), f(bf16_lo(v.w)), f(bf16_hi(v.w))));
}

// 2^(E - 133), exact down to the steps that no quantizer here writes.
__device__ __forceinline__ float mxi8_step(uint32_t e) {
  return e == 255u ? __uint_as_float(0x7FC00000u) : __builtin_amdgcn_ldexpf(1.0f, (int)e - 133);
}

// The 8 values of two code dwords as bf16 (exact).
__device__ __forceinline__ uint4 mxi8_values8(uint2 q, float step) {
  auto pair = [&](uint32_t w, int e) {
    return pack_bf16x2(code_f32(w, e) * step, code_f32(w, e + 1) * step);
  };
  return make_uint4(pair(q.x, 0), pair(q.x, 2), pair(q.y, 0), pair(q.y, 2));
}

// bf16 bits of the largest magnitude of a lane's 8 values, and of the 32 of a group of four lanes.
__device__ __forceinline__ uint32_t absmax16(uint4 v) {
  const uint32_t k = pk_max_u16(pk_max_u16(v.x & 0x7FFF7FFFu, v.y & 0x7FFF7FFFu),
                                pk_max_u16(v.z & 0x7FFF7FFFu, v.w & 0x7FFF7FFFu));
  return max(k & 0xFFFFu, k >> 16);
}
__device__ __forceinline__ uint32_t quad_max(uint32_t k) {
  k = max(k, (uint32_t)__builtin_amdgcn_mov_dpp((int)k, 0xB1, 0xF, 0xF, true));
  return max(k, (uint32_t)__builtin_amdgcn_mov_dpp((int)k, 0x4E, 0xF, 0xF, true));
}

}  // namespace bf8

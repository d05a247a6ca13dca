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

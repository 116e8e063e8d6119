// The 4-bit form of a paged cache's vectors.
//
// A group is 32 consecutive dims of a vector. With m its value of largest magnitude (the negative one of two),
//   s = -m / 8 rounded to bf16,  c = x / s rounded to a whole number of [-8, 7], plus 8 (8 where s is 0);  x ~ s (c - 8).
// m itself is then the code 0, so that all 16 codes are in use: on normal values the error is 0.086 of the values' size, 0.097 with
// s = max|x| / 7. A group that holds an infinity or a NaN is NaN: s is.
//
// Codes lie two to a byte, the low four bits first, four dims ("quads") to 16 bits, in an order of the attention's reads
// (paged_attention_int4.cu): there a lane's part of a vector is one run of bytes. With blocks of 128 dims (one block of D = 32 or
// 64), NG groups to a block, and quad i of 8 in group g:
//   K: the 16-bit word (i / 2 * NG + g) * 2 + i % 2 of the block (a lane of four: 8 dims of every group),
//   V: the 16-bit word i * NG + g (a lane of eight: 4 dims of every group).
#pragma once

#include "common.cuh"

namespace omni {

// The 16-bit word that holds dims 4u .. 4u + 3.
template <int D, bool KEYS>
OMNI_DEV int quad_at(int u) {
  constexpr int NG = D / 32 < 4 ? D / 32 : 4;
  const int b = u >> 5, g = (u & 31) >> 3, i = u & 7;
  return b * 32 + (KEYS ? ((i >> 1) * NG + g) * 2 + (i & 1) : i * NG + g);
}

OMNI_DEV float bf16_value(uint32_t bits) { return __uint_as_float(bits << 16); }

// The codes of four values under the scale s: x / s, one fp32 division, rounded to the nearest whole number of [-8, 7], plus 8.
OMNI_DEV uint32_t int4_codes(const float* x, float s) {
  uint32_t r = 0u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float c = s == 0.f ? 0.f : fminf(fmaxf(rintf(__fdiv_rn(x[i], s)), -8.f), 7.f);
    r |= (uint32_t)((int)c + 8) << (4 * i);
  }
  return r;
}

// The same codes of bf16 values, with inv = 1 / s (0 for s = 0; |s| at least kInt4Fast, so that it is a number). Quotients of two numbers
// of 8 bits near n + 1/2 (n < 8) are n + 1/2 or at least 2^-10 away from it: the numerator 2 X 2^d - (2 n + 1) S of the difference is
// a multiple of 1/2 and the denominator 2 S at most 510. So the product, 2^-18 off at most (the reciprocal by 2 units in the last
// place, the product by half of one, of up to 8), is rounded to multiples of 2^-14 first (by adding 768), which gives the ties back exactly
// and moves nothing across one.
constexpr float kInt4Fast = 0x1p-100f;
OMNI_DEV uint32_t int4_codes_bf16(const float* x, float inv) {
  uint32_t r = 0u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float q = __fsub_rn(__fadd_rn(__fmul_rn(x[i], inv), 768.f), 768.f);
    const float c = __fadd_rn(fminf(fmaxf(q, -8.f), 7.f), 12582920.f);  // 1.5 x 2^23 + 8: the code in the lowest bits
    r |= (__float_as_uint(c) & 15u) << (4 * i);
  }
  return r;
}

// Four codes' values (exact in fp32: 4 bits times bf16's 8).
OMNI_DEV void int4_values(uint32_t codes, float s, float* f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = s * (float)((int)((codes >> (4 * i)) & 15u) - 8);
}

// Four codes' values in bf16 (two words): c - 8 and the scale (bf16, in both halves) are exact operands, so the product is the fp32
// product rounded.
OMNI_DEV uint2 int4_values_bf16(uint32_t codes, uint32_t scale2) {
  const uint32_t lo = ((codes | codes << 12) & 0x000f000fu) | 0x43004300u;       // 128 + c of dims 0 and 1
  const uint32_t hi = ((codes >> 8 | codes << 4) & 0x000f000fu) | 0x43004300u;  // of dims 2 and 3
  uint2 r;
  asm("{\n\t.reg .b32 a, b;\n\t"
      "sub.rn.bf16x2 a, %2, %4;\n\t"
      "sub.rn.bf16x2 b, %3, %4;\n\t"
      "mul.rn.bf16x2 %0, a, %5;\n\t"
      "mul.rn.bf16x2 %1, b, %5;\n\t}"
      : "=r"(r.x), "=r"(r.y)
      : "r"(lo), "r"(hi), "r"(0x43084308u), "r"(scale2));
  return r;
}

}  // namespace omni

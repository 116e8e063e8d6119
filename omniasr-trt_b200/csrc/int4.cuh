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

// The codes of four values under the scale s.
OMNI_DEV uint32_t int4_codes(const float* x, float s) {
  uint32_t r = 0u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float c = s == 0.f ? 0.f : fminf(fmaxf(rintf(__fdiv_rn(x[i], s)), -8.f), 7.f);
    r |= (uint32_t)((int)c + 8) << (4 * i);
  }
  return r;
}

// Four codes' values (exact in fp32: 4 bits times bf16's 8).
OMNI_DEV void int4_values(uint32_t codes, float s, float* f) {
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = s * (float)((int)((codes >> (4 * i)) & 15u) - 8);
}

}  // namespace omni

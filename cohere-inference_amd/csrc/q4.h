// Vectors of 128 bf16 values held in 4 bits: four groups of 32 values, each with its largest magnitude m (bf16, exact:
// the values are bf16) and a code c = rint(7 x / m) in -7..7 per value (half to even; 0 where m = 0). The value held is
// c m / 7. 64 bytes of codes (byte j: dimension 2j in the low nibble, 2j + 1 in the high one, two's complement) and four
// maxima, 72 bytes in all (int8 with a scale: 132, bf16: 256). A group with a NaN or an infinity holds the maximum NaN
// and codes 0, so that what attends to it is NaN too.
//
// Why groups of 32 with a maximum each: a normal vector keeps 20.3 dB of signal over the rounding, with one maximum over
// 128 values 18.6 (the maximum of 128 is a fifth larger than that of 32, and a step is m / 7), for 6 bytes of 72. Why the
// maximum and not the step m / 7: it needs no rounding, so a code can be exact. 7 x is exact in fp32 (8 + 3 bits); 7 x / m is either k + 1/2 exactly or further
// from it than 1e-4 of its value (the numerators are 11-bit, the denominators 8-bit), so a quotient that is exact where
// it is representable gives the code of the exact quotient.
#pragma once
#include "common.h"

namespace cohere_q4 {

constexpr int HD = 128, GRP = 32, NG = HD / GRP, VB = HD / 2;  // head size, group, groups and code bytes a vector

// a group's maximum (its bits as an unsigned number, whose order is the magnitudes': a NaN or an infinity exceeds every
// finite value) as what its codes are computed with: 7 / m as hi + lo, hi of 15 bits, so that x hi is exact (8 + 15 bits)
// and fma(x, lo, x hi) is 7 x / m rounded once (lo has 24 bits more: a quotient that fp32 holds comes out as it is). Very
// small and very large maxima are scaled by a power of two with the values, to keep lo in the normal range.
struct Group {
  float hi, lo, scale;
  bool any;  // finite and not zero
  uint16_t store;  // the maximum as held
};

DEVI Group group_of(uint32_t mb) {
  Group g;
  g.any = mb != 0 && mb < 0x7f800000u;
  const float m = __uint_as_float(g.any ? mb : 0x3f800000u);
  g.scale = m < 0x1p-64f ? 0x1p64f : m > 0x1p64f ? 0x1p-64f : 1.f;
  const float ms = m * g.scale, inv = 1.f / ms;
  g.hi = __uint_as_float(__float_as_uint(7.f * inv) & 0xfffffe00u);
  g.lo = __builtin_fmaf(-g.hi, ms, 7.f) * inv;  // the remainder is exact: 15 + 8 bits below 7
  g.store = mb < 0x7f800000u ? (uint16_t)(mb >> 16) : (uint16_t)0x7fc0;
  return g;
}

// eight values' codes, the first in the lowest nibble. Adding 1.5 2^23 rounds to an integer k, half to even, in the sum's
// low bits (0x4B400000 + k); the eight sums are added up 4 bits apart, and what their constants add (0x3F400000 modulo
// 2^32) comes off with the bias of 8 a digit that makes every digit's borrow vanish.
DEVI uint32_t pack8(const Group& g, const float (&x)[8]) {
  float f[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = x[i];
  if (g.scale != 1.f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] *= g.scale;
  }
  uint32_t w = 0;
#pragma unroll
  for (int i = 7; i >= 0; --i) w = (w << 4) + __float_as_uint(__builtin_fmaf(f[i], g.lo, f[i] * g.hi) + 12582912.f);
  return g.any ? (w + (0x88888888u - 0x3F400000u)) ^ 0x88888888u : 0u;
}

// the code in nibble i (a constant) of a word
DEVI int code(uint32_t w, int i) { return (int)(w << (28 - 4 * i)) >> 28; }

// a group's step m / 7 as a sum of two fp32 numbers, and c m / 7 from it with one rounding that matters (the second
// number is 0 where the step is exact; c m / 7 is otherwise never halfway between two bf16 values)
struct Step {
  float hi, lo;
};
DEVI Step step_of(float m) {
  const float hi = m / 7.f;
  return {hi, __builtin_fmaf(-hi, 7.f, m) / 7.f};
}
DEVI float held(int c, const Step& s) { return __builtin_fmaf((float)c, s.hi, (float)c * s.lo); }

DEVI uint32_t max_u(uint32_t a, uint32_t b) { return a > b ? a : b; }
template <int CTRL>
DEVI uint32_t dpp_u(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
}
// over each quad of lanes, in every lane of it
DEVI uint32_t quad_max_u(uint32_t v) {
  v = max_u(v, dpp_u<DPP_XOR1>(v));
  return max_u(v, dpp_u<DPP_XOR2>(v));
}

// eight bf16 values as fp32, and the maximum of their magnitudes' bits
DEVI uint32_t unpack8(const uint4& u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  uint32_t mx = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    f[2 * k] = __uint_as_float(w[k] << 16);
    f[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
    mx = max_u(mx, max_u((w[k] << 16) & 0x7fffffffu, w[k] & 0x7fff0000u));
  }
  return mx;
}

}  // namespace cohere_q4

// Rows of keys and values held in 4 bits: what the kernels that write and read them share.
//
// A row is one token's d channels of one KV head, in groups of 32 (d is a multiple of 32).  With m the
// group's value of the largest magnitude (the positive one of two), its scale is
//   s = round5(-m / 8),   five significant bits, ties to even,
// its codes are c = the nearest whole number to x / s (ties to even) within -8 .. 7, and the row stands for
// c * s.  The signed scale puts m itself on code -8, the end of the range that has a code more, so a step is
// an eighth of the magnitude and not a seventh.  Five bits of scale cost at most 1/33 of m at the far end
// (a half of a code's half step, m / 16) and make every c * s a bfloat16 exactly (|c| <= 7 has three bits, 8 is
// a power of two): a row can be expanded to bfloat16 without a second rounding.  Whether x lies nearer to one code or the next
// is decided exactly: a border is (c + 1/2) s, nine significant bits at most, and a quotient in 32 bits
// falls on a border's own quotient only if x does.
// A group that holds a value that is not finite has the scale NaN, so that it shows where it is seen.
//
// Packing (u = c + 8 in 0 .. 15), G = d / 32 groups:
//   keys    32-bit words of eight channels: channel 32 g + 8 t + 2 j + e at bit 4 j + 16 e of word t * G + g, so
//           that (w >> 4 j) & 0x000f000f holds two neighbouring channels, the pair that an operand of a matrix
//           instruction takes where its inner axis runs along a row (scores), and a thread t of four
//           finds its word of every group side by side;
//   values  16-bit units of four channels: channel 32 g + 4 r + j at bit 4 j of unit r * G + g: units of two rows (two keys)
//           put side by side hold the pairs along the keys that the product with the weights takes.
// Pages: codes [pages, KV heads, page size, d / 2] bytes, scales [pages, KV heads, page size, G] bfloat16: the
// rows of one head and page lie one behind the other.
#pragma once

#include "common.cuh"

namespace q4 {

constexpr int kGroup = 32;

// x to five significant bits, ties to even (24 bits become 5: 19 go).
__device__ __forceinline__ float round5(float x) {
  const uint32_t bits = __float_as_uint(x);
  return __uint_as_float((bits + 0x3FFFFu + ((bits >> 19) & 1u)) & 0xFFF80000u);
}

// The codes (0 .. 15) of eight values in a group of scale s; a scale of 0 or NaN stands for itself whatever the code.  A product with 1 / s
// is near the quotient, and what is left of x beside that code's step, exact in 32 bits (x and the step are within a factor of two), says
// whether the next code is nearer, or as near and even.  Scales whose reciprocal is not a number divide.
__device__ __forceinline__ void codes_of(const float (&x)[8], float s, uint32_t (&code)[8]) {
  const bool none = s == 0.0f || s != s, tiny = fabsf(s) < 0x1p-120f;
  const float inverse = tiny ? 0.0f : __frcp_rn(s), half = 0.5f * fabsf(s);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float c;
    if (tiny) {
      c = none ? 0.0f : rintf(__fdiv_rn(x[i], s));
    } else {
      c = rintf(x[i] * inverse);
      const float left = fmaf(-c, s, x[i]), away = copysignf(1.0f, left * s);
      const bool odd = static_cast<int>(c) & 1;
      if (fabsf(left) > half || (fabsf(left) == half && odd)) c += away;
    }
    c = fminf(fmaxf(c, -8.0f), 7.0f);
    code[i] = none ? 8u : static_cast<uint32_t>(static_cast<int>(c) + 8);
  }
}

}  // namespace q4

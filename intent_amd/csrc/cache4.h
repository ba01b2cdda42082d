// Keys and values in 4 bits. A token's head of D elements is D / 8 words of eight codes, element e of a word at
// bit 16 (e mod 2) + 4 (e div 2), and ceil(D / 32) groups of 32 elements (the last may be shorter), each with a
// scale s and a lowest value m in f16, s in the low half of a word:
//   value = m + s code.
// The order puts the codes of two elements in the two halves of a word under one mask, so that a pair of f16
// comes out of one bitwise operation and two packed ones, in order.
#pragma once

#include "common.h"

namespace intent {

constexpr int kGroup4 = 32;

INTENT_DEVICE int code_bit(int e) { return 16 * (e & 1) + 4 * ((e & 7) >> 1); }

// Eight values in f32.
INTENT_DEVICE void widen4(uint32_t word, uint32_t pair, float (&v)[8]) {
  const f16x2 h = bit_cast<f16x2>(pair);
  const float s = (float)h[0], m = (float)h[1];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = __builtin_fmaf((float)(word >> code_bit(e) & 15u), s, m);
}

}  // namespace intent

// Cache rows in 4 bits, as the kernels write and read them.
//
// A row of one KV head is four groups of 32 dims; a group is a step s and a minimum m (bf16 each) and 32 codes c in 0 .. 15,
// and stands for the values m + s c. A slot's row of K (or V) is 8 heads x 64 bytes of codes, then 8 heads x 4 (s, m) pairs:
// 640 bytes (bf16: 2048), in pages [2 (K, V)][16 slots][640], so that rows move and pages are addressed as in the bf16 cache.
// Of a head's 16 code words, word 4 (b % 4) + b / 4 holds dims 8 b .. + 7: a lane that feeds a matrix instruction reads its part
// of all four groups as one 16-byte piece. Dim d sits at nibble d % 8 / 2 + 4 (d % 2) of its word, so that one shift and mask
// yields the codes of two neighbouring dims in the halves of a register.
#pragma once
#include "common.h"

namespace abkv {

constexpr int kHeadCodes4 = kHeadDim / 2;                    // bytes of a head's codes
constexpr int kParams4 = kHeadsKV * kHeadCodes4;             // offset of a slot's pairs
constexpr int kSlot4 = kParams4 + kHeadsKV * 16;             // 640
constexpr int kHalf4 = kPage * kSlot4;                       // V half of a page
constexpr int kPage4 = 2 * kHalf4;

__device__ __forceinline__ int code_word(int b) { return 4 * (b & 3) + (b >> 2); }      // word of dims 8 b .. + 7

// Quantises 32 dims that the four lanes of a quad hold, eight each: this lane's word of codes and the group's pair. x are bf16
// values, so the minimum is kept exactly; the step is the fp32 quotient (max - min) / 15 rounded to bf16 (2^-8 of it, at most
// 0.06 of a step over the 15 codes), and a code the nearest one. A group that holds a value that is not finite, or whose span
// is none, gets the step NaN and reads as NaN.
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], uint32_t& pair) {
  float lo = x[0], hi = x[0], bad = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
    bad += x[i] * 0.f;                                       // NaN of an infinity or NaN
  }
  lo = fminf(lo, dpp<kDppXor1>(lo));
  hi = fmaxf(hi, dpp<kDppXor1>(hi));
  bad += dpp<kDppXor1>(bad);
  lo = fminf(lo, dpp<kDppXor2>(lo));
  hi = fmaxf(hi, dpp<kDppXor2>(hi));
  bad += dpp<kDppXor2>(bad);
  const float span = hi - lo + bad;
  const uint32_t s16 = __builtin_bit_cast(uint16_t, (__bf16)(span / 15.f));
  if (!(span < INFINITY)) {
    pair = 0x7fc0;
    return 0;
  }
  pair = s16 | (__float_as_uint(lo) & 0xffff0000u);
  const float s = __uint_as_float(s16 << 16);
  uint32_t word = 0;
  if (s > 0.f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float c = fminf(rintf((x[i] - lo) / s), 15.f);
      word |= (uint32_t)c << (2 * i + ((i & 1) ? 14 : 0));   // nibble i / 2 + 4 (i % 2)
    }
  }
  return word;
}

}  // namespace abkv

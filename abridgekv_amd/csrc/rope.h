// RoPE positions of the abridged layout, shared by the kernels that rotate rows.
#pragma once
#include "common.h"

namespace abkv {

struct RopeLayout {
  long max_pos;                                // rows of the angle table
  int block_c, codes_k, log2_k;                // block_c == 0: positions are RoPE positions already
  int code_span;                               // code rows spread over in-block offsets [0, code_span)
};

// Logical position of period block_c + codes_k -> block * block_c + (offset < block_c ? offset : bitrev code offset over the
// code span, block_c minus a static retained tail), config/compresslm.py:192-216.
__device__ __forceinline__ long rope_position(const RopeLayout& a, long pos) {
  if (pos < 0) pos = 0;
  if (a.block_c > 0) {
    const long per = a.block_c + a.codes_k;
    const long blk = pos / per;
    const int w = (int)(pos - blk * per);
    long off = w;
    if (w >= a.block_c) {
      const unsigned k = (unsigned)(w - a.block_c);
      const unsigned rev = a.log2_k > 0 ? (__brev(k) >> (32 - a.log2_k)) : 0u;
      off = ((long)rev * a.code_span) / a.codes_k;
    }
    pos = blk * a.block_c + off;
  }
  return pos < a.max_pos ? pos : a.max_pos - 1;
}

// Fills a layout from an entry's arguments; false where they are out of range.
inline bool rope_layout(RopeLayout& a, long max_pos, int block_c, int codes_k, int code_span) {
  if (max_pos <= 0 || block_c < 0) return false;
  int log2_k = 0;
  if (code_span == 0) code_span = block_c;
  if (block_c > 0) {
    if (codes_k <= 0 || (codes_k & (codes_k - 1)) || codes_k > block_c || code_span < codes_k || code_span > block_c)
      return false;
    while ((1 << log2_k) < codes_k) ++log2_k;
  }
  a.max_pos = max_pos;
  a.block_c = block_c;
  a.codes_k = codes_k;
  a.log2_k = log2_k;
  a.code_span = code_span;
  return true;
}

}  // namespace abkv

// Where the prompt scores' query rows lie (prompt_scores_kernel). Plain integer code without GPU types, so a host build can check
// it over the strides that the entry accepts.
#pragma once
#include <stdint.h>

#include "mask_walk.h"

namespace abkv {

constexpr int kScoreQ = 32;                                  // query rows of an iteration

// Head strides of q [T, 32, 128] that keep score_piece in 32 bits (with token strides below 2^24: row_strides_ok).
ABKV_HD bool score_head_stride_ok(long q_sh) { return (q_sh >> 28) == 0; }

// Bytes from the iteration's first query row of the KV head's first query head to piece `piece` (8 elements) of LDS row `row`
// (head row / 32, query row row % 32, no further than query row `limit`). Unsigned: at the largest strides it passes 2^31.
ABKV_HD uint32_t score_piece(int row, int limit, uint32_t q_st, uint32_t q_sh, int piece) {
  const uint32_t q = (uint32_t)imin(row & (kScoreQ - 1), limit), h = (uint32_t)(row / kScoreQ);
  return (q * q_st + h * q_sh + 8u * (uint32_t)piece) * 2u;
}

}  // namespace abkv

// Host build of the prompt scores' query row offsets (csrc/score_rows.h).
#include "score_rows.h"

using namespace abkv;

extern "C" {
unsigned piece(int row, int limit, long q_st, long q_sh, int p) {
  return score_piece(row, limit, (uint32_t)q_st, (uint32_t)q_sh, p);
}
int head_stride_ok(long q_sh) { return score_head_stride_ok(q_sh); }
}

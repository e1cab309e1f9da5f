// Masking of score tiles under a sliding window with sinks (window_walk.h) and the arguments the dense kernels share.
#pragma once
#include "attn_tile.h"
#include "window_walk.h"

namespace abkv {

struct WindowArgs {
  const __bf16* q;  long q_sb, q_ss, q_sh;   // [B, S, 32, 128]; chunks: [T, 32, 128] (q_sb unused)
  const __bf16* k;  long k_sb, k_ss, k_sh;   // [B, S, 8, 128]
  const __bf16* v;  long v_sb, v_ss, v_sh;
  int B, S;
  const int32_t* seq_lens;                   // [B] rows of each sequence (nullptr: S); the rest is padding
  int window, sinks;
  float scale_log2;
  __bf16* out;      long o_sb, o_ss, o_sh;
  float* lse;                                // natural log, [B, 32, S]; chunks: [T, 32]; or nullptr
  int num_q_tiles;
  int group;                                 // tiles of one XCD in a row (window_tile)
};

// Workgroup -> (64-row tile, KV head, sequence). Workgroups go to the 8 XCDs round-robin by linear id; XCD x takes the tile
// groups x, x + 8, ..., of `group` consecutive tiles of a sequence with all KV heads each: neighbouring tiles read mostly the
// same rows of the other side, which then stay in one XCD's L2, and all of the rows' bytes, not one head's, so that its
// requests spread over all L2 channels. One KV head per XCD, as the compression mask's kernels place them (there every tile
// reads all codes), against this: B=2, 8192 rows, window 1024: forward 322 -> 294 us.
struct WindowTile {
  int tile, kvh, b;
};
__device__ __forceinline__ WindowTile window_tile(int tiles, int batch, int group) {
  const int total = tiles * batch, x = blockIdx.x % 8, i = blockIdx.x / 8;
  const int whole = total / (8 * group) * (8 * group);       // in whole rounds of groups; the rest evenly
  int t, kvh;
  if (i < whole) {
    const int in = i % (8 * group);
    kvh = in % kHeadsKV;
    t = (i / (8 * group) * 8 + x) * group + in / kHeadsKV;
  } else {
    const int rest = x * (total - whole) + (i - whole);
    kvh = rest % kHeadsKV;
    t = whole + rest / kHeadsKV;
  }
  return {t % tiles, kvh, t / tiles};
}

__device__ __forceinline__ int window_rows(const WindowArgs& a, int b) {
  return a.seq_lens ? min(max(a.seq_lens[b], 0), a.S) : a.S;
}

// Keys that a lane's query row sees: [lo, lo + len) and [0, sinks).
struct WindowLane {
  int lo;
  unsigned len;
  int sinks;
  // row: the query row's position; seen: false for rows that see nothing (past the sequence)
  __device__ __forceinline__ WindowLane(int row, bool seen, int window, int sinks_)
      : lo(max(row + 1 - window, 0)), len(seen ? row + 1 - lo : 0), sinks(seen ? min(sinks_, row + 1) : 0) {}
};

template <int H, class Walk>
__device__ __forceinline__ void tile_mask(floatx4 (&s)[2][2][H], int k0, const TileMask& tm, const WindowLane& lane,
                                          int j) {
  if (tm.mode == 0) return;                                 // (uniform)
  const int at = k0 + 4 * j, sinks = tm.mode == 2 ? lane.sinks : 0;
#pragma unroll
  for (int kk = 0; kk < 2; ++kk)
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int kv = at + 32 * kk + 16 * t + r;
        const bool ok = (unsigned)(kv - lane.lo) < lane.len || kv < sinks;
#pragma unroll
        for (int u = 0; u < H; ++u) s[kk][t][u][r] = ok ? s[kk][t][u][r] : -INFINITY;
      }
}

}  // namespace abkv

// Sliding-window attention with sinks as key ranges: row i sees key j when j <= i and (i - j < window or j < sinks). Which
// 64-key tiles a 64-row query tile reads and which query tiles read a key tile. Plain integer code without GPU types, so a
// host build can check it against the definition.
#pragma once
#include <stddef.h>

#include "mask_walk.h"

namespace abkv {

// Tiles that the rows q0 .. q_last (at most 64, q_last < n) read: the sinks' tiles, then those of the window, in key order
// and each once. The state is wave-uniform. Mode 0: every row sees every key, 1: each row its range, 2: its range and the
// sinks below it.
struct WindowWalk {
  int q0, q_last, window, sinks;
  int k, sink_end, win_begin;        // next tile's first key; keys [0, sink_end) and [win_begin, q_last] in whole tiles
  ABKV_HD WindowWalk(int q0_, int q_last_, int window_, int sinks_)
      : q0(q0_), q_last(q_last_), window(window_), sinks(sinks_), k(0) {
    win_begin = imax(q0 + 1 - window, 0) & ~(kBN - 1);
    sink_end = imin((imin(sinks, q_last + 1) + kBN - 1) & ~(kBN - 1), win_begin);
    if (sink_end == 0) k = win_begin;
  }
  ABKV_HD bool next(int& k0, TileMask& tm, bool) {
    if (k > q_last) return false;
    k0 = k;
    const int last = k0 + kBN - 1;
    tm.mode = last <= q0 && (k0 > q_last - window || last < sinks) ? 0 : k0 < sinks ? 2 : 1;
    k += kBN;
    if (k >= sink_end && k < win_begin) k = win_begin;
    return true;
  }
};

// The query tiles [first, near_end) whose windows can reach a key of the tile at k0, and [near_end, far_end) that see only
// its sinks (empty without sinks in the tile). n: rows of the sequence; all empty at k0 >= n.
struct WindowSpan {
  int first, near_end, far_end;
  ABKV_HD WindowSpan(int k0, int n, int window, int sinks) {
    const int tiles = (imax(n, 0) + kBM - 1) / kBM;
    first = imin(k0 / kBM, tiles);
    // the last key's last row: k0 + 63 + window - 1, below 2^31 for every window by the clamp to n
    const int reach = imin(window, imax(n, 1)) + k0 + kBN - 2;
    near_end = imax(first, imin(reach / kBM + 1, tiles));
    far_end = k0 < sinks ? imax(near_end, tiles) : near_end;
  }
};

// Work of the window's dK/dV launch: one item per key tile for its near query tiles, and for each tile that holds sinks
// `parts` more for the far ones, `part` query tiles each. The items of a sink tile leave fp32 sums in slots. More sink tiles
// than there are slots are enough items without parts: each then walks its near and far query tiles (sink_tiles 0).
// Query tiles (x 4 heads) a far part is worth starting for: with 8, us a forward and backward of three of up to 777 rows, window
// 129, 17 sinks 120 (with 4: 99), of 2048 rows, window 64 117 (96), of 1000 rows, 100 sinks 107 (86).
constexpr int kSinkPartMin = 4;
constexpr int kSinkSlots = 384;      // far parts of a launch, and sink tiles that have some, at most (64 KiB of sums each, per
                                     // KV head: slots for both, 384 MiB)
struct SinkPlan {
  int tiles, sink_tiles, part, parts;          // key tiles; those that hold sinks; query tiles per far part; parts a tile
  SinkPlan() = default;
  ABKV_HD SinkPlan(int seq_len, int batch, int window, int sinks) {
    tiles = (seq_len + kBN - 1) / kBN;
    const int near = imin((imin(window, seq_len) + kBN - 2) / kBM + 1, tiles);   // near tiles of a key tile, at most
    const int far = tiles - near;                                                // and the far ones (of the first tile)
    sink_tiles = far > 0 ? imin((imin(sinks, seq_len) + kBN - 1) / kBN, tiles) : 0;
    part = imax(kSinkPartMin, near);
    parts = 0;
    if ((long)sink_tiles * batch > kSinkSlots) sink_tiles = 0;
    if (sink_tiles == 0) return;
    const int most = imax(1, kSinkSlots / imax(1, sink_tiles * batch));          // parts of a tile, at most
    part = imax(part, (far + most - 1) / most);
    parts = (far + part - 1) / part;
  }
  ABKV_HD int items() const { return tiles + sink_tiles * parts; }               // per (KV head, sequence)
  ABKV_HD int slots() const { return sink_tiles * (parts + 1); }
  // Query tiles [first, end) of item z of a key tile (0: the near ones, and the far ones where the launch has no parts).
  ABKV_HD void range(const WindowSpan& span, int z, int& first, int& end) const {
    first = span.first;
    end = sink_tiles > 0 ? span.near_end : span.far_end;
    if (z > 0) {
      first = imin(span.near_end + (z - 1) * part, span.far_end);
      end = imin(first + part, span.far_end);
    }
  }
};

}  // namespace abkv

// Host build of the sliding window's key ranges and work plan (csrc/window_walk.h).
#include <stdint.h>

#include "window_walk.h"

using namespace abkv;

extern "C" {

// counts [n][n]: how often each (query, key) pair is visited as visible by the walk of the query tiles of rows q_base ..
// n - 1 (the first tile starts at q_base). Returns the tiles walked, or -1 for a tile out of range or out of order.
long window_counts(int n, int q_base, int window, int sinks, uint8_t* counts) {
  long tiles = 0;
  for (int q0 = q_base; q0 < n; q0 += kBM) {
    const int q_last = imin(q0 + kBM, n) - 1;
    WindowWalk walk(q0, q_last, window, sinks);
    int k0 = 0, before = -1;
    TileMask tm;
    for (bool first = true; walk.next(k0, tm, first); first = false) {
      if (k0 <= before || k0 % kBN || k0 >= n || k0 < 0) return -1;
      before = k0;
      ++tiles;
      for (int q = q0; q <= q_last; ++q) {
        const int lo = imax(q + 1 - window, 0), s = tm.mode == 2 ? imin(sinks, q + 1) : 0;
        const unsigned len = q + 1 - lo;
        for (int key = k0; key < imin(k0 + kBN, n); ++key)
          if (tm.mode == 0 || (unsigned)(key - lo) < len || key < s) counts[(long)q * n + key] += 1;
      }
    }
  }
  return tiles;
}

// counts [n][n]: how often each pair falls to a work item of the dK/dV launch for a sequence of n rows of seq_len, as its
// workgroups split them; -1 when a far part is out of its range.
long dkv_counts(int seq_len, int n, int batch, int window, int sinks, uint8_t* counts) {
  const SinkPlan p(seq_len, batch, window, sinks);
  if (p.slots() < p.sink_tiles || (p.parts > 1 && p.sink_tiles * batch <= kSinkSlots &&
                                   (long)p.sink_tiles * p.parts * batch > 2L * kSinkSlots))
    return -1;
  const int far_items = p.sink_tiles * p.parts;
  for (int item = 0; item < p.items(); ++item) {
    const int kt = item < far_items ? item / p.parts : item - far_items;
    const int z = item < far_items ? 1 + item % p.parts : 0;
    const int k0 = kt * kBN;
    const WindowSpan span(k0, n, window, sinks);
    int qt = span.first, end = span.near_end;
    if (z > 0) {
      qt = imin(span.near_end + (z - 1) * p.part, span.far_end);
      end = imin(qt + p.part, span.far_end);
    }
    if (end * kBM - kBM >= n && end > qt) return -1;
    for (; qt < end; ++qt)
      for (int q = qt * kBM; q < imin(qt * kBM + kBM, n); ++q)
        for (int key = k0; key < imin(k0 + kBN, n); ++key) {
          const unsigned rows = key < sinks ? n - key : imin(window, n - key);
          if ((unsigned)(q - key) < rows) counts[(long)q * n + key] += 1;
        }
  }
  return p.items();
}
}

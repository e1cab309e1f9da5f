// Host build of the sliding window's dK/dV work plan (csrc/window_walk.h).
#include <stdint.h>

#include "window_walk.h"

using namespace abkv;

extern "C" {

// Items, sink tiles, parts a tile and slots of a launch, per sequence.
void plan(int seq_len, int batch, int window, int sinks, int* out) {
  const SinkPlan p(seq_len, batch, window, sinks);
  out[0] = p.items();
  out[1] = p.sink_tiles;
  out[2] = p.parts;
  out[3] = p.slots();
}

// counts [tiles][tiles]: how often (key tile, query tile) is visited for a sequence of n rows.
void tile_counts(int seq_len, int n, int batch, int window, int sinks, uint8_t* counts) {
  const SinkPlan p(seq_len, batch, window, sinks);
  const int far = p.sink_tiles * p.parts;
  for (int item = 0; item < p.items(); ++item) {
    const int kt = item < far ? item / p.parts : item - far, z = item < far ? 1 + item % p.parts : 0;
    int qt, end;
    p.range(WindowSpan(kt * kBN, n, window, sinks), z, qt, end);
    for (; qt < end; ++qt) counts[(long)kt * p.tiles + qt] += 1;
  }
}
}

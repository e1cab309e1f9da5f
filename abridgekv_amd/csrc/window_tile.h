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

// Up to 32 sinks before a query tile's windows take half a tile of their own, outside the walk (a whole one costs a tenth of
// a query tile under a window of 512): 32 K rows and 32 V rows in one LDS tile. Sinks that the windows reach, or more of them,
// stay with the walk.
constexpr int kShortSinks = 32;
__device__ __forceinline__ bool short_sinks(int q0, int window, int sinks) {
  return sinks > 0 && sinks <= kShortSinks && q0 + 1 - window >= kBN;
}

// DMA of the sinks' rows (keys 0 .. 31, fewer than n_keys >= 64): K in rows 0 .. 31 of buf, V in rows 32 .. 63, by 8 waves.
template <class Rows>
__device__ __forceinline__ void issue_sinks(const Rows& rows, int n_keys, __bf16* buf, int w, int lane) {
  const auto src = rows.template src<2>(0, w & 3, n_keys);   // waves 4 .. 7: the V rows of the same keys
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int row = 8 * (w & 3) + 4 * n + (lane >> 4);
    const int chunk = (lane & 15) ^ (row & 15);              // (row + 32 swizzles alike)
    const __bf16* p = w < 4 ? rows.template addr<false>(src, row, chunk, n_keys)
                            : rows.template addr<true>(src, row, chunk, n_keys);
    __builtin_amdgcn_global_load_lds((const void*)p, ABKV_LDS(buf + (4 * (2 * w + n)) * kHeadDim), 16, 0, 0);
  }
}

// Scores of the 32 rows from row `first` of an LDS tile (tile_scores' first half).
template <int H>
__device__ __forceinline__ void half_scores(const __bf16* buf, int first, const bf16x8 (&qop)[H][4], floatx4 (&s)[2][H], int m16,
                                            int j) {
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int u = 0; u < H; ++u) s[t][u] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const bf16x8 kop = __builtin_bit_cast(bf16x8, lds16(buf, first + 16 * t + m16, 4 * i + j));
#pragma unroll
      for (int u = 0; u < H; ++u) s[t][u] = mfma16x16x32(kop, qop[u][i], s[t][u]);
    }
}

template <int H>
__device__ __forceinline__ bf16x8 pack_half(const floatx4 (&x)[2][H], int u) {
  u32x4 w;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    w[2 * t] = pack_bf16x2(x[t][u][0], x[t][u][1]);
    w[2 * t + 1] = pack_bf16x2(x[t][u][2], x[t][u][3]);
  }
  return __builtin_bit_cast(bf16x8, w);
}

// The sinks' share of a wave's columns as the start of its online softmax: o, m_run and the columns' weight sums l.
template <int H>
__device__ __forceinline__ void attend_sinks(const __bf16* buf, int sinks, const bf16x8 (&qop)[H][4], floatx4 (&o)[8][H],
                                             float (&m_run)[H], float (&l)[H], float scale_log2, int lane) {
  typedef short s8 __attribute__((ext_vector_type(8)));
  const bf16x8 ones = __builtin_bit_cast(bf16x8, s8{0x3f80, 0x3f80, 0x3f80, 0x3f80, 0x3f80, 0x3f80, 0x3f80, 0x3f80});
  const int m16 = lane & 15, j = lane >> 4;
  floatx4 s[2][H];
  half_scores<H>(buf, 0, qop, s, m16, j);
  bf16x8 pop[H];
#pragma unroll
  for (int u = 0; u < H; ++u) {
    float mx = -INFINITY;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[t][u][r] = 16 * t + 4 * j + r < sinks ? s[t][u][r] * scale_log2 : -INFINITY;
        mx = fmaxf(mx, s[t][u][r]);
      }
    m_run[u] = max_xor32(max_xor16(mx));
    const float m = m_run[u] == -INFINITY ? 0.f : m_run[u];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) s[t][u][r] = fast_exp2(s[t][u][r] - m);
    pop[u] = pack_half<H>(s, u);
  }
#pragma unroll
  for (int t = 0; t < 8; ++t) {
    const bf16x8 vop = vt_operand(buf, kShortSinks, t, lane);
#pragma unroll
    for (int u = 0; u < H; ++u) o[t][u] = mfma16x16x32(vop, pop[u], o[t][u]);
  }
#pragma unroll
  for (int u = 0; u < H; ++u) l[u] = mfma16x16x32(ones, pop[u], floatx4{0.f, 0.f, 0.f, 0.f})[0];
}

}  // namespace abkv

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
  uint8_t* low;                              // dense [B, S, 32, 128] or nullptr: what out's rounding left off (low_bytes)
  int num_q_tiles;
};

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

// Rows of a paged sequence that a query tile sees: keys below `sinks` and from `lo`, the first key of the tile's first row, on.
// The others of the tiles that it walks (before the windows, behind the sinks) may hold anything, or lie on pages that are no
// longer the sequence's: as the rows past its end they are not read, for a weight of 0 does not cancel a NaN.
struct PagedWindowRows : PagedRows {
  int lo, sinks;
  template <bool kV>
  __device__ __forceinline__ const __bf16* addr(const Src& t, int row, int chunk, int n_keys) const {
    const int key = t.k0 + row;
    const bool in = key < n_keys && (key >= lo || key < sinks);
    const __bf16* base = in ? t.blk + (row & 15) * kSlotElems : t.last;
    return base + ((kV ? kHalfElems : 0) + 8 * chunk);
  }
};

// Up to 32 sinks before a query tile's windows take half a tile of their own, outside the walk: 32 K rows and 32 V rows in one
// LDS tile. Sinks that the windows reach, or more of them, stay with the walk. (us of two sequences of 4096 rows with 4 sinks in
// the walk's whole tile / in this, windows of 64 52.9 / 51.2, 128 65.3 / 63.4, 512 106.6 / 103, 1024 149.4 / 146.)
constexpr int kShortSinks = 32;
__device__ __forceinline__ bool short_sinks(int q0, int window, int sinks) {
  return sinks > 0 && sinks <= kShortSinks && q0 + 1 - window >= kBN;
}

// DMA of the sinks' rows (keys 0 .. 31, fewer than n_keys >= 64; `rows` decides what stands for those past the sinks): K in rows
// 0 .. 31 of buf, V in rows 32 .. 63, by 4 waves.
template <class Rows>
__device__ __forceinline__ void issue_sinks(const Rows& rows, int n_keys, __bf16* buf, int w, int lane) {
  const auto src = rows.template src<4>(0, w & 1, n_keys);   // waves 2 and 3: the V rows of the same keys
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const int row = 16 * (w & 1) + 4 * n + (lane >> 4);
    const int chunk = (lane & 15) ^ (row & 15);              // (row + 32 swizzles alike)
    const __bf16* p = w < 2 ? rows.template addr<false>(src, row, chunk, n_keys)
                            : rows.template addr<true>(src, row, chunk, n_keys);
    __builtin_amdgcn_global_load_lds((const void*)p, ABKV_LDS(buf + (4 * (4 * w + n)) * kHeadDim), 16, 0, 0);
  }
}

// Scores of the 32 rows from row `first` of an LDS tile (tile_scores' first half).
template <int H>
__device__ __forceinline__ void half_scores(const __bf16* buf, int first, const bf16x8 (&qop)[H][4], floatx4 (&s)[2][H],
                                            int m16, int j) {
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

// The sinks' share of a wave's columns as the start of its online softmax: o, m_run and the columns' weight sums l (exact: this
// lane's part of those before the weights are rounded).
template <int H, bool kExact>
__device__ __forceinline__ void attend_sinks(const __bf16* buf, int sinks, const bf16x8 (&qop)[H][4], floatx4 (&o)[8][H],
                                             float (&m_run)[H], float (&l)[H], float (&exact)[H], float scale_log2, int lane) {
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
      for (int r = 0; r < 4; ++r) {
        s[t][u][r] = fast_exp2(s[t][u][r] - m);
        if constexpr (kExact) exact[u] += s[t][u][r];
      }
    pop[u] = pack_half<H>(s, u);
  }
#pragma unroll
  for (int t = 0; t < 8; ++t) {
    const bf16x8 vop = vt_operand(buf, kShortSinks, t, lane);
#pragma unroll
    for (int u = 0; u < H; ++u) o[t][u] = mfma16x16x32(vop, pop[u], o[t][u]);
  }
#pragma unroll
  for (int u = 0; u < H; ++u) {
    // every entry is the sum; their mean, or the compiler holds all four over the walk, in scratch
    const floatx4 sum = mfma16x16x32(ones, pop[u], floatx4{0.f, 0.f, 0.f, 0.f});
    l[u] = 0.5f * (sum[0] + sum[1]);
  }
}

// The first DMAs of a walk of at least one tile: K and V of tile 0, K of tile 1 (the first again where there is none).
template <int kWaves, class Rows, class Walk>
__device__ __forceinline__ void start_pair(const Rows& rows, Walk walk, int n_keys, __bf16* const (&K)[2],
                                           __bf16* const (&V)[2], int w, int lane) {
  int t = 0;
  TileMask m;
  walk.next(t, m, true);
  const auto s0 = rows.template src<16 / kWaves>(t, w, n_keys);
  issue_half<kWaves, false>(rows, s0, n_keys, K[0], w, lane);
  issue_half<kWaves, true>(rows, s0, n_keys, V[0], w, lane);
  walk.next(t, m, false);                                    // (t stays past the end)
  issue_half<kWaves, false>(rows, rows.template src<16 / kWaves>(t, w, n_keys), n_keys, K[1], w, lane);
}

// attend_tiles with two buffers each of K and V, tile m in K[m % 2] and V[m % 2], started by start_pair. Iteration n: wait for
// the DMAs of iteration n - 1 (K(n+1), V(n)), barrier, DMA K(n+2) and V(n+1) into the buffers that were read last, softmax of
// tile n beside the scores of tile n + 1, O += V(n) . P(n). The wait is the other workgroup's time: two share a CU.
// exact (kExact): this lane's part of the unrounded weight sums, rescaled from what it holds at the start.
template <int H, int kWaves, bool kExact, class Rows, class Walk, class Lane>
__device__ __forceinline__ void attend_pair(const Rows& rows, Walk& walk, int n_keys, __bf16* const (&K)[2],
                                            __bf16* const (&V)[2], const bf16x8 (&qop)[H][4], floatx4 (&o)[8][H],
                                            float (&m_run)[H], float (&l_run)[H], float (&exact)[H], const Lane& lane_mask,
                                            float scale_log2, int w, int lane) {
  constexpr int kPerWave = 16 / kWaves;
  const int m16 = lane & 15, j = lane >> 4;
  int t0 = 0, t1 = 0;                              // first keys of tiles n, n+1
  TileMask m0, m1;
  if (!walk.next(t0, m0, true)) return;
  t1 = t0;
  bool h1 = walk.next(t1, m1, false);
  static_assert(kWaves == 4, "the count that start_pair leaves behind K(0)");
  __asm__ volatile("s_waitcnt vmcnt(8)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  floatx4 sa[2][2][H], sb[2][2][H], lsum[H];
#pragma unroll
  for (int u = 0; u < H; ++u) lsum[u] = floatx4{0.f, 0.f, 0.f, 0.f};
  tile_scores<H>(K[0], qop, sa, m16, j);
  auto step = [&](floatx4 (&s_cur)[2][2][H], floatx4 (&s_nxt)[2][2][H], auto slot_c) -> bool {
    constexpr int slot = decltype(slot_c)::value;
    int t2 = t1;
    TileMask m2;
    const bool h2 = h1 && walk.next(t2, m2, false);
    const auto src_k = rows.template src<kPerWave>(h2 ? t2 : t0, w, n_keys);
    const auto src_v = rows.template src<kPerWave>(h1 ? t1 : t0, w, n_keys);
    __asm__ volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    issue_half<kWaves, false>(rows, src_k, n_keys, K[slot], w, lane);
    issue_half<kWaves, true>(rows, src_v, n_keys, V[1 - slot], w, lane);
    tile_mask<H, Walk>(s_cur, t0, m0, lane_mask, j);
    bf16x8 pop[2][H];
    tile_softmax<H, kExact>(s_cur, o, m_run, lsum, scale_log2, pop, exact);
    tile_scores<H>(K[1 - slot], qop, s_nxt, m16, j);         // (discarded after the last tile)
    tile_pv<H>(V[slot], pop, o, lsum, lane);
    if (!h1) return false;
    t0 = t1; m0 = m1;
    t1 = t2; m1 = m2; h1 = h2;
    return true;
  };
  for (;;) {
    if (!step(sa, sb, Slot<0>{})) break;
    if (!step(sb, sa, Slot<1>{})) break;
  }
  __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");       // no DMA may outlive the workgroup's LDS
#pragma unroll
  for (int u = 0; u < H; ++u) l_run[u] = lsum[u][0];
}

// What the bf16 rounding of an output leaves off, 256 times it in e5m2 (a lane's dims 32j .. 32j + 31 of head u). The backward's
// D = sum_d dO O takes it: with O rounded, D is off by about 2^-9 of a sum of 128 products, and over few keys, where dP and D
// nearly cancel, that is more than the rounding of dS: relative errors of dQ and dK (their own rounding gives 1.7e-3) of 2 rows
// 3.9e-3, of 8 2.9e-3, of 777 under a window of 129 2.5e-3; with it 2.4e-3 each. e5m2 keeps all but an eighth of it down to
// bf16's smallest values (beyond 57344 it saturates). Two of 4096 rows, window 512: 460 -> 477 us a forward and
// backward.
template <int H>
__device__ __forceinline__ void store_low(uint8_t* dst, const floatx4 (&o)[8][H], int u, int j, float inv) {
  const bool odd = j & 1;
  auto low = [](float x, uint32_t pair, bool hi) {
    const float r = hi ? bf16_hi(pair) : bf16_lo(pair);
    return fminf(fmaxf((x - r) * 256.f, -57344.f), 57344.f);
  };
  uint32_t w[8];                                             // [2p], [2p + 1]: dims 32j + 8p .. + 3, .. + 7
#pragma unroll
  for (int t = 0; t < 8; ++t) {
    const floatx4 x = o[t][u] * inv;
    const uint32_t p0 = pack_bf16x2(x[0], x[1]), p1 = pack_bf16x2(x[2], x[3]);
    int b = __builtin_amdgcn_cvt_pk_bf8_f32(low(x[0], p0, false), low(x[1], p0, true), 0, false);
    w[t] = __builtin_amdgcn_cvt_pk_bf8_f32(low(x[2], p1, false), low(x[3], p1, true), b, true);
  }
  // 16-byte piece 2j + h of the row is in half h of lane group j; after the swap half h holds pieces of its 64-byte run
  u32x4 v[2];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const auto r = __builtin_amdgcn_permlane32_swap(odd ? w[e ^ 1] : w[e], odd ? w[(4 + e) ^ 1] : w[4 + e], false, false);
    v[0][e] = r[0];
    v[1][e] = r[1];
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) *reinterpret_cast<u32x4*>(dst + 64 * h + 16 * (2 * (j & 1) + (j >> 1))) = v[h];
}
// Four of them (a dword), unscaled.
__device__ __forceinline__ floatx4 load_low(uint32_t w) {
  const auto a = __builtin_amdgcn_cvt_pk_f32_bf8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_bf8((int)w, true);
  return floatx4{a[0], a[1], b[0], b[1]};
}

}  // namespace abkv

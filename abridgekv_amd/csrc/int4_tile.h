// Attention tiles over a paged cache in 4 bits (int4.h), for the multi-query kernel (gfx950).
//
// The waves unpack a 64-key tile of codes into K and V tiles of fp16 in LDS, laid out as attn_tile.h's, and attend to them with
// v_mfma_f32_16x16x32_f16. fp16 keeps a value m + s c to 2^-11 of itself where bf16 (the type that the cache is written from)
// would round it a second time, to 2^-8; the weights gain as much, down to 2^-25 of the largest (kHeadroom). Its range is made up
// for by powers of two, which are exact:
//   K: 2^eK for each page, multiplied back into the page's scores;
//   Q: 2^eQ for each query row and head, likewise;
//   V: 2^eV for all of a walk, the largest need of its tiles so far; the output's sums are rescaled when it grows.
// An exponent is a multiple of 8 (it hardly ever moves), and leaves the largest value between 2^5 and 2^15.
//
// Wave w unpacks page w % 4 of K (waves 0 .. 3) or V (4 .. 7): 20 bytes a slot and head in place of 256, so that a tile costs each
// lane two 16-byte loads and about 80 VALU operations, beside 200 for its part of the softmax.
//
// A SIMD has one wave of either kind, and a tile is two phases of each: the vector unit's (softmax, unpacking) and the matrix
// unit's (products). The V waves are a phase behind, so that one wave's vector work runs beside the other's products; in step,
// they took turns at both units: 1.4 us a tile at the vector unit and 0.9 at the matrix unit came to 2.5 us, and then to 2.1
// (three chunks of 300 to 441 queries behind up to 8000 rows and a code step: 180 -> 160 us then, 169 now; with the two kinds on
// different SIMDs, 193).
#pragma once
#include "attn_tile.h"
#include "int4.h"

namespace abkv {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ floatx4 mfma16x16x32(const f16x8 a, const f16x8 b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// One sequence in the cache.
struct Int4Rows {
  const char* kv;
  int kvh;
  const int32_t* table;    // the sequence's page-table row
  int width;               // entries in the row
  int num_pages;
};

// A lane's part of a page: words 4 (lane % 4) .. + 3 of slot lane / 4, and the slot's four pairs.
struct Int4Part {
  u32x4 codes, pairs;
};
__device__ __forceinline__ Int4Part load_part(const Int4Rows& rows, int page, bool v, int lane) {
  const __attribute__((address_space(4))) int32_t* table = (const __attribute__((address_space(4))) int32_t*)rows.table;
  const int id = min(max(table[min(page, rows.width - 1)], 0), rows.num_pages - 1);
  const char* slot = rows.kv + (long)id * kPage4 + (v ? kHalf4 : 0) + (lane >> 2) * kSlot4;
  Int4Part p;
  p.codes = *reinterpret_cast<const u32x4*>(slot + rows.kvh * kHeadCodes4 + 16 * (lane & 3));
  p.pairs = *reinterpret_cast<const u32x4*>(slot + kParams4 + 16 * rows.kvh);
  return p;
}

constexpr int kLowestExp = -104;                             // (2^104 is still a float)

// A row's weights are 2^(score - ref), with ref kHeadroom below the running maximum, which moves when a weight would pass 2^15: so
// the largest lies between 2^kHeadroom and 2^15, the one at the walk's maximum so far among them. A weight is rounded to 2^-11 of
// itself down to 2^-25 of the largest; below, where fp16 has no finer steps, by up to 2^-36 of the largest, and the sum, taken of
// the rounded ones, by at most that for each row. (With weights up to 2^8 alone, a row that took most of the weight cost the
// others theirs from 2^-14 of it on. Less headroom moves ref less often: three chunks of 300 to 441 queries behind up to 8000
// rows and a code step take 168.6 us with 7, 169.1 with 11, 175.6 with 13; with scores of four times the spread 176, 185 and 191.)
constexpr int kHeadroom = 11;

// The exponent that values up to `bound` take.
__device__ __forceinline__ int range_exp(float bound) {
  const int e = (int)(__float_as_uint(bound) >> 23) - 127 - 14;           // (bound >= 0; infinity: 114, so 120)
  return max((e + 7) & ~7, kLowestExp);
}
__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
// A float's bits times 2^e for e << 23, from 2^-100 (so that -inf stays that, and no score that counts is as small) to 2^127. For
// the softmax scale times 2^(eQ + eK) it is called once, with both exponents (up to 240 << 23, an int): a part of the product may
// lie outside that range where the whole does not.
__device__ __forceinline__ float scaled_bits(int bits, int e23) {
  return __int_as_float(min(max(__builtin_elementwise_add_sat(bits, e23), 27 << 23), 254 << 23));
}

// The larger number; a NaN counts for nothing. (The instruction itself: fmaxf takes another one to quiet each operand.)
__device__ __forceinline__ float max_num(float a, float b) {
  float r;
  __asm__("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
// What no |value| of a page exceeds, in every lane: |m| + 15 |s|, at most three times the largest.
__device__ __forceinline__ float page_bound(const Int4Part& p) {
  float x[4];
#pragma unroll
  for (int g = 0; g < 4; ++g) x[g] = fmaf(15.f, fabsf(bf16_lo(p.pairs[g])), fabsf(bf16_hi(p.pairs[g])));
  float b = max_num(max_num(x[0], x[1]), max_num(x[2], x[3]));
  b = max_num(b, dpp<kDppHalfMirror>(b));                    // (the lanes of a quad have the same pairs)
  b = max_num(b, dpp<kDppMirror>(b));
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(b), __float_as_uint(b), false, false);
  b = max_num(__uint_as_float(r[0]), __uint_as_float(r[1]));
  const auto q = __builtin_amdgcn_permlane32_swap(__float_as_uint(b), __float_as_uint(b), false, false);
  return max_num(max_num(__uint_as_float(q[0]), __uint_as_float(q[1])), 0.f);
}

// Word 4 (lane % 4) + g of a lane's part, dims 32 g + 8 (lane % 4) .. + 7, as fp16 values times f to slot `row` of a tile.
__device__ __forceinline__ void unpack_word(const Int4Part& p, int g, float f, uint32_t mask, __bf16* tile, int row, int lane) {
  const _Float16 s = (_Float16)(bf16_lo(p.pairs[g]) * f), m = (_Float16)(bf16_hi(p.pairs[g]) * f);
  u32x4 x;
#pragma unroll
  for (int n = 0; n < 4; ++n) {                              // 1024 + c, c, m + s c: one rounding, of the last
    const uint32_t c = ((p.codes[g] >> (4 * n)) & mask) | 0x64006400u;
    const f16x2 code = __builtin_bit_cast(f16x2, c) - f16x2{(_Float16)1024.f, (_Float16)1024.f};
    x[n] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(code, f16x2{s, s}, f16x2{m, m}));
  }
  *reinterpret_cast<u32x4*>(tile + row * kHeadDim + 8 * ((4 * g + (lane & 3)) ^ (row & 15))) = x;
}

// attend_tiles over rows in 4 bits: same walk (contiguous tiles), masks, lanes and results. Phase A of tile n unpacks this wave's
// page of tile n + 1 and turns the scores of tile n into weights; phase B is O += V . P of tile n and the scores of tile n + 1. A
// barrier ends each. K waves take A(n) in phase 2 n, V waves in 2 n + 1, so what a buffer held is read for the last time:
//   K tile n - 1 by B(n - 2), in phases 2 n - 3 and 2 n - 2; the K waves put tile n + 1 in its place in phase 2 n;
//   V tile n - 1 by B(n - 1), in phases 2 n - 1 and 2 n; the V waves put tile n + 1 in its place in phase 2 n + 1.
template <int H, int kWaves, class Walk, class Lane>
__device__ __forceinline__ void attend_tiles_int4(const Int4Rows& rows, Walk& walk, int n_keys,
                                                  __bf16* const (&K)[kStages], __bf16* const (&V)[kStages],
                                                  const bf16x8 (&qop)[H][4], floatx4 (&o)[8][H], float (&m_run)[H],
                                                  float (&l_run)[H], const Lane& lane_mask, float scale_log2, int w, int lane) {
  static_assert(kWaves == 8 && kBN == 4 * kPage, "a wave a page of K or V");
  const int m16 = lane & 15, j = lane >> 4;
  const bool is_v = w >= 4;
  const int page = w & 3, row = 16 * page + (lane >> 2);
  const int tiles = walk.kt_end - walk.kt_begin;
  if (tiles <= 0) return;
  __shared__ __attribute__((aligned(16))) int k_exp[4][4];   // [tile % 4][page]: eK << 23
  __shared__ int v_need[2][4];                               // [tile % 2][page]

  f16x8 q[H][4];
  int q_exp[H];                                              // eQ << 23
#pragma unroll
  for (int u = 0; u < H; ++u) {
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int d = 0; d < 8; ++d) x = fmaxf(x, fabsf((float)qop[u][i][d]));
    const int e = range_exp(max_xor32(max_xor16(x)));
    const float f = exp2i(-e);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int d = 0; d < 8; ++d) q[u][i][d] = (_Float16)((float)qop[u][i][d] * f);
    q_exp[u] = e * (1 << 23);
  }

  // This wave's part of tile i of the walk; slots past the last key read as zeros (their weights are 0)
  auto load = [&](int i) {
    const int k0 = (walk.kt_begin + i) * kBN;
    Int4Part p = load_part(rows, (k0 >> 4) + page, is_v, lane);
    if (k0 + row >= n_keys) p.pairs = u32x4{0, 0, 0, 0};
    return p;
  };
  uint32_t mask = 0x000f000fu;                               // (in a register: and and or in one instruction)
  __asm__("" : "+v"(mask));
  auto needed = [&](int i) { return max(max(v_need[i & 1][0], v_need[i & 1][1]), max(v_need[i & 1][2], v_need[i & 1][3])); };
  auto unpack = [&](const Int4Part& p, int v_exp, int i, __bf16* k_to, __bf16* v_to) {
    int e = v_exp;
    if (!is_v) {
      e = range_exp(page_bound(p));
      if (lane == 0) k_exp[i & 3][page] = e * (1 << 23);
    }
    const float f = exp2i(-e);
    __bf16* const to = is_v ? v_to : k_to;
#pragma unroll
    for (int g = 0; g < 4; ++g) unpack_word(p, g, f, mask, to, row, lane);
  };
  auto announce = [&](const Int4Part& p, int i) {            // what a V wave's page of tile i needs
    if (!is_v) return;
    const int e = range_exp(page_bound(p));
    if (lane == 0) v_need[i & 1][page] = e;
  };
  float ref[H];                                              // the running maximum less kHeadroom
#pragma unroll
  for (int u = 0; u < H; ++u) ref[u] = -INFINITY;
  floatx4 s[2][2][H];
  auto scores = [&](const __bf16* buf) {
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int u = 0; u < H; ++u) s[kk][t][u] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const f16x8 kop = __builtin_bit_cast(f16x8, lds16(buf, 32 * kk + 16 * t + m16, 4 * i + j));
#pragma unroll
          for (int u = 0; u < H; ++u) s[kk][t][u] = mfma16x16x32(kop, q[u][i], s[kk][t][u]);
        }
  };
  // Ends a phase: this wave's LDS reads and writes are done (loads from memory stay in flight)
  auto end_phase = [] {
    __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    __asm__ volatile("" ::: "memory");
  };

  Int4Part part = load(0);
  announce(part, 0);
  __syncthreads();
  int v_exp = needed(0);
  unpack(part, v_exp, 0, K[0], V[0]);
  part = load(1);
  announce(part, 1);
  __syncthreads();
  scores(K[0]);
  floatx4 lsum[H];
#pragma unroll
  for (int u = 0; u < H; ++u) lsum[u] = floatx4{0.f, 0.f, 0.f, 0.f};
  const _Float16 one = (_Float16)1.f;
  const f16x8 ones = {one, one, one, one, one, one, one, one};

  int k0 = 0;
  TileMask tm;
  auto tile = [&](auto slot_c, int n) {
    constexpr int slot = decltype(slot_c)::value;
    // -- phase A
    const int v_now = max(v_exp, needed(n));
    if (v_now != v_exp) {
      const float f = exp2i(max(v_exp - v_now, -126));
#pragma unroll
      for (int u = 0; u < H; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i][u] *= f;
      v_exp = v_now;
    }
    typedef int i4 __attribute__((ext_vector_type(4)));
    const i4 ke = *reinterpret_cast<const i4*>(k_exp[n & 3]);
    unpack(part, is_v ? max(v_exp, needed(n + 1)) : 0, n + 1, K[slot ^ 1], V[slot ^ 1]);
    part = load(n + 2);
    walk.next(k0, tm, n == 0);
    tile_mask<H, Walk>(s, k0, tm, lane_mask, j);
    // online softmax, as tile_softmax: the log2 scores relative to ref, which moves when a weight would pass 2^15
    float neg_m[H];
    bool need = false;
#pragma unroll
    for (int u = 0; u < H; ++u) {
      neg_m[u] = ref[u] == -INFINITY ? 0.f : -ref[u];
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const float f = scaled_bits(__float_as_int(scale_log2), q_exp[u] + ke[2 * kk + t]);
#pragma unroll
          for (int r = 0; r < 4; ++r) s[kk][t][u][r] = fmaf(s[kk][t][u][r], f, neg_m[u]);
        }
      need |= lane_max(s, u) > (ref[u] == -INFINITY ? -INFINITY : 15.f);
    }
    if (__any(need)) {
#pragma unroll
      for (int u = 0; u < H; ++u) {
        const float tmax = max_xor32(max_xor16(lane_max(s, u)));
        const float r_new = fmaxf(ref[u], tmax - neg_m[u] - kHeadroom);
        const float alpha = r_new == -INFINITY ? 1.f : fast_exp2(ref[u] - r_new);
        const float d = r_new == -INFINITY ? 0.f : r_new + neg_m[u];
        ref[u] = r_new;
        lsum[u] *= alpha;
#pragma unroll
        for (int i = 0; i < 8; ++i) o[i][u] *= alpha;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
          for (int t = 0; t < 2; ++t) s[kk][t][u] -= d;
      }
    }
    f16x8 pop[2][H];
#pragma unroll
    for (int u = 0; u < H; ++u)
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
        for (int e = 0; e < 8; ++e) pop[kk][u][e] = (_Float16)fast_exp2(s[kk][e >> 2][u][e & 3]);
      }
    end_phase();
    // -- phase B
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const f16x8 vop = __builtin_bit_cast(f16x8, vt_operand(V[slot], 32 * kk, t, lane));
#pragma unroll
        for (int u = 0; u < H; ++u) o[t][u] = mfma16x16x32(vop, pop[kk][u], o[t][u]);
      }
#pragma unroll
      for (int u = 0; u < H; ++u) lsum[u] = mfma16x16x32(ones, pop[kk][u], lsum[u]);
    }
    scores(K[slot ^ 1]);                                     // (past the last tile: of zeros, or of another part's, discarded)
    announce(part, n + 2);
    end_phase();
  };
  if (is_v) end_phase();
  for (int n = 0;;) {
    tile(Slot<0>{}, n);
    if (++n >= tiles) break;
    tile(Slot<1>{}, n);
    if (++n >= tiles) break;
  }
  if (!is_v) end_phase();
  const float f = exp2i(v_exp - kHeadroom);
#pragma unroll
  for (int u = 0; u < H; ++u) {
    m_run[u] = ref[u] + kHeadroom;
    l_run[u] = lsum[u][0] * exp2i(-kHeadroom);
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i][u] *= f;
  }
}

}  // namespace abkv

// The paged cache in 4 bits (int4.h): rows written and read back, and single-token attention over it (gfx950).
#include "abridgekv_amd.h"
#include "int4.h"

#define ABKV_LDS(p) ((__attribute__((address_space(3))) void*)(p))

namespace abkv {

__device__ __forceinline__ u32x4 ld16b(const char* p) { return *reinterpret_cast<const u32x4*>(p); }

// -- rows in and out ----------------------------------------------------------------------------------------------------
struct Append4Args {
  const __bf16* k; long k_st, k_sh;            // [T, 8, 128]
  const __bf16* v; long v_st, v_sh;
  const int64_t* slot_mapping;                 // [T]; < 0 or past the cache = skip
  char* cache; long num_pages;
};

// Workgroup per token; thread: 8 dims of a head of K (the first 128 threads) or V. (1501 tokens: 4.8 us to write, 5.7 to read in
// fp32, the copy rate and a launch.)
__global__ __launch_bounds__(256) void kv_append4_kernel(Append4Args a) {
  const long t = blockIdx.x;
  const long slot = a.slot_mapping[t];
  if (slot < 0 || slot >= a.num_pages * kPage) return;       // (uniform)
  const int half = threadIdx.x >> 7, h = (threadIdx.x >> 4) & 7, b = threadIdx.x & 15;
  const __bf16* row = half ? a.v + t * a.v_st + h * a.v_sh : a.k + t * a.k_st + h * a.k_sh;
  const u32x4 w = *reinterpret_cast<const u32x4*>(row + 8 * b);
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = bf16_lo(w[i]);
    x[2 * i + 1] = bf16_hi(w[i]);
  }
  uint32_t pair;
  const uint32_t word = quantise8(x, pair);
  char* to = a.cache + slot / kPage * kPage4 + half * kHalf4 + slot % kPage * kSlot4;
  reinterpret_cast<uint32_t*>(to + h * kHeadCodes4)[code_word(b)] = word;
  if ((b & 3) == 0) reinterpret_cast<uint32_t*>(to + kParams4 + h * 16)[b >> 2] = pair;
}

// The eight values of a word and its group's pair.
__device__ __forceinline__ void values8(uint32_t word, uint32_t pair, float (&x)[8]) {
  const float s = bf16_lo(pair), m = bf16_hi(pair);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = fmaf(s, (float)((word >> (2 * i + ((i & 1) ? 14 : 0))) & 15), m);
}

// Rows by slot, as fp32 or bf16 [T, 8, 128]; a slot outside the cache reads as zeros. Threads as in kv_append4_kernel.
template <class T>
__global__ __launch_bounds__(256) void kv_read4_kernel(const char* cache, long num_pages, const int64_t* slot_mapping, T* k,
                                                       T* v) {
  const long t = blockIdx.x;
  const long slot = slot_mapping[t];
  const int half = threadIdx.x >> 7, h = (threadIdx.x >> 4) & 7, b = threadIdx.x & 15;
  float x[8] = {};
  if (slot >= 0 && slot < num_pages * kPage) {
    const char* from = cache + slot / kPage * kPage4 + half * kHalf4 + slot % kPage * kSlot4;
    values8(reinterpret_cast<const uint32_t*>(from + h * kHeadCodes4)[code_word(b)],
            reinterpret_cast<const uint32_t*>(from + kParams4 + h * 16)[b >> 2], x);
  }
  T* to = (half ? v : k) + (t * kHeadsKV + h) * kHeadDim + 8 * b;
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<floatx4*>(to) = floatx4{x[0], x[1], x[2], x[3]};
    *reinterpret_cast<floatx4*>(to + 4) = floatx4{x[4], x[5], x[6], x[7]};
  } else {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<u32x4*>(to) = w;
  }
}

// (Values: a conditional of two array elements would be their place, and the array in memory.)
__device__ __forceinline__ float pick(bool c, float a, float b) { return c ? a : b; }

// The middle of a group's values, m + 8 s.
__device__ __forceinline__ float middle(uint32_t pair) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pair), bf16x2{(__bf16)8.f, (__bf16)1.f}, 0.f, false);
}

// -- one token per sequence ---------------------------------------------------------------------------------------------
struct Decode4Args {
  const __bf16* q; long q_sb, q_sh;            // [B, 32, 128]
  const char* kv; int num_pages;
  const int32_t* block_table; long bt_stride;
  const int32_t* seq_lens;                     // [B]
  int split_pages, max_splits, max_pages;      // split_pages 0: shares
  int num_seqs, num_shares;
  int* prefix;                                 // shares: [B + 1] steps before each sequence, written by the first workgroup
  float scale_log2;
  __bf16* out; long o_sb, o_sh;                // [B, 32, 128]
  float* lse;                                  // [B, 32] or nullptr
  _Float16* part_o;                            // [parts, 32, 128]: a part's output / (l * scale)
  float* part_ml;                              // [parts, 32, 4]: m (log2 units), l, scale, unused
};                                             // parts: B x max_splits, or two for each share

__device__ __forceinline__ int rows_of(const Decode4Args& a, int b) {
  return max(min(a.seq_lens[b], a.max_pages * kPage), 0);
}
__device__ __forceinline__ int splits_of(const Decode4Args& a, int rows) {
  return max(1, ((rows + kPage - 1) / kPage + a.split_pages - 1) / a.split_pages);
}
__device__ __forceinline__ int steps_of(int rows) { return max(1, (rows + 2 * kPage - 1) / (2 * kPage)); }

// Codes of two neighbouring dims (nibbles n and n + 4 of a word) as the bf16 pair 128 + c: c lies in the low bits of the
// mantissa, so every code is exact, and the 128s leave with the sums.
// (mask in a vector register: with both constants literal the and and the or are instructions of their own)
__device__ __forceinline__ uint32_t code_pair(uint32_t w, int n, uint32_t mask) { return ((w >> (4 * n)) & mask) | 0x43004300u; }

// A wave per KV head. A workgroup walks its rows of a sequence 32 slots (two pages) at a time, the next step's rows on the way
// meanwhile.
//
// Scores: the four groups of 32 dims have their own steps and minima, so a score is the sum of four products:
//   x_j = sum_g (s_jg a_jg + m_jg Q_g),  a_jg = sum_{d in g} q_d c_jd,  Q_g = sum_{d in g} q_d.
// One MFMA tile has 16 columns where a KV head has 4 query heads: column 4 h + g holds query head h with the dims of group g
// alone (zero elsewhere), so that the four MFMAs of a tile leave a_jg in one accumulator and the sum over g is two DPP steps.
// Values: out_d = sum_j (p_j s_jg) (c_jd - 8) + sum_j p_j (m_jg + 8 s_jg): column 4 h + g of P^T carries p_j s_jg, and of the four
// accumulator rows 4 j + r of an output tile (words of the value rows, word % 4 its group) a lane keeps r = g: 8 dims in a row.
// The codes enter as 128 + c (code_pair): the score accumulator starts at -128 Q_g, and a row of -136s among the V tiles takes
// them, and the codes' middle, out of the output. p_j s_jg enters in two bf16 parts, itself and what its rounding leaves, so that
// it errs by 2^-16 of itself; everything else is exact or fp32. (One part: an output off by 0.0023 of itself in place of 0.0017,
// its own rounding to bf16; the second products, of the same codes, take 1.3 of 78 us over 64 sequences of 500 to 9500 rows, and
// no time over one of 32000.)
//
// What bounds the reads is the number of cache lines that a CU asks for (about one in six cycles), so a line should bring what it
// holds: a head's codes are half of one, its pairs an eighth. The workgroup's waves therefore fetch whole rows together, straight
// into LDS (a wave 5 of the step's 40 KB), one barrier a step. (64 sequences of 500 to 9500 rows, every wave its own pieces: 118
// us, of which 59 went with the pairs alone; the pairs shared, 99; whole rows, 94, nontemporal, 86, in equal shares, 73 without the
// merge: 410 MB at 5.6 TB/s, then beside 62 of vector work, to whose instructions the second parts have added a tenth. Three stages
// of LDS leave one workgroup a CU: 104 where two took 94.)
constexpr int kPairs4 = 16 * 4 * kHeadsKV, kCodes4 = 16 * kHeadsKV * 16;     // dwords of a page's pairs and codes (of K or V)
template <class T>
__device__ __forceinline__ const T& at4(const uint32_t* base, uint32_t bytes) {
  return *reinterpret_cast<const T*>(reinterpret_cast<const char*>(base) + bytes);
}
// The loads' cache policy: nontemporal, as every row is read once (64 sequences of 500 to 9500 rows: 98 -> 89 us, 256 of 500 to
// 3000: 136 -> 126).
constexpr int kOnce = 2;
// LDS of a step: parts K0 K1 V0 V1 (pages 0 and 1). Codes in rows of 32 16-byte chunks, slot by slot, chunk 4 head + word / 4 at
// place (chunk ^ slot): both kinds of reads below then take all banks. Pairs in rows of 8 chunks, a chunk a head: row 4 r + j is
// slot 4 j + r, its chunks at place (head ^ (j >> 1)).
struct Step4 {
  uint32_t codes[4][kCodes4];
  uint32_t pairs[4][kPairs4];
};
constexpr int kShareSteps = 64;                // steps of a share at most
constexpr int kShareSeqs = 64 * kHeadsKV;      // sequences of a launch in shares

// Pages [pg_begin, pg_end) of sequence b, at most 2 kShareSteps: its output (part < 0: that is all of the sequence) or a part.
__device__ __forceinline__ void decode4_piece(const Decode4Args& a, Step4& lds0, Step4& lds1, int b, int row_end, int pg_begin,
                                              int pg_end, long part_at) {
  const int kvh = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int lane = threadIdx.x & 63;
  __asm__("" : "+v"(lane));                                  // (what depends on it is not carried from piece to piece)
  const int m16 = lane & 15, j = lane >> 4;
  const int h = m16 >> 2, g = m16 & 3;

  // Page ids, lane l pages pg_begin + l and pg_begin + 64 + l
  const int32_t* bt = a.block_table + (long)b * a.bt_stride + pg_begin;
  int pid_l = 0, pid_h = 0;
  if (lane < pg_end - pg_begin) pid_l = min(max(bt[lane], 0), a.num_pages - 1);
  if (lane + 64 < pg_end - pg_begin) pid_h = min(max(bt[lane + 64], 0), a.num_pages - 1);

  // Q^T: dims 32 g + 8 j .. + 7 of head h, for the MFMA of group g
  bf16x8 qop[4];
  float qsum = 0.f;
  {
    const u32x4 w = *reinterpret_cast<const u32x4*>(a.q + (long)b * a.q_sb + (long)(kvh * kGroup + h) * a.q_sh + 32 * g + 8 * j);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      qop[i] = __builtin_bit_cast(bf16x8, g == i ? w : u32x4{0, 0, 0, 0});
      qsum += bf16_lo(w[i]) + bf16_hi(w[i]);
    }
    qsum = sum_xor32(sum_xor16(qsum));                       // Q_g
  }
  // Q_g in three bf16 parts (lane groups j = 0 .. 2), against a slot's pairs as they lie in the row: (s_0, m_0), .. (s_3, m_3).
  // One MFMA then leaves sum_g m_g Q_g, in the columns of g = 0.
  bf16x8 qmin;
  {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float v = __shfl(qsum, (lane & 48) + 4 * h + i, 64);   // Q_i of this head
      const float v0 = bf16_hi(__float_as_uint(v)), v1 = bf16_hi(__float_as_uint(v - v0));
      const float x = j == 0 ? v0 : j == 1 ? v1 : v - v0 - v1;
      w[i] = g == 0 && j < 3 ? __float_as_uint(x) & 0xffff0000u : 0u;
    }
    qmin = __builtin_bit_cast(bf16x8, w);
  }
  const float q128 = -128.f * qsum;
  typedef short s8 __attribute__((ext_vector_type(8)));
  const short n136 = (short)0xc308;                          // bf16 -136
  const bf16x8 minus = __builtin_bit_cast(bf16x8, s8{n136, n136, n136, n136, n136, n136, n136, n136});
  uint32_t mask = 0x000f000fu;
  __asm__("" : "+v"(mask));

  floatx4 o[8], off = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = floatx4{0.f, 0.f, 0.f, 0.f};
  float m_run = -INFINITY, l_run = 0.f, om = 0.f;            // om: sum of p_j (m_jg + 8 s_jg) over this lane's slots

  // What this wave fetches, of part wave / 2 (of K or V: part / 2; of page part % 2): slots 8 (wave % 2) .. + 7, two a load, and
  // rows 8 (wave % 2) .. + 7 of the pairs.
  const int part = kvh >> 1, rows8 = 8 * (kvh & 1);
  const int p_row = rows8 + (lane >> 3);
  uint32_t code_from = 16 * ((lane & 31) ^ (rows8 + (lane >> 5)));
  uint32_t pair_from = (4 * (p_row & 3) + (p_row >> 2)) * kSlot4 + kParams4 + 16 * ((lane & 7) ^ (p_row >> 1 & 1));
  const uint32_t slot_from = (lane >> 5) * kSlot4;
  const int last = pg_end - 1 - pg_begin;
  // Offsets as the instructions take them: 32 bits in a register beside a uniform base. (Pinned: made into 64-bit addresses
  // ahead of the loop they spill.)
  auto fetch = [&](Step4& to, int pg) {                      // (past the end: the last page again)
    const int at = min(pg + (part & 1) - pg_begin, last);
    const int id = at < 64 ? __builtin_amdgcn_readlane(pid_l, at) : __builtin_amdgcn_readlane(pid_h, at - 64);
    const char* from = a.kv + (long)id * kPage4 + (part >> 1) * kHalf4;
    __asm__("" : "+v"(pair_from), "+v"(code_from));
    __builtin_amdgcn_global_load_lds((const void*)(from + pair_from), ABKV_LDS(&to.pairs[part][32 * rows8]), 16, 0, kOnce);
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const uint32_t off = (code_from ^ 32 * n) + slot_from;
      __builtin_amdgcn_global_load_lds((const void*)(from + (rows8 + 2 * n) * kSlot4 + off),
                                       ABKV_LDS(&to.codes[part][128 * (rows8 + 2 * n)]), 16, 0, kOnce);
    }
  };
  // What it reads of a step, in bytes: K words 4 j .. + 3 of slot m16; word m16 of the V slots 4 j + e; group g's pairs of slots
  // 4 j + r; slot m16's pairs
  uint32_t k_at = 512 * m16 + 16 * ((4 * kvh + j) ^ m16);
  uint32_t v_at = 512 * 4 * j + 16 * ((4 * kvh + (m16 >> 2)) ^ (4 * j)) + 4 * (m16 & 3);           // (e: 512 e, the place ^ e)
  uint32_t pair_at = ((j * kHeadsKV + (kvh ^ (j >> 1))) * 4 + g) * 4;
  uint32_t row_at = ((4 * (m16 & 3) + (m16 >> 2)) * kHeadsKV + (kvh ^ (m16 >> 3))) * 16;
  // One step over the 32 slots from page pg on, which `cur` holds; the next step's rows go to nxt.
  auto step = [&](const Step4& cur, Step4& nxt, int pg) {
    __asm__ volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070);                      // (vmcnt(0) lgkmcnt(0), as a builtin: the compiler counts on from it)
    __builtin_amdgcn_s_barrier();                            // cur is whole, and nobody reads nxt any more
    __asm__ volatile("" ::: "memory");
    if (pg + 2 < pg_end) fetch(nxt, pg + 2);
    __asm__("" : "+v"(k_at), "+v"(v_at), "+v"(pair_at), "+v"(row_at));
    floatx4 s[2];
    u32x4 k[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) k[t] = at4<u32x4>(cur.codes[t], k_at);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      s[t] = floatx4{q128, q128, q128, q128};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t w = k[t][i];
        const u32x4 codes = {code_pair(w, 0, mask), code_pair(w, 1, mask), code_pair(w, 2, mask), code_pair(w, 3, mask)};
        s[t] = mfma16x16x32(__builtin_bit_cast(bf16x8, codes), qop[i], s[t]);
      }
    }
    floatx4 mq[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const u32x4 row = at4<u32x4>(cur.pairs[t], row_at);
      mq[t] = mfma16x16x32(__builtin_bit_cast(bf16x8, row), qmin, floatx4{0.f, 0.f, 0.f, 0.f});
    }
    uint32_t kp[2][4], vp[2][4];                             // pairs of group g of slots 4 j .. + 3 of the two pages
    uint32_t vw[8];                                          // word m16 of slots 4 j + e of page 0, then of page 1
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        kp[t][r] = at4<uint32_t>(cur.pairs[t] + r * 16 * kHeadsKV, pair_at);
        vp[t][r] = at4<uint32_t>(cur.pairs[2 + t] + r * 16 * kHeadsKV, pair_at);
        vw[4 * t + r] = at4<uint32_t>(cur.codes[2 + t] + 128 * r, v_at ^ 16 * r);
      }

    // Scores summed over the groups, i.e. the lanes of a quad, of which lane g keeps the slots e = 2 g, 2 g + 1 (of the order of
    // vw; page e / 4, slot 4 j + e % 4)
    float x[8], y[4], sv[2];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = fmaf(bf16_lo(kp[e >> 2][e & 3]), s[e >> 2][e & 3], mq[e >> 2][e & 3]);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] += dpp<kDppXor2>(x[e]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      y[e] = pick(g & 2, x[4 + e], x[e]);
      y[e] += dpp<kDppXor1>(y[e]);
    }
    sv[0] = pick(g & 1, y[2], y[0]);
    sv[1] = pick(g & 1, y[3], y[1]);
    if ((pg + 2) * kPage > row_end) {                        // rows past the end: whatever their slots hold
      __asm__ volatile("" ::: "memory");                     // (a branch: the last step's work, not every step's)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (pg * kPage + 8 * (g & 2) + 4 * j + 2 * (g & 1) + i >= row_end) sv[i] = -INFINITY;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (pg * kPage + 16 * (e >> 2) + 4 * j + (e & 3) >= row_end) vp[e >> 2][e & 3] = 0u;
    }
    const float mx = fmaxf(sv[0], sv[1]);
    // The maximum moves only when some row passes it by more than 8 (weights stay below 2^8)
    if (__any(mx * a.scale_log2 > m_run + 8.f)) {
      __asm__ volatile("" ::: "memory");
      float m_new = max_xor32(max_xor16(mx));
      m_new = fmaxf(m_new, dpp<kDppXor1>(m_new));
      m_new = fmaxf(m_run, fmaxf(m_new, dpp<kDppXor2>(m_new)) * a.scale_log2);
      const float alpha = m_new == -INFINITY ? 1.f : fast_exp2(m_run - m_new);
      m_run = m_new;
      l_run *= alpha;
      om *= alpha;
      off *= alpha;
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] *= alpha;
    }
    const float m_ref = m_run == -INFINITY ? 0.f : -m_run;
    const float pe[2] = {fast_exp2(fmaf(sv[0], a.scale_log2, m_ref)), fast_exp2(fmaf(sv[1], a.scale_log2, m_ref))};
    l_run += pe[0] + pe[1];
    float p[8];                                              // of all eight slots: lane e / 2 of the quad has it
    p[0] = dpp<0x00>(pe[0]);
    p[1] = dpp<0x00>(pe[1]);
    p[2] = dpp<0x55>(pe[0]);
    p[3] = dpp<0x55>(pe[1]);
    p[4] = dpp<0xaa>(pe[0]);
    p[5] = dpp<0xaa>(pe[1]);
    p[6] = dpp<0xff>(pe[0]);
    p[7] = dpp<0xff>(pe[1]);
    u32x4 pw, pl;                                            // p_j s_jg, and what its rounding leaves
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const uint32_t w0 = vp[e >> 2][e & 3], w1 = vp[e >> 2][(e & 3) + 1];
      om = fmaf(p[e], middle(w0), om);
      om = fmaf(p[e + 1], middle(w1), om);
      const float a0 = p[e] * bf16_lo(w0), a1 = p[e + 1] * bf16_lo(w1);
      pw[e / 2] = pack_bf16x2(a0, a1);
      pl[e / 2] = pack_bf16x2(a0 - bf16_lo(pw[e / 2]), a1 - bf16_hi(pw[e / 2]));
    }
    const bf16x8 pop = __builtin_bit_cast(bf16x8, pw), low = __builtin_bit_cast(bf16x8, pl);
    off = mfma16x16x32(minus, pop, off);
    off = mfma16x16x32(minus, low, off);
    uint32_t lo[4], hi[4];                                   // nibbles 0 .. 3 and 4 .. 7 of two slots
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      lo[n] = __builtin_amdgcn_perm(vw[2 * n + 1], vw[2 * n], 0x05040100u);
      hi[n] = __builtin_amdgcn_perm(vw[2 * n + 1], vw[2 * n], 0x07060302u);
    }
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const u32x4 ev = {code_pair(lo[0], n, mask), code_pair(lo[1], n, mask), code_pair(lo[2], n, mask), code_pair(lo[3], n, mask)};
      const u32x4 od = {code_pair(hi[0], n, mask), code_pair(hi[1], n, mask), code_pair(hi[2], n, mask), code_pair(hi[3], n, mask)};
      const bf16x8 even = __builtin_bit_cast(bf16x8, ev), odd = __builtin_bit_cast(bf16x8, od);
      o[2 * n] = mfma16x16x32(even, pop, o[2 * n]);
      o[2 * n + 1] = mfma16x16x32(odd, pop, o[2 * n + 1]);
      o[2 * n] = mfma16x16x32(even, low, o[2 * n]);
      o[2 * n + 1] = mfma16x16x32(odd, low, o[2 * n + 1]);
    }
  };
  if (pg_begin < pg_end) {
    fetch(lds0, pg_begin);
    for (int pg = pg_begin;;) {
      step(lds0, lds1, pg);
      if ((pg += 2) >= pg_end) break;
      step(lds1, lds0, pg);
      if ((pg += 2) >= pg_end) break;
    }
  }

  // This lane's 8 dims 32 g + 8 j .. + 7 of head h
  float l = sum_xor32(sum_xor16(l_run));
  l += dpp<kDppXor1>(l);
  l += dpp<kDppXor2>(l);
  om = sum_xor32(sum_xor16(om));
  const float inv = l > 0.f ? 1.f / l : l;                   // (a NaN stays one; no row: 0)
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float even = g & 2 ? o[i][2] : o[i][0], odd = g & 2 ? o[i][3] : o[i][1];
    x[i] = ((g & 1 ? odd : even) + off[0] + om) * inv;
  }
  const int head = kvh * kGroup + h, dim = 32 * g + 8 * j;
  if (part_at < 0) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<u32x4*>(a.out + (long)b * a.o_sb + (long)head * a.o_sh + dim) = w;
    if (a.lse != nullptr && g == 0 && j == 0)
      a.lse[(long)b * kHeadsQ + head] = l > 0.f ? (m_run + __log2f(l)) * 0.69314718055994531f : l == 0.f ? -INFINITY : l;
    return;
  }
  // Partials as the bf16 decode's: fp16 of the split's output, over a power of two that fits its largest value (F16Range)
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = fmaxf(amax, fabsf(x[i]));
  amax = fmaxf(amax, dpp<kDppXor1>(amax));
  amax = fmaxf(amax, dpp<kDppXor2>(amax));
  amax = max_xor32(max_xor16(amax));
  const F16Range range(amax);
  typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
  f16x8 w;
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = (_Float16)(x[i] * range.inv);
  const long at = part_at * kHeadsQ + head;
  *reinterpret_cast<f16x8*>(a.part_o + at * kHeadDim + dim) = w;
  if (g == 0 && j == 0) *reinterpret_cast<floatx4*>(a.part_ml + at * 4) = floatx4{m_run, l, range.scale, 0.f};
}

// Work goes out in one of two ways. Splits: workgroup (sequence, split) of split_pages pages. Shares: the steps of all sequences in
// a row, cut into num_shares equal parts, one a workgroup, which may end one sequence and begin others; at most its first and
// its last piece are parts of a sequence. The lengths are on the device, so each workgroup sums them itself.
template <bool kShares>
__global__ __launch_bounds__(64 * kHeadsKV, 4) void decode4_kernel(Decode4Args a) {
  __shared__ __attribute__((aligned(16))) Step4 lds0, lds1;
  if constexpr (!kShares) {
    // Linear grid, sequence by sequence; a sequence's splits start one further each time: workgroups go to the 8 XCDs
    // round-robin, and sequences end at different splits.
    const int b = blockIdx.x / a.max_splits, split = (blockIdx.x + b) % a.max_splits;
    const int row_end = rows_of(a, b);
    const int n_splits = splits_of(a, row_end);
    if (split >= n_splits) return;
    const int pg_begin = split * a.split_pages;
    decode4_piece(a, lds0, lds1, b, row_end, pg_begin, min((row_end + kPage - 1) / kPage, pg_begin + a.split_pages),
                  n_splits == 1 ? -1 : (long)b * a.max_splits + split);
  } else {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    // steps up to and with sequence t
    int* const sums = reinterpret_cast<int*>(&lds0);          // [8] of the waves, then the sequence and its first step
    const int mine = t < a.num_seqs ? steps_of(rows_of(a, t)) : 0;
    int upto = mine;
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) {
      const int v = __shfl_up(upto, k, 64);
      if (lane >= k) upto += v;
    }
    if (lane == 63) sums[wave] = upto;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int k = 0; k < kHeadsKV; ++k) {
      if (k < wave) upto += sums[k];
      total += sums[k];
    }
    total = __builtin_amdgcn_readfirstlane(total);
    const int share = (total + a.num_shares - 1) / a.num_shares;
    const int begin = blockIdx.x * share, end = min(begin + share, total);
    if (blockIdx.x == 0) {
      if (t < a.num_seqs) a.prefix[t] = upto - mine;
      if (t == 0) a.prefix[a.num_seqs] = total;
    }
    if (begin >= end) return;
    if (upto - mine <= begin && begin < upto) {
      sums[kHeadsKV] = t;
      sums[kHeadsKV + 1] = upto - mine;
    }
    __syncthreads();
    int b = __builtin_amdgcn_readfirstlane(sums[kHeadsKV]);
    int before = __builtin_amdgcn_readfirstlane(sums[kHeadsKV + 1]);
    for (int at = begin; at < end; ++b) {
      __syncthreads();                                       // (LDS is free again)
      const int rows = rows_of(a, b), steps = steps_of(rows);
      const int to = min(before + steps, end);
      const bool whole = at == before && to == before + steps;
      decode4_piece(a, lds0, lds1, b, rows, 2 * (at - before), min((rows + kPage - 1) / kPage, 2 * (to - before)),
                    whole ? -1 : 2l * blockIdx.x + (at != begin));
      at = to;
      before += steps;
    }
  }
}

// Joins the parts of a sequence: workgroup (head, sequence), kGroups groups of 16 lanes take the parts k = i, i + kGroups, ...,
// four at a time, a lane 8 dims; their sums meet in LDS. A pass is a trip to another XCD's memory, so many parts take more
// groups.
template <int kGroups>
__global__ __launch_bounds__(16 * kGroups) void decode4_merge_kernel(Decode4Args a) {
  const int head = blockIdx.x, b = blockIdx.y;
  long first;                                                // part 0; the others follow `second`, `apart` from each other
  long second, apart;
  int n;
  if (a.split_pages > 0) {
    n = splits_of(a, rows_of(a, b));
    first = (long)b * a.max_splits;
    second = first + 1;
    apart = 1;
  } else {
    const int total = a.prefix[a.num_seqs], share = (total + a.num_shares - 1) / a.num_shares;
    const int from = a.prefix[b], to = a.prefix[b + 1] - 1;
    const int w0 = from / share;
    n = to / share - w0 + 1;
    first = 2l * w0 + (from != w0 * share);
    second = 2l * w0 + 2;
    apart = 2;
  }
  if (n == 1) return;
  const int grp = threadIdx.x >> 4, c = threadIdx.x & 15;
  typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
  float M = -INFINITY, L = 0.f, acc[8] = {};
  for (int k0 = grp; k0 < n; k0 += 4 * kGroups) {
    floatx4 rec[4];
    f16x8 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {                            // (past the end: the last split again, without weight)
      const int k = min(k0 + u * kGroups, n - 1);
      const long from = (k == 0 ? first : second + (k - 1) * apart) * kHeadsQ + head;
      rec[u] = *reinterpret_cast<const floatx4*>(a.part_ml + from * 4);
      v[u] = *reinterpret_cast<const f16x8*>(a.part_o + from * kHeadDim + 8 * c);
    }
    float mn = M;
#pragma unroll
    for (int u = 0; u < 4; ++u) mn = fmaxf(mn, rec[u][0]);
    const float alpha = mn == -INFINITY ? 1.f : fast_exp2(M - mn);
    M = mn;
    L *= alpha;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] *= alpha;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (k0 + u * kGroups >= n) break;
      const float w = mn == -INFINITY ? rec[u][1] : fast_exp2(rec[u][0] - mn) * rec[u][1];
      L += w;
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[i] += (float)v[u][i] * (w * rec[u][2]);
    }
  }
  __shared__ float sm[kGroups], sl[kGroups], so[kGroups][kHeadDim + 4];
  if (c == 0) {
    sm[grp] = M;
    sl[grp] = L;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) so[grp][8 * c + i] = acc[i];
  __syncthreads();
  if (threadIdx.x >= kHeadDim) return;
  M = -INFINITY;
  L = 0.f;
  float x = 0.f;
#pragma unroll
  for (int i = 0; i < kGroups; ++i) M = fmaxf(M, sm[i]);
#pragma unroll
  for (int i = 0; i < kGroups; ++i) {
    const float f = sm[i] == M ? 1.f : fast_exp2(sm[i] - M);
    L += sl[i] * f;
    x += so[i][threadIdx.x] * f;
  }
  a.out[(long)b * a.o_sb + (long)head * a.o_sh + threadIdx.x] = (__bf16)(L == 0.f ? 0.f : x / L);
  if (a.lse != nullptr && threadIdx.x == 0)
    a.lse[(long)b * kHeadsQ + head] = L > 0.f ? (M + __log2f(L)) * 0.69314718055994531f : L == 0.f ? -INFINITY : L;
}

}  // namespace abkv

using namespace abkv;

constexpr int kMaxTokens = 0xFFFFFF;           // (256 threads each: work items of a launch fit 32 bits)

// Shares of a launch: a workgroup a CU while that takes at most 16 steps, else two, in as many rounds as kShareSteps needs.
static int decode4_shares(int num_seqs, int max_pages) {
  const long steps = (long)num_seqs * ((max_pages + 1) / 2);
  if (steps <= 256 * 16) return steps < 256 ? (int)steps : 256;
  return 512 * (int)((steps + 512 * kShareSteps - 1) / (512 * kShareSteps));
}

static bool rows16_ok(const void* p, long st, long sh) {
  return p != nullptr && ((uintptr_t)p & 15) == 0 && ((st | sh) & 7) == 0;
}

extern "C" {

int abkv_kv_append_int4(const void* key, long key_stride_t, long key_stride_h, const void* value, long value_stride_t,
                        long value_stride_h, const int64_t* slot_mapping, int num_tokens, void* kv_cache, int num_pages,
                        hipStream_t stream) {
  if (num_tokens <= 0) return 0;
  if (num_tokens > kMaxTokens || !rows16_ok(key, key_stride_t, key_stride_h) || !rows16_ok(value, value_stride_t, value_stride_h) ||
      slot_mapping == nullptr || !rows16_ok(kv_cache, 0, 0) || num_pages <= 0)
    return (int)hipErrorInvalidValue;
  const Append4Args a = {static_cast<const __bf16*>(key), key_stride_t, key_stride_h, static_cast<const __bf16*>(value),
                         value_stride_t, value_stride_h, slot_mapping, static_cast<char*>(kv_cache), num_pages};
  hipLaunchKernelGGL(kv_append4_kernel, dim3(num_tokens), dim3(256), 0, stream, a);
  return (int)hipGetLastError();
}

int abkv_kv_read_int4(const void* kv_cache, int num_pages, const int64_t* slot_mapping, int num_tokens, int f32, void* key,
                      void* value, hipStream_t stream) {
  if (num_tokens <= 0) return 0;
  if (num_tokens > kMaxTokens || !rows16_ok(kv_cache, 0, 0) || num_pages <= 0 || slot_mapping == nullptr || !rows16_ok(key, 0, 0) ||
      !rows16_ok(value, 0, 0))
    return (int)hipErrorInvalidValue;
  const char* cache = static_cast<const char*>(kv_cache);
  if (f32)
    hipLaunchKernelGGL(kv_read4_kernel<float>, dim3(num_tokens), dim3(256), 0, stream, cache, num_pages, slot_mapping,
                       static_cast<float*>(key), static_cast<float*>(value));
  else
    hipLaunchKernelGGL(kv_read4_kernel<__bf16>, dim3(num_tokens), dim3(256), 0, stream, cache, num_pages, slot_mapping,
                       static_cast<__bf16*>(key), static_cast<__bf16*>(value));
  return (int)hipGetLastError();
}

size_t abkv_decode_int4_workspace_size(int num_seqs, int max_pages_per_seq, int split_pages) {
  if (num_seqs <= 0 || max_pages_per_seq <= 0 || split_pages < 0) return 0;
  constexpr size_t kPart = kHeadsQ * (kHeadDim * sizeof(_Float16) + 4 * sizeof(float));
  if (split_pages == 0)
    return num_seqs > kShareSeqs ? 0
                                 : 2 * (size_t)decode4_shares(num_seqs, max_pages_per_seq) * kPart + (num_seqs + 1) * sizeof(int);
  const int splits = (max_pages_per_seq + split_pages - 1) / split_pages;
  return splits > 1 ? (size_t)num_seqs * splits * kPart : 0;
}

int abkv_decode_attn_int4(const void* q, long q_stride_seq, long q_stride_head, const void* kv_cache, int num_pages,
                          const int32_t* block_table, long block_table_stride, const int32_t* seq_lens, int num_seqs,
                          int max_pages_per_seq, int split_pages, float scale, void* out, long out_stride_seq,
                          long out_stride_head, float* lse, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  if (num_seqs <= 0) return 0;
  if (split_pages < 0 || (split_pages & 1) || split_pages > 64 || (split_pages == 0 && num_seqs > kShareSeqs) ||
      max_pages_per_seq <= 0 || max_pages_per_seq > (1 << 26) || num_pages <= 0 || block_table_stride < max_pages_per_seq ||
      num_seqs > 65535 || !softmax_scale_ok(scale) || !rows16_ok(q, q_stride_seq, q_stride_head) || !rows16_ok(kv_cache, 0, 0) ||
      block_table == nullptr || seq_lens == nullptr || !rows16_ok(out, out_stride_seq, out_stride_head))
    return (int)hipErrorInvalidValue;
  const size_t need = abkv_decode_int4_workspace_size(num_seqs, max_pages_per_seq, split_pages);
  if (need > 0 && (!rows16_ok(workspace, 0, 0) || workspace_bytes < need)) return (int)hipErrorInvalidValue;
  Decode4Args a;
  a.q = static_cast<const __bf16*>(q);
  a.q_sb = q_stride_seq;
  a.q_sh = q_stride_head;
  a.kv = static_cast<const char*>(kv_cache);
  a.num_pages = num_pages;
  a.block_table = block_table;
  a.bt_stride = block_table_stride;
  a.seq_lens = seq_lens;
  a.split_pages = split_pages;
  a.max_splits = split_pages ? (max_pages_per_seq + split_pages - 1) / split_pages : 0;
  a.max_pages = max_pages_per_seq;
  a.num_seqs = num_seqs;
  a.num_shares = split_pages ? 0 : decode4_shares(num_seqs, max_pages_per_seq);
  a.scale_log2 = scale * 1.4426950408889634f;
  a.out = static_cast<__bf16*>(out);
  a.o_sb = out_stride_seq;
  a.o_sh = out_stride_head;
  a.lse = lse;
  const size_t parts = split_pages ? (size_t)num_seqs * a.max_splits : 2 * (size_t)a.num_shares;
  a.part_o = static_cast<_Float16*>(workspace);
  a.part_ml = reinterpret_cast<float*>(a.part_o + parts * kHeadsQ * kHeadDim);
  a.prefix = reinterpret_cast<int*>(a.part_ml + parts * kHeadsQ * 4);
  const long groups = split_pages ? (long)num_seqs * a.max_splits : a.num_shares;
  if (groups * 64 * kHeadsKV > 0xFFFFFFFFL) return (int)hipErrorInvalidValue;
  if (split_pages) hipLaunchKernelGGL(decode4_kernel<false>, dim3((unsigned)groups), dim3(64 * kHeadsKV), 0, stream, a);
  else hipLaunchKernelGGL(decode4_kernel<true>, dim3((unsigned)groups), dim3(64 * kHeadsKV), 0, stream, a);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess || (split_pages && a.max_splits == 1)) return (int)err;
  const int most = split_pages ? a.max_splits : (a.num_shares + num_seqs - 1) / num_seqs;     // parts a sequence, about
  if (most > 64) hipLaunchKernelGGL(decode4_merge_kernel<64>, dim3(kHeadsQ, num_seqs), dim3(1024), 0, stream, a);
  else hipLaunchKernelGGL(decode4_merge_kernel<16>, dim3(kHeadsQ, num_seqs), dim3(256), 0, stream, a);
  return (int)hipGetLastError();
}

}  // extern "C"

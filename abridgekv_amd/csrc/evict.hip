// What a cache bounded by weight needs beside its attention (gfx950): the attention weights of a prompt's queries added up
// per cached row, and the eviction of the rows that weigh least. (A decode step's weights: decode_attn.hip.)
#include <algorithm>

#include "attn_tile.h"
#include "score_rows.h"

namespace abkv {

// ---------------------------------------------------------------------------------------------------------------------
// scores[r][KV head h][key j] += sum over h's four query heads u and the request's queries i >= j of
//                                exp(scale q_iu . k_jh - lse_iu),      query i at position kv_start[r] + i.
// A wave keeps 32 keys of one query head in registers as the MFMA's first operand. S^T = K . Q^T has a query per lane column:
// lse is one value a lane, and the sums over queries stay in the 8 accumulator positions until the end. A workgroup's 16 waves
// are the KV head's four query heads by four groups of 32 keys (kTiles = 2), or by two groups at alternate steps (kTiles = 1,
// where the longest workgroup would bound the launch). 32 query rows of the four heads at a time come into triple-buffered LDS
// by DMA. One owner per score: no atomics, the same bits every time.
// 1500 rows and 2048 behind 2048: 76 us a call among others, 800 TFLOP/s of visible pairs. Matrix units 30 % of the SIMDs'
// cycles, other vector work 43 %, 10 % both at once; the waves wait for rows and barriers 45 % of their time. A 16 x 64 step of
// MFMA, FMA, exponential and addition alone costs 419 cycles, here 640. Tried, against 94 us of this form at that time: query rows
// straight into operand registers 166 (64 bytes of each of 16 rows an instruction; without those loads 88); 64 keys a wave at
// two waves a SIMD, its three stages interleaved by hand, 95, with a step a barrier more 99.
// The requests and the tiles' order go with the launch's arguments (before, by an upload: two prompts 88 us a call, 64 queries
// behind 4000 rows 41; with it 83 and 21).
constexpr int kScoreRequests = 64, kScoreTiles = 640;        // of a launch (3.3 KiB of arguments)
struct PromptScoreArgs {
  const __bf16* q;  long q_st, q_sh;           // [T, 32, 128]
  const __bf16* kv; int num_pages;             // [pages, 2, 16, 8, 128]
  const int32_t* block_table; long bt_stride; int bt_width;      // (of the launch's first request)
  const float* lse;                            // [T, 32] natural log
  float* scores;  long s_sb, s_sh;             // [R, 8, rows] (of the launch's first request)
  float scale_log2;
  int32_t q_start[kScoreRequests + 1], kv_start[kScoreRequests];
  uint32_t tiles[kScoreTiles];                 // request << 24 | number of its tile of 64 * kTiles keys
};

// Sum over a row of 16 lanes, in each of them (DPP: no LDS).
__device__ __forceinline__ float sum16(float v) {
  auto add = [](float x, int y) { return x + __int_as_float(y); };
  v = add(v, __builtin_amdgcn_update_dpp(__float_as_int(v), __float_as_int(v), 0xB1, 0xF, 0xF, false));   // quad_perm 1,0,3,2
  v = add(v, __builtin_amdgcn_update_dpp(__float_as_int(v), __float_as_int(v), 0x4E, 0xF, 0xF, false));   // quad_perm 2,3,0,1
  v = add(v, __builtin_amdgcn_update_dpp(__float_as_int(v), __float_as_int(v), 0x141, 0xF, 0xF, false));  // row_half_mirror
  return add(v, __builtin_amdgcn_update_dpp(__float_as_int(v), __float_as_int(v), 0x140, 0xF, 0xF, false));   // row_mirror
}

constexpr int kScoreWaves = 16;
template <int kTiles>
__global__ __launch_bounds__(64 * kScoreWaves) void prompt_scores_kernel(PromptScoreArgs a) {
  constexpr int kSubs = 2 * kTiles, kPhases = kScoreWaves / kGroup / kSubs;
  constexpr int kElems = kGroup * kScoreQ * kHeadDim, kRows = kScoreQ * kGroup;
  __shared__ __attribute__((aligned(16))) __bf16 Q0[kElems], Q1[kElems], Q2[kElems];
  __shared__ __attribute__((aligned(16))) float L0[kRows], L1[kRows], L2[kRows];
  __shared__ float sums[kScoreWaves][32];
  __bf16* const Qb[3] = {Q0, Q1, Q2};
  float* const Lb[3] = {L0, L1, L2};
  const int kvh = blockIdx.x % kHeadsKV, tile = blockIdx.x / kHeadsKV;
  const uint32_t code = a.tiles[tile];
  const int r = code >> 24, first_key = (code & 0xffffffu) * (kBN * kTiles);
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, m16 = lane & 15, j = lane >> 4;
  const int t0 = a.q_start[r], nq = a.q_start[r + 1] - t0, kv0 = a.kv_start[r];
  const int n_keys = kv0 + nq;
  const int u = w & 3, sub = w >> 2 & (kSubs - 1), phase = w / (kGroup * kSubs);
  const int k0 = first_key + 32 * sub;                       // this wave's keys

  // iteration n: query rows 32n .. 32n + 31 of head h in LDS rows 32h .. (a wave's two DMAs: eight rows), and their lse as
  // [row][head] (eight waves write the same 16 rows' values). A lane's offset from the iteration's first row does not change,
  // so an iteration costs scalar arithmetic only; the last one re-reads the request's last row past its end (weight 0), and
  // so do the iterations issued past the last.
  const int last_iter = (nq - 1) / kScoreQ;
  const int half = w & 1, lrow = 16 * half + (lane >> 2);
  auto offset = [&](int i, int limit) {                      // bytes to the lane's piece of DMA i, rows up to `limit`
    const int row = 8 * w + 4 * i + j;                       // LDS row: head row / 32, query row % 32
    return score_piece(row, limit, (uint32_t)a.q_st, (uint32_t)a.q_sh, m16 ^ (row & 15));
  };
  unsigned off[2] = {offset(0, kScoreQ - 1), offset(1, kScoreQ - 1)}, off_l = (lrow * kHeadsQ + (lane & 3)) * 4;
  const char* const q_base = reinterpret_cast<const char*>(a.q + (long)t0 * a.q_st + (long)kvh * kGroup * a.q_sh);
  const char* const l_base = reinterpret_cast<const char*>(a.lse + (long)t0 * kHeadsQ + kvh * kGroup);
  auto issue = [&](int n, __bf16* qb, float* lb) {
    if (n >= last_iter) {                                    // (uniform, at the end of the walk)
      n = last_iter;
      const int limit = nq - 1 - kScoreQ * n;
      off[0] = offset(0, limit);
      off[1] = offset(1, limit);
      off_l = (min(lrow, limit) * kHeadsQ + (lane & 3)) * 4;
    }
    const char* const qp = q_base + (long)n * kScoreQ * a.q_st * 2;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      __builtin_amdgcn_global_load_lds((const void*)(qp + off[i]), ABKV_LDS(qb + 4 * (2 * w + i) * kHeadDim), 16, 0, 0);
    __builtin_amdgcn_global_load_lds((const void*)(l_base + (long)n * kScoreQ * kHeadsQ * 4 + off_l), ABKV_LDS(lb + 64 * half),
                                     4, 0, 0);
  };
  bf16x8 kop[2][4];
  floatx4 sum[2] = {floatx4{0.f, 0.f, 0.f, 0.f}, floatx4{0.f, 0.f, 0.f, 0.f}};
  auto work = [&](int row0, const __bf16* qb, const float* lb) {
    const int in = row0 & (kScoreQ - 1);                     // the step's first row in the iteration's rows
    const float l = lb[(in + m16) * kGroup + u];
    // rows past the request and rows that see nothing weigh 0, the latter (seldom there) whatever their scores
    const float l2 = row0 + m16 < nq && l > -INFINITY ? l * 1.4426950408889634f : INFINITY;
    const bool all = __all(l != -INFINITY);
    floatx4 s[2] = {floatx4{0.f, 0.f, 0.f, 0.f}, floatx4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bf16x8 qop = __builtin_bit_cast(bf16x8, lds16(qb, kScoreQ * u + in + m16, 4 * i + j));
#pragma unroll
      for (int t = 0; t < 2; ++t) s[t] = mfma16x16x32(kop[t][i], qop, s[t]);
    }
    const int before = l == -INFINITY ? -1 : kv0 + row0 + m16 - k0;          // keys 0 .. before of the wave's are seen
    if (all && kv0 + row0 >= k0 + 31) {                      // (uniform) all of them by all rows
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[t][e] += fast_exp2(fmaf(s[t][e], a.scale_log2, -l2));
    } else {
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = fast_exp2(fmaf(s[t][e], a.scale_log2, -l2));
          sum[t][e] += 16 * t + 4 * j + e <= before ? p : 0.f;
        }
    }
  };
  // the first query rows that see a key of the workgroup (a tile lies below n_keys, so some row does)
  int n = max(first_key - kv0, 0) / kScoreQ;
  const int end = last_iter + 1;
  if (n < end) {                                             // (uniform)
    // the keys through the third buffer: loaded straight into operand registers, the four heads' waves read them four times
    const PagedRows rows{a.kv + kvh * kHeadDim, a.block_table + (long)r * a.bt_stride, a.bt_width, a.num_pages};
#pragma unroll
    for (int t = 0; t < kTiles; ++t)
      issue_half<kScoreWaves, false>(rows, rows.template src<1>(min(first_key + kBN * t, n_keys - 1), w, n_keys), n_keys,
                                     Q2 + t * kTileElems, w, lane);
    issue(n, Q0, L0);
    issue(n + 1, Q1, L1);
    __asm__ volatile("s_waitcnt vmcnt(6)" ::: "memory");     // the keys; two iterations of three loads stay in flight
    __builtin_amdgcn_s_barrier();
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) kop[t][i] = __builtin_bit_cast(bf16x8, lds16(Q2, 32 * sub + 16 * t + m16, 4 * i + j));
    // Every iteration waits for this wave's three DMAs of it (the next one's stay in flight), then for the other waves', who
    // are then also done reading the buffer that the iteration after next takes.
    auto step = [&](auto slot_c) -> bool {
      constexpr int sl = decltype(slot_c)::value;
      __asm__ volatile("s_waitcnt vmcnt(3) lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      issue(n + 2, Qb[(sl + 2) % 3], Lb[(sl + 2) % 3]);
#pragma unroll
      for (int i = 0; i < 2; i += kPhases) work(kScoreQ * n + 16 * (phase + i), Qb[sl], Lb[sl]);
      return ++n < end;
    };
    for (;;) {
      if (!step(Slot<0>{})) break;
      if (!step(Slot<1>{})) break;
      if (!step(Slot<2>{})) break;
    }
    __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");     // no DMA may outlive the workgroup's LDS
  }
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float x = sum16(sum[t][e]);                      // over the query columns
      if (m16 == 0) sums[w][16 * t + 4 * j + e] = x;
    }
  __syncthreads();
  const int tid = threadIdx.x, key = first_key + tid;
  if (tid < kBN * kTiles && key < n_keys) {
    float x = 0.f;
#pragma unroll
    for (int p = 0; p < kPhases; ++p)
#pragma unroll
      for (int h = 0; h < kGroup; ++h) x += sums[h + kGroup * (tid / 32 + kSubs * p)][tid & 31];
    a.scores[(long)r * a.s_sb + (long)kvh * a.s_sh + key] += x;
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// Eviction. Per (layer, sequence, KV head): of n rows the best m = min(n, budget) are kept: rows of the first `sinks` and of
// the last `recent` tokens, then by score (ties: lowest slot; NaN below every number). Kept rows of slots >= m move into the
// evicted slots < m, both in ascending order, so a pass moves no more rows than it evicts and sources and destinations never
// meet: attention does not depend on the order of rows, and the tokens' indices travel in `positions`.
//
// One workgroup per (layer, sequence, head) does it all: keys that order as (held, score) in LDS; the m-th largest by up to
// four 8-bit digits of a histogram (no further than the rows that share its digits are kept all); each wave walks its own run
// of slots, so ranks among ties, holes and movers are ballot counts plus one prefix over the waves; then rows, scores and
// positions move. Bound by the latency of these phases for one sequence, by the moved rows (256-byte pieces) for a batch.
struct EvictArgs {
  __bf16* caches[16];
  int num_pages;
  const int32_t* block_table; long bt_stride;
  const int32_t* seq_lens;                     // [B]
  int max_rows;                                // bound on seq_lens (whole pages of the table row)
  float* scores;                               // [L, B, 8, rows_stride]
  int32_t* positions;                          // the same: token index of each row, < 0: appended since the last eviction
  long rows_stride;
  const int32_t* tokens;                       // [B] tokens seen
  int batch, budget, sinks, recent;
  int32_t* out_lens;                           // [B]
  uint32_t* work;                              // kSlots == 0: [L, B, 8, max_rows]
};

// Order-preserving key of a score; rows that are held above every score.
__device__ __forceinline__ uint32_t score_key(float x, bool held) {
  if (held) return 0xffffffffu;
  if (x != x) return 0u;
  const uint32_t u = __float_as_uint(x + 0.f);               // -0 and 0 tie
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kEvictMaxRows = 1 << 18;         // rows whose kept bits fit LDS beside the rest

template <int kSlots, int kWaves>
__global__ __launch_bounds__(64 * kWaves) void evict_kernel(EvictArgs a) {
  constexpr int kThreads = 64 * kWaves;
  constexpr int kCopies = 8;                                 // of the histogram: most scores share their first digit
  __shared__ uint32_t lds_keys[kSlots > 0 ? kSlots : 1];
  __shared__ uint64_t kept_bits[(kSlots > 0 ? kSlots : kEvictMaxRows) / 64];
  __shared__ uint32_t hist[256 * kCopies];
  __shared__ int counts[kWaves][2];
  __shared__ int pick[3];
  const int h = blockIdx.x % kHeadsKV;
  const int lb = blockIdx.x / kHeadsKV;
  const int b = lb % a.batch, layer = lb / a.batch;
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = max(min(a.seq_lens[b], a.max_rows), 0);
  const int m = min(n, a.budget);
  if (layer == 0 && h == 0 && tid == 0) a.out_lens[b] = m;
  if (n <= m) return;                                        // (uniform)
  const long at = ((long)lb * kHeadsKV + h) * a.rows_stride;
  float* const scores = a.scores + at;
  int32_t* const positions = a.positions + at;
  uint32_t* const keys = kSlots > 0 ? lds_keys : a.work + ((long)lb * kHeadsKV + h) * a.max_rows;
  const int tokens = a.tokens[b];
  // token index of a row (rows without one were appended one after the other)
  auto token_of = [&](int slot, int pos) { return pos < 0 ? tokens - (n - slot) : pos; };
  const int run = (n + kThreads - 1) / kThreads * 64;        // slots of a wave
  const int s0 = w * run, s1 = min(s0 + run, n);
  for (int s = s0 + lane; s < s1; s += 64) {
    const int t = token_of(s, positions[s]);
    keys[s] = score_key(scores[s], t < a.sinks || t >= tokens - a.recent);
  }
  // the m-th largest key, digit by digit from the top
  uint32_t prefix = 0, mask = 0;
  int want = m;                                              // rank of the key among those that share the prefix
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256 * kCopies; i += kThreads) hist[i] = 0;
    __syncthreads();
    for (int s = s0 + lane; s < s1; s += 64) {
      const uint32_t k = keys[s];
      if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift & 255u) * kCopies + (lane & (kCopies - 1))], 1u);
    }
    __syncthreads();
    if (w == 0) {                                            // lane l: digits 255 - 4l .. 252 - 4l
      int c[4], total = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        c[i] = 0;
        for (int e = 0; e < kCopies; ++e) c[i] += hist[(255 - 4 * lane - i) * kCopies + e];
        total += c[i];
      }
      int above = total;                                     // inclusive scan, then exclusive
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int up = __shfl_up(above, d, 64);
        above += lane >= d ? up : 0;
      }
      above -= total;
      if (want > above && want <= above + total) {           // one lane
        int i = 0;
        while (i < 3 && want > above + c[i]) above += c[i++];
        pick[0] = 255 - 4 * lane - i;
        pick[1] = want - above;
        pick[2] = i == 0 ? c[0] : i == 1 ? c[1] : i == 2 ? c[2] : c[3];
      }
    }
    __syncthreads();
    prefix |= (uint32_t)pick[0] << shift;
    mask |= 255u << shift;
    want = pick[1];
    if (want == pick[2]) break;                              // (uniform) all keys with these digits are kept
  }
  // kept: keys above the prefix, and the first `want` that equal it
  int ties = 0;
  for (int s = s0 + lane; s - lane < s1; s += 64) ties += __popcll(__ballot(s < s1 && (keys[min(s, n - 1)] & mask) == prefix));
  if (lane == 0) counts[w][0] = ties;
  __syncthreads();
  int rank = 0;
  for (int i = 0; i < w; ++i) rank += counts[i][0];
  __syncthreads();
  const uint64_t below = (1ull << lane) - 1;
  int holes = 0, movers = 0;
  for (int s = s0 + lane; s - lane < s1; s += 64) {
    const uint32_t k = keys[min(s, n - 1)] & mask;
    const uint64_t eq = __ballot(s < s1 && k == prefix);
    const bool keep = s < s1 && (k > prefix || (k == prefix && rank + __popcll(eq & below) < want));
    rank += __popcll(eq);
    const uint64_t kept = __ballot(keep);
    if (lane == 0) kept_bits[(s - lane) >> 6] = kept;
    holes += __popcll(__ballot(s < s1 && s < m && !keep));
    movers += __popcll(__ballot(keep && s >= m));
  }
  if (lane == 0) {
    counts[w][0] = holes;
    counts[w][1] = movers;
  }
  __syncthreads();                                           // every wave is done with the keys: their place takes the lists
  int hole_at = 0, mover_at = 0, total = 0;
  for (int i = 0; i < kWaves; ++i) {
    hole_at += i < w ? counts[i][0] : 0;
    mover_at += i < w ? counts[i][1] : 0;
    total += counts[i][0];
  }
  uint32_t* const to = keys;                                 // total <= min(m, n - m): both lists fit n entries
  uint32_t* const from = keys + total;
  for (int s = s0 + lane; s - lane < s1; s += 64) {
    const uint64_t kept = kept_bits[(s - lane) >> 6];
    const bool in = s < s1, keep = kept >> lane & 1;
    const uint64_t hole = __ballot(in && s < m && !keep), mover = __ballot(keep && s >= m);
    if (in && s < m && !keep) to[hole_at + __popcll(hole & below)] = s;
    if (keep && s >= m) from[mover_at + __popcll(mover & below)] = s;
    hole_at += __popcll(hole);
    mover_at += __popcll(mover);
    if (keep && s < m && positions[s] < 0) positions[s] = token_of(s, -1);
  }
  __syncthreads();
  for (int i = tid; i < total; i += kThreads) {
    const int src = from[i], dst = to[i];
    scores[dst] = scores[src];
    positions[dst] = token_of(src, positions[src]);
  }
  // rows: 16 lanes a row of K and of V, four moves in flight
  __bf16* const kv = a.caches[layer] + h * kHeadDim + 8 * (lane & 15);
  const int32_t* const bt = a.block_table + (long)b * a.bt_stride;
  auto row = [&](int slot) {
    const int page = min(max(bt[slot >> 4], 0), a.num_pages - 1);
    return kv + (long)page * kPageElems + (slot & 15) * kSlotElems;
  };
  constexpr int kGroups = kThreads / 16, kFlight = 4;
  for (int i0 = tid >> 4; i0 < total; i0 += kGroups * kFlight) {
    u32x4 x[kFlight][2];
#pragma unroll
    for (int f = 0; f < kFlight; ++f) {
      const __bf16* p = row(from[min(i0 + f * kGroups, total - 1)]);
      x[f][0] = *reinterpret_cast<const u32x4*>(p);
      x[f][1] = *reinterpret_cast<const u32x4*>(p + kHalfElems);
    }
#pragma unroll
    for (int f = 0; f < kFlight; ++f) {
      if (i0 + f * kGroups >= total) break;
      __bf16* p = row(to[i0 + f * kGroups]);
      *reinterpret_cast<u32x4*>(p) = x[f][0];
      *reinterpret_cast<u32x4*>(p + kHalfElems) = x[f][1];
    }
  }
  __syncthreads();                                           // scores and positions of the moved rows are read
  for (int s = m + tid; s < n; s += kThreads) {
    scores[s] = 0.f;
    positions[s] = -1;
  }
}

}  // namespace abkv

extern "C" {

int abkv_paged_prefill_scores(const void* q, long q_stride_tok, long q_stride_head, const void* kv_cache, int num_pages,
                              const int32_t* block_table, long block_table_stride, int table_width, const int32_t* q_start,
                              const int32_t* kv_start, int num_requests, int tile_keys, const float* lse, float* scores,
                              long scores_stride_req, long scores_stride_head, float scale, hipStream_t stream) {
  using namespace abkv;
  if (num_requests <= 0) return 0;
  if (q == nullptr || kv_cache == nullptr || block_table == nullptr || q_start == nullptr || kv_start == nullptr ||
      lse == nullptr || scores == nullptr || num_pages <= 0 || table_width <= 0 ||
      (tile_keys != kBN && tile_keys != 2 * kBN) || !row_strides_ok(q_stride_tok) || !score_head_stride_ok(q_stride_head) ||
      !softmax_scale_ok(scale))
    return (int)hipErrorInvalidValue;
  const long slots = std::min((long)table_width * kPage, 1L << 30);              // (tile numbers: 24 bits)
  for (int r = 0; r < num_requests; ++r)
    if (q_start[0] < 0 || q_start[r + 1] < q_start[r] || kv_start[r] < 0 ||
        (long)kv_start[r] + q_start[r + 1] - q_start[r] > slots)
      return (int)hipErrorInvalidValue;
  PromptScoreArgs a{};
  a.q = static_cast<const __bf16*>(q);
  a.q_st = q_stride_tok; a.q_sh = q_stride_head;
  a.kv = static_cast<const __bf16*>(kv_cache);
  a.num_pages = num_pages;
  a.bt_stride = block_table_stride;
  a.bt_width = table_width;
  a.lse = lse;
  a.s_sb = scores_stride_req; a.s_sh = scores_stride_head;
  a.scale_log2 = scale * 1.4426950408889634f;
  int count = 0;
  auto launch = [&]() -> hipError_t {
    const dim3 grid((unsigned)(count * kHeadsKV)), block(64 * kScoreWaves);
    count = 0;
    if (grid.x == 0) return hipSuccess;
    if (tile_keys == kBN) hipLaunchKernelGGL(prompt_scores_kernel<1>, grid, block, 0, stream, a);
    else hipLaunchKernelGGL(prompt_scores_kernel<2>, grid, block, 0, stream, a);
    return hipGetLastError();
  };
  for (int first = 0; first < num_requests; first += kScoreRequests) {
    const int n = std::min(num_requests - first, kScoreRequests);
    const int32_t* qs = q_start + first;
    const int32_t* ks = kv_start + first;
    a.block_table = block_table + (long)first * block_table_stride;
    a.scores = scores + (long)first * scores_stride_req;
    int most = 0, next[kScoreRequests] = {};
    for (int r = 0; r < n; ++r) {
      a.q_start[r] = qs[r];
      a.kv_start[r] = ks[r];
      most = std::max(most, qs[r + 1] - qs[r]);
    }
    a.q_start[n] = qs[n];
    // the tiles that most queries see first, to within a tile's keys: workgroups that start last are short
    for (long level = most; level > 0; level -= tile_keys)
      for (int r = 0; r < n; ++r) {
        const int rows = qs[r + 1] - qs[r];
        for (;; ++next[r]) {
          const long k0 = (long)next[r] * tile_keys;
          if (rows == 0 || k0 >= (long)ks[r] + rows || rows - std::max(k0 - ks[r], 0L) <= level - tile_keys) break;
          a.tiles[count++] = (uint32_t)r << 24 | (uint32_t)next[r];
          if (count < kScoreTiles) continue;
          const hipError_t err = launch();
          if (err != hipSuccess) return (int)err;
        }
      }
    const hipError_t err = launch();
    if (err != hipSuccess) return (int)err;
  }
  return 0;
}

size_t abkv_kv_evict_workspace_size(int num_layers, int num_seqs, int max_pages_per_seq) {
  if (num_layers <= 0 || num_seqs <= 0 || max_pages_per_seq <= 0) return 0;
  const size_t rows = (size_t)max_pages_per_seq * abkv::kPage;
  return rows <= 32768 ? 0 : (size_t)num_layers * num_seqs * abkv::kHeadsKV * rows * sizeof(uint32_t);
}

int abkv_kv_evict(void* const* layer_caches, int num_layers, int num_pages, const int32_t* block_table,
                  long block_table_stride, const int32_t* seq_lens, int num_seqs, int max_pages_per_seq, float* scores,
                  int32_t* positions, long rows_stride, const int32_t* num_tokens, int budget, int sinks, int recent,
                  int32_t* out_lens, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  using namespace abkv;
  if (num_seqs <= 0 || num_layers <= 0) return 0;
  if (num_layers > 16 || layer_caches == nullptr || block_table == nullptr || seq_lens == nullptr || scores == nullptr ||
      positions == nullptr || num_tokens == nullptr || out_lens == nullptr || num_pages <= 0 || max_pages_per_seq <= 0 ||
      max_pages_per_seq > kEvictMaxRows / kPage || block_table_stride < max_pages_per_seq || budget <= 0 || sinks < 0 ||
      recent < 0 || (long)sinks + recent > budget || rows_stride < (long)max_pages_per_seq * kPage)
    return (int)hipErrorInvalidValue;
  const size_t need = abkv_kv_evict_workspace_size(num_layers, num_seqs, max_pages_per_seq);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) return (int)hipErrorInvalidValue;
  const long grid = (long)num_layers * num_seqs * kHeadsKV;
  if (grid * 1024 > 0xFFFFFFFFL) return (int)hipErrorInvalidValue;
  EvictArgs a{};
  for (int l = 0; l < num_layers; ++l) {
    if (layer_caches[l] == nullptr) return (int)hipErrorInvalidValue;
    a.caches[l] = static_cast<__bf16*>(layer_caches[l]);
  }
  a.num_pages = num_pages;
  a.block_table = block_table;
  a.bt_stride = block_table_stride;
  a.seq_lens = seq_lens;
  a.max_rows = max_pages_per_seq * kPage;
  a.scores = scores;
  a.positions = positions;
  a.rows_stride = rows_stride;
  a.tokens = num_tokens;
  a.batch = num_seqs;
  a.budget = budget;
  a.sinks = sinks;
  a.recent = recent;
  a.out_lens = out_lens;
  a.work = static_cast<uint32_t*>(workspace);
  // 16 waves end a launch that fills the GPU once soonest; more workgroups a CU overlap one's selection with another's moves. us
  // with 16 / 8 / 4 waves (six layers): 1 sequence of 2560 rows 15.5 / 17.8 / 23.4, 8 29.7 / 32.3 / 38.3, 64 227 / 218 / 228; 64
  // of 600 rows 82 / 65 / 59. Above 4096 rows LDS holds one workgroup a CU.
  const dim3 g((unsigned)grid);
  if (a.max_rows <= 1024 && grid >= 1024) hipLaunchKernelGGL((evict_kernel<1024, 4>), g, dim3(256), 0, stream, a);
  else if (a.max_rows <= 4096 && grid >= 1024) hipLaunchKernelGGL((evict_kernel<4096, 8>), g, dim3(512), 0, stream, a);
  else if (a.max_rows <= 4096) hipLaunchKernelGGL((evict_kernel<4096, 16>), g, dim3(1024), 0, stream, a);
  else if (a.max_rows <= 32768) hipLaunchKernelGGL((evict_kernel<32768, 16>), g, dim3(1024), 0, stream, a);
  else hipLaunchKernelGGL((evict_kernel<0, 16>), g, dim3(1024), 0, stream, a);
  return (int)hipGetLastError();
}

}  // extern "C"

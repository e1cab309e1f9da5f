// What a cache bounded by weight needs beside its attention (gfx950): the attention weights of a prompt's queries added up
// per cached row, and the eviction of the rows that weigh least. (A decode step's weights: decode_attn.hip.)
#include "common.h"

namespace abkv {

// ---------------------------------------------------------------------------------------------------------------------
// scores[r][KV head h][key j] += sum over h's four query heads u and the request's queries i >= j of
//                                exp(scale q_iu . k_jh - lse_iu),      query i at position kv_start[r] + i.
// A workgroup takes 64 keys of a KV head, a wave one of the four query heads (kPhases waves take its query rows in turn).
// The wave keeps its 64 keys in registers as the MFMA's first operand (64 VGPRs), so a 16-row query operand, loaded from
// global memory straight into operand registers, feeds 16 MFMAs: no LDS, no barrier in the loop. S^T = K . Q^T has a query
// per lane column, so lse is one value a lane and the sums over queries stay in the 16 accumulator positions until the end.
// One owner per score: no atomics, the same bits every time. Bound by the exponentials: per 16 x 64 pairs 256 cycles of
// v_exp_f32 and 128 of FMAs and adds beside 256 of MFMA.
struct PromptScoreArgs {
  const __bf16* q;  long q_st, q_sh;           // [T, 32, 128]
  const __bf16* kv; int num_pages;             // [pages, 2, 16, 8, 128]
  const int32_t* block_table; long bt_stride; int bt_width;
  const int32_t* q_start;                      // [R + 1]
  const int32_t* kv_start;                     // [R]
  const int32_t* tile_req;                     // [tiles] request of each 64-key tile
  const int32_t* tile_k0;                      // [tiles] its first key
  const float* lse;                            // [T, 32] natural log
  float* scores;  long s_sb, s_sh;             // [R, 8, rows]
  float scale_log2;
};

constexpr int kScorePhases = 2;
__global__ __launch_bounds__(256 * kScorePhases) void prompt_scores_kernel(PromptScoreArgs a) {
  __shared__ float sums[4 * kScorePhases][kBN];
  const int kvh = blockIdx.x % kHeadsKV, tile = blockIdx.x / kHeadsKV;
  const int r = a.tile_req[tile], k0 = a.tile_k0[tile];
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, m16 = lane & 15, j = lane >> 4;
  const int t0 = a.q_start[r], nq = a.q_start[r + 1] - t0, kv0 = a.kv_start[r];
  const int n_keys = kv0 + nq;
  const int head = kvh * kGroup + (w & 3);

  bf16x8 kop[4][4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int key = k0 + 16 * t + m16;
    const int pg = min((k0 >> 4) + t, a.bt_width - 1);
    const int page = min(max(a.block_table[(long)r * a.bt_stride + pg], 0), a.num_pages - 1);
    const __bf16* row = a.kv + (long)page * kPageElems + m16 * kSlotElems + kvh * kHeadDim;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u32x4 x = *reinterpret_cast<const u32x4*>(row + 8 * (4 * i + j));
      if (key >= n_keys) x = u32x4{0, 0, 0, 0};              // stale bytes
      kop[t][i] = __builtin_bit_cast(bf16x8, x);
    }
  }
  floatx4 sum[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) sum[t] = floatx4{0.f, 0.f, 0.f, 0.f};

  const int steps = (nq + 15) >> 4;
  const int first = (max(k0 - kv0, 0) >> 4) + (w >> 2);      // the first query rows that see a key of the tile
  const __bf16* qh = a.q + (long)head * a.q_sh + 8 * j;
  u32x4 qn[4];
  float ln = 0.f;
  auto load = [&](int step) {
    const int tok = t0 + min(16 * step + m16, nq - 1);
    const __bf16* p = qh + (long)tok * a.q_st;
#pragma unroll
    for (int i = 0; i < 4; ++i) qn[i] = *reinterpret_cast<const u32x4*>(p + 32 * i);
    ln = a.lse[(long)tok * kHeadsQ + head];
  };
  if (first < steps) load(first);
  for (int step = first; step < steps; step += kScorePhases) {
    bf16x8 qop[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) qop[i] = __builtin_bit_cast(bf16x8, qn[i]);
    const int qi = 16 * step + m16;
    // rows past the request and rows that see nothing weigh 0
    const float l2 = qi < nq && ln > -INFINITY ? ln * 1.4426950408889634f : INFINITY;
    if (step + kScorePhases < steps) load(step + kScorePhases);
    floatx4 s[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) s[t] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int t = 0; t < 4; ++t) s[t] = mfma16x16x32(kop[t][i], qop[i], s[t]);
    const int before = kv0 + qi - k0;                        // keys 0 .. before of the tile are seen
    if (kv0 + 16 * step >= k0 + kBN - 1) {                   // (uniform) all of them by all rows
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[t][e] += fast_exp2(fmaf(s[t][e], a.scale_log2, -l2));
    } else {
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p = fast_exp2(fmaf(s[t][e], a.scale_log2, -l2));
          sum[t][e] += 16 * t + 4 * j + e <= before ? p : 0.f;
        }
    }
  }
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float x = sum[t][e];
#pragma unroll
      for (int m = 1; m < 16; m <<= 1) x += __shfl_xor(x, m, 64);
      if (m16 == 0) sums[w][16 * t + 4 * j + e] = x;
    }
  __syncthreads();
  const int key = k0 + threadIdx.x;
  if (threadIdx.x < kBN && key < n_keys) {
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < 4 * kScorePhases; ++i) x += sums[i][threadIdx.x];
    a.scores[(long)r * a.s_sb + (long)kvh * a.s_sh + key] += x;
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// Eviction. Per (layer, sequence, KV head): of n rows the best m = min(n, budget) are kept: rows of the first `sinks` and of
// the last `recent` tokens, then by score (ties: lowest slot; NaN below every number). Kept rows of slots >= m move into the
// evicted slots < m, both in ascending order, so a pass moves no more rows than it evicts and sources and destinations never
// meet: attention does not depend on the order of rows, and the tokens' indices travel in `positions`.
//
// One workgroup of 16 waves per (layer, sequence, head) does it all: keys that order as (held, score) in LDS; the m-th
// largest by four 8-bit digits of a histogram; each wave walks its own run of slots, so ranks among ties, holes and movers
// are ballot counts plus one prefix over 16 waves; then rows, scores and positions move. Bound by the latency of these
// phases for one sequence, by the moved rows for a batch.
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

constexpr int kEvictWaves = 16;
constexpr int kEvictMaxRows = 1 << 18;         // rows whose kept bits fit LDS beside the rest

template <int kSlots>
__global__ __launch_bounds__(64 * kEvictWaves) void evict_kernel(EvictArgs a) {
  constexpr int kThreads = 64 * kEvictWaves;
  constexpr int kCopies = 8;                                 // of the histogram: most scores share their first digit
  __shared__ uint32_t lds_keys[kSlots > 0 ? kSlots : 1];
  __shared__ uint64_t kept_bits[(kSlots > 0 ? kSlots : kEvictMaxRows) / 64];
  __shared__ uint32_t hist[256 * kCopies];
  __shared__ int counts[kEvictWaves][2];
  __shared__ uint32_t pick[2];
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
      }
    }
    __syncthreads();
    prefix |= pick[0] << shift;
    mask |= 255u << shift;
    want = pick[1];
  }
  // kept: keys above the prefix, and the first `want` that equal it
  int ties = 0;
  for (int s = s0 + lane; s - lane < s1; s += 64) ties += __popcll(__ballot(s < s1 && keys[min(s, n - 1)] == prefix));
  if (lane == 0) counts[w][0] = ties;
  __syncthreads();
  int rank = 0;
  for (int i = 0; i < w; ++i) rank += counts[i][0];
  __syncthreads();
  const uint64_t below = (1ull << lane) - 1;
  int holes = 0, movers = 0;
  for (int s = s0 + lane; s - lane < s1; s += 64) {
    const uint32_t k = keys[min(s, n - 1)];
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
  for (int i = 0; i < kEvictWaves; ++i) {
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
                              const int32_t* kv_start, const int32_t* tile_req, const int32_t* tile_k0, int num_tiles,
                              const float* lse, float* scores, long scores_stride_req, long scores_stride_head, float scale,
                              hipStream_t stream) {
  using namespace abkv;
  if (num_tiles <= 0) return 0;
  if (q == nullptr || kv_cache == nullptr || block_table == nullptr || q_start == nullptr || kv_start == nullptr ||
      tile_req == nullptr || tile_k0 == nullptr || lse == nullptr || scores == nullptr || num_pages <= 0 || table_width <= 0)
    return (int)hipErrorInvalidValue;
  const PromptScoreArgs a{static_cast<const __bf16*>(q), q_stride_tok, q_stride_head, static_cast<const __bf16*>(kv_cache),
                          num_pages, block_table, block_table_stride, table_width, q_start, kv_start, tile_req, tile_k0, lse,
                          scores, scores_stride_req, scores_stride_head, scale * 1.4426950408889634f};
  const long grid = (long)num_tiles * kHeadsKV;
  if (grid * 256 * kScorePhases > 0xFFFFFFFFL) return (int)hipErrorInvalidValue;
  hipLaunchKernelGGL(prompt_scores_kernel, dim3((unsigned)grid), dim3(256 * kScorePhases), 0, stream, a);
  return (int)hipGetLastError();
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
  if (grid * 64 * kEvictWaves > 0xFFFFFFFFL) return (int)hipErrorInvalidValue;
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
  // by the LDS the keys take: two workgroups a CU up to 4096 rows (their 32 waves), one above
  const dim3 g((unsigned)grid), t(64 * kEvictWaves);
  if (a.max_rows <= 4096) hipLaunchKernelGGL(evict_kernel<4096>, g, t, 0, stream, a);
  else if (a.max_rows <= 32768) hipLaunchKernelGGL(evict_kernel<32768>, g, t, 0, stream, a);
  else hipLaunchKernelGGL(evict_kernel<0>, g, t, 0, stream, a);
  return (int)hipGetLastError();
}

}  // extern "C"

// Attention under a sliding window with sinks (gfx950): whole prompts and prompt chunks over the paged cache.
//
//   row i sees key j when j <= i and (i - j < window or j < sinks), both inside the sequence;
//   out_i = sum_j softmax_j(scale q_i . k_j) v_j, rows that see nothing (padding) are 0 with lse -inf.
//
// The mask is evaluated from (window, sinks, the sequence's length): a query tile of 64 rows walks the tiles of the sinks,
// then the ceil((window + 63) / 64) (+ 1) tiles its rows' windows reach, and only tiles on an edge of a range are masked
// per element. The work of a row is bounded by the window, not by its position.
//
// A workgroup of 4 waves takes a query tile of two of a KV head's four query heads, a wave 16 rows x 2 heads (tiles and softmax
// as the compression mask's, attn_tile.h). Query rows and outputs are most of the bytes under a short window, and workgroups
// of one length all load, compute and store at the same times: two of them share a CU (two buffers each of K and V, 80 KiB), so
// that one's loads and stores run beside the other's products. Against one workgroup of 8 waves for all four heads, three
// buffers each, us a call of two sequences of 4096 rows under windows of 64 / 128 / 512 / 1024: 58 / 66 / 105 / 156 -> 48 / 57 /
// 99 / 147 (copies of the query rows and outputs alone: 27). Outputs in whole 64-byte runs (store_acc_rows) before it 66 / 73 /
// 112 / 160 -> 58 / 66 / 105 / 156. Long windows (8192 and 5000 rows, window
// 1024): matrix units 41 % of the SIMDs' cycles, other vector work 35 %, 10 % both at once; the waves are ready but not issued
// 37 % of their time and wait 26 %.
#include <algorithm>

#include "window_tile.h"

namespace abkv {

// Prompt chunks: request r's queries are rows q_start[r] .. q_start[r + 1] - 1 at positions kv_start[r] + i. The requests
// come with the launch's arguments (uploaded before it, four chunks of up to 512 cost 54 us a call, this 47.5), and a
// workgroup finds its own by bisection.
constexpr int kChunks = 64;                    // requests of a launch
struct ChunkArgs {
  static constexpr bool kPaged = true;
  const __bf16* kv; int num_pages;             // [pages, 2, 16, 8, 128]
  const int32_t* block_table; long bt_stride; int bt_width;      // (of the launch's first request)
  int requests;
  int32_t tile_start[kChunks], q_start[kChunks + 1], kv_start[kChunks];
};
struct DenseArgs {
  static constexpr bool kPaged = false;
};

// kLse: the call wants lse. The output is divided by the sum of its rounded weights, but lse takes the unrounded ones, up to 2^8
// under the running maximum's headroom: rounded, a few heavy keys would leave it up to 2^-8 off however many rows are visible
// (600 rows, one key 6 log2 units above the others: 2.3e-3, this 2e-6). The additions cost 4 % (two sequences of 8192 and 5000
// rows, window 1024: 244 -> 253 us), so calls without lse leave them out.
template <class Chunks, bool kLse>
__global__ __launch_bounds__(256, 2) void window_attn_kernel(WindowArgs a, Chunks c) {
  constexpr bool kPaged = Chunks::kPaged;
  constexpr int H = 2, kWaves = 4;
  __shared__ __attribute__((aligned(16))) __bf16 K0[kTileElems], K1[kTileElems], V0[kTileElems], V1[kTileElems];
  __shared__ __attribute__((aligned(16))) __bf16 Ks[kTileElems];           // the sinks, where they are few
  __bf16* const Kbuf[2] = {K0, K1};
  __bf16* const Vbuf[2] = {V0, V1};
  // KV head fastest: workgroups go to the 8 XCDs round-robin, so one XCD's L2 serves a head's rows to all its tiles. Then
  // the pair of heads and the query tile, the sequence last: with the sequence before them, a padded batch of two gives
  // every other workgroup little to do, and the dispatch, in turn over an XCD's parts as well, leaves half of them idle
  // (8192 and 5000 rows, window 1024: 321 us, this order 280, both with 8 waves).
  const int kvh = blockIdx.x % kHeadsKV;
  const int tile = blockIdx.x / (2 * kHeadsKV);
  int b, q0, kv0 = 0, t0 = 0, n, n_q;                        // n: keys; n_q: query rows of the sequence
  if constexpr (kPaged) {
    int end = c.requests;                                    // the last request whose tiles begin at or before this one
    for (b = 0; end - b > 1;) {
      const int mid = (b + end) / 2;
      if (c.tile_start[mid] <= tile) b = mid;
      else end = mid;
    }
    q0 = (tile - c.tile_start[b]) * kBM;
    t0 = c.q_start[b];
    n_q = c.q_start[b + 1] - t0;
    kv0 = c.kv_start[b];
    n = kv0 + n_q;
  } else {
    b = tile / a.num_q_tiles;
    q0 = (a.num_q_tiles - 1 - tile % a.num_q_tiles) * kBM;   // later (costlier) rows first
    n = n_q = window_rows(a, b);
  }
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int m16 = lane & 15, j = lane >> 4;
  const int hbase = H * (blockIdx.x / kHeadsKV & 1);         // first of the workgroup's heads in the GQA group
  const int qi = q0 + 16 * w + m16;                          // this lane's query row (MFMA column)
  const bool seen = qi < n_q;

  // (rows past the sequence: its last one, not stored)
  const long q_row = (kPaged ? (long)t0 * a.q_ss : (long)b * a.q_sb) + (long)min(qi, max(n_q - 1, 0)) * a.q_ss;
  bf16x8 qop[H][4];
#pragma unroll
  for (int u = 0; u < H; ++u)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __bf16* x = a.q + q_row + (long)(kvh * kGroup + hbase + u) * a.q_sh + 8 * (4 * i + j);
      qop[u][i] = __builtin_bit_cast(bf16x8, ld16g(x));
    }
  floatx4 o[8][H];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int u = 0; u < H; ++u) o[i][u] = floatx4{0.f, 0.f, 0.f, 0.f};
  float m_run[H], l_run[H], exact[H];
#pragma unroll
  for (int u = 0; u < H; ++u) {
    m_run[u] = -INFINITY;
    l_run[u] = exact[u] = 0.f;
  }
  if (q0 < n_q) {                                            // (uniform)
    const bool few = short_sinks(kv0 + q0, a.window, a.sinks);
    const int sinks = few ? 0 : a.sinks;                     // the walk's
    WindowWalk walk(kv0 + q0, kv0 + min(q0 + kBM, n_q) - 1, a.window, sinks);
    const WindowLane lm(kv0 + qi, seen, a.window, sinks);
    float m0[H], l0[H];                                      // the sinks' own
    auto attend = [&](const auto& rows) {
      if (few) issue_sinks(rows, n, Ks, w, lane);
      start_pair<kWaves>(rows, walk, n, Kbuf, Vbuf, w, lane);
      if (few) {
        __asm__ volatile("s_waitcnt vmcnt(12)" ::: "memory");    // (all but the first tiles')
        __builtin_amdgcn_s_barrier();
        attend_sinks<H, kLse>(Ks, a.sinks, qop, o, m_run, l0, exact, a.scale_log2, lane);
#pragma unroll
        for (int u = 0; u < H; ++u) m0[u] = m_run[u];
      }
      attend_pair<H, kWaves, kLse>(rows, walk, n, Kbuf, Vbuf, qop, o, m_run, l_run, exact, lm, a.scale_log2, w, lane);
#pragma unroll
      for (int u = 0; u < H; ++u)
        if (few) l_run[u] += l0[u] * fast_exp2(m0[u] - m_run[u]);
    };
    if constexpr (kPaged)
      attend(PagedWindowRows{{c.kv + kvh * kHeadDim, c.block_table + (long)b * c.bt_stride, c.bt_width, c.num_pages},
                             max(kv0 + q0 + 1 - a.window, 0), a.sinks});
    else
      attend(DenseRows<false>{a.k + (long)b * a.k_sb + (long)kvh * a.k_sh, a.v + (long)b * a.v_sb + (long)kvh * a.v_sh,
                              a.k_ss, a.v_ss});
  }
  if constexpr (kLse) {
#pragma unroll
    for (int u = 0; u < H; ++u) exact[u] = sum_xor32(sum_xor16(exact[u]));      // (before lanes leave)
  }
  if (qi >= (kPaged ? n_q : a.S)) return;
  const long o_row = kPaged ? (long)(t0 + qi) * a.o_ss : (long)b * a.o_sb + (long)qi * a.o_ss;
#pragma unroll
  for (int u = 0; u < H; ++u) {
    // padding rows (with o and l of unmasked tiles): 0, lse -inf. A row that sees keys has l > 0, or NaN scores.
    const float l = seen ? l_run[u] : 0.f;
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int head = kvh * kGroup + hbase + u;
    if (!seen)
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e][u] = floatx4{0.f, 0.f, 0.f, 0.f};
    store_acc_rows<H>(a.out + o_row + (long)head * a.o_sh, o, u, j, inv);
    if constexpr (!kPaged)
      if (a.low != nullptr) store_low<H>(a.low + (((long)b * a.S + qi) * kHeadsQ + head) * kHeadDim, o, u, j, inv);
    if (kLse && j == 0)
      a.lse[kPaged ? (long)(t0 + qi) * kHeadsQ + head : ((long)b * kHeadsQ + head) * a.S + qi] =
          l == 0.f ? -INFINITY : (m_run[u] + __log2f(exact[u])) * 0.69314718055994531f;
  }
}

}  // namespace abkv

extern "C" {

int abkv_window_attn(const void* q, long q_stride_b, long q_stride_s, long q_stride_h, const void* k, long k_stride_b,
                     long k_stride_s, long k_stride_h, const void* v, long v_stride_b, long v_stride_s, long v_stride_h,
                     int batch, int seq_len, const int32_t* seq_lens, int window, int sinks, float scale, void* out,
                     long out_stride_b, long out_stride_s, long out_stride_h, float* lse, void* out_low,
                     hipStream_t stream) {
  using namespace abkv;
  if (batch <= 0 || seq_len <= 0) return 0;
  if (q == nullptr || k == nullptr || v == nullptr || out == nullptr || window <= 0 || sinks < 0 ||
      !softmax_scale_ok(scale) || !row_strides_ok(q_stride_s, k_stride_s, v_stride_s))
    return (int)hipErrorInvalidValue;
  WindowArgs a;
  a.q = static_cast<const __bf16*>(q);
  a.q_sb = q_stride_b; a.q_ss = q_stride_s; a.q_sh = q_stride_h;
  a.k = static_cast<const __bf16*>(k);
  a.k_sb = k_stride_b; a.k_ss = k_stride_s; a.k_sh = k_stride_h;
  a.v = static_cast<const __bf16*>(v);
  a.v_sb = v_stride_b; a.v_ss = v_stride_s; a.v_sh = v_stride_h;
  a.B = batch;
  a.S = seq_len;
  a.seq_lens = seq_lens;
  a.window = window;
  a.sinks = sinks;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.out = static_cast<__bf16*>(out);
  a.o_sb = out_stride_b; a.o_ss = out_stride_s; a.o_sh = out_stride_h;
  a.lse = lse;
  a.low = static_cast<uint8_t*>(out_low);
  a.num_q_tiles = (seq_len - 1) / kBM + 1;
  const long grid = 2L * a.num_q_tiles * batch * kHeadsKV;
  if (grid * 256 > 0xFFFFFFFFL) return (int)hipErrorInvalidValue;
  const auto kernel = lse != nullptr ? window_attn_kernel<DenseArgs, true> : window_attn_kernel<DenseArgs, false>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(256), 0, stream, a, DenseArgs{});
  return (int)hipGetLastError();
}

int abkv_paged_prefill_attn_window(const void* q, long q_stride_tok, long q_stride_head, const void* kv_cache,
                                   int num_pages, const int32_t* block_table, long block_table_stride, int table_width,
                                   const int32_t* q_start, const int32_t* kv_start, int num_requests, int window, int sinks,
                                   float scale, void* out, long out_stride_tok, long out_stride_head, float* lse,
                                   hipStream_t stream) {
  using namespace abkv;
  if (num_requests <= 0) return 0;
  if (q == nullptr || kv_cache == nullptr || block_table == nullptr || q_start == nullptr || kv_start == nullptr ||
      out == nullptr || num_pages <= 0 || table_width <= 0 || window <= 0 || sinks < 0 || !softmax_scale_ok(scale) ||
      !row_strides_ok(q_stride_tok))
    return (int)hipErrorInvalidValue;
  const long slots = std::min((long)table_width * kPage, 1L << 30);              // (positions and their counts: 32 bits)
  for (int r = 0; r < num_requests; ++r)
    if (q_start[0] < 0 || q_start[r + 1] < q_start[r] || kv_start[r] < 0 ||
        (long)kv_start[r] + q_start[r + 1] - q_start[r] > slots)
      return (int)hipErrorInvalidValue;
  WindowArgs a{};
  a.q = static_cast<const __bf16*>(q);
  a.q_ss = q_stride_tok; a.q_sh = q_stride_head;
  a.window = window;
  a.sinks = sinks;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.out = static_cast<__bf16*>(out);
  a.o_ss = out_stride_tok; a.o_sh = out_stride_head;
  a.lse = lse;
  ChunkArgs c{};
  c.kv = static_cast<const __bf16*>(kv_cache);
  c.num_pages = num_pages;
  c.bt_stride = block_table_stride;
  c.bt_width = table_width;
  for (int first = 0; first < num_requests; first += kChunks) {
    c.block_table = block_table + (long)first * block_table_stride;
    c.requests = num_requests - first < kChunks ? num_requests - first : kChunks;
    long tiles = 0;
    for (int r = 0; r < c.requests; ++r) {
      c.tile_start[r] = (int32_t)tiles;
      c.q_start[r] = q_start[first + r];
      c.kv_start[r] = kv_start[first + r];
      tiles += ((long)q_start[first + r + 1] - q_start[first + r] + kBM - 1) / kBM;
    }
    c.q_start[c.requests] = q_start[first + c.requests];
    const long grid = 2 * tiles * kHeadsKV;
    if (grid * 256 > 0xFFFFFFFFL) return (int)hipErrorInvalidValue;
    if (grid == 0) continue;
    const auto kernel = lse != nullptr ? window_attn_kernel<ChunkArgs, true> : window_attn_kernel<ChunkArgs, false>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(256), 0, stream, a, c);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return (int)err;
  }
  return 0;
}

}  // extern "C"

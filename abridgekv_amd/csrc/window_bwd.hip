// Backward of attention under a sliding window with sinks (gfx950): dq, dk, dv from the forward's output and lse, as
// prefill_bwd.hip: P = exp2(S * scale * log2(e) - lse * log2(e)), dS = P o (dP - rowsum(dO o O)), dQ = scale * dS K,
// dK = scale * dS^T Q, dV = P^T dO, dK and dV summed over the KV head's four query heads.
//   window_bwd_dq_kernel    the forward's query tiles and key walk; dQ^T += K^T dS^T. Before it, each (row, query head)'s
//                           lse2 = lse * log2(e) and D = sum_d dO * O (O with the low part that its rounding left off,
//                           where the caller has it), which it leaves for the next kernel in rows padded to
//                           whole tiles (lse2 = +inf and D = 0 past the sequence, so that padding weighs 0)
//   window_bwd_dkv_kernel   a workgroup per 64 keys of a KV head over the query tiles whose windows reach them: the same
//                           count for every key tile. Keys among the sinks are seen by every later row as well: these far
//                           query tiles are cut into parts with workgroups of their own (SinkPlan), which leave fp32 sums
//                           in slots, and the last part of a tile to finish adds them up in part order. (Very many sink
//                           tiles: no parts.)
#include "bwd_tile.h"
#include "window_tile.h"

namespace abkv {

struct WindowBwdArgs {
  WindowArgs f;                               // q, k, v, geometry, scale_log2
  const __bf16* o;    long o_sb, o_ss, o_sh;  // forward output [B, S, 32, 128]
  const __bf16* dout; long g_sb, g_ss, g_sh;  // its gradient
  const float* lse;                           // [B, 32, S] natural log, from the forward
  float* lse2;                                // workspace [B, 32, Sp]
  float* dvec;                                // workspace [B, 32, Sp]
  int Sp;                                     // S rounded up to a multiple of 64
  int* done;                                  // [sink tiles x B x 8] finished parts
  float* slots;                               // [sink tiles x B][parts + 1][8][kSlotFloats]
  SinkPlan plan;
  float scale;
  __bf16* dq; long dq_sb, dq_ss, dq_sh;       // [B, S, 32, 128]
  __bf16* dk; long dk_sb, dk_ss, dk_sh;       // [B, S, 8, 128]
  __bf16* dv; long dv_sb, dv_ss, dv_sh;
};

constexpr int kWinSlotFloats = 2 * kBN * kHeadDim;          // dK and dV of a key tile, of one KV head

__global__ __launch_bounds__(512, 1) void window_bwd_dq_kernel(WindowBwdArgs a) {
  constexpr int H = 2, kWaves = 8;
  __shared__ __attribute__((aligned(16))) __bf16 K0[kTileElems], K1[kTileElems], V0[kTileElems], V1[kTileElems];
  __bf16* const Kb[2] = {K0, K1};
  __bf16* const Vb[2] = {V0, V1};
  const WindowArgs& f = a.f;
  const int kvh = blockIdx.x % kHeadsKV;
  const int tile = blockIdx.x / kHeadsKV;
  const int b = tile / f.num_q_tiles;                        // the forward's order
  const int q0 = (f.num_q_tiles - 1 - tile % f.num_q_tiles) * kBM;
  const int n = window_rows(f, b);
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int m16 = lane & 15, j = lane >> 4;
  const int hbase = H * (w & 1);
  const int qrow = q0 + 16 * (w >> 1) + m16;
  const bool seen = qrow < n;
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < a.plan.sink_tiles * f.B * kHeadsKV; i += 512) a.done[i] = 0;
  const DenseRows<false> rows{f.k + (long)b * f.k_sb + (long)kvh * f.k_sh, f.v + (long)b * f.v_sb + (long)kvh * f.v_sh,
                              f.k_ss, f.v_ss};
  WindowWalk walk(q0, min(q0 + kBM, n) - 1, f.window, f.sinks);
  int tc = 0;
  TileMask mc;
  const bool any = q0 < n && walk.next(tc, mc, true);        // (uniform)
  if (any) {                                                 // the first tile comes in beside the rows
    const auto s0 = rows.template src<2>(tc, w, n);
    issue_half<kWaves, false>(rows, s0, n, Kb[0], w, lane);
    issue_half<kWaves, true>(rows, s0, n, Vb[0], w, lane);
  }
  uint2 t[H][4] = {};                                        // what the rounding of O left off, if the caller has it
  if (f.low != nullptr) {
    const uint8_t* lp = f.low + (((long)b * f.S + min(qrow, f.S - 1)) * kHeadsQ + kvh * kGroup + hbase) * kHeadDim + 8 * j;
#pragma unroll
    for (int u = 0; u < H; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) t[u][i] = *reinterpret_cast<const uint2*>(lp + u * kHeadDim + 32 * i);
  }
  bf16x8 qop[H][4], gop[H][4];
  float l2[H], dd[H];
#pragma unroll
  for (int u = 0; u < H; ++u) {
    const int head = kvh * kGroup + hbase + u, r = min(qrow, f.S - 1);
    const __bf16* qp = f.q + (long)b * f.q_sb + (long)r * f.q_ss + (long)head * f.q_sh;
    const __bf16* gp = a.dout + (long)b * a.g_sb + (long)r * a.g_ss + (long)head * a.g_sh;
    const __bf16* op = a.o + (long)b * a.o_sb + (long)r * a.o_ss + (long)head * a.o_sh;
    float d = 0.f;                                           // dims 8 * (4i + j) .. + 7 of the row's dot product
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      u32x4 x = ld16g(qp + 8 * (4 * i + j)), y = ld16g(gp + 8 * (4 * i + j)), z = ld16g(op + 8 * (4 * i + j));
      if (!seen) x = y = z = u32x4{0, 0, 0, 0};
      qop[u][i] = __builtin_bit_cast(bf16x8, x);
      gop[u][i] = __builtin_bit_cast(bf16x8, y);
#pragma unroll
      for (int e = 0; e < 4; ++e) d += bf16_lo(y[e]) * bf16_lo(z[e]) + bf16_hi(y[e]) * bf16_hi(z[e]);
    }
    dd[u] = d;
    l2[u] = seen ? a.lse[((long)b * kHeadsQ + head) * f.S + r] * 1.4426950408889634f : INFINITY;
  }
  if (f.low != nullptr) {
#pragma unroll
    for (int u = 0; u < H; ++u) {
      float d = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const u32x4 y = __builtin_bit_cast(u32x4, gop[u][i]);
        const floatx4 t0 = load_low(t[u][i].x), t1 = load_low(t[u][i].y);
#pragma unroll
        for (int e = 0; e < 2; ++e)
          d += bf16_lo(y[e]) * t0[2 * e] + bf16_hi(y[e]) * t0[2 * e + 1] + bf16_lo(y[2 + e]) * t1[2 * e] +
               bf16_hi(y[2 + e]) * t1[2 * e + 1];
      }
      dd[u] += seen ? d * (1.f / 256) : 0.f;
    }
  }
#pragma unroll
  for (int u = 0; u < H; ++u) {
    dd[u] = sum_xor32(sum_xor16(dd[u]));
    if (j == 0) {
      const long wi = ((long)b * kHeadsQ + kvh * kGroup + hbase + u) * a.Sp + qrow;      // qrow < Sp
      a.lse2[wi] = l2[u];
      a.dvec[wi] = dd[u];
    }
  }
  floatx4 dq[8][H];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int u = 0; u < H; ++u) dq[i][u] = floatx4{0.f, 0.f, 0.f, 0.f};

  const WindowLane lm(qrow, seen, f.window, f.sinks);
  if (any) {
    // Double buffer as the masked prefill's dQ: wait for tile i, issue tile i + 1 (or re-load tile i past the end) into
    // the other buffer, compute tile i.
    auto step = [&](auto buf_c) -> bool {
      constexpr int sl = decltype(buf_c)::value;
      int tn = tc;
      TileMask mn;
      const bool hn = walk.next(tn, mn, false);
      const auto src = rows.template src<2>(hn ? tn : tc, w, n);
      __asm__ volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      issue_half<kWaves, false>(rows, src, n, Kb[1 - sl], w, lane);
      issue_half<kWaves, true>(rows, src, n, Vb[1 - sl], w, lane);
      floatx4 s[2][2][H], dp[2][2][H];
      tile_scores<H>(Kb[sl], qop, s, m16, j);
      tile_scores<H>(Vb[sl], gop, dp, m16, j);
      tile_mask<H, WindowWalk>(s, tc, mc, lm, j);
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int u = 0; u < H; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float pr = fast_exp2(fmaf(s[kk][t][u][r], f.scale_log2, -l2[u]));
              s[kk][t][u][r] = pr * (dp[kk][t][u][r] - dd[u]);
            }
      bf16x8 dsop[2][H];
      pack_tile_op<H>(s, dsop);
      tile_acc<H>(Kb[sl], dsop, dq, lane);
      if (!hn) return false;
      tc = tn;
      mc = mn;
      return true;
    };
    for (;;) {
      if (!step(Buf<0>{})) break;
      if (!step(Buf<1>{})) break;
    }
    __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }
  if (qrow >= f.S) return;
#pragma unroll
  for (int u = 0; u < H; ++u) {
    __bf16* dp = a.dq + (long)b * a.dq_sb + (long)qrow * a.dq_ss + (long)(kvh * kGroup + hbase + u) * a.dq_sh;
    store_acc_rows<H>(dp, dq, u, j, seen ? a.scale : 0.f);
  }
}

__global__ __launch_bounds__(256, 2) void window_bwd_dkv_kernel(WindowBwdArgs a) {
  constexpr int kWaves = 4;
  __shared__ __attribute__((aligned(16))) __bf16 Q0[kTileElems], Q1[kTileElems], G0[kTileElems], G1[kTileElems];
  __shared__ __attribute__((aligned(16))) float L0[kBN], L1[kBN], E0[kBN], E1[kBN];
  __bf16* const Qb[2] = {Q0, Q1};
  __bf16* const Gb[2] = {G0, G1};
  float* const Lb[2] = {L0, L1};
  float* const Eb[2] = {E0, E1};
  const WindowArgs& f = a.f;
  const int kvh = blockIdx.x % kHeadsKV;
  const int i = blockIdx.x / kHeadsKV;
  // the far parts of all sequences' sink tiles, then each sequence's key tiles for their near query tiles. (Sequences last, as
  // in the forward; us a forward and backward against sequences first: two of 1000 and 4096 rows, window 512: 400 / 427, both
  // of 4096 509 / 499.)
  const int far_items = a.plan.sink_tiles * a.plan.parts, far_all = far_items * f.B;
  const bool far = i < far_all;
  const int b = far ? i % f.B : (i - far_all) / a.plan.tiles;
  const int kt = far ? i / f.B / a.plan.parts : (i - far_all) % a.plan.tiles;
  const int z = far ? 1 + i / f.B % a.plan.parts : 0;        // part of the key tile (0: near)
  const int n = window_rows(f, b);
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  const int m16 = lane & 15, j = lane >> 4;
  const int k0 = kt * kBN;
  const int key = k0 + 16 * w + m16;                         // this lane's column
  const bool in = key < n;

  floatx4 dk[8][1], dv[8][1];
#pragma unroll
  for (int e = 0; e < 8; ++e) dk[e][0] = dv[e][0] = floatx4{0.f, 0.f, 0.f, 0.f};

  const WindowSpan span(k0, n, f.window, f.sinks);
  int qt_first, qt_end;
  a.plan.range(span, z, qt_first, qt_end);
  // The near query tiles in cyclic order from a multiple of `reach`, their number for an inner key tile: the workgroups of
  // neighbouring key tiles, which run at one time, then take the same query tile at the same step, and its rows come from
  // their XCD's L2 (from its own first tile on, a workgroup reads what its neighbour read a step before, when the other 60 of
  // the XCD have passed 8 MB: four times the fetches). us a forward and backward, two of 4096 rows, window 512: 463 -> 450;
  // four, window 1024: 1346 -> 1307.
  const int reach = (min(f.window, f.S) + kBN - 2) / kBM + 1;
  int left = qt_end - qt_first, qt = (qt_first + reach - 1) / reach * reach;
  if (z > 0 || qt >= qt_end) qt = qt_first;
  // rows that see this lane's key: from the key on, `rows` of them (past the sequence: none)
  const unsigned rows = !in ? 0u : (unsigned)(key < f.sinks ? n - key : min(f.window, n - key));
  int h = -1;
  auto next_pair = [&]() -> bool {                           // (query tile, head) pairs, head fastest
    if (++h == kGroup) {
      h = 0;
      if (++qt == qt_end) qt = qt_first;
      --left;
    }
    return left > 0;
  };
  // Q / dO rows of (qt, head) as the tile rows, lse2 / D rows beside them (waves 0 and 1, 4 bytes per lane)
  auto issue = [&](int pq, int ph, int sl_dst) {
    const int head = kvh * kGroup + ph;
    const DenseRows<false> src_rows{f.q + (long)b * f.q_sb + (long)head * f.q_sh,
                                    a.dout + (long)b * a.g_sb + (long)head * a.g_sh, f.q_ss, a.g_ss};
    const auto src = src_rows.template src<4>(pq * kBN, w, n);
    issue_half<kWaves, false>(src_rows, src, n, Qb[sl_dst], w, lane);
    issue_half<kWaves, true>(src_rows, src, n, Gb[sl_dst], w, lane);
    const long wi = ((long)b * kHeadsQ + head) * a.Sp + pq * kBN + lane;
    if (w == 0) __builtin_amdgcn_global_load_lds((const void*)(a.lse2 + wi), ABKV_LDS(Lb[sl_dst]), 4, 0, 0);
    if (w == 1) __builtin_amdgcn_global_load_lds((const void*)(a.dvec + wi), ABKV_LDS(Eb[sl_dst]), 4, 0, 0);
  };
  const bool any = next_pair();
  if (any) issue(qt, h, 0);                                  // the first rows come in beside the keys
  bf16x8 kop[4], vop[4];
  {
    const int r = min(key, f.S - 1);
    const __bf16* kp = f.k + (long)b * f.k_sb + (long)r * f.k_ss + (long)kvh * f.k_sh;
    const __bf16* vp = f.v + (long)b * f.v_sb + (long)r * f.v_ss + (long)kvh * f.v_sh;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      u32x4 x = ld16g(kp + 8 * (4 * e + j)), y = ld16g(vp + 8 * (4 * e + j));
      if (!in) x = y = u32x4{0, 0, 0, 0};
      kop[e] = __builtin_bit_cast(bf16x8, x);
      vop[e] = __builtin_bit_cast(bf16x8, y);
    }
  }
  if (any) {
    auto step = [&](auto buf_c) -> bool {
      constexpr int sl = decltype(buf_c)::value;
      const int q0 = qt * kBM;
      const bool hn = next_pair();
      __asm__ volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      if (hn) issue(qt, h, 1 - sl);
      floatx4 s[2][2][1], dp[2][2][1];
      dkv_scores(Qb[sl], Gb[sl], kop, vop, s, dp, m16, j);
      // wave-uniform: all 64 rows see all 64 keys (the rows lie inside the sequence, and the keys before them)
      const bool whole = q0 >= k0 + kBN - 1 && q0 + kBM <= n && (k0 + kBN <= f.sinks || q0 + kBM - 1 - k0 < f.window);
      if (whole) {
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const int r0 = 32 * kk + 16 * t + 4 * j;
            const floatx4 l4 = *reinterpret_cast<const floatx4*>(Lb[sl] + r0);
            const floatx4 e4 = *reinterpret_cast<const floatx4*>(Eb[sl] + r0);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float pr = fast_exp2(fmaf(s[kk][t][0][r], f.scale_log2, -l4[r]));
              s[kk][t][0][r] = pr;
              dp[kk][t][0][r] = pr * (dp[kk][t][0][r] - e4[r]);
            }
          }
      } else {
        const int at = q0 - key;                             // the tile's first row from the key's own
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const int r0 = 32 * kk + 16 * t + 4 * j;
            const floatx4 l4 = *reinterpret_cast<const floatx4*>(Lb[sl] + r0);
            const floatx4 e4 = *reinterpret_cast<const floatx4*>(Eb[sl] + r0);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const bool vis = (unsigned)(at + r0 + r) < rows;
              const float pr = vis ? fast_exp2(fmaf(s[kk][t][0][r], f.scale_log2, -l4[r])) : 0.f;
              s[kk][t][0][r] = pr;
              dp[kk][t][0][r] = vis ? pr * (dp[kk][t][0][r] - e4[r]) : 0.f;
            }
          }
      }
      bf16x8 pop[2][1], dsop[2][1];
      pack_tile_op<1>(s, pop);
      pack_tile_op<1>(dp, dsop);
      dkv_acc(Qb[sl], Gb[sl], pop, dsop, dk, dv, lane);
      return hn;
    };
    for (;;) {
      if (!step(Buf<0>{})) break;
      if (!step(Buf<1>{})) break;
    }
    __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
  }
  if (kt < a.plan.sink_tiles) {
    // sums of this part to its slot (lane order: whole 1 KiB runs); the part that finishes last adds the parts up in
    // order. Every slot's stores are released before the count and read after it is acquired (agent scope: the parts
    // may run on different XCDs). No part waits for another.
    __shared__ int finished;
    const long owner = (long)kt * f.B + b;
    floatx4* slot = reinterpret_cast<floatx4*>(a.slots) +
                    ((owner * (a.plan.parts + 1) * kHeadsKV + kvh) * kWaves + w) * (16 * 64) + lane;
    constexpr long kSlotStep = (long)kHeadsKV * kWinSlotFloats / 4;    // between the parts of a tile
    floatx4* mine = slot + z * kSlotStep;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      mine[64 * e] = dk[e][0];
      mine[64 * (8 + e)] = dv[e][0];
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "agent");
    __syncthreads();
    if (threadIdx.x == 0)
      finished = __hip_atomic_fetch_add(a.done + owner * kHeadsKV + kvh, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (finished != a.plan.parts) return;
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      dk[e][0] = slot[64 * e];
      dv[e][0] = slot[64 * (8 + e)];
    }
    for (int p = 0; p < a.plan.parts; ++p) {
      slot += kSlotStep;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        dk[e][0] += slot[64 * e];
        dv[e][0] += slot[64 * (8 + e)];
      }
    }
  }
  if (key >= f.S) return;                                    // (padding keys: sums of 0)
  __bf16* kp = a.dk + (long)b * a.dk_sb + (long)key * a.dk_ss + (long)kvh * a.dk_sh;
  __bf16* vp = a.dv + (long)b * a.dv_sb + (long)key * a.dv_ss + (long)kvh * a.dv_sh;
  store_acc_rows<1>(kp, dk, 0, j, in ? a.scale : 0.f);
  store_acc_rows<1>(vp, dv, 0, j, in ? 1.f : 0.f);
}

// Workspace: lse2, D (fp32 [B, 32, Sp] each), the counters, then the slots on a 16-byte boundary.
struct WindowBwdLayout {
  size_t dvec, done, slots, bytes;
  WindowBwdLayout(int batch, int seq_len, const SinkPlan& p) {
    const size_t rows = (size_t)batch * kHeadsQ * p.tiles * kBM * sizeof(float);
    dvec = rows;
    done = 2 * rows;
    slots = done + ((size_t)p.sink_tiles * batch * kHeadsKV * sizeof(int) + 255) / 256 * 256;
    bytes = slots + (size_t)p.slots() * batch * kHeadsKV * kWinSlotFloats * sizeof(float) + 16;
  }
};

}  // namespace abkv

extern "C" {

size_t abkv_window_bwd_workspace_size(int batch, int seq_len, int window, int sinks) {
  using namespace abkv;
  if (batch <= 0 || seq_len <= 0 || window <= 0 || sinks < 0) return 0;
  return WindowBwdLayout(batch, seq_len, SinkPlan(seq_len, batch, window, sinks)).bytes;
}

int abkv_window_attn_bwd(const void* q, long q_stride_b, long q_stride_s, long q_stride_h, const void* k, long k_stride_b,
                         long k_stride_s, long k_stride_h, const void* v, long v_stride_b, long v_stride_s,
                         long v_stride_h, const void* out, long out_stride_b, long out_stride_s, long out_stride_h,
                         const void* dout, long dout_stride_b, long dout_stride_s, long dout_stride_h, const float* lse,
                         const void* out_low, int batch, int seq_len, const int32_t* seq_lens, int window, int sinks, float scale, void* dq,
                         long dq_stride_b, long dq_stride_s, long dq_stride_h, void* dk, long dk_stride_b,
                         long dk_stride_s, long dk_stride_h, void* dv, long dv_stride_b, long dv_stride_s,
                         long dv_stride_h, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  using namespace abkv;
  if (batch <= 0 || seq_len <= 0) return 0;
  if (q == nullptr || k == nullptr || v == nullptr || out == nullptr || dout == nullptr || lse == nullptr ||
      dq == nullptr || dk == nullptr || dv == nullptr || window <= 0 || sinks < 0 ||
      !softmax_scale_ok(scale) || !row_strides_ok(q_stride_s, k_stride_s, v_stride_s, out_stride_s, dout_stride_s))
    return (int)hipErrorInvalidValue;
  const SinkPlan plan(seq_len, batch, window, sinks);
  const WindowBwdLayout lay(batch, seq_len, plan);
  if (workspace == nullptr || workspace_bytes < lay.bytes) return (int)hipErrorInvalidValue;
  WindowBwdArgs a;
  WindowArgs& f = a.f;
  f.q = static_cast<const __bf16*>(q);
  f.q_sb = q_stride_b; f.q_ss = q_stride_s; f.q_sh = q_stride_h;
  f.k = static_cast<const __bf16*>(k);
  f.k_sb = k_stride_b; f.k_ss = k_stride_s; f.k_sh = k_stride_h;
  f.v = static_cast<const __bf16*>(v);
  f.v_sb = v_stride_b; f.v_ss = v_stride_s; f.v_sh = v_stride_h;
  f.B = batch;
  f.S = seq_len;
  f.seq_lens = seq_lens;
  f.window = window;
  f.sinks = sinks;
  f.scale_log2 = scale * 1.4426950408889634f;
  f.out = nullptr; f.o_sb = f.o_ss = f.o_sh = 0;
  f.lse = nullptr;
  f.low = static_cast<uint8_t*>(const_cast<void*>(out_low));
  f.num_q_tiles = plan.tiles;
  a.o = static_cast<const __bf16*>(out);
  a.o_sb = out_stride_b; a.o_ss = out_stride_s; a.o_sh = out_stride_h;
  a.dout = static_cast<const __bf16*>(dout);
  a.g_sb = dout_stride_b; a.g_ss = dout_stride_s; a.g_sh = dout_stride_h;
  a.lse = lse;
  a.Sp = plan.tiles * kBM;
  char* ws = static_cast<char*>(workspace);
  a.lse2 = reinterpret_cast<float*>(ws);
  a.dvec = reinterpret_cast<float*>(ws + lay.dvec);
  a.done = reinterpret_cast<int*>(ws + lay.done);
  char* slots = ws + lay.slots;
  a.slots = reinterpret_cast<float*>(slots + (-reinterpret_cast<uintptr_t>(slots) & 15));
  a.plan = plan;
  a.scale = scale;
  a.dq = static_cast<__bf16*>(dq);
  a.dq_sb = dq_stride_b; a.dq_ss = dq_stride_s; a.dq_sh = dq_stride_h;
  a.dk = static_cast<__bf16*>(dk);
  a.dk_sb = dk_stride_b; a.dk_ss = dk_stride_s; a.dk_sh = dk_stride_h;
  a.dv = static_cast<__bf16*>(dv);
  a.dv_sb = dv_stride_b; a.dv_ss = dv_stride_s; a.dv_sh = dv_stride_h;
  const long gq = (long)f.num_q_tiles * batch * kHeadsKV;
  const long gk = (long)plan.items() * batch * kHeadsKV;
  if (gq * 512 > 0xFFFFFFFFL || gk * 256 > 0xFFFFFFFFL) return (int)hipErrorInvalidValue;
  hipLaunchKernelGGL(window_bwd_dq_kernel, dim3((unsigned)gq), dim3(512), 0, stream, a);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return (int)err;
  hipLaunchKernelGGL(window_bwd_dkv_kernel, dim3((unsigned)gk), dim3(256), 0, stream, a);
  return (int)hipGetLastError();
}

}  // extern "C"

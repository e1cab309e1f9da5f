// Tile products of the attention backward kernels (gfx950): the masked prefill's (prefill_bwd.hip) and the sliding
// window's (window_bwd.hip).
#pragma once
#include "attn_tile.h"

namespace abkv {

// acc[t][u] += A^T . B^T over one 64-row tile: A^T operands by LDS transpose reads of the tile, B^T the packed bf16
// operands (the forward's PV step without its row sums). acc[t][u][r] = dim 32j + 4 * acc_tile(t, j) + r of column
// (u, m16), j = lane >> 4.
template <int H>
__device__ __forceinline__ void tile_acc(const __bf16* buf, const bf16x8 (&op)[2][H], floatx4 (&acc)[8][H], int lane) {
#pragma unroll
  for (int kk = 0; kk < 2; ++kk)
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      const bf16x8 a = vt_operand(buf, 32 * kk, t, lane);
#pragma unroll
      for (int u = 0; u < H; ++u) acc[t][u] = mfma16x16x32(a, op[kk][u], acc[t][u]);
    }
}

// bf16 MFMA operand of a 64-row score tile x[kk][t][u][r] (row 32kk + 16t + 4j + r): k-index e < 4 is row
// 32kk + 4j + e, e >= 4 row 32kk + 16 + 4j + e - 4 (the order vt_operand reads the tile in).
template <int H>
__device__ __forceinline__ void pack_tile_op(const floatx4 (&x)[2][2][H], bf16x8 (&op)[2][H]) {
#pragma unroll
  for (int u = 0; u < H; ++u)
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      u32x4 pw;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        pw[2 * t] = pack_bf16x2(x[kk][t][u][0], x[kk][t][u][1]);
        pw[2 * t + 1] = pack_bf16x2(x[kk][t][u][2], x[kk][t][u][3]);
      }
      op[kk][u] = __builtin_bit_cast(bf16x8, pw);
    }
}

template <int N>
struct Buf {
  static constexpr int value = N;
};

// S = Q K^T and dP = dO V^T of a wave's 16 keys over one staged tile (32 ds_read_b128, 32 MFMAs). The two products
// are interleaved and the reads run eight ahead of the MFMAs: at 2 waves per SIMD the other wave alone cannot cover
// an LDS round trip per MFMA.
__device__ __forceinline__ void dkv_scores(const __bf16* Qbuf, const __bf16* Gbuf, const bf16x8 (&kop)[4],
                                           const bf16x8 (&vop)[4], floatx4 (&s)[2][2][1], floatx4 (&dp)[2][2][1],
                                           int m16, int j) {
#pragma unroll
  for (int kk = 0; kk < 2; ++kk)
#pragma unroll
    for (int t = 0; t < 2; ++t) s[kk][t][0] = dp[kk][t][0] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const bf16x8 qa = __builtin_bit_cast(bf16x8, lds16(Qbuf, 32 * kk + 16 * t + m16, 4 * i + j));
        const bf16x8 ga = __builtin_bit_cast(bf16x8, lds16(Gbuf, 32 * kk + 16 * t + m16, 4 * i + j));
        s[kk][t][0] = mfma16x16x32(qa, kop[i], s[kk][t][0]);
        dp[kk][t][0] = mfma16x16x32(ga, vop[i], dp[kk][t][0]);
      }
  // scheduling groups (mask 0x100 LDS reads, 0x008 MFMA): 8 reads, then one MFMA per read, then the last 8 MFMAs
  __builtin_amdgcn_sched_group_barrier(0x100, 8, 0);
#pragma unroll
  for (int n = 0; n < 24; ++n) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
  }
  __builtin_amdgcn_sched_group_barrier(0x008, 8, 0);
}

// dV^T += dO^T P and dK^T += Q^T dS over one staged tile (the forward's PV step twice, interleaved; 64 transposed
// reads, 32 MFMAs), the reads running ahead of the MFMAs as in dkv_scores.
__device__ __forceinline__ void dkv_acc(const __bf16* Qbuf, const __bf16* Gbuf, const bf16x8 (&pop)[2][1],
                                        const bf16x8 (&dsop)[2][1], floatx4 (&dk)[8][1], floatx4 (&dv)[8][1],
                                        int lane) {
#pragma unroll
  for (int kk = 0; kk < 2; ++kk)
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      const bf16x8 ga = vt_operand(Gbuf, 32 * kk, t, lane);
      const bf16x8 qa = vt_operand(Qbuf, 32 * kk, t, lane);
      dv[t][0] = mfma16x16x32(ga, pop[kk][0], dv[t][0]);
      dk[t][0] = mfma16x16x32(qa, dsop[kk][0], dk[t][0]);
    }
  __builtin_amdgcn_sched_group_barrier(0x100, 8, 1);
#pragma unroll
  for (int n = 0; n < 28; ++n) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 1);
    __builtin_amdgcn_sched_group_barrier(0x100, 2, 1);
  }
  __builtin_amdgcn_sched_group_barrier(0x008, 4, 1);
}

}  // namespace abkv

// RMS norms of queries and keys for each head, and the position rotation in the same pass (gfx950).
//
// A head row x [128] with norm weight w and the angles of its token (64 cosines c and sines s, NeoX halves):
//   r = 1 / sqrt(mean(x^2) + eps),  y = w x r,  out[i] = y[i] c[i] - y[i + 64] s[i],  out[i + 64] = y[i + 64] c[i] + y[i] s[i].
// Backward, from the gradient of out: dy = the inverse rotation of it, g = w dy,
//   dx = r (g - x r^2 mean(g x)),  dw = sum over rows of dy x r.
// Everything between the loads and the stores is fp32 and rounded once (the norm and rotation as separate operations round to
// bf16 between them). Without weights (both null) the rows are only rotated.
//
// Bound by memory: a row is read once and written once. A row lies in 8 lanes, lane i with dims 8 i .. + 7 and 64 + 8 i .. + 7,
// both members of its rotation pairs, so a wave holds 8 rows, its loads are whole 16-byte pieces and the sums over a row are
// three DPP steps.
// Measured, inputs from memory: 2048 tokens appended 10.6 us (4.8 TB/s, what a copy reaches); training, two sequences of 4096 in
// bf16: forward 33 us (168 MB, 5.1 TB/s), backward 57 (252 MB, 4.4 TB/s).
#include "abridgekv_amd.h"
#include "int4.h"
#include "rope.h"

namespace abkv {

constexpr int kHeadSets = (kHeadsQ + kHeadsKV) / 8;          // sets of 8 heads of a token: four of queries, one of keys

// The 16 dims of a row that a lane holds.
struct Piece {
  float lo[8], hi[8];
};

__device__ __forceinline__ void ld8(const __bf16* p, float (&x)[8]) {
  const u32x4 w = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = bf16_lo(w[i]);
    x[2 * i + 1] = bf16_hi(w[i]);
  }
}
__device__ __forceinline__ void ld8(const float* p, float (&x)[8]) {
  const floatx4 a = *reinterpret_cast<const floatx4*>(p), b = *reinterpret_cast<const floatx4*>(p + 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[i] = a[i];
    x[4 + i] = b[i];
  }
}
__device__ __forceinline__ u32x4 pack8(const float (&x)[8]) {
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
  return w;
}
__device__ __forceinline__ void st8(__bf16* p, const float (&x)[8]) { *reinterpret_cast<u32x4*>(p) = pack8(x); }
__device__ __forceinline__ void st8(float* p, const float (&x)[8]) {
  *reinterpret_cast<floatx4*>(p) = floatx4{x[0], x[1], x[2], x[3]};
  *reinterpret_cast<floatx4*>(p + 4) = floatx4{x[4], x[5], x[6], x[7]};
}
template <class T>
__device__ __forceinline__ Piece ld_piece(const T* row, int i) {
  Piece p;
  ld8(row + 8 * i, p.lo);
  ld8(row + 64 + 8 * i, p.hi);
  return p;
}
template <class T>
__device__ __forceinline__ void st_piece(T* row, int i, const Piece& p) {
  st8(row + 8 * i, p.lo);
  st8(row + 64 + 8 * i, p.hi);
}
// A weight or a table of either type.
__device__ __forceinline__ Piece ld_piece_as(const void* row, bool f32, int i) {
  return f32 ? ld_piece(static_cast<const float*>(row), i) : ld_piece(static_cast<const __bf16*>(row), i);
}

// Sum over the 8 lanes of a row.
__device__ __forceinline__ float row_sum(float v) {
  v += dpp<kDppXor1>(v);
  v += dpp<kDppXor2>(v);
  return v + dpp<kDppHalfMirror>(v);
}
__device__ __forceinline__ float sum_squares(const Piece& x) {
  float v = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) v = fmaf(x.lo[i], x.lo[i], fmaf(x.hi[i], x.hi[i], v));
  return v;
}

// The norm (w: the weight, or null for none) and the rotation of a row, in place. The fused operations are written out, so that
// every kernel here leaves the same bits.
__device__ __forceinline__ void norm_rotate(Piece& x, const Piece* w, float eps, const float (&c)[8], const float (&s)[8]) {
  if (w != nullptr) {
    const float r = 1.f / sqrtf(fmaf(row_sum(sum_squares(x)), 1.f / kHeadDim, eps));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x.lo[i] *= r * w->lo[i];
      x.hi[i] *= r * w->hi[i];
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = x.lo[i], b = x.hi[i];
    x.lo[i] = fmaf(a, c[i], -(b * s[i]));
    x.hi[i] = fmaf(b, c[i], a * s[i]);
  }
}

// -- a serving step's rows: queries out, keys and values into the cache ---------------------------------------------------
struct NormAppendArgs : RopeLayout {
  const __bf16* q; long q_st, q_sh;            // [T, 32, 128]
  const __bf16* k; long k_st, k_sh;            // [T, 8, 128]
  const __bf16* v; long v_st, v_sh;            // [T, 8, 128]
  const int64_t* positions;                    // [T]
  const float* cos_sin;                        // [max_pos, 128]: cos of the 64 frequencies, then sin
  const void *wq, *wk;                         // [128] bf16 or fp32, or null: no norms
  bool w_f32;
  float eps;
  __bf16* out; long o_st, o_sh;                // [T, 32, 128]; may be q
  const int64_t* slot_mapping;                 // [T]; < 0 or past the cache = skip
  char* cache; long num_pages;                 // [num_pages, 2, 16, 8, 128] bf16, or [num_pages, 2, 16, 640] bytes
};

// A row of the 4-bit cache from the bf16 values of x (head h, lane i of the row's eight).
__device__ __forceinline__ void store_row4(char* slot, int h, int i, const Piece& x) {
  uint32_t lo_pair, hi_pair;
  const uint32_t lo = quantise8(x.lo, lo_pair), hi = quantise8(x.hi, hi_pair);
  uint32_t* codes = reinterpret_cast<uint32_t*>(slot + h * kHeadCodes4);
  codes[code_word(i)] = lo;
  codes[code_word(8 + i)] = hi;
  if ((i & 3) == 0) {                                        // lanes 0 .. 3 hold groups 0 and 2, lanes 4 .. 7 groups 1 and 3
    uint32_t* pairs = reinterpret_cast<uint32_t*>(slot + kParams4 + h * 16);
    pairs[i >> 2] = lo_pair;
    pairs[2 + (i >> 2)] = hi_pair;
  }
}

// One workgroup per token, a wave per set of 8 heads: the key heads' wave stores the value rows too. A decode step has a few
// tokens and is as long as one wave's chain of loads, so the sets go side by side.
template <bool kInt4>
__global__ __launch_bounds__(64 * kHeadSets) void norm_append_kernel(NormAppendArgs a) {
  const long t = blockIdx.x;
  const int set = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, h = lane >> 3, i = lane & 7;
  const bool keys = set == kHeadSets - 1;
  const long slot = keys ? a.slot_mapping[t] : 0;
  Piece x = ld_piece(keys ? a.k + t * a.k_st + h * a.k_sh : a.q + t * a.q_st + (long)(8 * set + h) * a.q_sh, i);
  const float* cs = a.cos_sin + rope_position(a, a.positions[t]) * kHeadDim;
  float c[8], s[8];
  ld8(cs + 8 * i, c);
  ld8(cs + 64 + 8 * i, s);
  if (a.wq != nullptr) {
    const Piece w = ld_piece_as(keys ? a.wk : a.wq, a.w_f32, i);
    norm_rotate(x, &w, a.eps, c, s);
  } else {
    norm_rotate(x, nullptr, 0.f, c, s);
  }
  if (!keys) {
    st_piece(a.out + t * a.o_st + (long)(8 * set + h) * a.o_sh, i, x);
    return;
  }
  if (slot < 0 || slot >= a.num_pages * kPage) return;
  const __bf16* v = a.v + t * a.v_st + h * a.v_sh;
  if constexpr (kInt4) {
    char* to = a.cache + slot / kPage * kPage4 + slot % kPage * kSlot4;
#pragma unroll
    for (int d = 0; d < 8; ++d) {                            // the row as a bf16 cache would hold it
      x.lo[d] = (float)(__bf16)x.lo[d];
      x.hi[d] = (float)(__bf16)x.hi[d];
    }
    store_row4(to, h, i, x);
    store_row4(to + kHalf4, h, i, ld_piece(v, i));
  } else {
    __bf16* to = reinterpret_cast<__bf16*>(a.cache) + slot / kPage * kPageElems + slot % kPage * kSlotElems + h * kHeadDim;
    const u32x4 v0 = *reinterpret_cast<const u32x4*>(v + 8 * i), v1 = *reinterpret_cast<const u32x4*>(v + 64 + 8 * i);
    st_piece(to, i, x);
    *reinterpret_cast<u32x4*>(to + kHalfElems + 8 * i) = v0;
    *reinterpret_cast<u32x4*>(to + kHalfElems + 64 + 8 * i) = v1;
  }
}

// -- a training step's rows -------------------------------------------------------------------------------------------
struct Rows4 {                                 // [batch, seq, heads, 128], dims contiguous
  void* p;
  long sb, ss, sh;
};
struct NormRopeArgs {
  Rows4 q, k;
  Rows4 dq_out, dk_out;                        // backward: gradients of the outputs
  void *q_to, *k_to;                           // outputs (forward) or gradients (backward), dense
  const void *cos, *sin;                       // [batch or 1, seq, 128] (the first 64 of a row are read)
  long a_sb, a_ss;                             // (a_sb 0: shared by the batch)
  bool a_f32;
  const void *wq, *wk;
  bool w_f32;
  float eps;
  long tokens;
  int seq;
  float* parts;                                // backward: [workgroups][2][128] sums for the weights' gradients
};

template <class T>
__device__ __forceinline__ const T* head_row(const Rows4& r, long b, long s, int h) {
  return static_cast<const T*>(r.p) + b * r.sb + s * r.ss + h * r.sh;
}

constexpr int kTokenWaves = 4;

// A wave per token: its angles once, then the five sets of heads.
template <class T>
__global__ __launch_bounds__(64 * kTokenWaves) void norm_rope_kernel(NormRopeArgs a) {
  const int lane = threadIdx.x & 63, h = lane >> 3, i = lane & 7;
  const long t = (long)blockIdx.x * kTokenWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (t >= a.tokens) return;
  const long b = t / a.seq, s = t - b * a.seq;
  Piece x[kHeadSets];
#pragma unroll
  for (int n = 0; n < kHeadSets; ++n)
    x[n] = n < 4 ? ld_piece(head_row<T>(a.q, b, s, 8 * n + h), i) : ld_piece(head_row<T>(a.k, b, s, h), i);
  float c[8], sn[8];
  const long at = b * a.a_sb + s * a.a_ss + 8 * i;
  if (a.a_f32) {
    ld8(static_cast<const float*>(a.cos) + at, c);
    ld8(static_cast<const float*>(a.sin) + at, sn);
  } else {
    ld8(static_cast<const __bf16*>(a.cos) + at, c);
    ld8(static_cast<const __bf16*>(a.sin) + at, sn);
  }
  Piece w = ld_piece_as(a.wq, a.w_f32, i);
#pragma unroll
  for (int n = 0; n < kHeadSets; ++n) {
    if (n == 4) w = ld_piece_as(a.wk, a.w_f32, i);
    norm_rotate(x[n], &w, a.eps, c, sn);
    T* to = n < 4 ? static_cast<T*>(a.q_to) + (t * kHeadsQ + 8 * n + h) * kHeadDim
                  : static_cast<T*>(a.k_to) + (t * kHeadsKV + h) * kHeadDim;
    st_piece(to, i, x[n]);
  }
}

// Backward: workgroups walk the tokens, a wave a token at a time, and keep the weights' sums in registers; each leaves its sums
// in a part of its own, which norm_weights_kernel adds in a fixed order.
template <class T>
__global__ __launch_bounds__(64 * kTokenWaves) void norm_rope_bwd_kernel(NormRopeArgs a) {
  const int lane = threadIdx.x & 63, h = lane >> 3, i = lane & 7;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Piece wq = ld_piece_as(a.wq, a.w_f32, i), wk = ld_piece_as(a.wk, a.w_f32, i);
  Piece sums[2] = {};
  for (long t = (long)blockIdx.x * kTokenWaves + wave; t < a.tokens; t += (long)gridDim.x * kTokenWaves) {
    const long b = t / a.seq, s = t - b * a.seq;
    float c[8], sn[8];
    const long at = b * a.a_sb + s * a.a_ss + 8 * i;
    if (a.a_f32) {
      ld8(static_cast<const float*>(a.cos) + at, c);
      ld8(static_cast<const float*>(a.sin) + at, sn);
    } else {
      ld8(static_cast<const __bf16*>(a.cos) + at, c);
      ld8(static_cast<const __bf16*>(a.sin) + at, sn);
    }
#pragma unroll
    for (int n = 0; n < kHeadSets; ++n) {
      const bool keys = n == 4;
      const Piece x = ld_piece(keys ? head_row<T>(a.k, b, s, h) : head_row<T>(a.q, b, s, 8 * n + h), i);
      Piece g = ld_piece(keys ? head_row<T>(a.dk_out, b, s, h) : head_row<T>(a.dq_out, b, s, 8 * n + h), i);
      const Piece& w = keys ? wk : wq;
      Piece& sum = sums[keys];
      const float r = 1.f / sqrtf(row_sum(sum_squares(x)) * (1.f / kHeadDim) + a.eps);
      float gx = 0.f;
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        const float lo = g.lo[d] * c[d] + g.hi[d] * sn[d], hi = g.hi[d] * c[d] - g.lo[d] * sn[d];
        sum.lo[d] += lo * (x.lo[d] * r);
        sum.hi[d] += hi * (x.hi[d] * r);
        g.lo[d] = lo * w.lo[d];
        g.hi[d] = hi * w.hi[d];
        gx += g.lo[d] * x.lo[d] + g.hi[d] * x.hi[d];
      }
      const float m = row_sum(gx) * (1.f / kHeadDim) * r * r;
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        g.lo[d] = r * (g.lo[d] - x.lo[d] * m);
        g.hi[d] = r * (g.hi[d] - x.hi[d] * m);
      }
      T* to = keys ? static_cast<T*>(a.k_to) + (t * kHeadsKV + h) * kHeadDim
                   : static_cast<T*>(a.q_to) + (t * kHeadsQ + 8 * n + h) * kHeadDim;
      st_piece(to, i, g);
    }
  }
  // over the wave's 8 rows (lanes i, i + 8, ...), then over the waves
  __shared__ float red[kTokenWaves][2][kHeadDim];
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int d = 0; d < 8; ++d) {
      float lo = sums[k].lo[d], hi = sums[k].hi[d];
      lo += __shfl_xor(lo, 8, 64);
      hi += __shfl_xor(hi, 8, 64);
      lo = sum_xor32(sum_xor16(lo));
      hi = sum_xor32(sum_xor16(hi));
      if (h == 0) {
        red[wave][k][8 * i + d] = lo;
        red[wave][k][64 + 8 * i + d] = hi;
      }
    }
  __syncthreads();
  float v = 0.f;
  for (int w = 0; w < kTokenWaves; ++w) v += red[w][threadIdx.x >> 7][threadIdx.x & 127];
  a.parts[(long)blockIdx.x * 2 * kHeadDim + threadIdx.x] = v;
}
static_assert(64 * kTokenWaves == 2 * kHeadDim, "a thread for each of the two weights' dims");

// The weights' gradients from the workgroups' parts: workgroup of 16 dims, 16 threads a dim.
__global__ __launch_bounds__(256) void norm_weights_kernel(const float* parts, int n, void* dwq, void* dwk, bool f32) {
  __shared__ float red[16][17];
  const int c = threadIdx.x & 15, r = threadIdx.x >> 4;
  const int dim = 16 * blockIdx.x + c;                       // of the two weights' 256
  float v = 0.f;
#pragma unroll 8
  for (int p = r; p < n; p += 16) v += parts[(long)p * 2 * kHeadDim + dim];
  red[r][c] = v;
  __syncthreads();
  if (r != 0) return;
  v = 0.f;
#pragma unroll
  for (int k = 0; k < 16; ++k) v += red[k][c];
  void* to = dim < kHeadDim ? dwq : dwk;
  if (f32) static_cast<float*>(to)[dim % kHeadDim] = v;
  else static_cast<__bf16*>(to)[dim % kHeadDim] = (__bf16)v;
}

// Workgroups of the backward: three a CU, what its registers let a CU hold; fewer where tokens are few. Calls in a row, with the
// weights' launch, for 512, 768 and 1024 workgroups (a third of these in a second round): two sequences of 4096 tokens in bf16,
// eight sets of inputs in turn 66, 57 and 72 us, one set again and again, part of which the last-level cache then holds, 48, 47
// and 56; eight of 8192, three sets 494, 399 and 513.
inline int bwd_groups(long tokens) {
  const long n = (tokens + kTokenWaves - 1) / kTokenWaves;
  return n < 768 ? (int)n : 768;
}

}  // namespace abkv

using namespace abkv;

static bool rows_ok(const void* p, long a, long b, long c, int elem) {
  return p != nullptr && (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ((a | b | c) * elem) % 16 == 0;
}
static bool norm_args(NormRopeArgs& a, int f32, const void* q, long q_sb, long q_ss, long q_sh, const void* k, long k_sb,
                      long k_ss, long k_sh, int batch, int seq, const void* q_weight, const void* k_weight, int weight_f32,
                      float eps, const void* cos, const void* sin, long angle_sb, long angle_ss, int angle_f32, void* q_to,
                      void* k_to) {
  const int e = f32 ? 4 : 2, ae = angle_f32 ? 4 : 2;
  if (!rows_ok(q, q_sb, q_ss, q_sh, e) || !rows_ok(k, k_sb, k_ss, k_sh, e) || !rows_ok(cos, angle_sb, angle_ss, 0, ae) ||
      !rows_ok(sin, angle_sb, angle_ss, 0, ae) || !rows_ok(q_weight, 0, 0, 0, 2) || !rows_ok(k_weight, 0, 0, 0, 2) ||
      !rows_ok(q_to, 0, 0, 0, 2) || !rows_ok(k_to, 0, 0, 0, 2) || !(eps >= 0.f))
    return false;
  a.q = Rows4{const_cast<void*>(q), q_sb, q_ss, q_sh};
  a.k = Rows4{const_cast<void*>(k), k_sb, k_ss, k_sh};
  a.q_to = q_to;
  a.k_to = k_to;
  a.cos = cos;
  a.sin = sin;
  a.a_sb = angle_sb;
  a.a_ss = angle_ss;
  a.a_f32 = angle_f32 != 0;
  a.wq = q_weight;
  a.wk = k_weight;
  a.w_f32 = weight_f32 != 0;
  a.eps = eps;
  a.tokens = (long)batch * seq;
  a.seq = seq;
  a.parts = nullptr;
  return (a.tokens + kTokenWaves - 1) / kTokenWaves <= 0x00FFFFFFL;
}

extern "C" {

int abkv_qk_norm_rope_append(const void* q, long q_stride_t, long q_stride_h, const void* key, long key_stride_t,
                             long key_stride_h, const void* value, long value_stride_t, long value_stride_h,
                             const int64_t* positions, int num_tokens, const void* q_weight, const void* k_weight,
                             int weight_f32, float eps, int block_c, int codes_k, int code_span, const float* cos_sin,
                             long max_pos, const int64_t* slot_mapping, void* kv_cache, int num_pages, int int4, void* q_out,
                             long out_stride_t, long out_stride_h, hipStream_t stream) {
  if (num_tokens <= 0) return 0;
  NormAppendArgs a;
  if (!rows_ok(q, q_stride_t, q_stride_h, 0, 2) || !rows_ok(key, key_stride_t, key_stride_h, 0, 2) ||
      !rows_ok(value, value_stride_t, value_stride_h, 0, 2) || !rows_ok(q_out, out_stride_t, out_stride_h, 0, 2) ||
      !rows_ok(cos_sin, 0, 0, 0, 4) || !rows_ok(kv_cache, 0, 0, 0, 2) || positions == nullptr || slot_mapping == nullptr ||
      num_pages <= 0 || (q_weight == nullptr) != (k_weight == nullptr) ||
      (q_weight != nullptr && (!rows_ok(q_weight, 0, 0, 0, 2) || !rows_ok(k_weight, 0, 0, 0, 2))) || !(eps >= 0.f) ||
      !rope_layout(a, max_pos, block_c, codes_k, code_span))
    return (int)hipErrorInvalidValue;
  a.q = static_cast<const __bf16*>(q);
  a.q_st = q_stride_t;
  a.q_sh = q_stride_h;
  a.k = static_cast<const __bf16*>(key);
  a.k_st = key_stride_t;
  a.k_sh = key_stride_h;
  a.v = static_cast<const __bf16*>(value);
  a.v_st = value_stride_t;
  a.v_sh = value_stride_h;
  a.positions = positions;
  a.cos_sin = cos_sin;
  a.wq = q_weight;
  a.wk = k_weight;
  a.w_f32 = weight_f32 != 0;
  a.eps = eps;
  a.out = static_cast<__bf16*>(q_out);
  a.o_st = out_stride_t;
  a.o_sh = out_stride_h;
  a.slot_mapping = slot_mapping;
  a.cache = static_cast<char*>(kv_cache);
  a.num_pages = num_pages;
  if (int4) hipLaunchKernelGGL(norm_append_kernel<true>, dim3(num_tokens), dim3(64 * kHeadSets), 0, stream, a);
  else hipLaunchKernelGGL(norm_append_kernel<false>, dim3(num_tokens), dim3(64 * kHeadSets), 0, stream, a);
  return (int)hipGetLastError();
}

int abkv_qk_norm_rope(int f32, const void* q, long q_stride_b, long q_stride_s, long q_stride_h, const void* k,
                      long k_stride_b, long k_stride_s, long k_stride_h, int batch, int seq_len, const void* q_weight,
                      const void* k_weight, int weight_f32, float eps, const void* cos, const void* sin, long angle_stride_b,
                      long angle_stride_s, int angle_f32, void* q_out, void* k_out, hipStream_t stream) {
  if (batch <= 0 || seq_len <= 0) return 0;
  NormRopeArgs a;
  if (!norm_args(a, f32, q, q_stride_b, q_stride_s, q_stride_h, k, k_stride_b, k_stride_s, k_stride_h, batch, seq_len,
                 q_weight, k_weight, weight_f32, eps, cos, sin, angle_stride_b, angle_stride_s, angle_f32, q_out, k_out))
    return (int)hipErrorInvalidValue;
  const dim3 grid((unsigned)((a.tokens + kTokenWaves - 1) / kTokenWaves)), block(64 * kTokenWaves);
  if (f32) hipLaunchKernelGGL(norm_rope_kernel<float>, grid, block, 0, stream, a);
  else hipLaunchKernelGGL(norm_rope_kernel<__bf16>, grid, block, 0, stream, a);
  return (int)hipGetLastError();
}

size_t abkv_qk_norm_rope_bwd_workspace_size(int batch, int seq_len) {
  if (batch <= 0 || seq_len <= 0) return 0;
  return (size_t)bwd_groups((long)batch * seq_len) * 2 * kHeadDim * sizeof(float);
}

int abkv_qk_norm_rope_bwd(int f32, const void* q, long q_stride_b, long q_stride_s, long q_stride_h, const void* k,
                          long k_stride_b, long k_stride_s, long k_stride_h, const void* dq_out, long dqo_stride_b,
                          long dqo_stride_s, long dqo_stride_h, const void* dk_out, long dko_stride_b, long dko_stride_s,
                          long dko_stride_h, int batch, int seq_len, const void* q_weight, const void* k_weight,
                          int weight_f32, float eps, const void* cos, const void* sin, long angle_stride_b,
                          long angle_stride_s, int angle_f32, void* dq, void* dk, void* dq_weight, void* dk_weight,
                          void* workspace, size_t workspace_bytes, hipStream_t stream) {
  if (batch <= 0 || seq_len <= 0) return 0;
  NormRopeArgs a;
  const int e = f32 ? 4 : 2;
  if (!norm_args(a, f32, q, q_stride_b, q_stride_s, q_stride_h, k, k_stride_b, k_stride_s, k_stride_h, batch, seq_len,
                 q_weight, k_weight, weight_f32, eps, cos, sin, angle_stride_b, angle_stride_s, angle_f32, dq, dk) ||
      !rows_ok(dq_out, dqo_stride_b, dqo_stride_s, dqo_stride_h, e) ||
      !rows_ok(dk_out, dko_stride_b, dko_stride_s, dko_stride_h, e) || dq_weight == nullptr || dk_weight == nullptr ||
      workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 3) ||
      workspace_bytes < abkv_qk_norm_rope_bwd_workspace_size(batch, seq_len))
    return (int)hipErrorInvalidValue;
  a.dq_out = Rows4{const_cast<void*>(dq_out), dqo_stride_b, dqo_stride_s, dqo_stride_h};
  a.dk_out = Rows4{const_cast<void*>(dk_out), dko_stride_b, dko_stride_s, dko_stride_h};
  a.parts = static_cast<float*>(workspace);
  const int groups = bwd_groups(a.tokens);
  if (f32) hipLaunchKernelGGL(norm_rope_bwd_kernel<float>, dim3(groups), dim3(64 * kTokenWaves), 0, stream, a);
  else hipLaunchKernelGGL(norm_rope_bwd_kernel<__bf16>, dim3(groups), dim3(64 * kTokenWaves), 0, stream, a);
  const hipError_t err = hipGetLastError();
  if (err != hipSuccess) return (int)err;
  hipLaunchKernelGGL(norm_weights_kernel, dim3(2 * kHeadDim / 16), dim3(256), 0, stream, a.parts, groups, dq_weight, dk_weight,
                     a.w_f32);
  return (int)hipGetLastError();
}

}  // extern "C"

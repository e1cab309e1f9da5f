// Log probabilities of given tokens from logits, with the entropy and the most likely alternatives, and the gradient (gfx950).
//
// x = logits / temperature, m = max x, l = sum exp(x - m):  log p_v = x_v - m - ln l,  H = ln l - (sum exp(x - m) (x - m)) / l.
// Gradient of g log p_t + h H:  dlogits_v = (p_v (-g - h (log p_v + H)) + g [v = t]) / temperature.
//
// The forward reads a row once: every thread keeps a running maximum m, l and e = sum exp(x - m) (x - m) (fp32; sums of up to a
// few hundred terms a thread, then in a tree), which meet at the end. Rows are split over workgroups when they are few; a
// second launch joins the splits. Logits below -1e25 (banned tokens: -inf, or the type's lowest value) weigh nothing; a NaN or
// +inf makes its row NaN.
//
// Alternatives: the n-th largest of a wave's thread maxima bounds the n-th largest logit from below, and so does the largest of
// the waves' bounds. Only the threads whose maximum reaches it read their part again and collect what reaches it in LDS; every
// candidate counts how many come before it (higher, or equal at a lower index). More candidates than the list holds (rows of many
// equal logits) are found one after the other instead.
//
// Bound by memory: 2 (bf16) or 4 bytes a logit, beside one exponential and ten other operations.
// Measured: 2048 rows of 131072 logits in bf16, forward 84 to 104 us (537 MB, 5.2 to 6.4 TB/s), gradient 172 to 181 (1.07 GB,
// 6 TB/s); one row in fp32 with 5 alternatives 5.2 + 3.4 us over 64 workgroups.
#include "abridgekv_amd.h"
#include "common.h"

namespace abkv {

constexpr int kRowThreads = 512;
constexpr int kTopMax = 32;                    // alternatives a row
constexpr int kListMax = 1024;                 // candidates in LDS
constexpr int kMergeMax = 2048;                // candidates of a row's splits
// Stands for -inf and whatever lies below it (a mask of the type's lowest value), so that exp(x - m) (x - m), and that times a
// count, is 0 and not NaN. Temperatures up to 1e20 leave it no weight, and the reciprocals of those from 1e-30 on are floats, with
// room for a gradient.
constexpr float kLowest = -1.0e25f;
inline bool temperature_ok(float t) { return t >= 1e-30f && t <= 1e20f; }
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.69314718055994531f;

struct LogprobArgs {
  const void* logits;          // [T, V] rows `stride` elements apart
  long stride;
  int vocab;
  const int64_t* targets;      // [T]; outside [0, vocab): the row has no target (log probability 0)
  float inv_t;                 // 1 / temperature
  int top;
  float* logprob;              // [T]
  float* entropy;              // [T] or nullptr
  float* stats;                // [T, 3]: max logit, ln of the weights' sum, entropy; or nullptr
  int64_t* top_ids;            // [T, top]
  float* top_logprobs;         // [T, top]
  int splits, split_vecs;      // workgroups a row, 16-byte pieces each
  float* part;                 // [T, splits, 3]: m, l, e of a split
  uint64_t* part_top;          // [T, splits, top] keys, 0: none
};

template <class T>
struct Vec;
template <>
struct Vec<__bf16> {
  static constexpr int n = 8;
  static __device__ __forceinline__ void ld(const __bf16* p, float (&x)[8]) {
    const u32x4 w = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = bf16_lo(w[i]);
      x[2 * i + 1] = bf16_hi(w[i]);
    }
  }
};
template <>
struct Vec<float> {
  static constexpr int n = 4;
  static __device__ __forceinline__ void ld(const float* p, float (&x)[4]) {
    const floatx4 w = __builtin_nontemporal_load(reinterpret_cast<const floatx4*>(p));
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = w[i];
  }
};

// Elements of a row before its first 16-byte boundary, whole pieces behind them; the rest is the tail.
template <class T>
struct RowShape {
  int head, vecs;
  __device__ __forceinline__ RowShape(const T* row, int vocab) {
    head = min((int)((16 - ((uintptr_t)row & 15)) & 15) / (int)sizeof(T), vocab);
    vecs = (vocab - head) / Vec<T>::n;
  }
};

// Order of logits as unsigned numbers; a NaN comes below everything, as -inf does.
__device__ __forceinline__ uint32_t order_key(float x) {
  x = fmaxf(x, -INFINITY);
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float order_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
// Keys sort by logit, then by the lower index.
__device__ __forceinline__ uint64_t top_key(float x, int v) { return (uint64_t)order_key(x + 0.f) << 32 | (uint32_t)~v; }

// m (of the logits), l and e (of logits times c = log2(e) / temperature, e in units of the logits).
struct Running {
  float m, l, e;
};
__device__ __forceinline__ Running joined(const Running& a, const Running& b, float c) {
  Running r;
  r.m = fmaxf(a.m, b.m);
  const float da = a.m - r.m, db = b.m - r.m;
  const float fa = fast_exp2(da * c), fb = fast_exp2(db * c);
  r.l = a.l * fa + b.l * fb;
  r.e = fa * (a.e + da * a.l) + fb * (b.e + db * b.l);
  return r;
}
__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, dpp<kDppXor1>(v));
  v = fmaxf(v, dpp<kDppXor2>(v));
  v = fmaxf(v, dpp<kDppHalfMirror>(v));
  v = fmaxf(v, dpp<kDppMirror>(v));
  return max_xor32(max_xor16(v));
}
__device__ __forceinline__ float wave_sum(float v) {
  v += dpp<kDppXor1>(v);
  v += dpp<kDppXor2>(v);
  v += dpp<kDppHalfMirror>(v);
  v += dpp<kDppMirror>(v);
  return sum_xor32(sum_xor16(v));
}
// The lanes' sums in one, in every lane.
__device__ __forceinline__ Running wave_joined(const Running& a, float c) {
  Running r;
  r.m = wave_max(a.m);
  const float d = a.m - r.m, f = fast_exp2(d * c);
  r.l = wave_sum(a.l * f);
  r.e = wave_sum(f * (a.e + d * a.l));
  return r;
}
template <int N, bool kEntropy>
__device__ __forceinline__ void take(Running& st, const float (&raw)[N], float c) {
  float x[N], mx = st.m;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    x[i] = raw[i] < kLowest ? kLowest : raw[i];              // (NaN stays)
    mx = fmaxf(mx, x[i]);
  }
  const float d = st.m - mx, f = fast_exp2(d * c);
  if constexpr (kEntropy) st.e = f * (st.e + d * st.l);
  st.l *= f;
  st.m = mx;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float y = x[i] - mx, p = fast_exp2(y * c);
    st.l += p;
    if constexpr (kEntropy) st.e += p * y;
  }
}

// The row's outputs from its whole sums, by one thread.
template <class T>
__device__ __forceinline__ float finish_row(const LogprobArgs& a, long t, const T* row, Running st) {
  // (a row without any logit that weighs, or with a weight that is not a number, has no probabilities)
  const float log_l = st.m > kLowest ? logf(st.l) : NAN;
  const float h = log_l - st.e / st.l * a.inv_t;
  const int64_t target = a.targets[t];
  float lp = 0.f;
  if (target >= 0 && target < a.vocab) lp = ((float)row[target] - st.m) * a.inv_t - log_l;
  a.logprob[t] = lp;
  if (a.entropy != nullptr) a.entropy[t] = h;
  if (a.stats != nullptr) {
    a.stats[3 * t] = st.m;
    a.stats[3 * t + 1] = log_l;
    a.stats[3 * t + 2] = h;
  }
  return log_l;
}
__device__ __forceinline__ void store_top(const LogprobArgs& a, long t, int rank, uint64_t key, float m, float log_l) {
  a.top_ids[t * a.top + rank] = (int)~(uint32_t)key;
  a.top_logprobs[t * a.top + rank] = (order_value((uint32_t)(key >> 32)) - m) * a.inv_t - log_l;
}

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
  v = max(v, dpp<kDppXor1>(v));
  v = max(v, dpp<kDppXor2>(v));
  v = max(v, dpp<kDppHalfMirror>(v));
  v = max(v, dpp<kDppMirror>(v));
  v = max(v, (uint32_t)__shfl_xor((int)v, 16, 64));
  return max(v, (uint32_t)__shfl_xor((int)v, 32, 64));
}
__device__ __forceinline__ uint64_t wave_max64(uint64_t v) {
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) {
    const uint64_t o = (uint64_t)__shfl_xor((unsigned long long)v, k, 64);
    v = o > v ? o : v;
  }
  return v;
}

// Workgroup (row, split), splits next to each other. The elements of a thread: pieces v0 + tid, v0 + tid + 512, ...; the head's
// with the first split, the tail's with the last.
template <class T, bool kEntropy>
__global__ __launch_bounds__(kRowThreads) void logprob_kernel(LogprobArgs a) {
  constexpr int N = Vec<T>::n, kWaves = kRowThreads / 64;
  const long t = blockIdx.x / a.splits;
  const int split = blockIdx.x % a.splits, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const T* row = static_cast<const T*>(a.logits) + t * a.stride;
  const RowShape<T> shape(row, a.vocab);
  const int v0 = split * a.split_vecs, v1 = min(shape.vecs, v0 + a.split_vecs);
  const float c = a.inv_t * kLog2e;
  // the one head or tail element of a thread, if any (a head and a tail hold fewer than 8 elements each)
  int lone = -1;
  if (split == 0 && tid < shape.head) lone = tid;
  const int tail = shape.head + shape.vecs * N;
  if (split == a.splits - 1 && tid >= 64 && tid - 64 < a.vocab - tail) lone = tail + tid - 64;

  Running st{kLowest, 0.f, 0.f};
  const T* body = row + shape.head;
  for (int v = v0 + tid; v < v1; v += kRowThreads) {
    float x[N];
    Vec<T>::ld(body + (long)v * N, x);
    take<N, kEntropy>(st, x, c);
  }
  if (lone >= 0) {
    const float x[1] = {(float)row[lone]};
    take<1, kEntropy>(st, x, c);
  }
  const float mine = st.m;                                   // this thread's largest (kLowest for -inf and none)
  st = wave_joined(st, c);
  __shared__ Running wave_st[kWaves];
  __shared__ float row_m, row_log_l;
  if (lane == 0) wave_st[wave] = st;
  __syncthreads();
  if (tid == 0) {
    st = wave_st[0];
    for (int w = 1; w < kWaves; ++w) st = joined(st, wave_st[w], c);
    if (a.splits == 1) {
      row_m = st.m;
      row_log_l = finish_row(a, t, row, st);
    } else {
      float* p = a.part + (t * a.splits + split) * 3;
      p[0] = st.m;
      p[1] = st.l;
      p[2] = st.e;
    }
  }
  if (a.top == 0) return;

  __shared__ uint64_t list[kListMax];
  __shared__ uint64_t wave_best[kWaves];
  __shared__ float bounds[kWaves];
  __shared__ int count;
  float bound = mine;                                        // the top-th largest of this wave's maxima, then of all waves' ones
  float left = mine;
  for (int k = 0; k < a.top; ++k) {
    bound = wave_max(left);
    if (lane == __ffsll(__ballot(left == bound)) - 1) left = -INFINITY;
  }
  if (lane == 0) bounds[wave] = bound;
  if (tid == 0) count = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) bound = fmaxf(bound, bounds[w]);
  const float lowest = bound > kLowest ? bound : -INFINITY;  // (kLowest: fewer threads than `top` hold a finite logit)
  auto each = [&](auto&& f) {                                // every element of this thread
    for (int v = v0 + tid; v < v1; v += kRowThreads) {
      float x[N];
      Vec<T>::ld(body + (long)v * N, x);
#pragma unroll
      for (int i = 0; i < N; ++i) f(x[i], shape.head + v * N + i);
    }
    if (lone >= 0) f((float)row[lone], lone);
  };
  if (mine >= bound)
    each([&](float x, int v) {
      if (fmaxf(x, -INFINITY) >= lowest) {
        const int at = atomicAdd(&count, 1);
        if (at < kListMax) list[at] = top_key(x, v);
      }
    });
  __syncthreads();
  const int n = count;
  uint64_t* out = a.part_top + (t * a.splits + split) * a.top;
  if (n <= kListMax) {
    for (int i = tid; i < n; i += kRowThreads) {
      const uint64_t key = list[i];
      int rank = 0;
      for (int k = 0; k < n; ++k) rank += list[k] > key;
      if (rank >= a.top) continue;
      if (a.splits == 1) store_top(a, t, rank, key, row_m, row_log_l);
      else out[rank] = key;
    }
    if (a.splits > 1)
      for (int i = n + tid; i < a.top; i += kRowThreads) out[i] = 0;
    return;
  }
  uint64_t last = ~0ull;
  for (int rank = 0; rank < a.top; ++rank) {                 // the largest key below the last one, again and again
    uint64_t best = 0;
    each([&](float x, int v) {
      const uint64_t key = top_key(x, v);
      if (key < last && key > best) best = key;
    });
    best = wave_max64(best);
    if (lane == 0) wave_best[wave] = best;
    __syncthreads();
    for (int w = 0; w < kWaves; ++w) best = wave_best[w] > best ? wave_best[w] : best;
    __syncthreads();
    last = best;
    if (tid == 0) {
      if (a.splits == 1) store_top(a, t, rank, best, row_m, row_log_l);
      else out[rank] = best;
    }
  }
}

// Joins the splits of a row: workgroup per row.
template <class T>
__global__ __launch_bounds__(256) void logprob_join_kernel(LogprobArgs a) {
  const long t = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63;
  const T* row = static_cast<const T*>(a.logits) + t * a.stride;
  const float c = a.inv_t * kLog2e;
  __shared__ uint64_t list[kMergeMax];
  const int n = a.splits * a.top;                            // at most kMergeMax (the host's choice of splits)
  for (int i = tid; i < n; i += 256) list[i] = a.part_top[t * n + i];
  Running st{kLowest, 0.f, 0.f};
  if (tid < a.splits) {                                      // (at most 64 splits)
    const float* p = a.part + (t * a.splits + tid) * 3;
    st = Running{p[0], p[1], p[2]};
  }
  __syncthreads();
  if (tid >= 64) return;
  st = wave_joined(st, c);
  float log_l = 0.f;
  if (lane == 0) log_l = finish_row(a, t, row, st);
  log_l = __shfl(log_l, 0, 64);
  // Every split's candidates lie in order, and a split's come before the next one's: the largest of the splits' first ones, at the
  // first split that has it, again and again.
  const uint64_t* next = list + (lane < a.splits ? lane * a.top : 0);
  int left = lane < a.splits ? a.top : 0;
  for (int rank = 0; rank < a.top; ++rank) {
    const uint64_t key = left > 0 ? *next : 0;
    const uint32_t best = wave_max_u32((uint32_t)(key >> 32));
    if (lane != __ffsll(__ballot((uint32_t)(key >> 32) == best)) - 1) continue;
    store_top(a, t, rank, key, st.m, log_l);
    ++next;
    --left;
  }
}

// -- the gradient -----------------------------------------------------------------------------------------------------
struct LogprobBwdArgs {
  const void* logits;
  long stride;
  int vocab, chunks;
  const int64_t* targets;
  float inv_t;
  const float* stats;          // [T, 3]
  const float* dlogprob;       // [T] or nullptr
  const float* dentropy;       // [T] or nullptr
  void* grad;                  // [T, V] rows `grad_stride` elements apart
  long grad_stride;
};

template <class T>
struct Grad {
  float m, c, a, b, log2_l;
  // p (-g - h (ln p + H)) / temperature, with ln p = y ln 2, y = (x - m) c - log2 l
  __device__ __forceinline__ float operator()(float x) const {
    float y = ((x < kLowest ? kLowest : x) - m) * c - log2_l;
    y = y < -1000.f ? -1000.f : y;                           // (weighs nothing; its product with b stays finite)
    return fast_exp2(y) * (a + b * y);
  }
};

constexpr int kBwdVecs = 4;    // pieces a thread

// Workgroup (row, chunk of 256 x 4 pieces), chunks next to each other; the head's and tail's elements go with chunk 0.
template <class T>
__global__ __launch_bounds__(256) void logprob_bwd_kernel(LogprobBwdArgs a) {
  constexpr int N = Vec<T>::n;
  const long t = blockIdx.x / a.chunks;
  const int chunk = blockIdx.x % a.chunks, tid = threadIdx.x;
  const T* row = static_cast<const T*>(a.logits) + t * a.stride;
  T* to = static_cast<T*>(a.grad) + t * a.grad_stride;
  const RowShape<T> shape(row, a.vocab);
  int64_t target = a.targets[t];
  if (target < 0 || target >= a.vocab) target = -1;
  const float g = a.dlogprob != nullptr && target >= 0 ? a.dlogprob[t] : 0.f;
  const float h = a.dentropy != nullptr ? a.dentropy[t] : 0.f;
  const float* stats = a.stats + 3 * t;
  Grad<T> f;
  f.m = stats[0];
  f.c = a.inv_t * kLog2e;
  f.log2_l = stats[1] * kLog2e;
  f.a = (-g - h * stats[2]) * a.inv_t;
  f.b = -h * a.inv_t * kLn2;
  const float hit = g * a.inv_t;
  const int tgt = (int)target;
  const T* body = row + shape.head;
  const bool aligned = (((uintptr_t)(to + shape.head)) & 15) == 0;
  const int first = chunk * 256 * kBwdVecs + tid;
  float x[kBwdVecs][N];
#pragma unroll
  for (int k = 0; k < kBwdVecs; ++k)
    if (first + 256 * k < shape.vecs) Vec<T>::ld(body + (long)(first + 256 * k) * N, x[k]);
#pragma unroll
  for (int k = 0; k < kBwdVecs; ++k) {
    const int v = first + 256 * k;
    if (v >= shape.vecs) break;
    const int at = shape.head + v * N;
#pragma unroll
    for (int i = 0; i < N; ++i) x[k][i] = f(x[k][i]) + (at + i == tgt ? hit : 0.f);
    if (aligned) {
      if constexpr (N == 8) {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(x[k][2 * i], x[k][2 * i + 1]);
        __builtin_nontemporal_store(w, reinterpret_cast<u32x4*>(to + at));
      } else {
        __builtin_nontemporal_store(floatx4{x[k][0], x[k][1], x[k][2], x[k][3]}, reinterpret_cast<floatx4*>(to + at));
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) to[at + i] = (T)x[k][i];
    }
  }
  if (chunk != 0) return;
  const int tail = shape.head + shape.vecs * N;
  int lone = -1;
  if (tid < shape.head) lone = tid;
  if (tid >= 64 && tid - 64 < a.vocab - tail) lone = tail + tid - 64;
  if (lone >= 0) to[lone] = (T)(f((float)row[lone]) + (lone == tgt ? hit : 0.f));
}

// Splits of a row: as many workgroups as fill the GPU twice over, of at least 512 pieces each, and as many as the join's list
// holds.
static int logprob_splits(int tokens, int vocab, int elem, int top) {
  const long vecs = ((long)vocab * elem + 15) / 16;
  long n = tokens >= 512 ? 1 : (1024 + tokens - 1) / tokens;
  const long most = (vecs + kRowThreads - 1) / kRowThreads;
  n = n < most ? n : most;
  n = n < 64 ? n : 64;
  if (top > 0) n = n < kMergeMax / top ? n : kMergeMax / top;
  return n < 1 ? 1 : (int)n;
}

}  // namespace abkv

using namespace abkv;

constexpr long kMaxGroups = 0xFFFFFFFFL;       // work items of a launch fit 32 bits

template <class T>
static void launch_logprobs(const LogprobArgs& a, int tokens, bool entropy, hipStream_t stream) {
  if (entropy) hipLaunchKernelGGL((logprob_kernel<T, true>), dim3(tokens * a.splits), dim3(kRowThreads), 0, stream, a);
  else hipLaunchKernelGGL((logprob_kernel<T, false>), dim3(tokens * a.splits), dim3(kRowThreads), 0, stream, a);
  if (a.splits > 1) hipLaunchKernelGGL(logprob_join_kernel<T>, dim3(tokens), dim3(256), 0, stream, a);
}

extern "C" {

size_t abkv_token_logprobs_workspace_size(int num_tokens, int vocab, int f32, int top) {
  if (num_tokens <= 0 || vocab <= 0 || top < 0) return 0;
  const int splits = logprob_splits(num_tokens, vocab, f32 ? 4 : 2, top);
  return splits == 1 ? 0 : (size_t)num_tokens * splits * (top * sizeof(uint64_t) + 4 * sizeof(float));
}

int abkv_token_logprobs(int f32, const void* logits, long stride, int num_tokens, int vocab, const int64_t* targets,
                        float temperature, int top, float* logprob, float* entropy, float* stats, int64_t* top_ids,
                        float* top_logprobs, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  if (num_tokens <= 0) return 0;
  const int elem = f32 ? 4 : 2;
  if (vocab <= 0 || vocab > (1 << 30) || num_tokens > kMaxGroups / kRowThreads / 2 || logits == nullptr ||
      ((uintptr_t)logits & (elem - 1)) || targets == nullptr || logprob == nullptr || !temperature_ok(temperature) || top < 0 ||
      top > kTopMax || top > vocab || (top > 0 && (top_ids == nullptr || top_logprobs == nullptr)) ||
      (num_tokens > 1 && stride < vocab))
    return (int)hipErrorInvalidValue;
  const size_t need = abkv_token_logprobs_workspace_size(num_tokens, vocab, f32, top);
  if (need > 0 && (workspace == nullptr || ((uintptr_t)workspace & 7) || workspace_bytes < need))
    return (int)hipErrorInvalidValue;
  LogprobArgs a;
  a.logits = logits;
  a.stride = stride;
  a.vocab = vocab;
  a.targets = targets;
  a.inv_t = 1.f / temperature;
  a.top = top;
  a.logprob = logprob;
  a.entropy = entropy;
  a.stats = stats;
  a.top_ids = top_ids;
  a.top_logprobs = top_logprobs;
  a.splits = logprob_splits(num_tokens, vocab, elem, top);
  const int n = 16 / elem;
  const int vecs = (vocab + n - 1) / n;                      // at least the whole pieces of any row
  a.split_vecs = (vecs + a.splits - 1) / a.splits;
  a.part_top = static_cast<uint64_t*>(workspace);
  a.part = reinterpret_cast<float*>(a.part_top + (size_t)num_tokens * a.splits * top);
  const bool with_entropy = entropy != nullptr || stats != nullptr;
  if (f32) launch_logprobs<float>(a, num_tokens, with_entropy, stream);
  else launch_logprobs<__bf16>(a, num_tokens, with_entropy, stream);
  return (int)hipGetLastError();
}

int abkv_token_logprobs_bwd(int f32, const void* logits, long stride, int num_tokens, int vocab, const int64_t* targets,
                            float temperature, const float* stats, const float* dlogprob, const float* dentropy, void* dlogits,
                            long grad_stride, hipStream_t stream) {
  if (num_tokens <= 0) return 0;
  const int elem = f32 ? 4 : 2;
  if (vocab <= 0 || vocab > (1 << 30) || logits == nullptr || dlogits == nullptr ||
      (((uintptr_t)logits | (uintptr_t)dlogits) & (elem - 1)) || targets == nullptr || stats == nullptr ||
      !temperature_ok(temperature) || (num_tokens > 1 && (stride < vocab || grad_stride < vocab)))
    return (int)hipErrorInvalidValue;
  LogprobBwdArgs a;
  a.logits = logits;
  a.stride = stride;
  a.vocab = vocab;
  a.targets = targets;
  a.inv_t = 1.f / temperature;
  a.stats = stats;
  a.dlogprob = dlogprob;
  a.dentropy = dentropy;
  a.grad = dlogits;
  a.grad_stride = grad_stride;
  const int n = 16 / elem, vecs = (vocab + n - 1) / n;
  a.chunks = (vecs + 256 * kBwdVecs - 1) / (256 * kBwdVecs);
  if ((long)a.chunks * num_tokens > kMaxGroups / 256) return (int)hipErrorInvalidValue;
  const dim3 grid((unsigned)(a.chunks * num_tokens));
  if (f32) hipLaunchKernelGGL(logprob_bwd_kernel<float>, grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL(logprob_bwd_kernel<__bf16>, grid, dim3(256), 0, stream, a);
  return (int)hipGetLastError();
}

}  // extern "C"

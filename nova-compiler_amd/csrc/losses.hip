// Losses over token log-probabilities, beside nova.sce: token_logp, the
// clipped policy loss with a KL term, and the paired preference loss, each
// with the gradient of the logits.  For a row x with label y
//   lse = log sum exp x,  lp = x[y] - lse,  d lp / d x = onehot(y) - exp(x - lse).
//
// All are HBM-bound.  A row is held on chip (in registers, 16 bytes at a time)
// between the maximum, the sum and the gradient, so the policy loss reads the
// logits once and writes the gradient once.  The preference loss knows a row's
// slope only when both sequences of the pair are summed, so its gradient is
// a second pass over the logits, from the last row to the first: some of the rows
// read last are still cached beyond the L2s (8192 x 50304 bf16 326 us, 361 from the
// first row on; 4096 x 32000 bf16 100 either way, 2048 x 50304 f32 169 and 166).
//
// 16-bit logits are widened exactly; maxima, sums and log-probabilities are
// f32, sums over rows 64 bits; the gradient is rounded once, to the logits'
// type.
//
// Measured, of the bytes that have to move: policy loss 8192 x 50304 f32, 80% of
// the rows valid, 525 us (5.65 TB/s, 0.87 of the copy's 6.5); bf16 263 us;
// token_logp 8192 x 50304 190 us in f32 (6.95 TB/s), 96 us in bf16; preference
// loss 8192 x 50304 bf16, 70% valid, 327 us (4.3 TB/s counting the logits once,
// 6.1 as read).  Small calls are their launches' time on the host.
#include <hip/hip_runtime.h>

#include <math.h>

#include "gemm_common.h"
#include "wave.h"

namespace nova_hip {
namespace {

using gemm::u32x4;

constexpr float kL2e = 1.4426950408889634f;

// kPairs: kLogp ahead of a second pass over the logits.
enum Mode { kLogp, kPairs, kPolicy };

struct RowArgs {
  const void *logits;
  void *grad;  // may be null
  const int32_t *labels;
  const float *old_logp, *ref_logp, *advantage, *weight;  // policy; ref may be null
  float *logp, *lse, *row_loss, *slope;                   // each may be null
  int64_t sx, sg;                                         // row strides (elements)
  int rows, C;
  float lo, hi, kl, grad_scale;
};

typedef uint32_t u32x4_at4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4_at2 __attribute__((ext_vector_type(4), aligned(2)));

// One 16-byte chunk of a row: 4 f32 or 8 16-bit values, at any alignment of
// the elements' own.
template <int DT>
struct Chunk {
  static constexpr int kE = DT == NOVA_HIP_DT_F32 ? 4 : 8;
  typedef typename std::conditional<DT == NOVA_HIP_DT_F32, float, uint16_t>::type T;

  static __device__ __forceinline__ u32x4 load(const T *p) {
    if constexpr (DT == NOVA_HIP_DT_F32)
      return __builtin_nontemporal_load(reinterpret_cast<const u32x4_at4 *>(p));
    else return __builtin_nontemporal_load(reinterpret_cast<const u32x4_at2 *>(p));
  }
  // With KEEP the line stays in the caches for a second pass.
  template <bool KEEP>
  static __device__ __forceinline__ u32x4 load_as(const T *p) {
    if constexpr (!KEEP) return load(p);
    else if constexpr (DT == NOVA_HIP_DT_F32) return *reinterpret_cast<const u32x4_at4 *>(p);
    else return *reinterpret_cast<const u32x4_at2 *>(p);
  }
  static __device__ __forceinline__ void store(T *p, u32x4 v) {
    if constexpr (DT == NOVA_HIP_DT_F32)
      __builtin_nontemporal_store(v, reinterpret_cast<u32x4_at4 *>(p));
    else __builtin_nontemporal_store(v, reinterpret_cast<u32x4_at2 *>(p));
  }
  static __device__ __forceinline__ u32x4 none() {
    const uint32_t w = DT == NOVA_HIP_DT_F32 ? 0xff800000u : DT == NOVA_HIP_DT_BF16 ? 0xff80ff80u : 0xfc00fc00u;
    return u32x4{w, w, w, w};
  }
  static __device__ __forceinline__ float at(const u32x4 &v, int e) {
    if constexpr (DT == NOVA_HIP_DT_F32) return __uint_as_float(v[e]);
    else if constexpr (DT == NOVA_HIP_DT_BF16)
      return __uint_as_float(e & 1 ? v[e >> 1] & 0xffff0000u : v[e >> 1] << 16);
    else return (float)__builtin_bit_cast(gemm::f16x2v, (uint32_t)v[e >> 1])[e & 1];
  }
  static __device__ __forceinline__ float widen(T x) {
    if constexpr (DT == NOVA_HIP_DT_F32) return x;
    else if constexpr (DT == NOVA_HIP_DT_BF16) return __uint_as_float((uint32_t)x << 16);
    else return (float)__builtin_bit_cast(_Float16, x);
  }
  static __device__ __forceinline__ T narrow(float x) {
    if constexpr (DT == NOVA_HIP_DT_F32) return x;
    else if constexpr (DT == NOVA_HIP_DT_BF16) return gemm::to_bf16(x);
    else return gemm::to_f16(x);
  }
  // f(e) for the kE values, packed.
  template <typename F>
  static __device__ __forceinline__ u32x4 make(F f) {
    u32x4 v;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (DT == NOVA_HIP_DT_F32) v[j] = __float_as_uint(f(j));
      else if constexpr (DT == NOVA_HIP_DT_BF16) v[j] = gemm::pack_bf16(f(2 * j), f(2 * j + 1));
      else v[j] = gemm::pack_f16(f(2 * j), f(2 * j + 1));
    }
    return v;
  }
};

// The packed row is what stays in registers from one phase to the next: without
// this the compiler keeps 16-bit rows widened, twice the registers.
template <int NC>
__device__ __forceinline__ void keep(u32x4 (&v)[NC]) {
#pragma unroll
  for (int i = 0; i < NC; ++i) asm volatile("" : "+v"(v[i]));
}

// Over the TH threads of a workgroup (or one wave), in a fixed order.
template <int TH, bool MAX>
__device__ __forceinline__ float group_reduce(float v, float *red) {
  v = MAX ? wave_max(v) : wave_sum(v);
  if constexpr (TH > 64) {
    __syncthreads();  // the last use of red is over
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < TH / 64; ++i) v = MAX ? fmaxf(v, red[i]) : v + red[i];
  }
  return v;
}

// exp(x - m) as exp2 of one rounded product; m finite.
__device__ __forceinline__ float exp_diff(float x, float m) {
  return __builtin_amdgcn_exp2f((x - m) * kL2e);
}

// A row's inputs.  Every thread reads them ahead of the reductions' barriers, so
// that logp and row_loss may be written over them.
struct Row {
  float old_logp, ref_logp, advantage, weight;
  __device__ __forceinline__ void load(const RowArgs &a, int row) {
    old_logp = a.old_logp[row];
    ref_logp = a.ref_logp ? a.ref_logp[row] : 0.0f;
    advantage = a.advantage[row];
    weight = a.weight[row];
  }
};

// A row's slope d loss / d lp and its loss, from its log-probability.
__device__ __forceinline__ void policy_row(const RowArgs &a, const Row &in, float lp, float &loss,
                                           float &slope) {
  const float w = in.weight, adv = in.advantage;
  const float ratio = expf(lp - in.old_logp);
  const float plain = ratio * adv;
  // fminf / fmaxf drop a NaN, which the products with the ratio bring back.
  const float clipped = fminf(fmaxf(ratio, a.lo), a.hi) * adv;
  const bool take = !(clipped < plain);  // the clip's gradient is zero where it is the lesser
  float l = -(take ? plain : clipped);
  float g = take ? -plain : 0.0f;
  if (ratio != ratio) l = g = ratio;
  if (a.ref_logp) {
    const float d = in.ref_logp - lp;
    // exp(d) - 1 - d cancels near 0: expm1.
    const float em1 = expm1f(d);
    l += a.kl * (em1 - d);
    g -= a.kl * em1;
  }
  // Weight 0: nothing of an infinite or NaN loss either.
  loss = w == 0.0f ? 0.0f : w * l;
  slope = w == 0.0f ? 0.0f : w * g;
}

template <int DT, int TH>
__device__ __forceinline__ void zero_row(typename Chunk<DT>::T *g, int C, int tid) {
  typedef Chunk<DT> X;
  const int nc = C / X::kE, tail = C - nc * X::kE;
  for (int c = tid; c < nc; c += TH) X::store(g + (int64_t)c * X::kE, u32x4{0, 0, 0, 0});
  if (tid < tail) g[(int64_t)nc * X::kE + tid] = typename X::T(0);
}

// TH threads per row, NC chunks per thread; TH == 64: four rows a workgroup.
template <int DT, int TH, int NC, int MODE>
__global__ __launch_bounds__(TH == 64 ? 256 : TH, TH >= 512 ? 4 : 1) void logp_row_kernel(RowArgs a) {
  typedef Chunk<DT> X;
  typedef typename X::T T;
  __shared__ float red[TH > 64 ? TH / 64 : 1];
  const int tid = TH == 64 ? threadIdx.x & 63 : threadIdx.x;
  const int row = TH == 64 ? blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
  if (row >= a.rows) return;
  const int y = __builtin_amdgcn_readfirstlane(a.labels[row]);
  const bool skip = y < 0 || (MODE == kPolicy && y >= a.C && a.weight[row] == 0.0f);
  const T *x = static_cast<const T *>(a.logits) + row * a.sx;
  T *g = a.grad ? static_cast<T *>(a.grad) + row * a.sg : nullptr;
  const int nc = a.C / X::kE, tail = a.C - nc * X::kE;
  if (skip) {
    // No part of the loss: the logits are not read.
    if (tid == 0) {
      if (a.logp) a.logp[row] = 0.0f;
      if (a.lse) a.lse[row] = 0.0f;
      if (a.slope) a.slope[row] = 0.0f;
      if (MODE == kPolicy) a.row_loss[row] = 0.0f;
    }
    if (MODE == kPolicy && g) zero_row<DT, TH>(g, a.C, tid);
    return;
  }
  Row in = {};
  if constexpr (MODE == kPolicy) in.load(a, row);
  u32x4 v[NC];
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const int c = tid + TH * i;
    v[i] = c < nc ? X::template load_as<MODE == kPairs>(x + c * X::kE) : X::none();  // -inf: no part of the sum
  }
  float xt = -INFINITY;  // this thread's value behind the last chunk
  if (tid < tail) xt = X::widen(x[nc * X::kE + tid]);
  const float xy = y < a.C ? X::widen(x[y]) : __builtin_nanf("");

  float m = xt;
#pragma unroll
  for (int i = 0; i < NC; ++i)
#pragma unroll
    for (int e = 0; e < X::kE; ++e) m = fmaxf(m, X::at(v[i], e));
  keep(v);
  m = group_reduce<TH, true>(m, red);
  const float mm = m == -INFINITY ? 0.0f : m;  // a row of nothing but -inf: sum 0, lse -inf
  float s = tid < tail ? exp_diff(xt, mm) : 0.0f;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    float p = 0.0f;
#pragma unroll
    for (int e = 0; e < X::kE; ++e) p += exp_diff(X::at(v[i], e), mm);
    s += p;
  }
  keep(v);
  s = group_reduce<TH, false>(s, red);
  const float ls = logf(s), lse = mm + ls;
  const float lp = (xy - mm) - ls;
  if constexpr (MODE != kPolicy) {
    if (tid == 0) {
      if (a.logp) a.logp[row] = lp;
      if (a.lse) a.lse[row] = lse;
      if (a.slope) a.slope[row] = 0.0f;
    }
    return;
  } else {
    float loss, slope;
    policy_row(a, in, lp, loss, slope);
    if (tid == 0) {
      a.logp[row] = lp;
      a.row_loss[row] = loss;
    }
    if (!g) return;
    if (in.weight == 0.0f) return zero_row<DT, TH>(g, a.C, tid);
    slope *= a.grad_scale;
    const float k = -slope / s;
    auto value = [&](float xv, int col) __attribute__((always_inline)) {
      const float p = k * exp_diff(xv, mm);
      return col == y ? p + slope : p;
    };
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int c = tid + TH * i;
      if (c < nc)
        X::store(g + c * X::kE,
                 X::make([&](int e) { return value(X::at(v[i], e), c * X::kE + e); }));
    }
    if (tid < tail) g[nc * X::kE + tid] = X::narrow(value(xt, nc * X::kE + tid));
  }
}

// Rows beyond the registers: one pass with a running maximum and sum, a second
// one for the gradient.
template <int DT, int MODE>
__global__ __launch_bounds__(512) void logp_long_kernel(RowArgs a) {
  typedef Chunk<DT> X;
  typedef typename X::T T;
  constexpr int TH = 512;
  __shared__ float red[TH / 64];
  const int tid = threadIdx.x, row = blockIdx.x;
  const int y = __builtin_amdgcn_readfirstlane(a.labels[row]);
  const bool skip = y < 0 || (MODE == kPolicy && y >= a.C && a.weight[row] == 0.0f);
  const T *x = static_cast<const T *>(a.logits) + row * a.sx;
  T *g = a.grad ? static_cast<T *>(a.grad) + row * a.sg : nullptr;
  const int nc = a.C / X::kE, tail = a.C - nc * X::kE;
  if (skip) {
    if (tid == 0) {
      if (a.logp) a.logp[row] = 0.0f;
      if (a.lse) a.lse[row] = 0.0f;
      if (a.slope) a.slope[row] = 0.0f;
      if (MODE == kPolicy) a.row_loss[row] = 0.0f;
    }
    if (MODE == kPolicy && g) zero_row<DT, TH>(g, a.C, tid);
    return;
  }
  Row in = {};
  if constexpr (MODE == kPolicy) in.load(a, row);
  const float xt = tid < tail ? X::widen(x[(int64_t)nc * X::kE + tid]) : -INFINITY;
  const float xy = y < a.C ? X::widen(x[y]) : __builtin_nanf("");
  float m = xt, s = tid < tail && xt > -INFINITY ? 1.0f : 0.0f;
  if (xt != xt) s = xt;
#pragma unroll 4
  for (int c = tid; c < nc; c += TH) {
    const u32x4 v = X::template load_as<MODE != kLogp>(x + (int64_t)c * X::kE);
    float t = X::at(v, 0);
#pragma unroll
    for (int e = 1; e < X::kE; ++e) t = fmaxf(t, X::at(v, e));
    if (t > m) {
      s *= m == -INFINITY ? (s != s ? s : 0.0f) : exp_diff(m, t);
      m = t;
    }
    const float mu = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int e = 0; e < X::kE; ++e) s += exp_diff(X::at(v, e), mu);
  }
  const float mg = group_reduce<TH, true>(m, red);
  const float mm = mg == -INFINITY ? 0.0f : mg;
  s = m == -INFINITY ? (s != s ? s : 0.0f) : s * exp_diff(m, mm);
  s = group_reduce<TH, false>(s, red);
  const float ls = logf(s), lse = mm + ls;
  const float lp = (xy - mm) - ls;
  if constexpr (MODE != kPolicy) {
    if (tid == 0) {
      if (a.logp) a.logp[row] = lp;
      if (a.lse) a.lse[row] = lse;
      if (a.slope) a.slope[row] = 0.0f;
    }
  } else {
    float loss, slope;
    policy_row(a, in, lp, loss, slope);
    if (tid == 0) {
      a.logp[row] = lp;
      a.row_loss[row] = loss;
    }
    if (!g) return;
    if (in.weight == 0.0f) return zero_row<DT, TH>(g, a.C, tid);
    slope *= a.grad_scale;
    const float k = -slope / s;
    auto value = [&](float xv, int64_t col) __attribute__((always_inline)) {
      const float p = k * exp_diff(xv, mm);
      return col == y ? p + slope : p;
    };
#pragma unroll 4
    for (int c = tid; c < nc; c += TH) {
      const u32x4 v = X::load(x + (int64_t)c * X::kE);
      X::store(g + (int64_t)c * X::kE,
               X::make([&](int e) { return value(X::at(v, e), (int64_t)c * X::kE + e); }));
    }
    if (tid < tail) {
      const int64_t col = (int64_t)nc * X::kE + tid;
      g[col] = X::narrow(value(xt, col));
    }
  }
}

// out[0] = sum of v[0 .. n) * scale by TH threads, in 64 bits: each its own
// stride, then the threads in the order of a fixed tree.
template <int TH>
__device__ __forceinline__ void sum_losses(const float *v, int n, double scale, float *out) {
  __shared__ double part[TH];
  double s = 0.0;
  for (int i = threadIdx.x; i < n; i += TH) s += (double)v[i];
  part[threadIdx.x] = s;
  for (int d = TH / 2; d > 0; d >>= 1) {
    __syncthreads();
    if (threadIdx.x < d) part[threadIdx.x] += part[threadIdx.x + d];
  }
  if (threadIdx.x == 0) out[0] = (float)(part[0] * scale);
}
__global__ __launch_bounds__(1024) void loss_sum_kernel(const float *v, int n, double scale,
                                                        float *out) {
  sum_losses<1024>(v, n, scale, out);
}

struct PairArgs {
  const float *logp;  // [R]
  float *slope;       // [R]
  const int32_t *off;
  const float *ref;
  float *seq_logp, *pair_loss;
  int R, P;
  double beta, smoothing, grad_scale;
};

// One workgroup per pair: sums of its two sequences' log-probabilities (64
// bits, fixed order), the pair's loss, and its rows' slopes.
__global__ __launch_bounds__(256) void preference_pair_kernel(PairArgs a) {
  __shared__ double part[256];
  const int pair = blockIdx.x, tid = threadIdx.x;
  // Ahead of the barriers: seq_logp may be written over them.
  const float ref0 = a.ref[2 * pair], ref1 = a.ref[2 * pair + 1];
  double seq[2];
  int s[2], e[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    s[j] = min(max(a.off[2 * pair + j], 0), a.R);
    e[j] = min(max(a.off[2 * pair + j + 1], 0), a.R);
    double x = 0.0;
    for (int i = s[j] + tid; i < e[j]; i += 256) x += (double)a.logp[i];
    __syncthreads();
    part[tid] = x;
    for (int d = 128; d > 0; d >>= 1) {
      __syncthreads();
      if (tid < d) part[tid] += part[tid + d];
    }
    __syncthreads();
    seq[j] = part[0];
  }
  const double h = a.beta * ((seq[0] - (double)ref0) - (seq[1] - (double)ref1));
  const double soft = log1p(exp(-fabs(h)));
  const double neg = 1.0 / (1.0 + exp(h));  // sigmoid(-h)
  const double c = a.beta * (a.smoothing * (1.0 - neg) - (1.0 - a.smoothing) * neg) / a.P;
  if (tid < 2) a.seq_logp[2 * pair + tid] = (float)seq[tid];
  if (tid == 0)
    a.pair_loss[pair] = (float)((1.0 - a.smoothing) * (soft + fmax(-h, 0.0)) +
                                a.smoothing * (soft + fmax(h, 0.0)));
  const float up = (float)(c * a.grad_scale);
#pragma unroll
  for (int j = 0; j < 2; ++j)
    for (int i = s[j] + tid; i < e[j]; i += 256) a.slope[i] = j ? -up : up;
}

struct GradArgs {
  const void *logits;
  void *grad;
  const int32_t *labels;
  const float *logp, *lse, *slope;
  int64_t sx, sg;
  int rows, C, pairs;
  const float *pair_loss;
  float *loss;
};

// grad[row] = slope (onehot(label) - exp(x - lse)), from the last row to the
// first.  The first workgroup also sums the pairs' losses (a launch of its own
// would take longer than a small call's other kernels).
template <int DT, int TH>
__global__ __launch_bounds__(TH == 64 ? 256 : TH) void logits_grad_kernel(GradArgs a) {
  typedef Chunk<DT> X;
  typedef typename X::T T;
  const int tid = TH == 64 ? threadIdx.x & 63 : threadIdx.x;
  if (blockIdx.x == 0)
    sum_losses<TH == 64 ? 256 : TH>(a.pair_loss, a.pairs, 1.0 / (double)a.pairs, a.loss);
  const int r = TH == 64 ? blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x;
  if (r >= a.rows) return;
  const int row = a.rows - 1 - r;
  const int y = a.labels[row];
  const float slope = y < 0 ? 0.0f : a.slope[row], lse = a.lse[row];
  const T *x = static_cast<const T *>(a.logits) + row * a.sx;
  T *g = static_cast<T *>(a.grad) + row * a.sg;
  const int nc = a.C / X::kE, tail = a.C - nc * X::kE;
  const bool none = slope == 0.0f;  // the logits are not read
  // log p = x - lse, or (x - x[y]) + lp where that is the smaller number: an lse
  // of 10^4 is rounded by 2^-11, and the probabilities with it.
  float pivot = lse, add = 0.0f;
  if (fabsf(lse) > 64.0f && !none && y < a.C && fabsf(a.logp[row]) < fabsf(lse)) {
    pivot = X::widen(x[y]);
    add = a.logp[row];
  }
  auto value = [&](float xv, int64_t col) __attribute__((always_inline)) {
    const float p = -slope * __builtin_amdgcn_exp2f(((xv - pivot) + add) * kL2e);
    return col == y ? p + slope : p;
  };
#pragma unroll 4
  for (int c = tid; c < nc; c += TH) {
    u32x4 o = {0, 0, 0, 0};
    if (!none) {
      const u32x4 v = X::template load_as<true>(x + (int64_t)c * X::kE);
      o = X::make([&](int e) { return value(X::at(v, e), (int64_t)c * X::kE + e); });
    }
    X::store(g + (int64_t)c * X::kE, o);
  }
  if (tid < tail) {
    const int64_t col = (int64_t)nc * X::kE + tid;
    g[col] = none ? T(0) : X::narrow(value(X::widen(x[col]), col));
  }
}

template <int DT, int MODE>
void launch_rows_t(const RowArgs &a, hipStream_t s) {
  const int chunks = (a.C + Chunk<DT>::kE - 1) / Chunk<DT>::kE;
  const unsigned g = (unsigned)a.rows, g4 = (unsigned)((a.rows + 3) / 4);
  auto go = [&](auto th, auto nc) {
    constexpr int TH = decltype(th)::value, NC = decltype(nc)::value;
    hipLaunchKernelGGL((logp_row_kernel<DT, TH, NC, MODE>), dim3(TH == 64 ? g4 : g),
                       dim3(TH == 64 ? 256 : TH), 0, s, a);
  };
  using std::integral_constant;
#define NOVA_ROWS(TH, NC) go(integral_constant<int, TH>(), integral_constant<int, NC>())
  // With a gradient to write, few wide workgroups per CU serve HBM better (1024
  // threads at 8192 x 50304 f32, 8192 x 50304 bf16, 4096 x 32000 f32: 526, 270
  // and 172 us; 512 threads: 554, 278 and 178); to read alone, narrower ones
  // (8192 x 50304 bf16 97 us, 105 with 1024; 4096 x 32000 bf16 29 and 36).
  if (chunks <= 64 * 4) NOVA_ROWS(64, 4);
  else if (chunks <= 256 * 4) NOVA_ROWS(256, 4);
  else if (chunks <= 512 * 4) NOVA_ROWS(512, 4);
  else if (chunks <= 512 * 8) NOVA_ROWS(512, 8);
  else if (chunks <= 1024 * 8) {
    if constexpr (MODE == kPolicy) NOVA_ROWS(1024, 8);
    else if (chunks <= 512 * 13) NOVA_ROWS(512, 13);
    else NOVA_ROWS(512, 16);
  } else if (chunks <= 1024 * 13) NOVA_ROWS(1024, 13);
  else hipLaunchKernelGGL((logp_long_kernel<DT, MODE>), dim3(g), dim3(512), 0, s, a);
#undef NOVA_ROWS
}
template <int MODE>
int32_t launch_rows(const RowArgs &a, int dt, const char *what, hipStream_t s) {
  if (dt == NOVA_HIP_DT_F32) launch_rows_t<NOVA_HIP_DT_F32, MODE>(a, s);
  else if (dt == NOVA_HIP_DT_BF16) launch_rows_t<NOVA_HIP_DT_BF16, MODE>(a, s);
  else launch_rows_t<NOVA_HIP_DT_F16, MODE>(a, s);
  return check_hip(hipGetLastError(), what);
}

int32_t launch_loss_sum(const float *v, int64_t n, double scale, float *out, const char *what,
                        hipStream_t s) {
  hipLaunchKernelGGL(loss_sum_kernel, dim3(1), dim3(1024), 0, s, v, (int)n, scale, out);
  return check_hip(hipGetLastError(), what);
}

RowArgs row_args(const TokenLossProblem &p) {
  RowArgs a = {};
  a.logits = p.logits;
  a.grad = p.grad;
  a.labels = p.labels;
  a.sx = p.sx;
  a.sg = p.sg;
  a.rows = (int)p.rows;
  a.C = (int)p.C;
  return a;
}

int32_t in_range(const TokenLossProblem &p, const char *w) {
  if (p.rows > 0x7fffffff - (1 << 20) || p.C > 0x7fffffff - (1 << 20))
    return fail(NOVA_HIP_ERANGE, "%s: rows or classes exceed 2^31 - 2^20", w);
  // A grid's dimension holds less than 2^32 threads: 64 to a row of 1024 f32 or
  // 2048 16-bit classes, at most 1024 to longer ones.
  const int64_t threads = p.C <= (p.dt == NOVA_HIP_DT_F32 ? 1024 : 2048) ? 64 : 1024;
  if (p.rows * threads >= (int64_t)1 << 32)
    return fail(NOVA_HIP_ERANGE, "%s: %lld rows of %lld classes are more than one grid holds", w,
                (long long)p.rows, (long long)p.C);
  return NOVA_HIP_SUCCESS;
}

template <int DT>
void launch_grad_t(const GradArgs &a, hipStream_t s) {
  // A wave per row as long as four strides of it cover the row; 1024 threads to
  // the longest (8192 x 50304 bf16: 324 us, 330 with 512, 341 with 256).
  if (a.C <= 256 * Chunk<DT>::kE)
    hipLaunchKernelGGL((logits_grad_kernel<DT, 64>), dim3((unsigned)((a.rows + 3) / 4)), dim3(256), 0,
                       s, a);
  else if (a.C <= 2048 * Chunk<DT>::kE)
    hipLaunchKernelGGL((logits_grad_kernel<DT, 512>), dim3((unsigned)a.rows), dim3(512), 0, s, a);
  else
    hipLaunchKernelGGL((logits_grad_kernel<DT, 1024>), dim3((unsigned)a.rows), dim3(1024), 0, s, a);
}

}  // namespace

int32_t launch_token_logp(const TokenLossProblem &p, float *logp, float *lse, hipStream_t s) {
  int32_t rc = in_range(p, "token_logp");
  if (rc || p.rows == 0) return rc;
  RowArgs a = row_args(p);
  a.logp = logp;
  a.lse = lse;
  return launch_rows<kLogp>(a, p.dt, "token_logp launch", s);
}

int32_t launch_policy_loss(const PolicyProblem &p, hipStream_t s) {
  int32_t rc = in_range(p.t, "policy_loss");
  if (rc) return rc;
  RowArgs a = row_args(p.t);
  a.old_logp = p.old_logp;
  a.ref_logp = p.ref_logp;
  a.advantage = p.advantage;
  a.weight = p.weight;
  a.logp = p.logp;
  a.row_loss = p.row_loss;
  a.lo = 1.0f - p.clip_low;
  a.hi = 1.0f + p.clip_high;
  a.kl = p.kl_coef;
  a.grad_scale = p.grad_scale;
  if (p.t.rows > 0 && (rc = launch_rows<kPolicy>(a, p.t.dt, "policy_loss launch", s))) return rc;
  return launch_loss_sum(p.row_loss, p.t.rows, 1.0, p.loss, "policy_loss sum launch", s);
}

int32_t launch_preference_loss(const PreferenceProblem &p, hipStream_t s) {
  int32_t rc = in_range(p.t, "preference_loss");
  if (rc) return rc;
  RowArgs a = row_args(p.t);
  a.grad = nullptr;
  a.logp = p.logp;
  a.lse = p.lse;
  a.slope = p.slope;
  const bool grad = p.t.grad && p.t.rows > 0;
  if (p.t.rows > 0 && (rc = grad ? launch_rows<kPairs>(a, p.t.dt, "preference_loss launch", s)
                                 : launch_rows<kLogp>(a, p.t.dt, "preference_loss launch", s)))
    return rc;
  const PairArgs b = {p.logp, p.slope, p.offsets, p.ref_logp, p.seq_logp, p.pair_loss,
                      (int)p.t.rows, (int)p.pairs, p.beta, p.smoothing, p.grad_scale};
  hipLaunchKernelGGL(preference_pair_kernel, dim3((unsigned)p.pairs), dim3(256), 0, s, b);
  if ((rc = check_hip(hipGetLastError(), "preference_loss pair launch"))) return rc;
  if (!grad)
    return launch_loss_sum(p.pair_loss, p.pairs, 1.0 / (double)p.pairs, p.loss,
                           "preference_loss sum launch", s);
  const GradArgs g = {p.t.logits, p.t.grad, p.t.labels, p.logp, p.lse, p.slope, p.t.sx, p.t.sg,
                      (int)p.t.rows, (int)p.t.C, (int)p.pairs, p.pair_loss, p.loss};
  if (p.t.dt == NOVA_HIP_DT_F32) launch_grad_t<NOVA_HIP_DT_F32>(g, s);
  else if (p.t.dt == NOVA_HIP_DT_BF16) launch_grad_t<NOVA_HIP_DT_BF16>(g, s);
  else launch_grad_t<NOVA_HIP_DT_F16>(g, s);
  return check_hip(hipGetLastError(), "preference_loss gradient launch");
}

}  // namespace nova_hip

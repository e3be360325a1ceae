// Rotary positions, the norm of query and key heads in front of them, its
// backward pass, and the same rotation on the way into a paged cache.
//
// A head's row of D values is rotated pair by pair: with angle t = position f_i,
//   a' = s (a cos t - b sin t),   b' = s (b cos t + a sin t),
// the pair i being values (i, i + R / 2) of the row (halves) or (2 i, 2 i + 1)
// (interleaved), i < R / 2; values from R on stay.  The norm ahead of it is
//   y = x r w,   r = (mean x^2 + eps)^-1/2,
// and backward, with g the gradient rotated back and t = g w:
//   dx = r (t - x r^2 mean(t x)),   dw = sum over rows of g x r.
//
// All of it is bound by HBM: a row is read and written once.  A workgroup takes one to
// kMaxTB tokens with all their heads (see shape_of), issues the loads of its rows, works
// out the tokens' sines and cosines meanwhile, once, into LDS, and ends: angles are taken
// in 64 bits (in 32 an angle of 10^5 is off by 4e-3).  A row belongs to L = 1 .. 32 lanes,
// each with a "slot" of two 16-byte chunks that hold whole pairs, so that the rotation
// needs no exchange between lanes and the norm log2 L of them.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "gemm_common.h"
#include "wave.h"

namespace nova_hip {
namespace pos {
namespace {

constexpr int kMaxThreads = 512;  // of a workgroup forward
constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kMaxTB = 8;  // tokens whose angles a workgroup holds at once
// Rows of a lane whose loads are on their way together (1 / 2, cold: 8120 tokens of 32 + 8
// heads of 128 normed 32.8 / 33.8 us, into the cache 37.4 / 37.2; 8192 of 12 heads of 64 in
// f32, 32 values rotated, warm, 10.4 / 9.6).  They and the stores are such that the caches
// keep nothing for: 8120 tokens of 40 heads of 128, cold, in 30.0 us against 34.7, where they
// still lie in a cache 30.4 against 27.1.
constexpr int kAhead = 2;
constexpr int kMaxPairs = kMaxHeadDim / 2;

// n / d for n < 1024 by inverse(d): the product lies above n 2^22 / d by n at most, which is
// less than 2^22 / d up to d = 4096; beyond, n < d and the product stays below 2^22.
static_assert(kMaxTB * kMaxPairs <= 1024 && kMaxThreads <= 1024, "what is divided");
inline uint32_t inverse(int d) { return (1u << 22) / (uint32_t)d + 1; }
__device__ __forceinline__ int divided(int n, uint32_t inverse) {
  return (int)(((uint32_t)n * inverse) >> 22);
}

// A lane group's rows among tokens of `heads` each: every groups-th, from its own.
struct Steps {
  int heads, dt, dh;  // a step is of dt tokens and dh heads
  uint32_t by_heads;
  Steps() = default;
  Steps(int groups, int heads)
      : heads(heads), dt(heads ? groups / heads : 0), dh(heads ? groups % heads : 0),
        by_heads(heads ? inverse(heads) : 0) {}
};
struct Walk {
  int t, h;
  __device__ __forceinline__ Walk(int group, const Steps &s)
      : t(divided(group, s.by_heads)), h(group - t * s.heads) {}
  __device__ __forceinline__ void next(const Steps &s) {
    t += s.dt;
    h += s.dh;
    if (h >= s.heads) {
      h -= s.heads;
      ++t;
    }
  }
};

// A token's and a head's stride in 16 bytes: two products of 32 bits make a row's place
// (of 64 they cost the backward pass as much as its arithmetic).
struct Strides {
  uint32_t t, h;
  __device__ __forceinline__ int64_t at(int token, int head) const {
    return (int64_t)(((uint64_t)(uint32_t)token * t + (uint64_t)(uint32_t)head * h) << 4);
  }
};

// One operand's rows and where they go.
struct Rows {
  const char *src;
  char *dst;
  const void *w;  // the norm's weight
  Strides from, to;
  int heads;
};

struct Paged {
  const int *off, *lens, *table;
  int64_t sp[2], ss[2];  // page and row strides of k and v in bytes
  int64_t stb;           // the table's row stride
  int B, width, pages;
  uint32_t page;
};

struct Args {
  Rows rows[3];  // paged: queries, keys, values
  Paged paged;
  const int *positions;
  const float *freqs;
  float scale, eps;
  int T, D, R, TB, L, log_l, w_dt, threads;
  Steps steps;  // of all rows together
  uint32_t by_pairs;
  bool inverse;
};

template <int DT>
__device__ __forceinline__ float widen(uint32_t h) {
  if constexpr (DT == NOVA_HIP_DT_BF16) return __uint_as_float(h << 16);
  else return (float)__builtin_bit_cast(_Float16, (uint16_t)h);
}

// V values, 16 or 8 bytes.
template <int DT, int V>
struct Chunk {
  typedef uint32_t raw __attribute__((ext_vector_type(DT == NOVA_HIP_DT_F32 ? V : V / 2)));
  static __device__ __forceinline__ void widen_to(const raw &r, float (&x)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if constexpr (DT == NOVA_HIP_DT_F32) x[i] = __uint_as_float(r[i]);
      else x[i] = widen<DT>(i & 1 ? r[i / 2] >> 16 : r[i / 2] & 0xffffu);
    }
  }
  static __device__ __forceinline__ raw load(const char *p) {
    return __builtin_nontemporal_load(reinterpret_cast<const raw *>(p));
  }
  static __device__ __forceinline__ void store(char *p, const float (&x)[V]) {
    raw r;
    if constexpr (DT == NOVA_HIP_DT_F32) {
#pragma unroll
      for (int i = 0; i < V; ++i) r[i] = __float_as_uint(x[i]);
    } else {
#pragma unroll
      for (int i = 0; i < V / 2; ++i)
        r[i] = DT == NOVA_HIP_DT_BF16 ? gemm::pack_bf16(x[2 * i], x[2 * i + 1])
                                      : gemm::pack_f16(x[2 * i], x[2 * i + 1]);
    }
    __builtin_nontemporal_store(r, reinterpret_cast<raw *>(p));
  }
};

// A lane's slot of a row: its two chunks of V values, in elements from the row's
// start, and which of them are there and rotated.  Halves: chunk j < R / 2 V goes with
// the chunk R / 2 values on; what is left (all, when pairs are interleaved) lies in two
// runs, so that neighbouring lanes load neighbouring chunks.
struct Slot {
  int e[2];
  bool has[2], rot[2];
};
template <int V, bool INTER>
__device__ __forceinline__ Slot slot_of(int j, int D, int R) {
  Slot s;
  const int np = INTER ? 0 : R / 2 / V, run = (D / V - 2 * np + 1) / 2;
  const bool pair = j < np;
  s.e[0] = (pair ? j : np + j) * V;
  s.e[1] = pair ? s.e[0] + R / 2 : j - np < run ? s.e[0] + run * V : D;
  if (!pair && j - np >= run) s.e[0] = D;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    s.has[i] = s.e[i] < D;
    s.rot[i] = INTER ? s.e[i] < R : pair;
  }
  return s;
}

// Cosine and sine of a token's angle, times the scale.
__device__ __forceinline__ void angle(double position, float freq, float scale, bool inverse,
                                      float &c, float &s) {
  double turns = position * (double)freq * 0.15915494309189533577;
  turns = 2.0 * (turns - __builtin_rint(turns));
  const float x = (float)turns, rest = (float)(turns - (double)x) * 3.14159265f;
  float sx, cx;
  sincospif(x, &sx, &cx);
  c = scale * __builtin_fmaf(-sx, rest, cx);
  s = (inverse ? -scale : scale) * __builtin_fmaf(cx, rest, sx);
}

// The angles of tokens 0 .. nt - 1 by a workgroup: cs[t][i] and cs[t][kMaxPairs + i].
template <typename Position>
__device__ __forceinline__ void angles(float (&cs)[kMaxTB][2 * kMaxPairs], int nt, int pairs,
                                       uint32_t by_pairs, const float *freqs, float scale, bool inverse,
                                       Position position) {
  for (int i = threadIdx.x; i < nt * pairs; i += blockDim.x) {
    const int t = divided(i, by_pairs), k = i - t * pairs;
    float c, s;
    angle(position(t), freqs[k], scale, inverse, c, s);
    cs[t][k] = c;
    cs[t][kMaxPairs + k] = s;
  }
}

// V values of LDS, from a multiple of four.
template <int V>
__device__ __forceinline__ void load_floats(const float *p, float (&x)[V]) {
  typedef float four __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int i = 0; i < V / 4; ++i) {
    const four v = *reinterpret_cast<const four *>(p + 4 * i);
#pragma unroll
    for (int k = 0; k < 4; ++k) x[4 * i + k] = v[k];
  }
}

// Rotates the slot's values by the token's angles.
template <int V, bool INTER>
__device__ __forceinline__ void rotate(const Slot &sl, const float *cs, float (&x)[2][V]) {
  if constexpr (INTER) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (!sl.rot[k]) continue;
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        const float c = cs[sl.e[k] / 2 + i], s = cs[kMaxPairs + sl.e[k] / 2 + i];
        const float a = x[k][2 * i], b = x[k][2 * i + 1];
        x[k][2 * i] = a * c - b * s;
        x[k][2 * i + 1] = b * c + a * s;
      }
    }
  } else {
    if (!sl.rot[0]) return;
    float c[V], s[V];
    load_floats(cs + sl.e[0], c);
    load_floats(cs + kMaxPairs + sl.e[0], s);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float a = x[0][i], b = x[1][i];
      x[0][i] = a * c[i] - b * s[i];
      x[1][i] = b * c[i] + a * s[i];
    }
  }
}

// Sum over the L lanes of a row (L a power of two up to 32): in quads, then with the
// mirrored lane, all on DPP but the last.
__device__ __forceinline__ float row_sum(float v, int L) {
  if (L > 1) v += dpp_mov<0xB1>(v);   // quad_perm [1,0,3,2]
  if (L > 2) v += dpp_mov<0x4E>(v);   // quad_perm [2,3,0,1]
  if (L > 4) v += dpp_mov<0x141>(v);  // row_half_mirror
  if (L > 8) v += dpp_mov<0x140>(v);  // row_mirror
  if (L > 16) v += __shfl_xor(v, 16);
  return v;
}
__device__ __forceinline__ void row_sums(float &v, float &u, int L) {
#define NOVA_POS_ADD(c) v += dpp_mov<c>(v), u += dpp_mov<c>(u)
  if (L > 1) NOVA_POS_ADD(0xB1);
  if (L > 2) NOVA_POS_ADD(0x4E);
  if (L > 4) NOVA_POS_ADD(0x141);
  if (L > 8) NOVA_POS_ADD(0x140);
#undef NOVA_POS_ADD
  if (L > 16) v += __shfl_xor(v, 16), u += __shfl_xor(u, 16);
}

// Where a new token goes: its position and the byte offsets of its rows in the
// pages, -1 where it is not stored, position kNowhere outside every sequence.
struct Place {
  int64_t position, at[2];
};
constexpr int64_t kNowhere = INT64_MIN;

// By a whole wave; every lane gets the result.  64 sequences are probed at a
// time.  Whatever the offsets, lengths and table hold, a place lies inside the
// pages or is none.
__device__ __forceinline__ Place place_of(const Paged &p, int t, int T) {
  const int lane = threadIdx.x & 63;
  Place r = {kNowhere, {-1, -1}};
  // The sequences whose end lies behind t are counted out: offsets do not fall.
  int lo = 0, n = p.B;
  while (n > 0) {
    const int step = (n + 63) / 64, i = min(lo + (lane + 1) * step, lo + n);
    const bool behind = lane * step < n && p.off[i] <= t;
    const int c = __builtin_popcountll(__ballot(behind));
    if (step == 1) {
      lo += c;
      break;
    }
    const int skip = min(c * step, n);
    lo += skip;
    n = min(step, n - skip);
  }
  if (lo >= p.B) return r;
  const int s = p.off[lo], e = min(p.off[lo + 1], T);
  if (s > t || e <= t) return r;
  r.position = (int64_t)p.lens[lo] - (e - t);
  if (r.position < 0) return r;
  const int64_t page = r.position / p.page;
  if (page >= p.width) return r;
  const int id = p.table[lo * p.stb + page];
  if (id < 0 || id >= p.pages) return r;
  const int row = (int)(r.position - page * p.page);
#pragma unroll
  for (int k = 0; k < 2; ++k) r.at[k] = id * p.sp[k] + row * p.ss[k];
  return r;
}

template <int DT, int V, bool INTER, bool NORM, bool PAGED>
__global__ __launch_bounds__(kMaxThreads) void positions_kernel(Args a) {
  __shared__ __attribute__((aligned(16))) float cs[kMaxTB][2 * kMaxPairs];
  // Both weights: as registers they would cost more than the rows.
  __shared__ __attribute__((aligned(16))) float weights[NORM ? 2 : 1][NORM ? kMaxHeadDim : 1];
  __shared__ Place place[PAGED ? kMaxTB : 1];
  typedef Chunk<DT, V> C;
  constexpr int kSize = DT == NOVA_HIP_DT_F32 ? 4 : 2;
  const int t0 = blockIdx.x * a.TB, nt = min(a.TB, a.T - t0);
  const int j = threadIdx.x & (a.L - 1);
  const Slot sl = slot_of<V, INTER>(j, a.D, a.R);
  const float mean = 1.0f / (float)a.D;
  // A row's operand (queries, keys, values one behind the other) and head in it.
  auto part_of = [&](int h, int &head) __attribute__((always_inline)) {
    const int h1 = a.rows[0].heads, h2 = h1 + a.rows[1].heads;
    const int part = h < h1 ? 0 : h < h2 ? 1 : 2;
    head = part == 0 ? h : part == 1 ? h - h1 : h - h2;
    return part;
  };
  typename C::raw raw[kAhead][2] = {};
  auto fetch = [&](Walk w) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u, w.next(a.steps)) {
      if (w.t >= nt) continue;
      int head;
      const int part = part_of(w.h, head);
      const Rows &r = part == 0 ? a.rows[0] : part == 1 ? a.rows[1] : a.rows[2];
      const char *src = r.src + r.from.at(t0 + w.t, head);
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (sl.has[k])
          raw[u][k] = C::load(src + sl.e[k] * kSize);
    }
  };
  Walk w(threadIdx.x >> a.log_l, a.steps);
  fetch(w);
  if constexpr (NORM) {
    // (Zeros behind the row, where absent chunks point: only rows that no lane lacks reach 256.)
    for (int d = threadIdx.x; d < kMaxHeadDim; d += blockDim.x) {
      weights[0][d] = d < a.D && a.rows[0].heads ? gemm::bias_at(a.rows[0].w, a.w_dt, d) : 0.0f;
      weights[1][d] = d < a.D && a.rows[1].heads ? gemm::bias_at(a.rows[1].w, a.w_dt, d) : 0.0f;
    }
  }
  if constexpr (PAGED) {
    for (int t = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); t < nt; t += blockDim.x / 64) {
      const Place p = place_of(a.paged, t0 + t, a.T);
      if ((threadIdx.x & 63) == 0) place[t] = p;
    }
    __syncthreads();
  }
  angles(cs, nt, a.R / 2, a.by_pairs, a.freqs, a.scale, a.inverse, [&](int t) {
    if constexpr (PAGED) return (double)place[t].position;
    else return (double)a.positions[t0 + t];
  });
  __syncthreads();
  while (__ballot(w.t < nt)) {  // (whole waves: the lanes of a row stay together)
    Walk now = w;
#pragma unroll
    for (int u = 0; u < kAhead; ++u, now.next(a.steps)) {
      if (u && !__ballot(now.t < nt)) break;
      int head;
      const int part = part_of(now.h, head), t = min(now.t, nt - 1);
      float x[2][V];
#pragma unroll
      for (int k = 0; k < 2; ++k) C::widen_to(raw[u][k], x[k]);
      if constexpr (NORM) {
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int i = 0; i < V; ++i) sum = __builtin_fmaf(x[k][i], x[k][i], sum);
        const float r = rsqrtf(__builtin_fmaf(row_sum(sum, a.L), mean, a.eps));
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float weight[V];
          load_floats(&weights[part][0] + sl.e[k], weight);
#pragma unroll
          for (int i = 0; i < V; ++i) x[k][i] *= r * weight[i];
        }
      }
      if (!PAGED || part < 2) rotate<V, INTER>(sl, cs[t], x);
      const Rows &r = part == 0 ? a.rows[0] : part == 1 ? a.rows[1] : a.rows[2];
      int64_t at = r.to.at(t0 + t, head);
      bool write = now.t < nt;
      if constexpr (PAGED) {
        const int64_t page = part == 0 ? 0 : part == 1 ? place[t].at[0] : place[t].at[1];
        at += page;  // (the pages' stride of a token is zero)
        write = write && place[t].position != kNowhere && page >= 0;
      }
      if (write) {
        char *dst = r.dst + at;
#pragma unroll
        for (int k = 0; k < 2; ++k)
          if (sl.has[k]) C::store(dst + sl.e[k] * kSize, x[k]);
      }
    }
    w = now;
    fetch(w);
  }
}

struct BackwardArgs {
  // Per operand: x, the gradient of its result, its own.
  struct Part {
    const char *x, *g;
    char *dx;
    const void *w;
    float *partial, *dw;  // [blocks][D], [D]
    Strides xs, gs, ds;
    int heads, blocks;
    Steps steps;
  } part[2];
  const int *positions;
  const float *freqs;
  float scale, eps;
  int T, D, R, TB, L, log_l, w_dt;
  uint32_t by_pairs;
};

// A workgroup takes a run of TB tokens, the queries' rows and then the keys' by the same
// angles, and every gridDim.x-th run on.  A lane keeps its share of the weight's gradient
// in registers until an operand's rows of a run end, a column's thread the sums of runs.
// Bound by what is on its way to a CU, so by its waves: chunks of four values to a lane
// at every type leave room for five waves to a SIMD (8120 tokens of 40 heads of 128 in
// bf16, 249 MB, cold, with the sums behind: 57.3 us, 4.3 TB/s, vector units 63 % busy; 65536
// tokens 5.1; chunks of eight: 62 with four waves, 73 with three; runs of four tokens: 67).
// In f32, 499 MB, vector units are 30 % busy and HBM is the bound (105 us warm, 4.8 TB/s).
// Five waves cost 4 registers to scratch in f32 and 2 in bf16 interleaved: the latter takes
// as long as bf16 in halves, which has none there (kernel alone 50.0 and 50.4 us).
template <int DT, bool INTER>
__global__ __launch_bounds__(kThreads, 5) void qk_norm_backward_kernel(BackwardArgs a) {
  constexpr int V = 4;
  __shared__ __attribute__((aligned(16))) float cs[kMaxTB][2 * kMaxPairs];
  __shared__ __attribute__((aligned(16))) float weights[2][kMaxHeadDim];
  __shared__ float box[kWaves][kMaxHeadDim], total[2][kMaxHeadDim];  // (a column to a thread)
  typedef Chunk<DT, V> C;
  constexpr int kSize = DT == NOVA_HIP_DT_F32 ? 4 : 2;
  const int j = threadIdx.x & (a.L - 1);
  const Slot sl = slot_of<V, INTER>(j, a.D, a.R);
  const float mean = 1.0f / (float)a.D;
  int t0 = 0, nt = 0;
  typename C::raw rx[2] = {}, rg[2] = {};
  auto fetch = [&](const BackwardArgs::Part &p, const Walk &at) __attribute__((always_inline)) {
    if (at.t >= nt) return;
    const char *x = p.x + p.xs.at(t0 + at.t, at.h), *y = p.g + p.gs.at(t0 + at.t, at.h);
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (sl.has[k]) {
        rx[k] = C::load(x + sl.e[k] * kSize);
        rg[k] = C::load(y + sl.e[k] * kSize);
      }
  };
  // (An operand without heads has its walk behind the last token.)
  auto walk = [&](int kind) __attribute__((always_inline)) {
    Walk w(threadIdx.x >> a.log_l, a.part[kind].steps);
    if (a.part[kind].heads == 0) w.t = nt;
    return w;
  };
  const int first = blockIdx.y, last = gridDim.y > 1 ? first : 1;
  // (Zeros behind the row, where absent chunks point: only rows that no lane lacks reach 256.)
#pragma unroll
  for (int kind = 0; kind < 2; ++kind)
    weights[kind][threadIdx.x] = (int)threadIdx.x < a.D && a.part[kind].heads
                                     ? gemm::bias_at(a.part[kind].w, a.w_dt, threadIdx.x) : 0.0f;
  total[0][threadIdx.x] = total[1][threadIdx.x] = 0.0f;
  for (int run = blockIdx.x; run < (a.T + a.TB - 1) / a.TB; run += gridDim.x) {
    t0 = run * a.TB;
    nt = min(a.TB, a.T - t0);
    Walk at = walk(first);
    fetch(a.part[first], at);
    angles(cs, nt, a.R / 2, a.by_pairs, a.freqs, a.scale, true,
           [&](int t) { return (double)a.positions[t0 + t]; });
    __syncthreads();
#pragma unroll 1
    for (int kind = first; kind <= last; ++kind) {
      const BackwardArgs::Part &p = a.part[kind];
      const float *weight = weights[kind];
      float dw[2][V] = {};
      while (__ballot(at.t < nt)) {  // (whole waves: the lanes of a row stay together)
        float x[2][V], d[2][V];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          C::widen_to(rx[k], x[k]);
          C::widen_to(rg[k], d[k]);
        }
        rotate<V, INTER>(sl, cs[min(at.t, nt - 1)], d);
        float xx = 0.0f, tx = 0.0f, t[2][V];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          load_floats(weight + sl.e[k], t[k]);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            t[k][i] *= d[k][i];
            xx = __builtin_fmaf(x[k][i], x[k][i], xx);
            tx = __builtin_fmaf(t[k][i], x[k][i], tx);
          }
        }
        row_sums(xx, tx, a.L);
        const float r = rsqrtf(__builtin_fmaf(xx, mean, a.eps)), m = tx * mean * r * r;
        if (at.t < nt) {
          char *dx = p.dx + p.ds.at(t0 + at.t, at.h);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
              const float n = x[k][i] * r;
              dw[k][i] = __builtin_fmaf(d[k][i], n, dw[k][i]);
              x[k][i] = __builtin_fmaf(-n, m, r * t[k][i]);
            }
            if (sl.has[k]) C::store(dx + sl.e[k] * kSize, x[k]);
          }
        }
        at.next(p.steps);
        fetch(p, at);
      }
      if (kind < last) {
        at = walk(1);
        fetch(a.part[1], at);
      }
      if (p.heads == 0) continue;
      // The lanes with the same slot, then the waves in order.
      const int lane = threadIdx.x & 63;
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          for (int d = a.L; d < 64; d <<= 1) dw[k][i] += __shfl_xor(dw[k][i], d);
          if (lane < a.L && sl.has[k]) box[threadIdx.x >> 6][sl.e[k] + i] = dw[k][i];
        }
      __syncthreads();
      if ((int)threadIdx.x < a.D)
        total[kind][threadIdx.x] +=
            (box[0][threadIdx.x] + box[1][threadIdx.x]) + (box[2][threadIdx.x] + box[3][threadIdx.x]);
      __syncthreads();
    }
  }
  if ((int)threadIdx.x >= a.D) return;
  for (int kind = first; kind <= last; ++kind)
    if (a.part[kind].heads)
      a.part[kind].partial[(int64_t)blockIdx.x * a.D + threadIdx.x] = total[kind][threadIdx.x];
}

// The workgroups' sums of eight columns: every 128th row, then those in order.
__global__ __launch_bounds__(1024) void qk_norm_weight_kernel(BackwardArgs a) {
  __shared__ float box[16][8];
  const BackwardArgs::Part &p = a.part[blockIdx.y];
  const int c = threadIdx.x & 7, d = blockIdx.x * 8 + c;  // D is a multiple of 8
  float sum = 0.0f;
#pragma unroll 8
  for (int i = threadIdx.x >> 3; i < p.blocks; i += 128) sum += p.partial[(int64_t)i * a.D + d];
  // The eight rows of a wave, then the waves.
  sum += __shfl_xor(sum, 8);
  sum += __shfl_xor(sum, 16);
  sum += __shfl_xor(sum, 32);
  if ((threadIdx.x & 63) < 8) box[threadIdx.x >> 6][c] = sum;
  __syncthreads();
  if (threadIdx.x >= 8) return;
  sum = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) sum += box[i][c];
  p.dw[d] = sum;
}

__global__ void rotary_frequencies_kernel(float *freqs, int n, double base, double factor, double low,
                                          double high, double original) {
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n) return;
  const double f = pow(base, -(double)i / n);
  double keep = 0.0;
  if (original > 0.0)
    keep = fmin(fmax((original * f * 0.15915494309189533577 - low) / (high - low), 0.0), 1.0);
  freqs[i] = (float)(f * (keep + (1.0 - keep) / factor));
}

// Values to a chunk: 16 bytes, or 8 of 16-bit halves that are no multiple of that.
int chunk_values(int dt, int R, bool interleaved) {
  return dt == NOVA_HIP_DT_F32 || (!interleaved && R % 16) ? 4 : 8;
}
// Lanes to a row.
int lanes_of(int D, int V) {
  int L = 1;
  while (L < (D / V + 1) / 2) L <<= 1;
  return L;
}

template <int DT, int V, bool INTER>
void launch_rows(const Args &a, bool norm, bool paged, hipStream_t s) {
  const dim3 grid((unsigned)((a.T + a.TB - 1) / a.TB)), block((unsigned)a.threads);
  if constexpr (DT != NOVA_HIP_DT_F32) {
    if (paged) {
      hipLaunchKernelGGL((positions_kernel<DT, V, INTER, false, true>), grid, block, 0, s, a);
      return;
    }
  }
  if (norm) hipLaunchKernelGGL((positions_kernel<DT, V, INTER, true, false>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((positions_kernel<DT, V, INTER, false, false>), grid, block, 0, s, a);
}
template <int DT>
void launch_back(const BackwardArgs &a, bool interleaved, hipStream_t s) {
  const unsigned runs = (unsigned)std::max(a.part[0].blocks, a.part[1].blocks);
  // Few runs: a workgroup for each operand (333 tokens of 24 heads of 80: 8.8 us against 10.6).
  const dim3 grid(runs, runs <= 512 ? 2 : 1);
  if (runs && interleaved)
    hipLaunchKernelGGL((qk_norm_backward_kernel<DT, true>), grid, dim3(kThreads), 0, s, a);
  else if (runs)
    hipLaunchKernelGGL((qk_norm_backward_kernel<DT, false>), grid, dim3(kThreads), 0, s, a);
  hipLaunchKernelGGL(qk_norm_weight_kernel, dim3((unsigned)a.D / 8, 2), dim3(1024), 0, s, a);
}

// Calls f<DT, V, INTER>() of a problem.
template <typename F>
void dispatch(int dt, int R, bool interleaved, F f) {
  using std::integral_constant;
  const bool wide = chunk_values(dt, R, interleaved) == 8;
#define NOVA_POS_CASE(DT_, V_, I_) \
  f(integral_constant<int, DT_>{}, integral_constant<int, V_>{}, integral_constant<bool, I_>{})
  if (dt == NOVA_HIP_DT_F32) {
    if (interleaved) NOVA_POS_CASE(NOVA_HIP_DT_F32, 4, true);
    else NOVA_POS_CASE(NOVA_HIP_DT_F32, 4, false);
  } else if (dt == NOVA_HIP_DT_BF16) {
    if (interleaved) NOVA_POS_CASE(NOVA_HIP_DT_BF16, 8, true);
    else if (wide) NOVA_POS_CASE(NOVA_HIP_DT_BF16, 8, false);
    else NOVA_POS_CASE(NOVA_HIP_DT_BF16, 4, false);
  } else {
    if (interleaved) NOVA_POS_CASE(NOVA_HIP_DT_F16, 8, true);
    else if (wide) NOVA_POS_CASE(NOVA_HIP_DT_F16, 8, false);
    else NOVA_POS_CASE(NOVA_HIP_DT_F16, 4, false);
  }
#undef NOVA_POS_CASE
}

// Tokens and threads of a workgroup.  Few tokens: one, a thread to each of its lanes (32
// tokens of 40 heads of 128 normed: 3.9 us, with 256 threads 4.6).  Else up to two rows to a
// lane of 256 threads at most, what leaves the fewest lanes idle: short workgroups keep
// what the chip works on at a time together (8120 tokens of 40 heads of 128, cold, one
// token to 192 threads 30.5 us, 5.4 TB/s; two to 256 32.5, to 384 38.6; 8192 of 12 heads of
// 64 in f32, four to 192 9.6, six to 256 12.5).
void shape_of(int64_t T, int heads, int L, int &TB, int &threads) {
  const int64_t lanes = heads * L;
  TB = 1;
  threads = (int)std::min<int64_t>(kMaxThreads, (lanes + 63) / 64 * 64);
  if (T < 1024) return;
  const int64_t most = std::min<int64_t>(kMaxTB, T / 1024);
  double fill = 0.0;
  for (int64_t n = 1; n == 1 || (n <= most && n * lanes <= 512); ++n) {
    const int64_t rows = (n * lanes + 255) / 256;
    const int64_t t = ((n * lanes + rows - 1) / rows + 63) / 64 * 64;
    const double f = (double)(n * lanes) / (double)(rows * t);
    if (f >= fill) fill = f, TB = (int)n, threads = (int)t;
  }
}

// An operand's strides; false where they do not fit.
bool strides_of(const AttentionOperand &o, int size, Strides &s) {
  s = {(uint32_t)(o.st * size / 16), (uint32_t)(o.sh * size / 16)};
  return o.st * size / 16 == s.t && o.sh * size / 16 == s.h;
}
int32_t too_far(const char *what) {
  return fail(NOVA_HIP_ERANGE, "%s: tokens or heads 2^36 bytes apart", what);
}

}  // namespace
}  // namespace pos

int32_t launch_rotary_frequencies(float *freqs, int64_t n, double base, double factor, double low,
                                  double high, double original, hipStream_t s) {
  if (n == 0) return NOVA_HIP_SUCCESS;
  hipLaunchKernelGGL(pos::rotary_frequencies_kernel, dim3((unsigned)((n + 63) / 64)), dim3(64), 0, s,
                     freqs, (int)n, base, factor, low, high, original);
  return check_hip(hipGetLastError(), "rotary_frequencies launch");
}

int32_t launch_positions(const PositionProblem &p, hipStream_t s) {
  pos::Args a = {};
  const int size = dtype_size(p.dt);
  int heads = 0;
  for (int i = 0; i < 3; ++i) {
    const PositionRows &r = p.rows[i];
    heads += (int)r.heads;
    a.rows[i] = {static_cast<const char *>(r.src.p), static_cast<char *>(r.dst.p), r.w, {}, {},
                 (int)r.heads};
    if (p.T == 0 || r.heads == 0) continue;  // (strides of nothing)
    if (!pos::strides_of(r.src, size, a.rows[i].from) || !pos::strides_of(r.dst, size, a.rows[i].to))
      return pos::too_far(p.what);
  }
  if (p.T == 0 || heads == 0 || p.D == 0) return NOVA_HIP_SUCCESS;
  if (p.paged) {
    const PagedCache &c = *p.paged;
    a.paged = {c.offsets, c.lengths, c.table, {c.k.sp * size, c.v.sp * size},
               {c.k.st * size, c.v.st * size}, c.stable, (int)c.B, (int)c.width, (int)c.pages,
               (uint32_t)c.page};
  }
  a.positions = p.positions;
  a.freqs = p.freqs;
  a.scale = p.scale;
  a.eps = p.eps;
  a.T = (int)p.T;
  a.D = (int)p.D;
  a.R = (int)p.R;
  a.w_dt = p.w_dt;
  a.inverse = p.inverse;
  a.L = pos::lanes_of(a.D, pos::chunk_values(p.dt, a.R, p.interleaved));
  a.log_l = __builtin_ctz(a.L);
  pos::shape_of(p.T, heads, a.L, a.TB, a.threads);
  a.steps = pos::Steps(a.threads / a.L, heads);
  a.by_pairs = a.R ? pos::inverse(a.R / 2) : 0;
  // A grid's dimension holds less than 2^32 threads.
  if ((p.T + a.TB - 1) / a.TB >= 1 << 24)
    return fail(NOVA_HIP_ERANGE, "%s: %lld tokens of %d heads exceed 2^24 workgroups", p.what,
                (long long)p.T, heads);
  pos::dispatch(p.dt, a.R, p.interleaved, [&](auto dt, auto v, auto inter) {
    pos::launch_rows<dt.value, v.value, inter.value>(a, p.norm, p.paged != nullptr, s);
  });
  return check_hip(hipGetLastError(), "positions launch");
}

// Tokens to a run of the backward pass, and workgroups: up to five to a CU, all with the
// same number of runs.
static int backward_run(int64_t T) {
  return (int)std::max<int64_t>(1, std::min<int64_t>(pos::kMaxTB, T / 512));
}
static int64_t backward_blocks(int64_t T, int64_t heads) {
  if (T == 0 || heads == 0) return 0;
  const int64_t runs = (T + backward_run(T) - 1) / backward_run(T), turns = (runs + 1279) / 1280;
  return (runs + turns - 1) / turns;
}
int64_t qk_norm_backward_scratch(int64_t T, int64_t heads, int64_t kv_heads, int64_t D) {
  return (backward_blocks(T, heads) + backward_blocks(T, kv_heads)) * D;
}

int32_t launch_qk_norm_backward(const QkNormBackwardProblem &p, hipStream_t s) {
  if (p.D == 0) return NOVA_HIP_SUCCESS;
  pos::BackwardArgs a = {};
  const int size = dtype_size(p.dt);
  a.D = (int)p.D;
  a.R = (int)p.R;
  a.L = pos::lanes_of(a.D, 4);
  a.log_l = __builtin_ctz(a.L);
  a.by_pairs = a.R ? pos::inverse(a.R / 2) : 0;
  float *scratch = p.scratch;
  for (int i = 0; i < 2; ++i) {
    const auto &q = p.part[i];
    const int64_t blocks = backward_blocks(p.T, q.heads);
    a.part[i] = {static_cast<const char *>(q.x.p), static_cast<const char *>(q.g.p),
                 static_cast<char *>(q.dx.p), q.w, scratch, q.dw, {}, {}, {}, (int)q.heads, (int)blocks,
                 pos::Steps(pos::kThreads / a.L, (int)q.heads)};
    scratch += blocks * p.D;
    if (blocks == 0) continue;
    if (!pos::strides_of(q.x, size, a.part[i].xs) || !pos::strides_of(q.g, size, a.part[i].gs) ||
        !pos::strides_of(q.dx, size, a.part[i].ds))
      return pos::too_far("qk_norm_rotary_backward");
  }
  a.positions = p.positions;
  a.freqs = p.freqs;
  a.scale = p.scale;
  a.eps = p.eps;
  a.T = (int)p.T;
  a.w_dt = p.w_dt;
  a.TB = backward_run(p.T);
  if (p.dt == NOVA_HIP_DT_F32) pos::launch_back<NOVA_HIP_DT_F32>(a, p.interleaved, s);
  else if (p.dt == NOVA_HIP_DT_BF16) pos::launch_back<NOVA_HIP_DT_BF16>(a, p.interleaved, s);
  else pos::launch_back<NOVA_HIP_DT_F16>(a, p.interleaved, s);
  return check_hip(hipGetLastError(), "qk_norm_rotary_backward launch");
}

}  // namespace nova_hip

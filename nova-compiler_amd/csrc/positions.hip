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
// All of it is bound by HBM: a row is read and written once.  A row belongs to
// L = 1 .. 32 neighbouring lanes, each with a "slot" of two 16-byte chunks that
// hold whole pairs, so that the rotation needs no exchange between lanes and the
// norm log2 L of them.  A workgroup takes a few tokens with all their heads and
// works out their sines and cosines once, into LDS: angles are taken in 64 bits
// (in 32 an angle of 10^5 is off by 4e-3) and only their fraction of a turn is
// rounded.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "gemm_common.h"

namespace nova_hip {
namespace pos {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTB = 8;  // tokens whose angles a workgroup holds at once
constexpr int kMaxPairs = kMaxHeadDim / 2;

// One operand's rows and where they go (strides in bytes).
struct Rows {
  const char *src;
  char *dst;
  const void *w;  // the norm's weight
  int64_t st, sh, dt, dh;
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
  int T, D, R, TB, L, NS, heads, w_dt;  // heads: of all rows together
  bool inverse;
};

template <int DT>
__device__ __forceinline__ float widen(uint32_t h) {
  if constexpr (DT == NOVA_HIP_DT_BF16) return __uint_as_float(h << 16);
  else return (float)__builtin_bit_cast(_Float16, (uint16_t)h);
}

// V values at p, 16 or 8 bytes.
template <int DT, int V>
__device__ __forceinline__ void load(const char *p, float (&x)[V]) {
  if constexpr (DT == NOVA_HIP_DT_F32) {
    static_assert(V == 4, "16 bytes");
    const gemm::f32x4 r = *reinterpret_cast<const gemm::f32x4 *>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = r[i];
  } else {
    uint32_t r[V / 2];
    if constexpr (V == 8) {
      const gemm::u32x4 v = *reinterpret_cast<const gemm::u32x4 *>(p);
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = v[i];
    } else {
      const gemm::u32x2 v = *reinterpret_cast<const gemm::u32x2 *>(p);
      r[0] = v[0];
      r[1] = v[1];
    }
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      x[2 * i] = widen<DT>(r[i] & 0xffffu);
      x[2 * i + 1] = widen<DT>(r[i] >> 16);
    }
  }
}
template <int DT, int V>
__device__ __forceinline__ void store(char *p, const float (&x)[V]) {
  if constexpr (DT == NOVA_HIP_DT_F32) {
    *reinterpret_cast<gemm::f32x4 *>(p) = gemm::f32x4{x[0], x[1], x[2], x[3]};
  } else {
    uint32_t r[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; ++i)
      r[i] = DT == NOVA_HIP_DT_BF16 ? gemm::pack_bf16(x[2 * i], x[2 * i + 1])
                                    : gemm::pack_f16(x[2 * i], x[2 * i + 1]);
    if constexpr (V == 8) *reinterpret_cast<gemm::u32x4 *>(p) = gemm::u32x4{r[0], r[1], r[2], r[3]};
    else *reinterpret_cast<gemm::u32x2 *>(p) = gemm::u32x2{r[0], r[1]};
  }
}

// A lane's slot of a row: its two chunks of V values, in elements from the row's
// start, and which of them are there and rotated.  Halves: chunk j < R / 2 V goes
// with the chunk R / 2 values on; what is not rotated lies in pairs of neighbours,
// as all chunks do when pairs are interleaved.
struct Slot {
  int e[2];
  bool has[2], rot[2];
};
template <int V, bool INTER>
__device__ __forceinline__ Slot slot_of(int j, int D, int R) {
  Slot s;
  const int np = R / 2 / V;
  const bool pair = !INTER && j < np;
  s.e[0] = (pair ? j : 2 * j) * V;
  s.e[1] = pair ? s.e[0] + R / 2 : s.e[0] + V;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    s.has[i] = s.e[i] < D;
    s.rot[i] = INTER ? s.e[i] < R : pair;
  }
  return s;
}

// Sines and cosines of a token, times the scale: cs[i] and cs[kMaxPairs + i].
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

// Rotates the slot's values by the token's table.
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
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float c = cs[sl.e[0] + i], s = cs[kMaxPairs + sl.e[0] + i];
      const float a = x[0][i], b = x[1][i];
      x[0][i] = a * c - b * s;
      x[1][i] = b * c + a * s;
    }
  }
}

// Sum over the L lanes of a row (L a power of two up to 32).
__device__ __forceinline__ float row_sum(float v, int L) {
  for (int d = 1; d < L; d <<= 1) v += __shfl_xor(v, d);
  return v;
}

template <int V>
__device__ __forceinline__ void load_weight(const void *w, int dt, const Slot &sl, float (&x)[2][V]) {
#pragma unroll
  for (int k = 0; k < 2; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) x[k][i] = sl.has[k] ? gemm::bias_at(w, dt, sl.e[k] + i) : 0.0f;
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
__global__ __launch_bounds__(kThreads) void positions_kernel(Args a) {
  __shared__ float cs[kMaxTB][2 * kMaxPairs];
  __shared__ Place place[PAGED ? kMaxTB : 1];
  constexpr int kSize = DT == NOVA_HIP_DT_F32 ? 4 : 2;
  const int t0 = blockIdx.x * a.TB, nt = min(a.TB, a.T - t0), pairs = a.R / 2;
  if constexpr (PAGED) {
    for (int t = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); t < nt; t += kThreads / 64) {
      const Place p = place_of(a.paged, t0 + t, a.T);
      if ((threadIdx.x & 63) == 0) place[t] = p;
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < nt * pairs; i += kThreads) {
    const int t = i / pairs, k = i - t * pairs;
    double at;
    if constexpr (PAGED) at = (double)place[t].position;
    else at = (double)a.positions[t0 + t];
    float c, s;
    angle(at, a.freqs[k], a.scale, a.inverse, c, s);
    cs[t][k] = c;
    cs[t][kMaxPairs + k] = s;
  }
  __syncthreads();

  const int j = threadIdx.x & (a.L - 1), group = threadIdx.x / a.L, groups = kThreads / a.L;
  const Slot sl = slot_of<V, INTER>(j, a.D, a.R);
  float w[2][2][V] = {};
  if constexpr (NORM) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (a.rows[i].heads) load_weight<V>(a.rows[i].w, a.w_dt, sl, w[i]);
  }
  const float mean = 1.0f / (float)a.D;
  const int ht = groups / a.heads, hr = groups - ht * a.heads;
  int t = group / a.heads, h = group - t * a.heads;
  for (; t < nt;) {
    int part = 0, head = h;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (part == i && head >= a.rows[i].heads) {
        head -= a.rows[i].heads;
        ++part;
      }
    const Rows &r0 = a.rows[0], &r1 = a.rows[1], &r2 = a.rows[2];
    const char *src = part == 0 ? r0.src : part == 1 ? r1.src : r2.src;
    char *dst = part == 0 ? r0.dst : part == 1 ? r1.dst : r2.dst;
    const int64_t st = part == 0 ? r0.st : part == 1 ? r1.st : r2.st;
    const int64_t sh = part == 0 ? r0.sh : part == 1 ? r1.sh : r2.sh;
    const int64_t dh = part == 0 ? r0.dh : part == 1 ? r1.dh : r2.dh;
    src += (t0 + t) * st + head * sh;
    bool write = true;
    if constexpr (PAGED) {
      if (part == 0) {
        write = place[t].position != kNowhere;
        dst += (t0 + t) * r0.dt + head * dh;
      } else {
        const int64_t at = place[t].at[part - 1];
        write = at >= 0;
        dst += at + head * dh;
      }
    } else {
      dst += (t0 + t) * (part == 0 ? r0.dt : r1.dt) + head * dh;
    }
    float x[2][V];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (sl.has[k]) load<DT, V>(src + sl.e[k] * kSize, x[k]);
      else
#pragma unroll
        for (int i = 0; i < V; ++i) x[k][i] = 0.0f;
    }
    if constexpr (NORM) {
      float sum = 0.0f;
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) sum = __builtin_fmaf(x[k][i], x[k][i], sum);
      const float r = rsqrtf(__builtin_fmaf(row_sum(sum, a.L), mean, a.eps));
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) x[k][i] *= r * (part == 0 ? w[0][k][i] : w[1][k][i]);
    }
    if (!PAGED || part < 2) rotate<V, INTER>(sl, cs[t], x);
    if (write) {
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (sl.has[k]) store<DT, V>(dst + sl.e[k] * kSize, x[k]);
    }
    t += ht;
    h += hr;
    if (h >= a.heads) {
      h -= a.heads;
      ++t;
    }
  }
}

struct BackwardArgs {
  // Per operand: x, its gradient's source, the gradient (strides in bytes).
  struct Part {
    const char *x, *g;
    char *dx;
    const void *w;
    float *partial, *dw;  // [blocks][D], [D]
    int64_t xt, xh, gt, gh, dt, dh;
    int heads, blocks;
  } part[2];
  const int *positions;
  const float *freqs;
  float scale, eps;
  int T, D, R, TB, L, NS, w_dt;
};

// Workgroup b < part[0].blocks takes every blocks-th run of TB tokens of the
// queries, the others the keys'.  A lane keeps its slot's weights and its share
// of their gradient in registers.
template <int DT, int V, bool INTER>
__global__ __launch_bounds__(kThreads) void qk_norm_backward_kernel(BackwardArgs a) {
  __shared__ float cs[kMaxTB][2 * kMaxPairs];
  __shared__ float box[kThreads / 64][kMaxHeadDim];
  constexpr int kSize = DT == NOVA_HIP_DT_F32 ? 4 : 2;
  const int kind = (int)blockIdx.x >= a.part[0].blocks ? 1 : 0;
  const BackwardArgs::Part &p = a.part[kind];
  const int block = blockIdx.x - (kind ? a.part[0].blocks : 0);
  const int pairs = a.R / 2;
  const int j = threadIdx.x & (a.L - 1), group = threadIdx.x / a.L, groups = kThreads / a.L;
  const Slot sl = slot_of<V, INTER>(j, a.D, a.R);
  float w[2][V], dw[2][V] = {};
  load_weight<V>(p.w, a.w_dt, sl, w);
  const float mean = 1.0f / (float)a.D;
  const int ht = groups / p.heads, hr = groups - ht * p.heads;
  for (int64_t t0 = (int64_t)block * a.TB; t0 < a.T; t0 += (int64_t)p.blocks * a.TB) {
    const int nt = (int)min((int64_t)a.TB, a.T - t0);
    __syncthreads();
    for (int i = threadIdx.x; i < nt * pairs; i += kThreads) {
      const int t = i / pairs, k = i - t * pairs;
      float c, s;
      angle((double)a.positions[t0 + t], a.freqs[k], a.scale, true, c, s);
      cs[t][k] = c;
      cs[t][kMaxPairs + k] = s;
    }
    __syncthreads();
    int t = group / p.heads, h = group - t * p.heads;
    while (t < nt) {
      const char *xp = p.x + (t0 + t) * p.xt + h * p.xh, *gp = p.g + (t0 + t) * p.gt + h * p.gh;
      float x[2][V], g[2][V];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (sl.has[k]) {
          load<DT, V>(xp + sl.e[k] * kSize, x[k]);
          load<DT, V>(gp + sl.e[k] * kSize, g[k]);
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) x[k][i] = g[k][i] = 0.0f;
        }
      }
      rotate<V, INTER>(sl, cs[t], g);
      float xx = 0.0f, tx = 0.0f;
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          xx = __builtin_fmaf(x[k][i], x[k][i], xx);
          tx = __builtin_fmaf(g[k][i] * w[k][i], x[k][i], tx);
        }
      const float r = rsqrtf(__builtin_fmaf(row_sum(xx, a.L), mean, a.eps));
      const float m = row_sum(tx, a.L) * mean * r * r;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          dw[k][i] = __builtin_fmaf(g[k][i], x[k][i] * r, dw[k][i]);
          x[k][i] = r * __builtin_fmaf(-x[k][i], m, g[k][i] * w[k][i]);
        }
        if (sl.has[k]) store<DT, V>(p.dx + (t0 + t) * p.dt + h * p.dh + sl.e[k] * kSize, x[k]);
      }
      t += ht;
      h += hr;
      if (h >= p.heads) {
        h -= p.heads;
        ++t;
      }
    }
  }
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
    p.partial[(int64_t)block * a.D + threadIdx.x] =
        (box[0][threadIdx.x] + box[1][threadIdx.x]) + (box[2][threadIdx.x] + box[3][threadIdx.x]);
}

// The workgroups' sums of 32 columns: eight rows at a time, then those in order.
__global__ __launch_bounds__(kThreads) void qk_norm_weight_kernel(BackwardArgs a) {
  __shared__ float box[8][32];
  const BackwardArgs::Part &p = a.part[blockIdx.y];
  const int c = threadIdx.x & 31, r = threadIdx.x >> 5, d = blockIdx.x * 32 + c;
  float sum = 0.0f;
  if (d < a.D) {
#pragma unroll 8
    for (int i = r; i < p.blocks; i += 8) sum += p.partial[(int64_t)i * a.D + d];
  }
  box[r][c] = sum;
  __syncthreads();
  if (r || d >= a.D) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) sum += box[i][c];
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
void shape(int D, int V, int &NS, int &L) {
  NS = (D / V + 1) / 2;
  for (L = 1; L < NS;) L <<= 1;
}

template <int DT, int V, bool INTER>
void launch_rows(const Args &a, bool norm, bool paged, hipStream_t s) {
  const dim3 grid((unsigned)((a.T + a.TB - 1) / a.TB)), block(kThreads);
  if constexpr (DT != NOVA_HIP_DT_F32) {
    if (paged) {
      hipLaunchKernelGGL((positions_kernel<DT, V, INTER, false, true>), grid, block, 0, s, a);
      return;
    }
  }
  if (norm) hipLaunchKernelGGL((positions_kernel<DT, V, INTER, true, false>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((positions_kernel<DT, V, INTER, false, false>), grid, block, 0, s, a);
}
template <int DT, int V, bool INTER>
void launch_back(const BackwardArgs &a, hipStream_t s) {
  const unsigned grid = (unsigned)(a.part[0].blocks + a.part[1].blocks);
  if (grid) hipLaunchKernelGGL((qk_norm_backward_kernel<DT, V, INTER>), dim3(grid), dim3(kThreads), 0, s, a);
  hipLaunchKernelGGL(qk_norm_weight_kernel, dim3((unsigned)((a.D + 31) / 32), 2), dim3(kThreads), 0, s, a);
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

// Tokens to a workgroup: one while they do not give every CU four, up to eight.
int tokens_per_block(int64_t T) { return (int)std::min<int64_t>(kMaxTB, std::max<int64_t>(1, T / 1024)); }

Rows rows_of(const PositionRows &r, int size) {
  return {static_cast<const char *>(r.src.p), static_cast<char *>(r.dst.p), r.w,
          r.src.st * size, r.src.sh * size, r.dst.st * size, r.dst.sh * size, (int)r.heads};
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
  for (int i = 0; i < 3; ++i) {
    a.rows[i] = pos::rows_of(p.rows[i], size);
    a.heads += (int)p.rows[i].heads;
  }
  if (p.T == 0 || a.heads == 0 || p.D == 0) return NOVA_HIP_SUCCESS;
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
  a.TB = pos::tokens_per_block(p.T);
  // A grid's dimension holds less than 2^32 threads.
  if ((p.T + a.TB - 1) / a.TB >= 1 << 24)
    return fail(NOVA_HIP_ERANGE, "%s: %lld tokens exceed 2^27 - 8", p.what, (long long)p.T);
  a.w_dt = p.w_dt;
  a.inverse = p.inverse;
  pos::shape(a.D, pos::chunk_values(p.dt, a.R, p.interleaved), a.NS, a.L);
  pos::dispatch(p.dt, a.R, p.interleaved, [&](auto dt, auto v, auto inter) {
    pos::launch_rows<dt.value, v.value, inter.value>(a, p.norm, p.paged != nullptr, s);
  });
  return check_hip(hipGetLastError(), "positions launch");
}

// Workgroups of the backward pass over `heads` heads of T tokens, of all `all`.
static int64_t backward_blocks(int64_t T, int64_t heads, int64_t all) {
  if (T == 0 || heads == 0) return 0;
  const int64_t TB = pos::tokens_per_block(T);
  return std::min((T + TB - 1) / TB, std::max<int64_t>(1, 1024 * heads / all));
}
int64_t qk_norm_backward_scratch(int64_t T, int64_t heads, int64_t kv_heads, int64_t D) {
  return (backward_blocks(T, heads, heads + kv_heads) + backward_blocks(T, kv_heads, heads + kv_heads)) * D;
}

int32_t launch_qk_norm_backward(const QkNormBackwardProblem &p, hipStream_t s) {
  if (p.D == 0) return NOVA_HIP_SUCCESS;
  pos::BackwardArgs a = {};
  const int size = dtype_size(p.dt);
  float *scratch = p.scratch;
  const int64_t all = p.part[0].heads + p.part[1].heads;
  for (int i = 0; i < 2; ++i) {
    const auto &q = p.part[i];
    const int64_t blocks = backward_blocks(p.T, q.heads, all);
    a.part[i] = {static_cast<const char *>(q.x.p), static_cast<const char *>(q.g.p),
                 static_cast<char *>(q.dx.p), q.w, scratch, q.dw,
                 q.x.st * size, q.x.sh * size, q.g.st * size, q.g.sh * size,
                 q.dx.st * size, q.dx.sh * size, (int)q.heads, (int)blocks};
    scratch += blocks * p.D;
  }
  a.positions = p.positions;
  a.freqs = p.freqs;
  a.scale = p.scale;
  a.eps = p.eps;
  a.T = (int)p.T;
  a.D = (int)p.D;
  a.R = (int)p.R;
  a.TB = pos::tokens_per_block(p.T);
  a.w_dt = p.w_dt;
  pos::shape(a.D, pos::chunk_values(p.dt, a.R, p.interleaved), a.NS, a.L);
  pos::dispatch(p.dt, a.R, p.interleaved, [&](auto dt, auto v, auto inter) {
    pos::launch_back<dt.value, v.value, inter.value>(a, s);
  });
  return check_hip(hipGetLastError(), "qk_norm_rotary_backward launch");
}

}  // namespace nova_hip

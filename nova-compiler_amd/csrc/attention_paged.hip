// Attention of chunks of new tokens over a paged cache: the queries of sequence
// b are the packed rows offsets[b] .. offsets[b + 1], its keys and values the
// first lengths[b] rows of its pages, the new tokens' own among them.
//
// The query heads of a group read the same keys, so a tile's rows are (token,
// head of the group) pairs: row r is token r / group, head r % group, and keys
// and values are read once for the group.  The products, the running maximum and
// sum and the LDS tiles are those of the packed forward (attention.hip).
//
// Two forms.  Chunks: four waves of 32 rows share tiles of 64 keys.  Up to 32 rows
// per sequence (single tokens): a wave per split of the keys, tiles of 32, without
// a barrier; bound by HBM.  Either cuts the keys of a tile of rows into splits of
// `chunk` where there are few tiles; a tile whose rows see at most one split
// writes its result, the others' sums go to the caller's scratch and
// paged_join_kernel adds them in order.
//
// Keys come by DMA into LDS.  Where a page holds whole loads (rows that are a
// multiple of the 4 or 8 of one instruction) its address is a scalar: 64 entries of
// the table lie in a register, and a buffer of the load's rows that are there makes
// the others zero.  Other page sizes go through registers, a row's address per lane.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attention.h"
#include "wave.h"

namespace nova_hip {
namespace attn {
namespace {

struct PagedArgs {
  const uint16_t *q, *k, *v;
  uint16_t *o;
  float *lse;      // [heads][T] with row stride slse, or null
  float *partial;  // [T][heads][splits][D + 2]: sum, then m c and l (splits > 1)
  const int *off, *lens, *table;
  Rows sq, so;
  int64_t skp, skt, skh, svp, svt, svh, stb, slse;
  double per_page;  // 1 / page
  int T, B, heads, kv_heads, group, D, page, pages, width, cap;  // cap: rows of a sequence
  int tiles, splits, chunk;
  float c;  // scale log2 e
  bool causal;
  bool whole;  // a load's rows lie in one page
};

constexpr float kSlack = 8.0f;  // as in the packed forward
template <int DT>
constexpr float kUp = DT == NOVA_HIP_DT_F16 ? 7.0f : 0.0f;

// A sequence's new tokens and cache rows, whatever offsets and lengths hold.
struct Seq {
  int s, n, len;
  // Keys that a token of it sees.
  __device__ __forceinline__ int seen(int token, bool causal) const {
    return causal ? max(0, min(len, len - n + token + 1)) : len;
  }
};
__device__ __forceinline__ Seq seq_of(const PagedArgs &a, int b) {
  Seq q;
  q.s = min(max(a.off[b], 0), a.T);
  q.n = max(min(a.off[b + 1], a.T), q.s) - q.s;
  q.len = min(max(a.lens[b], 0), a.cap);
  return q;
}

// Tile t of the sequences' tiles of BM rows (n group rows each): the sequence, or
// -1, and the tile's index in it.  Wave-uniform.  The order and the two searches
// are find_tile's.
__device__ __forceinline__ int find_rows(const PagedArgs &a, int BM, int t, int &index) {
  const int lane = threadIdx.x & 63;
  if (a.B <= 64) {
    int n = 0;
    if (lane < a.B) {
      const int s = min(max(a.off[lane], 0), a.T), e = max(s, min(a.off[lane + 1], a.T));
      n = ((e - s) * a.group + BM - 1) / BM;
    }
    auto above = [&](int k) __attribute__((always_inline)) { return wave_sum_int(max(0, n - k)); };
    if (above(0) <= t) return -1;
    int level = 0, bit = 1;
    while (bit < (1 << 25) && above(bit) > t) bit <<= 1;
    for (bit >>= 1; bit > 0; bit >>= 1)
      if (above(level + bit) > t) level += bit;
    const int k = t - above(level + 1);
    const uint64_t has = __ballot(n > level);
    const int rank = __builtin_amdgcn_mbcnt_hi((uint32_t)(has >> 32),
                                               __builtin_amdgcn_mbcnt_lo((uint32_t)has, 0));
    const uint64_t hit = __ballot(n > level && rank == k);
    if (!hit) return -1;
    index = level;
    return __builtin_ctzll(hit);
  }
  // Sequence b's tiles are numbered from off[b] group / BM + b.
  t = a.T * a.group / BM + a.B - 1 - t;
  int lo = 0, n = a.B;
  for (;;) {
    const int step = (n + 63) / 64, b = lo + lane * step;
    const bool at = lane * step < n && min(max(a.off[b], 0), a.T) * a.group / BM + b <= t;
    const int c = __builtin_popcountll(__ballot(at));
    if (c == 0) return -1;
    lo += (c - 1) * step;
    n = min(step, n - (c - 1) * step);
    if (step == 1) break;
  }
  const Seq q = seq_of(a, lo);
  index = __builtin_amdgcn_readfirstlane(t - (q.s * a.group / BM + lo));
  if (index < 0 || index >= (q.n * a.group + BM - 1) / BM) return -1;
  return __builtin_amdgcn_readfirstlane(lo);
}

// NW waves of 32 rows each.
template <int DT, int DP, int NW>
__global__ __launch_bounds__(64 * NW, NW == 1 ? 1 : 2) void attention_paged_kernel(PagedArgs a) {
  constexpr int CH = kPitch<DP>, BN = NW == 1 ? 32 : 64, kTile = BN * CH * 16;
  constexpr int kRows = 64 / CH;               // rows of one DMA instruction
  constexpr int kN = BN / kRows / NW;          // instructions of a wave and tile
  __shared__ __attribute__((aligned(1024))) char sk0_[kTile], sk1_[kTile], sv0_[kTile], sv1_[kTile];
  lds_char *const sk0 = (lds_char *)sk0_, *const sk1 = (lds_char *)sk1_;
  lds_char *const sv0 = (lds_char *)sv0_, *const sv1 = (lds_char *)sv1_;
  const int lane = threadIdx.x & 63;
  const int wave = NW == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int kh, b, index = 0, split;
  if constexpr (NW == 1) {
    kh = blockIdx.x;
    b = blockIdx.y;
    split = blockIdx.z;
  } else {
    int tile;
    unit_of(blockIdx.x, a.kv_heads, a.tiles, a.causal, kh, tile);
    split = blockIdx.y;
    b = find_rows(a, 32 * NW, tile, index);
    if (b < 0) return;
  }
  const Seq seq = seq_of(a, b);
  const int row0 = index * 32 * NW, R = NW == 1 ? min(seq.n, 32 / a.group) * a.group : seq.n * a.group;
  if (R <= row0) return;
  const int vis = seq.seen((min(row0 + 32 * NW, R) - 1) / a.group, a.causal);
  const int from = split * a.chunk, to = min(vis, from + a.chunk);
  if (split > 0 && from >= vis) return;
  const bool direct = vis <= a.chunk;

  const int q0 = row0 + 32 * wave, qn = min(32, R - q0);  // this wave's rows, maybe none
  const int row = min(q0 + (lane & 31), R - 1), token = row / a.group;
  const int head = kh * a.group + row - token * a.group;
  const bool mine = (lane & 31) < qn;
  const int end = mine ? min(to, seq.seen(token, a.causal)) : 0;  // the keys this lane's row sees
  // ... and those that the wave's first and last rows see.
  const int least = qn > 0 ? min(to, seq.seen(q0 / a.group, a.causal)) : 0;
  const int most = qn > 0 ? min(to, seq.seen((q0 + qn - 1) / a.group, a.causal)) : 0;
  u32x4 qf[DP / 16];
  {
    const uint16_t *p = a.q + (seq.s + token) * a.sq.t + head * a.sq.h;
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
      const int d = 16 * s + 8 * (lane >> 5);
      qf[s] = u32x4{0, 0, 0, 0};
      if (mine && d < a.D) qf[s] = *reinterpret_cast<const u32x4 *>(p + d);
    }
  }

  const int *table = a.table + b * a.stb;
  const uint16_t *kp = a.k + kh * a.skh, *vp = a.v + kh * a.svh;
  // (key + 1/2) / page in 64 bits lies at least 1 / (2 page) from a whole number,
  // far more than it can be off.
  auto page_of = [&](int key) __attribute__((always_inline)) {
    return (int)(((double)key + 0.5) * a.per_page);
  };
  int first = 0, ids = 0;  // entries first .. first + 63 of the table
  bool loaded = false;
  auto fetch = [&](int t, lds_char *sk, lds_char *sv) __attribute__((always_inline)) {
    const int k0 = from + t * BN;
    if (a.whole) {
      const int p0 = __builtin_amdgcn_readfirstlane(page_of(k0));
      const int p1 = __builtin_amdgcn_readfirstlane(page_of(min(k0 + BN, to) - 1));
      if (!loaded || p1 >= first + 64) {
        loaded = true;
        first = p0;
        ids = min(max(table[min(p0 + lane, a.width - 1)], 0), a.pages - 1);
      }
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int r0 = (i * NW + wave) * kRows, key = k0 + r0, n = min(to - key, kRows);
        const int pg = __builtin_amdgcn_readfirstlane(page_of(min(key, to - 1)));
        const int id = __builtin_amdgcn_readlane(ids, pg - first);
        const int r = key - pg * a.page;
        const __amdgpu_buffer_rsrc_t rk =
            make_rsrc(kp + id * a.skp + r * a.skt, n > 0 ? (uint32_t)(((n - 1) * a.skt + a.D) * 2) : 0u);
        const __amdgpu_buffer_rsrc_t rv =
            make_rsrc(vp + id * a.svp + r * a.svt, n > 0 ? (uint32_t)(((n - 1) * a.svt + a.D) * 2) : 0u);
        const int lr = lane / CH, ch = (lane & (CH - 1)) ^ swz<CH>(r0 + lr);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rk, (lds_void *)(sk + r0 * CH * 16), 16,
            ch * 8 < a.D ? (uint32_t)(lr * a.skt + ch * 8) * 2u : kOOB, 0, 0, NW == 1 ? 2 : 0);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rv, (lds_void *)(sv + r0 * CH * 16), 16,
            ch * 8 < a.D ? (uint32_t)(lr * a.svt + ch * 8) * 2u : kOOB, 0, 0, NW == 1 ? 2 : 0);
      }
    } else {
      typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
      u32x4 x[kN], y[kN];
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int r0 = (i * NW + wave) * kRows, lr = lane / CH, key = k0 + r0 + lr;
        const int ch = (lane & (CH - 1)) ^ swz<CH>(r0 + lr);
        x[i] = y[i] = u32x4{0, 0, 0, 0};
        if (key < to && ch * 8 < a.D) {
          const int pg = page_of(key), r = key - pg * a.page;
          const int id = min(max(table[pg], 0), a.pages - 1);
          x[i] = *reinterpret_cast<const u32x4 *>(kp + id * a.skp + r * a.skt + ch * 8);
          y[i] = *reinterpret_cast<const u32x4 *>(vp + id * a.svp + r * a.svt + ch * 8);
        }
      }
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int r0 = (i * NW + wave) * kRows;
        *(lds_u32x4 *)(sk + r0 * CH * 16 + lane * 16) = x[i];
        *(lds_u32x4 *)(sv + r0 * CH * 16 + lane * 16) = y[i];
      }
    }
  };

  f32x16 acc[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i) acc[i] = f32x16{};
  float mc = -INFINITY, l = 0.0f;  // m c and this lane's share of the sum
  auto step = [&](int t, const lds_char *sk, const lds_char *sv) __attribute__((always_inline)) {
    const int k0 = from + t * BN;
    if (k0 >= most) return;  // wave-uniform
    if constexpr (NW > 1) __builtin_amdgcn_iglp_opt(0);
    f32x16 s[BN / 32];
#pragma unroll
    for (int i = 0; i < BN / 32; ++i) {
      s[i] = f32x16{};
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk)
        s[i] = mfma_32x32x16<DT>(read_row_frag(sk, row_frag<CH>(32 * i, kk, lane)), qf[kk], s[i]);
    }
    if (k0 + BN > least || qn < 32) {
      keep_branch();
#pragma unroll
      for (int i = 0; i < BN / 32; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (k0 + 32 * i + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3) >= end) s[i][r] = -INFINITY;
    }
    float m = s[0][0];
#pragma unroll
    for (int i = 0; i < BN / 32; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) m = fmaxf(m, s[i][r]);
    m = both_max(m) * a.c;
    if (__ballot(m > mc + kSlack)) {
      const float to_m = fmaxf(m, mc), f = mc == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mc - to_m);
      mc = to_m;
      l *= f;
#pragma unroll
      for (int i = 0; i < DP / 32; ++i) acc[i] *= f;
    }
    const float up = kUp<DT> - (mc == -INFINITY ? 0.0f : mc);
#pragma unroll
    for (int i = 0; i < BN / 32; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[i][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][r], a.c, up));
        l += s[i][r];
      }
#pragma unroll
    for (int i = 0; i < BN / 32; ++i)
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        // Weights round to the operands' type, as in the packed forward.
        const u32x4 pf = pack_frag<DT>(s[i], kk);
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
          acc[db] = mfma_32x32x16<DT>(read_col_frag<CH>(sv, 32 * i + 16 * kk, 32 * db, lane), pf,
                                      acc[db]);
      }
  };
  const int nt = (max(to - from, 0) + BN - 1) / BN;
  if constexpr (NW > 1) {
    // One barrier per tile: behind it the tile just fetched is whole and the
    // other stage has no reader left.
    auto sync = [&]() __attribute__((always_inline)) {
      __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's DMA has landed
      __syncthreads();
    };
    if (nt > 0) fetch(0, sk0, sv0);
    for (int t = 0; t < nt; t += 2) {
      sync();
      if (t + 1 < nt) fetch(t + 1, sk1, sv1);
      step(t, sk0, sv0);
      if (t + 1 >= nt) break;
      sync();
      if (t + 2 < nt) fetch(t + 2, sk0, sv0);
      step(t + 1, sk1, sv1);
    }
  } else {
    // A stage is refilled when the reads of it have returned, and read when all
    // but the next stage's loads have landed.
    constexpr int kInFlight = 2 * kN;
    auto landed = [&](bool more) __attribute__((always_inline)) {
      __builtin_amdgcn_sched_barrier(0);
      if (more) __builtin_amdgcn_s_waitcnt(0x0F70 | (kInFlight & 15) | ((kInFlight >> 4) << 14));
      else __builtin_amdgcn_s_waitcnt(0x0F70);
      __builtin_amdgcn_sched_barrier(0);
    };
    auto drained = [&]() __attribute__((always_inline)) {
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
      __builtin_amdgcn_sched_barrier(0);
    };
    if (nt > 0) fetch(0, sk0, sv0);
    for (int t = 0; t < nt; t += 2) {
      const bool two = t + 1 < nt;
      drained();
      if (two) fetch(t + 1, sk1, sv1);
      landed(two && a.whole);
      step(t, sk0, sv0);
      if (!two) break;
      const bool three = t + 2 < nt;
      drained();
      if (three) fetch(t + 2, sk0, sv0);
      landed(three && a.whole);
      step(t + 1, sk1, sv1);
    }
  }
  l = both_sum(l);
  if (qn <= 0) return;
  if (direct) {
    // A row that sees no key is zero, its lse -inf.
    store_row<DT, DP>(acc, l == 0.0f ? 0.0f : 1.0f / l,
                      a.o + (seq.s + token) * a.so.t + head * a.so.h, mine, a.D, lane);
    if (a.lse && lane < qn)
      a.lse[head * a.slse + seq.s + token] =
          l == 0.0f ? -INFINITY : (mc + (__log2f(l) - kUp<DT>)) * kLn2;
    return;
  }
  if (!mine) return;
  float *p = a.partial + (((int64_t)(seq.s + token) * a.heads + head) * a.splits + split) * (a.D + 2);
#pragma unroll
  for (int db = 0; db < DP / 32; ++db)
#pragma unroll
    for (int r = 0; r < 16; r += 2) {
      const int d = 32 * db + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
      if (d < a.D) *reinterpret_cast<float2 *>(p + d) = float2{acc[db][r], acc[db][r + 1]};
    }
  if (lane < 32) *reinterpret_cast<float2 *>(p + a.D) = float2{mc, l};
}

// The sequence of a token, or -1: 64 sequences are probed at a time.
__device__ __forceinline__ int sequence_of(const PagedArgs &a, int t) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = a.B;
  while (n > 0) {
    const int step = (n + 63) / 64, i = min(lo + (lane + 1) * step, lo + n);
    const int c = __builtin_popcountll(__ballot(lane * step < n && a.off[i] <= t));
    if (step == 1) {
      lo += c;
      break;
    }
    const int skip = min(c * step, n);
    lo += skip;
    n = min(step, n - skip);
  }
  return lo < a.B ? lo : -1;
}

// One workgroup per (token, head) whose tile of BM rows left sums of several
// splits: to their largest maximum, added in split order within each wave's share
// (splits w, w + 4, ...), then the four shares in order.
template <int DT>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs a, int BM) {
  __shared__ float smax[4], ssum[4], sx[4][128];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int t = blockIdx.x / a.heads, head = blockIdx.x - t * a.heads;
  const int b = sequence_of(a, t);
  if (b < 0) return;
  const Seq seq = seq_of(a, b);
  const int token = t - seq.s;
  if (token < 0 || token >= seq.n) return;
  // As the rows' tile decided it.
  const int R = BM == 32 ? min(seq.n, 32 / a.group) * a.group : seq.n * a.group;
  const int row = token * a.group + head % a.group;
  if (row >= R) return;
  const int vis = seq.seen((min(row / BM * BM + BM, R) - 1) / a.group, a.causal);
  if (vis <= a.chunk) return;
  const int n = (vis + a.chunk - 1) / a.chunk;
  const float *p = a.partial + ((int64_t)t * a.heads + head) * a.splits * (a.D + 2);
  float mx = -INFINITY;
  for (int i = threadIdx.x; i < n; i += 256) mx = fmaxf(mx, p[(int64_t)i * (a.D + 2) + a.D]);
  mx = wave_max(mx);
  if (lane == 0) smax[wave] = mx;
  __syncthreads();
  mx = fmaxf(fmaxf(smax[0], smax[1]), fmaxf(smax[2], smax[3]));
  float sum = 0.0f, x0 = 0.0f, x1 = 0.0f;
  const int d = 2 * lane;
#pragma unroll 8
  for (int i = wave; i < n; i += 4) {
    const float *r = p + (int64_t)i * (a.D + 2);
    const float2 ml = *reinterpret_cast<const float2 *>(r + a.D);
    const float2 v = *reinterpret_cast<const float2 *>(r + min(d, a.D - 2));
    const float f = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - mx);
    sum = __builtin_fmaf(ml.y, f, sum);
    x0 = __builtin_fmaf(v.x, f, x0);
    x1 = __builtin_fmaf(v.y, f, x1);
  }
  sx[wave][d] = x0;
  sx[wave][d + 1] = x1;
  if (lane == 0) ssum[wave] = sum;
  __syncthreads();
  if (wave) return;
  sum = (ssum[0] + ssum[1]) + (ssum[2] + ssum[3]);
  x0 = (sx[0][d] + sx[1][d]) + (sx[2][d] + sx[3][d]);
  x1 = (sx[0][d + 1] + sx[1][d + 1]) + (sx[2][d + 1] + sx[3][d + 1]);
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  if (d < a.D)
    *reinterpret_cast<uint32_t *>(a.o + t * a.so.t + head * a.so.h + d) = pack<DT>(x0 * inv, x1 * inv);
  if (a.lse && lane == 0)
    a.lse[head * a.slse + t] = sum == 0.0f ? -INFINITY : (mx + (__log2f(sum) - kUp<DT>)) * kLn2;
}

template <int DT, int DP>
void launch_paged_t(const PagedArgs &a, bool narrow, hipStream_t s) {
  if (narrow)
    hipLaunchKernelGGL((attention_paged_kernel<DT, DP, 1>),
                       dim3((unsigned)a.kv_heads, (unsigned)a.B, (unsigned)a.splits), dim3(64), 0, s, a);
  else
    hipLaunchKernelGGL((attention_paged_kernel<DT, DP, 4>),
                       dim3((unsigned)(a.tiles * a.kv_heads), (unsigned)a.splits), dim3(256), 0, s, a);
}
template <int DT>
int32_t launch_paged(const PagedArgs &a, bool narrow, hipStream_t s) {
  if (a.D <= 32) launch_paged_t<DT, 32>(a, narrow, s);
  else if (a.D <= 64) launch_paged_t<DT, 64>(a, narrow, s);
  else if (a.D <= 96) launch_paged_t<DT, 96>(a, narrow, s);
  else launch_paged_t<DT, 128>(a, narrow, s);
  const int32_t rc = check_hip(hipGetLastError(), "paged_attention launch");
  if (rc || a.splits <= 1) return rc;
  hipLaunchKernelGGL(paged_join_kernel<DT>, dim3((unsigned)(a.T * a.heads)), dim3(256), 0, s, a,
                     narrow ? 32 : 128);
  return check_hip(hipGetLastError(), "paged_attention join launch");
}

// The form of a call, its tiles of rows and its splits.
struct Plan {
  bool narrow;
  int64_t tiles, chunk, splits;
};
Plan plan_of(int64_t T, int64_t B, int64_t heads, int64_t kv_heads, int64_t rows, int64_t max_queries) {
  Plan p;
  const int64_t group = heads / kv_heads;
  p.narrow = max_queries * group <= 32 && B <= 0xffff;
  if (p.narrow) {
    p.tiles = 0;
    // As for the padded cache (attention_decode.hip).
    const int64_t all = B * rows * kv_heads;
    const int64_t keys = std::max(std::min<int64_t>(512, all / 2048), std::min<int64_t>(2048, all / 8192));
    p.chunk = std::max<int64_t>(64, (std::max(keys, rows / 32768) + 63) / 64 * 64);
  } else {
    // Two workgroups to a CU, four rounds of them at most.
    p.tiles = B <= 64 ? std::min(T * group, T * group / 128 + B) : T * group / 128 + B;
    const int64_t units = p.tiles * kv_heads;
    const int64_t splits = std::max<int64_t>(1, std::min(2048 / units, rows / 512));
    p.chunk = std::max<int64_t>(64, ((rows + splits - 1) / splits + 63) / 64 * 64);
  }
  p.splits = std::max<int64_t>(1, (rows + p.chunk - 1) / p.chunk);
  return p;
}

}  // namespace
}  // namespace attn

int64_t paged_attention_scratch(int64_t T, int64_t B, int64_t heads, int64_t kv_heads, int64_t D,
                                int64_t rows, int64_t max_queries) {
  const attn::Plan p = attn::plan_of(T, B, heads, kv_heads, rows, max_queries);
  return p.splits <= 1 ? 0 : T * heads * p.splits * (D + 2);
}

int32_t launch_paged_attention(const PagedAttentionProblem &p, hipStream_t s) {
  const PagedCache &c = p.c;
  if (p.T == 0 || p.heads == 0 || c.D == 0 || c.B == 0) return NOVA_HIP_SUCCESS;
  attn::PagedArgs a = {};
  a.q = static_cast<const uint16_t *>(p.q.p);
  a.k = static_cast<const uint16_t *>(c.k.p);
  a.v = static_cast<const uint16_t *>(c.v.p);
  a.o = static_cast<uint16_t *>(p.o.p);
  a.lse = p.lse;
  a.slse = p.slse;
  a.partial = p.partial;
  a.off = c.offsets;
  a.lens = c.lengths;
  a.table = c.table;
  a.sq = {p.q.st, p.q.sh};
  a.so = {p.o.st, p.o.sh};
  a.skp = c.k.sp; a.skt = c.k.st; a.skh = c.k.sh;
  a.svp = c.v.sp; a.svt = c.v.st; a.svh = c.v.sh;
  a.stb = c.stable;
  a.per_page = 1.0 / (double)c.page;
  a.T = (int)p.T;
  a.B = (int)c.B;
  a.heads = (int)p.heads;
  a.kv_heads = (int)c.kv_heads;
  a.group = (int)(p.heads / c.kv_heads);
  a.D = (int)c.D;
  a.page = (int)c.page;
  a.pages = (int)c.pages;
  a.width = (int)c.width;
  a.cap = (int)(c.width * c.page);
  const attn::Plan plan = attn::plan_of(p.T, c.B, p.heads, c.kv_heads, a.cap, p.max_queries);
  // Rows are counted in 32 bits, a grid's dimension holds less than 2^32 threads.
  if (p.T * p.heads >= (1LL << 31) - (1 << 20) || plan.tiles * c.kv_heads >= 1 << 24 ||
      (plan.splits > 1 && p.T * p.heads >= 1 << 24))
    return fail(NOVA_HIP_ERANGE, "paged_attention: %lld tokens of %lld heads in %lld sequences",
                (long long)p.T, (long long)p.heads, (long long)c.B);
  a.tiles = (int)plan.tiles;
  a.splits = (int)plan.splits;
  a.chunk = (int)plan.chunk;
  a.c = p.scale * attn::kLog2e;
  a.causal = p.causal;
  a.whole = c.page % (c.D <= 64 ? 8 : 4) == 0;
  return p.dt == NOVA_HIP_DT_BF16 ? attn::launch_paged<NOVA_HIP_DT_BF16>(a, plan.narrow, s)
                                  : attn::launch_paged<NOVA_HIP_DT_F16>(a, plan.narrow, s);
}

}  // namespace nova_hip

// Attention of one query per sequence over a padded cache: the form for
// single tokens.  Bound by HBM: keys and values are read once, for all query
// heads of their group together (the group's heads are the MFMA's columns).
//
// A cache of up to 1024 rows is one workgroup's per sequence and key head: its
// waves take a part each and join their sums through LDS, in one launch (see
// kJoined).  A longer cache is cut into splits of `chunk` keys; a workgroup of one
// wave takes one split of one sequence and key head, 32 keys at a time through a
// two-stage ring in LDS filled by DMA, without a barrier.  (Two waves sharing a
// split joined their sums through LDS and took 2% longer.)  With more than
// one split the sums go to the caller's scratch, and attention_join_kernel adds
// them in a fixed order.
//
// Measured: 32 sequences of 1500 to 8192 rows, 597 MB of keys and values, in
// 104 us (5.7 TB/s); 8 of 131072 in 685 us (6.3 TB/s).  Without the products
// (the DMA alone) it takes the same: the loads are the time.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attention.h"
#include "wave.h"

namespace nova_hip {
namespace attn {
namespace {

struct DecodeArgs {
  const uint16_t *q, *k, *v;
  uint16_t *o;
  float *lse;      // [B][heads] with row stride slse, or null
  float *partial;  // [B][heads][splits][D + 2]: sum, then m c and l (splits > 1)
  const int *lens;
  int64_t sqb, sqh, sob, soh, slse;
  int64_t skb, skt, skh, svb, svt, svh;
  int S, heads, group, D, chunk;
  int splits;  // 0 where one workgroup's waves take a sequence and join
  float c;
};

constexpr int kBN = 32;
// f16 weights, at most 1, are taken times 2^15: one that rounds to zero is under
// 2^-40 of the largest in its part of the cache, not 2^-25 (see the forward).
template <int DT>
constexpr float kUp = DT == NOVA_HIP_DT_F16 ? 15.0f : 0.0f;

template <int DT, int DP, int NW>
__global__ __launch_bounds__(64 * NW) void attention_decode_kernel(DecodeArgs a) {
  constexpr int CH = kPitch<DP>, kTile = kBN * CH * 16;
  const int lane = threadIdx.x & 63;
  const int wave = NW == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  __shared__ float sm[NW][32], sl[NW][32];
  __shared__ __attribute__((aligned(1024))) char sk0_[NW * kTile];
  lds_char *const sk0 = (lds_char *)sk0_ + wave * kTile;
  __shared__ __attribute__((aligned(1024))) char sk1_[NW * kTile];
  lds_char *const sk1 = (lds_char *)sk1_ + wave * kTile;
  __shared__ __attribute__((aligned(1024))) char sv0_[NW * kTile];
  lds_char *const sv0 = (lds_char *)sv0_ + wave * kTile;
  __shared__ __attribute__((aligned(1024))) char sv1_[NW * kTile];
  lds_char *const sv1 = (lds_char *)sv1_ + wave * kTile;
  const int b = blockIdx.y, split = NW == 1 ? blockIdx.z : wave;
  const int blocks = (a.group + 31) / 32;  // of 32 query heads
  const int kh = blockIdx.x / blocks, h0 = kh * a.group + 32 * (blockIdx.x - kh * blocks);
  const int hn = min(32, (kh + 1) * a.group - h0);
  const int len = __builtin_amdgcn_readfirstlane(min(max(a.lens[b], 0), a.S));
  const int from = split * a.chunk, to = min(len, from + a.chunk);
  if (NW == 1 && from >= len && split > 0) return;  // nothing here; the join does not read it

  const uint16_t *kp = a.k + b * a.skb + kh * a.skh, *vp = a.v + b * a.svb + kh * a.svh;

  // A wave's own loads: 64 lanes cover 64 / CH rows at a time.
  constexpr int kN = kBN * CH / 64, kStep = 64 / CH;
  const int row = lane / CH;
  auto fetch = [&](int t, lds_char *sk, lds_char *sv) __attribute__((always_inline)) {
    const int k0 = from + t * kBN, n = min(to - k0, kBN);
    const __amdgpu_buffer_rsrc_t rk = make_rsrc(
        kp + (int64_t)k0 * a.skt, n > 0 ? (uint32_t)(((n - 1) * a.skt + a.D) * 2) : 0u);
    const __amdgpu_buffer_rsrc_t rv = make_rsrc(
        vp + (int64_t)k0 * a.svt, n > 0 ? (uint32_t)(((n - 1) * a.svt + a.D) * 2) : 0u);
    // Read once by the whole chip: the nontemporal hint (1 in aux bit 1) keeps
    // them from pushing each other through the L2s (32 sequences of 1500 to
    // 8192 rows: 122 -> 105 us; 8 of 131072: 757 -> 688 us).
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int r = i * kStep + row, c = (lane & (CH - 1)) ^ swz<CH>(r);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rk, (lds_void *)(sk + i * 1024), 16,
          c * 8 < a.D ? (uint32_t)(r * a.skt + c * 8) * 2u : kOOB, 0, 0, 2);
    }
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int r = i * kStep + row, c = (lane & (CH - 1)) ^ swz<CH>(r);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rv, (lds_void *)(sv + i * 1024), 16,
          c * 8 < a.D ? (uint32_t)(r * a.svt + c * 8) * 2u : kOOB, 0, 0, 2);
    }
  };
  const int nb = (max(to - from, 0) + kBN - 1) / kBN;
  if (nb > 0) fetch(0, sk0, sv0);
  u32x4 qf[DP / 16];
  load_cols<DP>(qf, a.q + b * a.sqb + h0 * a.sqh, a.sqh, hn, a.D, lane);

  f32x16 acc[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i) acc[i] = f32x16{};
  float mc = -INFINITY, l = 0.0f;
  auto step = [&](int t, const lds_char *sk, const lds_char *sv) __attribute__((always_inline)) {
    const int k0 = from + t * kBN;
    f32x16 s = {};
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk)
      s = mfma_32x32x16<DT>(read_row_frag(sk, row_frag<CH>(0, kk, lane)), qf[kk], s);
    if (k0 + kBN > to) {
      keep_branch();
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (k0 + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3) >= to) s[r] = -INFINITY;
    }
    float m = s[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) m = fmaxf(m, s[r]);
    m = fmaxf(mc, both_max(m) * a.c);
    if (__ballot(m > mc)) {
      const float f = mc == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mc - m);
      mc = m;
      l *= f;
#pragma unroll
      for (int i = 0; i < DP / 32; ++i) acc[i] *= f;
    }
    const float up = kUp<DT> - (mc == -INFINITY ? 0.0f : mc);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], a.c, up));
      l += s[r];
    }
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      // Weights round to the operands' type: half a step of it, as much as the
      // result's own.  (As two numbers each, the second the first's remainder, the
      // result has its own rounding alone: off by 1.66e-3 of itself in bf16 and not
      // by 2.2e-3, in 111 against 107 us as above.)
      const u32x4 pf = pack_frag<DT>(s, kk);
#pragma unroll
      for (int db = 0; db < DP / 32; ++db)
        acc[db] = mfma_32x32x16<DT>(read_col_frag<CH>(sv, 16 * kk, 32 * db, lane), pf, acc[db]);
    }
  };
  // A stage is refilled when the reads of it have returned.
  constexpr int kInFlight = 2 * kN;  // DMA instructions of one stage
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
  for (int t = 0; t < nb; t += 2) {
    const bool two = t + 1 < nb;
    drained();
    if (two) fetch(t + 1, sk1, sv1);
    landed(two);
    step(t, sk0, sv0);
    if (!two) break;
    const bool three = t + 2 < nb;
    drained();
    if (three) fetch(t + 2, sk0, sv0);
    landed(three);
    step(t + 1, sk1, sv1);
  }

  l = both_sum(l);
  if constexpr (NW > 1) {
    // Join the waves: to the largest of their maxima, then in wave order, each
    // handing its sums over through its part of the ring.
    if (lane < 32) {
      sm[wave][lane] = mc;
      sl[wave][lane] = l;
    }
    __syncthreads();
    const int c = lane & 31;
    float mx = sm[0][c];
#pragma unroll
    for (int i = 1; i < NW; ++i) mx = fmaxf(mx, sm[i][c]);
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < NW; ++i)  // 0 times a NaN stays one: all scores of a wave may be NaN
      l += sl[i][c] *
           (sm[i][c] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sm[i][c] - mx));
    const float f = mc == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mc - mx);
    mc = mx;
    static_assert(kTile >= 64 * 16 * 4, "a block of 32 x 32 sums");
    lds_float *const box = (lds_float *)sk0 + lane;
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) {
      if (db) __syncthreads();
      if (wave) {
#pragma unroll
        for (int r = 0; r < 16; ++r) box[64 * r] = acc[db][r] * f;
      }
      __syncthreads();
      if (wave == 0) {
        acc[db] *= f;
#pragma unroll
        for (int i = 1; i < NW; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[db][r] += box[i * (kTile / 4) + 64 * r];
      }
    }
    if (wave) return;
  }
  if (NW > 1 || a.splits == 1) {
    store_rows<DT, DP>(acc, l == 0.0f ? 0.0f : 1.0f / l, a.o + b * a.sob + h0 * a.soh, a.soh, hn,
                       a.D, lane);
    if (a.lse && lane < hn)
      a.lse[b * a.slse + h0 + lane] = l == 0.0f ? -INFINITY : (mc + (__log2f(l) - kUp<DT>)) * kLn2;
    return;
  }
  const int col = lane & 31;
  if (col >= hn) return;
  float *p = a.partial + (((int64_t)b * a.heads + h0 + col) * a.splits + split) * (a.D + 2);
#pragma unroll
  for (int db = 0; db < DP / 32; ++db)
#pragma unroll
    for (int r = 0; r < 16; r += 2) {
      const int d = 32 * db + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
      if (d < a.D) *reinterpret_cast<float2 *>(p + d) = float2{acc[db][r], acc[db][r + 1]};
    }
  if (lane < 32) *reinterpret_cast<float2 *>(p + a.D) = float2{mc, l};
}

// One workgroup per (sequence, head): the splits' sums to their largest
// maximum, added in split order within each wave's quarter (splits w, w + 4,
// ...), then the four quarters in order.
template <int DT>
__global__ __launch_bounds__(256) void attention_join_kernel(DecodeArgs a) {
  __shared__ float smax[4], ssum[4], sx[4][128];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = blockIdx.x, b = blockIdx.y;
  const int len = min(max(a.lens[b], 0), a.S);
  const int n = max(1, (len + a.chunk - 1) / a.chunk);
  const float *p = a.partial + ((int64_t)b * a.heads + h) * a.splits * (a.D + 2);
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
    *reinterpret_cast<uint32_t *>(a.o + b * a.sob + h * a.soh + d) = pack<DT>(x0 * inv, x1 * inv);
  if (a.lse && lane == 0)
    a.lse[b * a.slse + h] = sum == 0.0f ? -INFINITY : (mx + (__log2f(sum) - kUp<DT>)) * kLn2;
}

// Cache rows that the form takes whose waves join by themselves.  One launch costs
// the host 4 us less than two, but one workgroup is slower than many splits, the
// more so the longer the cache.  Two launches / one, us, of eager calls and of
// replays of a captured graph, where the host's part is none:
//   1 x 512 rows, 6 heads of 64                17.3 / 12.8    7.4 /  6.7
//   1 x 1024                                   17.0 / 12.7    8.1 /  8.6
//   1 x 2048                                   17.3 / 13.1    7.8 / 12.2
//   1 x 512, 32 heads in groups of 4 of 128    17.3 / 13.0    9.2 / 11.1
//   1 x 1024                                   17.6 / 16.6    9.9 / 16.4
//   1 x 1536                                   17.5 / 21.1   10.5 / 21.1
//   32 x 1024                                  30.0 / 24.3   30.1 / 24.4
//   32 x 2048                                  51.4 / 43.6   51.8 / 43.3
//   64 x 1024, 6 of 64                         19.9 / 21.9   19.6 / 22.0
// Eager calls of one sequence gain up to 1024 rows of 128 and 2000 of 64, replays up
// to about 350 and 768.
constexpr int kJoined = 1024;
// Its waves: what the LDS of a CU holds.
constexpr int waves_joined(int64_t D) { return D <= 64 ? 8 : 4; }

template <int DT, int DP>
void launch_decode_t(const DecodeArgs &a, dim3 grid, hipStream_t s) {
  constexpr int NW = waves_joined(DP);
  if (a.splits == 0)
    hipLaunchKernelGGL((attention_decode_kernel<DT, DP, NW>), grid, dim3(64 * NW), 0, s, a);
  else
    hipLaunchKernelGGL((attention_decode_kernel<DT, DP, 1>), grid, dim3(64), 0, s, a);
}
template <int DT>
int32_t launch_decode(const DecodeArgs &a, dim3 grid, hipStream_t s) {
  if (a.D <= 32) launch_decode_t<DT, 32>(a, grid, s);
  else if (a.D <= 64) launch_decode_t<DT, 64>(a, grid, s);
  else if (a.D <= 96) launch_decode_t<DT, 96>(a, grid, s);
  else launch_decode_t<DT, 128>(a, grid, s);
  const int32_t rc = check_hip(hipGetLastError(), "attention_decode launch");
  if (rc || a.splits <= 1) return rc;
  hipLaunchKernelGGL(attention_join_kernel<DT>, dim3((unsigned)a.heads, grid.y), dim3(256), 0, s, a);
  return check_hip(hipGetLastError(), "attention_decode join launch");
}

}  // namespace
}  // namespace attn

// Keys per split, a multiple of 64.  A wave per split, 1024 of them resident
// (four per CU by LDS): short splits for parallelism while the cache is
// small, at most 512 keys while there are fewer than eight rounds of them (long
// ones leave a ragged batch's last round idle), longer beyond.  Measured at 64
// / 128 / 256 / 512 / 1024 keys, heads 32 and 8 of 128, us:
//   1 x 8192 rows                13.9 / 13.8 / 17.6 / 27.6 / 45.5
//   8 x 8192                     69.2 / 57.7 / 51.5 / 48.5 / 50.8
//   32 x 1500 .. 8192 of 8192     151 /  128 /  114 /  103 /  116
//   8 x 131072                   1007 /  878 /  797 /  755 /  685
static int64_t decode_chunk(int64_t B, int64_t S, int64_t kv_heads) {
  const int64_t all = B * S * kv_heads;
  const int64_t keys = std::max(std::min<int64_t>(512, all / 2048), std::min<int64_t>(2048, all / 8192));
  // At most 32768 splits (a dimension of the grid).
  return std::max<int64_t>(64, (std::max(keys, S / 32768) + 63) / 64 * 64);
}

int64_t attention_decode_scratch(int64_t B, int64_t S, int64_t heads, int64_t kv_heads, int64_t D) {
  if (S <= attn::kJoined) return 0;
  const int64_t chunk = decode_chunk(B, S, kv_heads), splits = (S + chunk - 1) / chunk;
  return splits <= 1 ? 0 : B * heads * splits * (D + 2);
}

int32_t launch_attention_decode(const AttentionDecodeProblem &p, hipStream_t s) {
  if (p.B == 0 || p.heads == 0 || p.D == 0) return NOVA_HIP_SUCCESS;
  const int64_t B = p.B, S = p.S, H = p.heads, G = p.kv_heads, run = 2 * p.D;
  const Extent q = {"q", p.q, run, {B, H, 1}, {2 * p.sqb, 2 * p.sqh, 0}},
               k = {"k", p.k, S ? run : 0, {B, S, G}, {2 * p.skb, 2 * p.skt, 2 * p.skh}},
               v = {"v", p.v, S ? run : 0, {B, S, G}, {2 * p.svb, 2 * p.svt, 2 * p.svh}},
               out = {"out", p.o, run, {B, H, 1}, {2 * p.sob, 2 * p.soh, 0}},
               lse = {"lse", p.lse, p.lse ? 4 * H : 0, {B, 1, 1}, {4 * p.slse, 0, 0}};
  int32_t rc;
  if ((rc = check_apart("attention_decode", out, {q, k, v})) ||
      (rc = check_apart("attention_decode", lse, {q, k, v, out})))
    return rc;
  attn::DecodeArgs a;
  a.q = static_cast<const uint16_t *>(p.q);
  a.k = static_cast<const uint16_t *>(p.k);
  a.v = static_cast<const uint16_t *>(p.v);
  a.o = static_cast<uint16_t *>(p.o);
  a.lse = p.lse;
  a.partial = p.partial;
  a.lens = p.lens;
  a.sqb = p.sqb; a.sqh = p.sqh;
  a.sob = p.sob; a.soh = p.soh;
  a.slse = p.slse;
  a.skb = p.skb; a.skt = p.skt; a.skh = p.skh;
  a.svb = p.svb; a.svt = p.svt; a.svh = p.svh;
  a.S = (int)p.S;
  a.heads = (int)p.heads;
  a.group = (int)(p.heads / p.kv_heads);
  a.D = (int)p.D;
  if (p.S <= attn::kJoined) {
    const int64_t waves = attn::waves_joined(p.D);
    a.chunk = (int)std::max<int64_t>(32, ((p.S + waves - 1) / waves + 31) / 32 * 32);
    a.splits = 0;
  } else {
    a.chunk = (int)decode_chunk(p.B, p.S, p.kv_heads);
    a.splits = (int)((p.S + a.chunk - 1) / a.chunk);
  }
  a.c = p.scale * attn::kLog2e;
  // Splits outermost: sequences shorter than the cache leave the last splits
  // empty, and with splits innermost a power of two of them put every first
  // split on the same XCD (32 sequences of 300 rows in a cache of 8192, splits
  // of 512: 90 us, 16 with the order below).
  const dim3 grid((unsigned)(p.kv_heads * ((a.group + 31) / 32)), (unsigned)p.B,
                  (unsigned)std::max(1, a.splits));
  return p.dt == NOVA_HIP_DT_BF16 ? attn::launch_decode<NOVA_HIP_DT_BF16>(a, grid, s)
                                  : attn::launch_decode<NOVA_HIP_DT_F16>(a, grid, s);
}

}  // namespace nova_hip

// Attention of packed sequences, forward:  O = softmax(scale Q K^T) V per
// sequence and head, lse = log sum exp of each row's scaled scores.
//
// One pass over the keys with the running maximum m and sum l of the softmax:
// a row's accumulators are sums of exp2((s - m) c) v, c = scale log2 e, which
// a larger m multiplies by exp2((m_old - m) c).  m follows the scores only
// when one is more than 2^8 above it (the factor is exact either way, and
// f32 sums and 16-bit weights have that much room), so most tiles multiply no
// accumulator.
//
// Four waves hold 32 queries each and stream tiles of 64 keys and values through
// a two-stage ring in LDS filled by DMA; two workgroups share a CU at D = 128
// (230 registers), so that one's exponentials run beside the other's products.
// What bounds it: at D = 128 the products and the softmax, which hardly overlap
// (counters, packed causal 1 to 4096 tokens: the matrix cores 49% busy and the
// vector units 55% of the time; 8192 causal tokens, 32 heads: 535 us, 1.03 PFLOP/s,
// where a plain 8192^3 product of the library reaches 1.40 and a 4096^3 one 1.17);
// at D = 64 the exponentials and the rest of the softmax (2 x 4096 tokens, 32
// heads: 334 us, 0.82 PFLOP/s).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attention.h"

namespace nova_hip {
namespace attn {
namespace {

struct FwdArgs {
  const uint16_t *q, *k, *v;
  uint16_t *o;
  float *lse;  // [heads][Tq] with row stride slse, or null
  const int *q_off, *k_off;
  Rows sq, sk, sv, so;
  int64_t slse;
  int Tq, Tk, B, heads, group, D, tiles;  // group: query heads per key head
  float c;                                // scale * log2(e)
};

constexpr int kWaves = 4, kBM = 32 * kWaves, kBN = 64;
constexpr float kSlack = 8.0f;  // m c may lag the largest score by this much
// f16 weights are taken times 2^7: with the slack they stay under 2^15, and one
// that rounds to zero is under 2^-32 of a row's largest, not 2^-25.  Thousands of
// the latter behind one key far above them are a part of the result that f16
// shows (2^-11): 4095 keys of weight 2^-25.2 together weigh 2^-13.2, and more
// where their values are the larger ones.
template <int DT>
constexpr float kUp = DT == NOVA_HIP_DT_F16 ? 7.0f : 0.0f;

// KS groups of four waves share a tile of queries: group g takes the tiles of
// keys g, g + KS, ... through a ring of its own, and the groups' sums are joined
// at the end.  Two where the chip holds every tile of queries at once and waits
// for the longest (see launch_fwd).
template <int DT, int DP, bool CAUSAL, int KS>
__global__ __launch_bounds__(64 * kWaves * KS, 2) void attention_fwd_kernel(FwdArgs a) {
  constexpr int CH = kPitch<DP>, kTile = kBN * CH * 16;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % kWaves;
  const int part = KS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / kWaves;
  __shared__ float sm[KS > 1 ? kWaves : 1][32], sl[KS > 1 ? kWaves : 1][32];
  __shared__ __attribute__((aligned(1024))) char sk0_[KS * kTile];
  lds_char *const sk0 = (lds_char *)sk0_ + part * kTile;
  __shared__ __attribute__((aligned(1024))) char sk1_[KS * kTile];
  lds_char *const sk1 = (lds_char *)sk1_ + part * kTile;
  __shared__ __attribute__((aligned(1024))) char sv0_[KS * kTile];
  lds_char *const sv0 = (lds_char *)sv0_ + part * kTile;
  __shared__ __attribute__((aligned(1024))) char sv1_[KS * kTile];
  lds_char *const sv1 = (lds_char *)sv1_ + part * kTile;
  int head, tile;
  unit_of(blockIdx.x, a.heads, a.tiles, CAUSAL, head, tile);
  Tile at;
  if (!find_tile(a.q_off, a.k_off, a.B, a.Tq, a.Tk, kBM, tile, at)) return;
  const int row0 = at.index * kBM, qs = at.s, qe = at.e, ks = at.os, ke = at.oe;
  const int Lq = qe - qs, Lk = ke - ks;
  // Query i sees keys 0 .. i + Lk - Lq.
  const int shift = Lk - Lq;
  const int keys = CAUSAL ? min(Lk, max(0, row0 + kBM + shift)) : Lk;
  const int nt = (keys + kBN - 1) / kBN;

  const int q0 = row0 + 32 * wave, qn = min(32, Lq - q0);  // this wave's rows, maybe none
  u32x4 qf[DP / 16];
  load_cols<DP>(qf, a.q + (qs + q0) * a.sq.t + head * a.sq.h, a.sq.t, qn, a.D, lane);

  const uint16_t *kp = a.k + ks * a.sk.t + (head / a.group) * a.sk.h;
  const uint16_t *vp = a.v + ks * a.sv.t + (head / a.group) * a.sv.h;
  TileLoad<kBN, CH, kWaves> lk, lv;
  lk.init(a.sk.t, a.D);
  lv.init(a.sv.t, a.D);

  f32x16 acc[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i) acc[i] = f32x16{};
  float mc = -INFINITY, l = 0.0f;  // m c and this lane's share of the sum
  const int last = q0 + (lane & 31) + shift;  // causal: the last key this lane's row sees

  auto fetch = [&](int t, lds_char *sk, lds_char *sv) __attribute__((always_inline)) {
    lk.load(kp + (int64_t)t * kBN * a.sk.t, a.sk.t, Lk - t * kBN, a.D, sk);
    lv.load(vp + (int64_t)t * kBN * a.sv.t, a.sv.t, Lk - t * kBN, a.D, sv);
  };
  auto step = [&](int t, const lds_char *sk, const lds_char *sv) __attribute__((always_inline)) {
    const int k0 = t * kBN;
    if (qn <= 0 || (CAUSAL && k0 > q0 + qn - 1 + shift)) return;  // wave-uniform
    __builtin_amdgcn_iglp_opt(0);  // a product, an LDS read, a product, ...: 2% at D = 128
    f32x16 s[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      s[i] = f32x16{};
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk)
        s[i] = mfma_32x32x16<DT>(read_row_frag(sk, row_frag<CH>(32 * i, kk, lane)), qf[kk], s[i]);
    }
    if (k0 + kBN > Lk || (CAUSAL && k0 + kBN - 1 > q0 + shift)) {
      keep_branch();
      const int end = CAUSAL ? min(Lk, last + 1) : Lk;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (k0 + 32 * i + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3) >= end) s[i][r] = -INFINITY;
    }
    float m = s[0][0];
#pragma unroll
    for (int r = 0; r < 16; ++r) m = fmaxf(m, fmaxf(s[0][r], s[1][r]));
    m = both_max(m) * a.c;
    if (__ballot(m > mc + kSlack)) {
      const float to = fmaxf(m, mc), f = mc == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mc - to);
      mc = to;
      l *= f;
#pragma unroll
      for (int i = 0; i < DP / 32; ++i) acc[i] *= f;
    }
    const float up = kUp<DT> - (mc == -INFINITY ? 0.0f : mc);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[i][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i][r], a.c, up));
        l += s[i][r];
      }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        // The weights round to the operands' type for the product (the sum l
        // takes them in f32): half a step of it, as much as the result's own.
        const u32x4 pf = pack_frag<DT>(s[i], kk);
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
          acc[db] = mfma_32x32x16<DT>(read_col_frag<CH>(sv, 32 * i + 16 * kk, 32 * db, lane), pf,
                                      acc[db]);
      }
  };
  // One barrier per tile: behind it the tile just fetched is whole and the
  // other stage has no reader left.
  auto sync = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0): this wave's DMA has landed
    __syncthreads();
  };
  // Every group takes as many turns; one behind the last tile does nothing.
  const int nu = (nt + KS - 1) / KS;
  auto turn = [&](int u, const lds_char *sk, const lds_char *sv) __attribute__((always_inline)) {
    if (KS == 1 || u * KS + part < nt) step(u * KS + part, sk, sv);
  };
  if (nu > 0) fetch(part, sk0, sv0);
  for (int u = 0; u < nu; u += 2) {
    sync();
    if (u + 1 < nu) fetch((u + 1) * KS + part, sk1, sv1);
    turn(u, sk0, sv0);
    if (u + 1 >= nu) break;
    sync();
    if (u + 2 < nu) fetch((u + 2) * KS + part, sk0, sv0);
    turn(u + 1, sk1, sv1);
  }
  l = both_sum(l);
  if constexpr (KS > 1) {
    static_assert(KS == 2 && KS * kTile >= kWaves * 64 * 16 * 4, "one block of each wave's sums");
    lds_float *const box = (lds_float *)(lds_char *)sk0_ + wave * 1024 + lane;
    __syncthreads();
    if (part == 1 && lane < 32) {
      sm[wave][lane] = mc;
      sl[wave][lane] = l;
    }
    float mine = 0.0f, other = 0.0f;  // factors of the two groups' sums
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) {
      if (i) __syncthreads();
      if (part == 1) {
#pragma unroll
        for (int r = 0; r < 16; ++r) box[64 * r] = acc[i][r];
      }
      __syncthreads();
      if (part == 0) {
        if (i == 0) {
          const float m1 = sm[wave][lane & 31], to = fmaxf(mc, m1);
          mine = mc == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mc - to);
          other = m1 == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m1 - to);
          l = l * mine + sl[wave][lane & 31] * other;
          mc = to;
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] = acc[i][r] * mine + box[64 * r] * other;
      }
    }
    if (part == 1) return;
  }
  if (qn <= 0) return;
  // A row that sees no key is zero, its lse -inf.
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  store_rows<DT, DP>(acc, inv, a.o + (qs + q0) * a.so.t + head * a.so.h, a.so.t, qn, a.D, lane);
  if (a.lse && lane < qn)
    a.lse[head * a.slse + qs + q0 + lane] = l == 0.0f ? -INFINITY : (mc + (__log2f(l) - kUp<DT>)) * kLn2;
}

template <int DT, int DP, int KS>
void launch_fwd_k(const FwdArgs &a, bool causal, unsigned grid, hipStream_t s) {
  if (causal)
    hipLaunchKernelGGL((attention_fwd_kernel<DT, DP, true, KS>), dim3(grid), dim3(64 * kWaves * KS),
                       0, s, a);
  else
    hipLaunchKernelGGL((attention_fwd_kernel<DT, DP, false, KS>), dim3(grid), dim3(64 * kWaves * KS),
                       0, s, a);
}
template <int DT, int DP>
void launch_fwd(const FwdArgs &a, bool causal, unsigned grid, hipStream_t s) {
  // Two groups while one workgroup of them per CU (of causal ones, whose work
  // differs, two at D <= 64) holds all tiles.  One group against two, us: 1000
  // causal tokens of 6 heads of 64 18.1 / 15.6, packed 1 to 4096 of these heads
  // (426 tiles) 62.7 / 50.2, 3000 of 8 heads of 128 57.9 / 47.1; beyond, 4 x
  // 1024 of 12 heads of 128 (432 tiles) 37.6 / 45.0.
  // Not for sequences of less than eight tiles of keys in the mean, which lose
  // to the join what they gain (8 x 197 of 12 heads of 64: 8.7 / 9.2).
  const unsigned few = causal && a.D <= 64 ? 512 : 256;
  if (grid <= few && a.Tk / a.B >= 8 * kBN) launch_fwd_k<DT, DP, 2>(a, causal, grid, s);
  else launch_fwd_k<DT, DP, 1>(a, causal, grid, s);
}
template <int DT>
void launch_fwd(const FwdArgs &a, bool causal, unsigned grid, hipStream_t s) {
  if (a.D <= 32) launch_fwd<DT, 32>(a, causal, grid, s);
  else if (a.D <= 64) launch_fwd<DT, 64>(a, causal, grid, s);
  else if (a.D <= 96) launch_fwd<DT, 96>(a, causal, grid, s);
  else launch_fwd<DT, 128>(a, causal, grid, s);
}

}  // namespace
}  // namespace attn

int32_t launch_attention(const AttentionProblem &p, hipStream_t s) {
  if (p.Tq == 0 || p.heads == 0 || p.D == 0 || p.B == 0) return NOVA_HIP_SUCCESS;
  attn::FwdArgs a;
  a.q = static_cast<const uint16_t *>(p.q.p);
  a.k = static_cast<const uint16_t *>(p.k.p);
  a.v = static_cast<const uint16_t *>(p.v.p);
  a.o = static_cast<uint16_t *>(p.o.p);
  a.lse = p.lse;
  a.slse = p.slse;
  a.q_off = p.q_off;
  a.k_off = p.k_off;
  a.sq = {p.q.st, p.q.sh};
  a.sk = {p.k.st, p.k.sh};
  a.sv = {p.v.st, p.v.sh};
  a.so = {p.o.st, p.o.sh};
  a.Tq = (int)p.Tq;
  a.Tk = (int)p.Tk;
  a.B = (int)p.B;
  a.heads = (int)p.heads;
  a.group = (int)(p.heads / p.kv_heads);
  a.D = (int)p.D;
  a.c = p.scale * attn::kLog2e;
  const int64_t tiles = attn::tile_bound(p.Tq, p.B, attn::kBM);
  // A grid's dimension holds less than 2^32 threads.
  if (tiles * p.heads >= 1 << 24)
    return fail(NOVA_HIP_ERANGE, "attention: %lld tiles of %lld heads exceed 2^24 - 1",
                (long long)tiles, (long long)p.heads);
  const Extent q = extent("q", p.q, p.Tq, p.heads, p.D), k = extent("k", p.k, p.Tk, p.kv_heads, p.D),
               v = extent("v", p.v, p.Tk, p.kv_heads, p.D),
               out = extent("out", p.o, p.Tq, p.heads, p.D),
               lse = {"lse", p.lse, p.lse ? 4 * p.Tq : 0, {p.heads, 1, 1}, {4 * p.slse, 0, 0}};
  int32_t rc;
  if ((rc = check_apart("attention", out, {q, k, v})) ||
      (rc = check_apart("attention", lse, {q, k, v, out})))
    return rc;
  a.tiles = (int)tiles;
  const unsigned grid = (unsigned)(tiles * p.heads);
  if (p.dt == NOVA_HIP_DT_BF16) attn::launch_fwd<NOVA_HIP_DT_BF16>(a, p.causal, grid, s);
  else attn::launch_fwd<NOVA_HIP_DT_F16>(a, p.causal, grid, s);
  return check_hip(hipGetLastError(), "attention launch");
}

}  // namespace nova_hip

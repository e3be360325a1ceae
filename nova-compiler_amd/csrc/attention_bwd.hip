// Backward of attention over packed sequences (attention.hip), from the
// forward's result and log-sum-exp:  P = exp(scale S - lse),
//   dV = P^T dO,  dP = dO V^T,  dS = P o (dP - delta),  delta = rowsum(dO o O),
//   dQ = scale dS K,  dK = scale dS^T Q.
//
// Two kernels, each recomputing P and dP for itself, so that every sum is made
// in a fixed order: no atomics, the same bits on every run, and the gradients of
// keys shared by a group of query heads are summed over the group inside the
// workgroup (or, where its queries are split into runs, over the runs in order
// by a third kernel).  That is seven products where five are the least.
// attention_dq_kernel holds 32 queries per wave and streams keys and values; it
// also writes the rows' two constants (lse in base 2, delta), which
// attention_dkv_kernel, behind it on the stream, reads while it holds keys and
// values and streams Q and dO.
//
// What bounds them at D = 128 (2 x 4096 tokens, 32 heads, not causal): products and
// exponentials that overlap in part for dQ (755 us, 1.09 PFLOP/s of its three
// products; counters: the matrix cores 51% busy, the vector units 36%), the issue
// of one wave per SIMD for dK and dV (1045 us, 1.05 of four; 49% and 30%).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attention.h"
#include "wave.h"

namespace nova_hip {
namespace attn {
namespace {

struct BwdArgs {
  const uint16_t *q, *k, *v, *o, *go;
  const float *lse;
  uint16_t *dq, *dk, *dv;
  float *rows;  // [2][heads][Tq]: lse log2 e, -delta
  float *partial;  // [key heads][tiles][splits][wave][dK, dV][DP / 2][lane] (splits > 1)
  const int *q_off, *k_off;
  Rows sq, sk, sv, so, sgo, sdq, sdk, sdv;
  int64_t slse;
  int Tq, Tk, B, heads, group, D, tiles, splits;
  int least;        // tiles of queries in a run
  float share;      // and the part of the batch's work that it takes at least
  bool last_first;  // the last runs are launched first
  float c, scale;
};

typedef __attribute__((address_space(3))) const gemm::f32x4 lds_f32x4;

constexpr int kWaves = 4, kBM = 32 * kWaves, kBN = 64;

// Floats of one wave's dK and dV.
template <int DP>
constexpr int64_t kPartial = DP * 64;

// f16 weights take a factor 2^8 in the product for dV (they are at most 1, and
// in long rows most lie under 2^-14, where f16 has fewer bits), taken back at
// the store; bf16 has f32's exponents and needs none.
template <int DT>
constexpr float kWeightLog2 = DT == NOVA_HIP_DT_F16 ? 8.0f : 0.0f;

// f16 dS is as small as the gradient that came in (a mean over thousands of
// tokens: under 2^-24, where f16 has nothing left) and as large as its loss scale
// makes it, so each column of a product with it (a lane and its partner) has a
// factor 2^up of its own, which its sums carry until they are complete.  It starts
// at 2^40, and is lowered, with the sums so far, where a value would pass 2^15: the
// largest comes to [2^5, 2^6) then, so that what rounds to zero is under 2^-30 of
// the column's largest.  (Factors of two are exact.)  bf16 has f32's exponents.
constexpr float kUp = 40.0f;
template <int DP>
__device__ __forceinline__ void fit_f16(f32x16 &ds, f32x16 (&acc)[DP / 32], float &up) {
  float t = 0.0f;
#pragma unroll
  for (int r = 0; r < 16; ++r) t = fmaxf(t, fabsf(ds[r]));
  if (__ballot(t > 32768.0f)) {
    keep_branch();
    t = both_max(t);
    const int by = t > 32768.0f && t < INFINITY ? 6 - __builtin_amdgcn_frexp_expf(t) : 0;
    const float f = __builtin_amdgcn_ldexpf(1.0f, by);
    up += (float)by;
    ds *= f;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) acc[i] *= f;
  }
}
// Takes the factor back.
template <int DT, int DP>
__device__ __forceinline__ void unfit(f32x16 (&acc)[DP / 32], float up) {
  if constexpr (DT == NOVA_HIP_DT_F16) {
    const float f = __builtin_amdgcn_ldexpf(1.0f, -(int)up);
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) acc[i] *= f;
  }
}

// sum over d of a row's products, the row held as load_cols gives it.
template <int DT, int DP>
__device__ __forceinline__ float row_dot(const u32x4 (&x)[DP / 16], const u32x4 (&y)[DP / 16]) {
  float s = 0.0f;
#pragma unroll
  for (int i = 0; i < DP / 16; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (DT == NOVA_HIP_DT_BF16) {
        s = __builtin_fmaf(__uint_as_float(x[i][j] << 16), __uint_as_float(y[i][j] << 16), s);
        s = __builtin_fmaf(__uint_as_float(x[i][j] & 0xffff0000u),
                           __uint_as_float(y[i][j] & 0xffff0000u), s);
      } else {
        const auto a = __builtin_bit_cast(gemm::f16x2v, (uint32_t)x[i][j]);
        const auto b = __builtin_bit_cast(gemm::f16x2v, (uint32_t)y[i][j]);
        s = __builtin_fmaf((float)a[0], (float)b[0], s);
        s = __builtin_fmaf((float)a[1], (float)b[1], s);
      }
    }
  return both_sum(s);
}

// Adds the second group of waves' sums to the first's, block by block through
// 16 KB of LDS, all of whose readers are done when every wave has come here.
template <int DP>
__device__ __forceinline__ void add_group(f32x16 (&acc)[DP / 32], lds_char *lds, int wave, int part,
                                          int lane) {
  lds_float *const box = (lds_float *)lds + wave * 1024 + lane;
#pragma unroll
  for (int i = 0; i < DP / 32; ++i) {
    __syncthreads();
    if (part == 1) {
#pragma unroll
      for (int r = 0; r < 16; ++r) box[64 * r] = acc[i][r];
    }
    __syncthreads();
    if (part == 0) {
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][r] += box[64 * r];
    }
  }
}

// KS groups of four waves share a tile of queries, as in the forward: group g
// takes the tiles of keys g, g + KS, ... and the groups' sums are added at the end.
template <int DT, int DP, bool CAUSAL, int KS>
__global__ __launch_bounds__(64 * kWaves * KS, 2) void attention_dq_kernel(BwdArgs a) {
  constexpr int CH = kPitch<DP>, kTile = kBN * CH * 16;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % kWaves;
  const int part = KS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / kWaves;
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
  Tile place;
  if (!find_tile(a.q_off, a.k_off, a.B, a.Tq, a.Tk, kBM, tile, place)) return;
  const int row0 = place.index * kBM, qs = place.s, qe = place.e, ks = place.os, ke = place.oe;
  const int Lq = qe - qs, Lk = ke - ks, shift = Lk - Lq;
  const int keys = CAUSAL ? min(Lk, max(0, row0 + kBM + shift)) : Lk;
  const int nt = (keys + kBN - 1) / kBN;

  const int q0 = row0 + 32 * wave, qn = min(32, Lq - q0);
  u32x4 qf[DP / 16], gf[DP / 16];
  load_cols<DP>(qf, a.q + (qs + q0) * a.sq.t + head * a.sq.h, a.sq.t, qn, a.D, lane);
  load_cols<DP>(gf, a.go + (qs + q0) * a.sgo.t + head * a.sgo.h, a.sgo.t, qn, a.D, lane);
  float nl = 0.0f, delta;
  {
    u32x4 of[DP / 16];
    load_cols<DP>(of, a.o + (qs + q0) * a.so.t + head * a.so.h, a.so.t, qn, a.D, lane);
    delta = row_dot<DT, DP>(gf, of);
  }
  const int64_t at = (int64_t)head * a.Tq + qs + q0 + (lane & 31);
  if ((lane & 31) < qn) {
    const float lse = a.lse[head * a.slse + qs + q0 + (lane & 31)];
    // A row without keys (lse -inf): every weight is masked below.
    nl = lse == -INFINITY ? 0.0f : lse * kLog2e;
    if (lane < 32 && part == 0) {
      a.rows[at] = nl - kWeightLog2<DT>;
      a.rows[(int64_t)a.heads * a.Tq + at] = -delta;
    }
  }

  const uint16_t *kp = a.k + ks * a.sk.t + (head / a.group) * a.sk.h;
  const uint16_t *vp = a.v + ks * a.sv.t + (head / a.group) * a.sv.h;
  TileLoad<kBN, CH, kWaves> lk, lv;
  lk.init(a.sk.t, a.D);
  lv.init(a.sv.t, a.D);
  f32x16 acc[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i) acc[i] = f32x16{};
  float up = DT == NOVA_HIP_DT_F16 ? kUp : 0.0f;  // of dS, see fit_f16
  const int last = q0 + (lane & 31) + shift;

  auto fetch = [&](int t, lds_char *sk, lds_char *sv) __attribute__((always_inline)) {
    lk.load(kp + (int64_t)t * kBN * a.sk.t, a.sk.t, Lk - t * kBN, a.D, sk);
    lv.load(vp + (int64_t)t * kBN * a.sv.t, a.sv.t, Lk - t * kBN, a.D, sv);
  };
  auto step = [&](int t, const lds_char *sk, const lds_char *sv) __attribute__((always_inline)) {
    const int k0 = t * kBN;
    if (qn <= 0 || (CAUSAL && k0 > q0 + qn - 1 + shift)) return;
    const bool edge = k0 + kBN > Lk || (CAUSAL && k0 + kBN - 1 > q0 + shift);
    const int end = CAUSAL ? min(Lk, last + 1) : Lk;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      f32x16 s = {}, dp = {};
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk) {
        s = mfma_32x32x16<DT>(read_row_frag(sk, row_frag<CH>(32 * i, kk, lane)), qf[kk], s);
        dp = mfma_32x32x16<DT>(read_row_frag(sv, row_frag<CH>(32 * i, kk, lane)), gf[kk], dp);
      }
      const float add = up - nl;
#pragma unroll
      for (int r = 0; r < 16; ++r)
        s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], a.c, add)) * (dp[r] - delta);
      if (edge) {
        keep_branch();
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (k0 + 32 * i + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3) >= end) s[r] = 0.0f;
      }
      if constexpr (DT == NOVA_HIP_DT_F16) fit_f16<DP>(s, acc, up);
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const u32x4 sf = pack_frag<DT>(s, kk);  // dS rounds to the operands' type
#pragma unroll
        for (int db = 0; db < DP / 32; ++db)
          acc[db] = mfma_32x32x16<DT>(read_col_frag<CH>(sk, 32 * i + 16 * kk, 32 * db, lane), sf,
                                      acc[db]);
      }
    }
  };
  auto sync = [&]() __attribute__((always_inline)) {
    __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
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
  unfit<DT, DP>(acc, up);
  if constexpr (KS > 1) {
    static_assert(KS == 2, "one group hands its sums to the other");
    add_group<DP>(acc, (lds_char *)sk0_, wave, part, lane);
    if (part == 1) return;
  }
  if (qn <= 0) return;
  store_rows<DT, DP>(acc, a.scale, a.dq + (qs + q0) * a.sdq.t + head * a.sdq.h, a.sdq.t, qn, a.D,
                     lane);
}

// Runs that the `total` tiles of queries of a tile of keys are split into: none
// shorter than the least, nor than a.share of the batch's work, which the offsets
// give.  Two kernels must come to the same number, so no product here can be
// fused with a sum but the one that is.
template <bool CAUSAL>
__device__ __forceinline__ int runs_of(const BwdArgs &a, int total) {
  if (a.splits == 1) return 1;
  const int lane = threadIdx.x & 63;
  float work = 0.0f;
  for (int b = lane; b < a.B; b += 64) {
    const float k = (float)a.k_off[b + 1] - (float)a.k_off[b];
    const float q = (float)a.q_off[b + 1] - (float)a.q_off[b];
    work = __builtin_fmaf(k, q, work);
  }
  work = wave_sum(work) * (CAUSAL ? 0.5f : 1.0f) / (kBM * kBN) * (float)a.heads;
  const int length = max(a.least, (int)fminf(fmaxf(work, 0.0f) * a.share, 1e9f));
  return __builtin_amdgcn_readfirstlane(min(a.splits, max(1, total / length)));
}

// The first query of a sequence that sees a key from row0 on.
template <bool CAUSAL>
__device__ __forceinline__ int first_query(int row0, int Lq, int Lk) {
  return CAUSAL ? min(Lq, max(0, row0 - (Lk - Lq))) : 0;
}

// 128 keys, 32 to a wave, x the queries that see them in every query head of the
// group: `total` tiles of 64 queries, or, where tiles of keys alone are too few
// or too uneven for the chip, one of up to `splits` runs of them; the runs' sums
// then go to scratch and attention_dkv_join_kernel adds them in order.  (The run
// that ends last adding them, behind a fence, made the L2s write back and forget:
// 680 -> 1470 us packed as below.)  Runs are the grid's outer dimension, so that
// those which a shorter tile has not got lie together: between the others they
// keep whole shader engines idle (8192 tokens, 32 heads in groups of 4 of 128,
// two runs at most: 1755 us, 2394 the other way).
//
// At D = 128 the keys, the values and the two gradients of a wave's 32 keys
// take 192 registers, so one wave runs per SIMD (two at D <= 64).  What then
// bounds it is the issue of one wave: of 4400 cycles per tile of 64 queries
// 2048 are the products, 2400 go by issuing instructions (counters).  Hence
// few of them: masked tiles in a loop of their own, the heads' and tiles'
// pointers advanced and not computed, dP's sum started from -delta.
template <int DT, int DP, bool CAUSAL>
__global__ __launch_bounds__(64 * kWaves, DP <= 64 ? 2 : 1) void attention_dkv_kernel(BwdArgs a) {
  constexpr int CH = kPitch<DP>, kTile = kBN * CH * 16;
  __shared__ __attribute__((aligned(1024))) char sq0_[kTile];
  lds_char *const sq0 = (lds_char *)sq0_;
  __shared__ __attribute__((aligned(1024))) char sq1_[kTile];
  lds_char *const sq1 = (lds_char *)sq1_;
  __shared__ __attribute__((aligned(1024))) char sg0_[kTile];
  lds_char *const sg0 = (lds_char *)sg0_;
  __shared__ __attribute__((aligned(1024))) char sg1_[kTile];
  lds_char *const sg1 = (lds_char *)sg1_;
  __shared__ __attribute__((aligned(1024))) float sc0_[2 * kBN];  // the tile's row constants
  lds_float *const sc0 = (lds_float *)sc0_;
  __shared__ __attribute__((aligned(1024))) float sc1_[2 * kBN];
  lds_float *const sc1 = (lds_float *)sc1_;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kv_heads = a.heads / a.group;
  int kh, tile;
  if ((int)blockIdx.x >= kv_heads * a.tiles) return;
  unit_of(blockIdx.x, kv_heads, a.tiles, CAUSAL, kh, tile);
  const int split = a.last_first ? a.splits - 1 - blockIdx.y : blockIdx.y;
  const int unit = kh * a.tiles + tile;
  Tile place;
  if (!find_tile(a.k_off, a.q_off, a.B, a.Tk, a.Tq, kBM, tile, place)) return;
  // Causal: the first keys have the most queries.
  const int row0 = (place.tiles - 1 - place.index) * kBM;
  const int qs = place.os, qe = place.oe, ks = place.s, ke = place.e;
  const int Lq = qe - qs, Lk = ke - ks, shift = Lk - Lq;
  // Causal: key j is seen by the queries j - shift and on.
  const int first = first_query<CAUSAL>(row0, Lq, Lk);
  const int nt = (Lq - first + kBN - 1) / kBN, total = nt * a.group;
  // The first `nm` of a head's tiles of queries hold some that do not see all of
  // the keys.  Every head's come first, the others behind them, in a loop of
  // its own without masks.
  const int nm = CAUSAL ? min(nt, max(0, (row0 + kBM - shift - first + kBN - 2) / kBN)) : 0;
  const int masked = nm * a.group;
  const int runs = runs_of<CAUSAL>(a, total);
  if (split >= runs) return;
  const int from = (int)((int64_t)total * split / runs);
  const int to = (int)((int64_t)total * (split + 1) / runs);

  const int k0 = row0 + 32 * wave, kn = min(32, Lk - k0);
  u32x4 kf[DP / 16], vf[DP / 16];
  load_cols<DP>(kf, a.k + (int64_t)(ks + k0) * a.sk.t + kh * a.sk.h, a.sk.t, kn, a.D, lane);
  load_cols<DP>(vf, a.v + (int64_t)(ks + k0) * a.sv.t + kh * a.sv.h, a.sv.t, kn, a.D, lane);
  TileLoad<kBN, CH, kWaves> lq, lg;
  lq.init(a.sq.t, a.D);
  lg.init(a.sgo.t, a.D);
  float up = DT == NOVA_HIP_DT_F16 ? kUp : 0.0f;  // of dS, see fit_f16
  f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i) dk[i] = dv[i] = f32x16{};

  // Tiles [lo, hi) of the part of each head's tiles [j0, j1).
  auto run = [&](auto mask, int lo, int hi, int j0, int j1) __attribute__((always_inline)) {
    constexpr bool kMask = decltype(mask)::value;
    if (lo >= hi) return;
    // The next tile to fetch, and (masked) the next to compute: head of the
    // group and tile.
    int fg = lo / (j1 - j0), fj = j0 + lo - fg * (j1 - j0), cj = fj;
    auto fetch = [&](lds_char *sq, lds_char *sg, lds_float *sc) __attribute__((always_inline)) {
      const int q0 = first + fj * kBN, head = kh * a.group + fg, left = Lq - q0;
      lq.load(a.q + (int64_t)(qs + q0) * a.sq.t + head * a.sq.h, a.sq.t, left, a.D, sq);
      lg.load(a.go + (int64_t)(qs + q0) * a.sgo.t + head * a.sgo.h, a.sgo.t, left, a.D, sg);
      // Rows behind the sequence read zero: with q and dO zero there too, they
      // add nothing.
      if (wave < 2) {
        const float *p = a.rows + ((int64_t)wave * a.heads + head) * a.Tq + qs + q0;
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<float *>(p), (short)0, min(left, kBN) * 4, 0x00020000);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void *)(sc + kBN * wave), 4, lane * 4, 0,
                                                 0, 0);
      }
      if (++fj == j1) {
        fj = j0;
        ++fg;
      }
    };
    auto step = [&](const lds_char *sq, const lds_char *sg, const lds_float *sc)
        __attribute__((always_inline)) {
      const int q0 = first + cj * kBN;
      if (kMask && ++cj == j1) cj = j0;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (kMask && q0 + 32 * i + 31 + shift < k0) continue;  // none of these sees these keys
        __builtin_amdgcn_iglp_opt(0);  // a product, an LDS read, a product, ...
        f32x16 s = {}, dp;
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const gemm::f32x4 de = *(lds_f32x4 *)(sc + kBN + 32 * i + 8 * r4 + 4 * (lane >> 5));
#pragma unroll
          for (int e = 0; e < 4; ++e) dp[4 * r4 + e] = de[e];
        }
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
          s = mfma_32x32x16<DT>(read_row_frag(sq, row_frag<CH>(32 * i, kk, lane)), kf[kk], s);
          dp = mfma_32x32x16<DT>(read_row_frag(sg, row_frag<CH>(32 * i, kk, lane)), vf[kk], dp);
        }
        // From the weights' factor to that of dS.
        const float down =
            DT == NOVA_HIP_DT_F16 ? __builtin_amdgcn_exp2f(up - kWeightLog2<DT>) : 1.0f;
        // Rows of this block from which on the lane's key is seen.
        const int seen = kMask ? k0 + (lane & 31) - shift - q0 - 32 * i - 4 * (lane >> 5) : 0;
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const gemm::f32x4 nl = *(lds_f32x4 *)(sc + 32 * i + 8 * r4 + 4 * (lane >> 5));
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int r = 4 * r4 + e;
            s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], a.c, -nl[e]));
            dp[r] = s[r] * (DT == NOVA_HIP_DT_F16 ? dp[r] * down : dp[r]);
            if constexpr (kMask)
              if (8 * (r >> 2) + (r & 3) < seen) s[r] = dp[r] = 0.0f;
          }
        }
        if constexpr (DT == NOVA_HIP_DT_F16) fit_f16<DP>(dp, dk, up);
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
          // Weights and dS round to the operands' type for these products.
          const u32x4 pf = pack_frag<DT>(s, kk), sf = pack_frag<DT>(dp, kk);
#pragma unroll
          for (int db = 0; db < DP / 32; ++db) {
            dv[db] = mfma_32x32x16<DT>(read_col_frag<CH>(sg, 32 * i + 16 * kk, 32 * db, lane), pf,
                                       dv[db]);
            dk[db] = mfma_32x32x16<DT>(read_col_frag<CH>(sq, 32 * i + 16 * kk, 32 * db, lane), sf,
                                       dk[db]);
          }
        }
      }
    };
    auto sync = [&]() __attribute__((always_inline)) {
      __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
      __syncthreads();
    };
    fetch(sq0, sg0, sc0);
    for (int u = lo; u < hi; u += 2) {
      if constexpr (DP > 64) {
        // The gradients stay in the accumulation registers: left to the compiler
        // they moved between the files in each tile (2 x 4096 tokens, not causal,
        // 32 heads of 128: 1310 -> 1045 us).
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) asm volatile("" : "+a"(dk[i]), "+a"(dv[i]));
      }
      sync();
      if (u + 1 < hi) fetch(sq1, sg1, sc1);
      step(sq0, sg0, sc0);
      if (u + 1 >= hi) break;
      sync();
      if (u + 2 < hi) fetch(sq0, sg0, sc0);
      step(sq1, sg1, sc1);
    }
    __syncthreads();  // stage 0 has no reader left
  };
  if constexpr (CAUSAL) run(std::true_type(), from, min(to, masked), 0, nm);
  run(std::false_type(), max(from - masked, 0), to - masked, nm, nt);
  if (kn <= 0) return;
  unfit<DT, DP>(dk, up);
  if (runs > 1) {
    float *p = a.partial + (((int64_t)unit * a.splits + split) * kWaves + wave) * kPartial<DP> + lane;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        p[(16 * i + r) * 64] = dk[i][r];
        p[(DP / 2 + 16 * i + r) * 64] = dv[i][r];
      }
    return;
  }
  store_rows<DT, DP>(dk, a.scale, a.dk + (int64_t)(ks + k0) * a.sdk.t + kh * a.sdk.h, a.sdk.t, kn,
                     a.D, lane);
  store_rows<DT, DP>(dv, DT == NOVA_HIP_DT_F16 ? 1.0f / 256.0f : 1.0f,
                     a.dv + (int64_t)(ks + k0) * a.sdv.t + kh * a.sdv.h, a.sdv.t, kn, a.D, lane);
}

// The sums of a tile of keys from those of its splits, in split order.
template <int DT, int DP, bool CAUSAL>
__global__ __launch_bounds__(64 * kWaves) void attention_dkv_join_kernel(BwdArgs a) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int w = blockIdx.x, kh = w / a.tiles;
  Tile place;
  if (!find_tile(a.k_off, a.q_off, a.B, a.Tk, a.Tq, kBM, w - kh * a.tiles, place)) return;
  const int ks = place.s, ke = place.e;
  const int row0 = (place.tiles - 1 - place.index) * kBM;
  const int k0 = row0 + 32 * wave, kn = min(32, ke - ks - k0);
  if (kn <= 0) return;
  const int Lq = place.oe - place.os, first = first_query<CAUSAL>(row0, Lq, ke - ks);
  const int runs = runs_of<CAUSAL>(a, (Lq - first + kBN - 1) / kBN * a.group);
  if (runs == 1) return;
  f32x16 x[DP / 32];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const float *p = a.partial + ((int64_t)w * a.splits * kWaves + wave) * kPartial<DP> +
                     half * (DP / 2 * 64) + lane;
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) x[i][r] = p[(16 * i + r) * 64];
    for (int s = 1; s < runs; ++s) {
      p += (int64_t)kWaves * kPartial<DP>;
#pragma unroll
      for (int i = 0; i < DP / 32; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) x[i][r] += p[(16 * i + r) * 64];
    }
    if (half == 0)
      store_rows<DT, DP>(x, a.scale, a.dk + (ks + k0) * a.sdk.t + kh * a.sdk.h, a.sdk.t, kn, a.D,
                         lane);
    else
      store_rows<DT, DP>(x, DT == NOVA_HIP_DT_F16 ? 1.0f / 256.0f : 1.0f,
                         a.dv + (ks + k0) * a.sdv.t + kh * a.sdv.h, a.sdv.t, kn, a.D, lane);
  }
}

template <int DT, int DP, bool CAUSAL>
int32_t launch_bwd_t(BwdArgs a, int64_t q_tiles, int64_t k_tiles, hipStream_t s) {
  if (q_tiles > 0) {
    a.tiles = (int)q_tiles;
    const unsigned grid = (unsigned)(q_tiles * a.heads);
    // Two groups while the tiles' number is within the workgroups of one group that
    // the chip holds (two per CU) and the longest tile decides.  At D > 64 it holds
    // 256 of two groups, so that causal batches of more take a second round, of
    // their shortest tiles: still less than the longest's turns.  The whole backward
    // with one group and with two, us, causal:
    //   2048 tokens, 8 heads of 128 (136 tiles); 3000, 12 (288)    115 / 102, 179 / 160
    //   4096, 8 of 128 (264); 8192, 6 (390)                        221 / 194, 481 / 430
    //   2 x 2048, 12 of 128 (408); 4 x 1024, 12 (432)              141 / 132, 85.5 / 88.1
    //   packed 1 to 4096, 6 of 128 (426); of 96                    214 / 185, 168 / 152
    //   8 x 1024, 7 of 128 (504); of 96                            92.6 / 97.3, 75.7 / 79.1
    //   4096, 8 of 64 (264); packed 1 to 4096, 6 of 64 (426)       114 / 105, 134 / 122
    //   4 x 1024, 12 of 64 (432); 8 x 1024, 6 of 64 (432)          46.2 / 48.2, 46.5 / 48.3
    // so equal sequences of 1024 lose 3 to 5% by what packed batches of as many
    // tokens gain 9 to 13% by.  Beyond, 8 x 1024 not causal of 6 heads of 64 (432
    // tiles) 65 / 76.  Short sequences lose it to the join (8 x 512 of 6 heads of 64
    // 27.1 / 27.9).
    if (grid <= (CAUSAL ? 512 : 256) && a.Tk / a.B >= 10 * kBN)
      hipLaunchKernelGGL((attention_dq_kernel<DT, DP, CAUSAL, 2>), dim3(grid), dim3(128 * kWaves), 0,
                         s, a);
    else
      hipLaunchKernelGGL((attention_dq_kernel<DT, DP, CAUSAL, 1>), dim3(grid), dim3(64 * kWaves), 0,
                         s, a);
    const int32_t rc = check_hip(hipGetLastError(), "attention_backward launch");
    if (rc) return rc;
  }
  if (k_tiles > 0) {
    a.tiles = (int)k_tiles;
    const unsigned grid = (unsigned)(k_tiles * (a.heads / a.group));
    hipLaunchKernelGGL((attention_dkv_kernel<DT, DP, CAUSAL>),
                       dim3(a.splits > 1 ? (grid + 7) / 8 * 8 : grid, a.splits), dim3(64 * kWaves),
                       0, s, a);
    if (a.splits > 1) {
      const int32_t rc = check_hip(hipGetLastError(), "attention_backward launch");
      if (rc) return rc;
      hipLaunchKernelGGL((attention_dkv_join_kernel<DT, DP, CAUSAL>), dim3(grid),
                         dim3(64 * kWaves), 0, s, a);
    }
  }
  return check_hip(hipGetLastError(), "attention_backward launch");
}
template <int DT, int DP>
int32_t launch_bwd_c(const BwdArgs &a, bool causal, int64_t qt, int64_t kt, hipStream_t s) {
  return causal ? launch_bwd_t<DT, DP, true>(a, qt, kt, s) : launch_bwd_t<DT, DP, false>(a, qt, kt, s);
}
template <int DT>
int32_t launch_bwd(const BwdArgs &a, bool causal, int64_t qt, int64_t kt, hipStream_t s) {
  if (a.D <= 32) return launch_bwd_c<DT, 32>(a, causal, qt, kt, s);
  if (a.D <= 64) return launch_bwd_c<DT, 64>(a, causal, qt, kt, s);
  if (a.D <= 96) return launch_bwd_c<DT, 96>(a, causal, qt, kt, s);
  return launch_bwd_c<DT, 128>(a, causal, qt, kt, s);
}

}  // namespace
}  // namespace attn

namespace {
int64_t padded_dim(int64_t D) { return D <= 32 ? 32 : D <= 64 ? 64 : D <= 96 ? 96 : 128; }
int64_t tile_bound(int64_t T, int64_t B) { return attn::tile_bound(T, B, attn::kBM); }

// Runs of queries that tiles of keys are split into, where the longest of them
// would keep the chip waiting.  The host knows the sequences' number and tokens;
// `most` follows from them, and the device splits those tiles that are long.
// With fewer tiles than the chip takes at once (256, 512 at D <= 64), up to four
// runs, or eight for very few tiles; with up to four times as many, causal, two,
// the last ones first (the longest tiles have them).
//
// A run has `least` tiles of 64 queries at least: 8 where tiles are few or long in
// time (D > 64), else 16.  And at least a slot's share of the batch's work, of which
// causal tiles, the longest twice the mean, take a half (a quarter / a half, us,
// packed 568 tiles as below 687 / 674, 2 x 4096 tokens of 8 heads of 128 312 / 283)
// and the others, as long as their sequence, all (a half / all: 4 x 2048 of 6 heads
// of 64 134 / 116, 8 x 1024 of 3 of 128 90 / 73, packed 1 to 4096 of 6 of 64 199 /
// 187).  Where the tiles are just more than the chip takes, halves of all of them
// fill it evenly (2 x 8192 of 16 in groups of 8 of 128, 260 tiles: 2380 / 1800).
//
// Nothing is split where no sequence is likely to be long enough: two runs of 16 or
// three of 8 in the geometric mean of all sequences of one length and one that has
// all tokens.  The host cannot tell these apart, so equal sequences pay for the
// join's launch (3 us, 6 at D > 64) and packed ones of the same number gain.  The
// whole backward without runs and with them, us, causal unless said otherwise:
//   8 x 1024 / 1 to 4096 packed, 6 heads of 64 (432, 426 tiles)  49.3 / 52.1, 122 / 116
//   9 x 1024, 4 x 2048, 6 of 64                                   54.7 / 58.0, 73.6 / 78.3
//   4000 and seven shorter to 50, 6 of 64                         117 / 99
//   8 x 1024 / 1 to 4096 packed, 3 of 128                         65 / 71, 192 / 163
//   8 x 1024, 4 x 2048 / 1 to 4096 packed, 8 of 128               89 / 96, 146 / 162, 236 / 241
//   1 to 4096 packed, 32 in groups of 4 of 128 (568)              720 / 666
//   8 x 1024, 8 in groups of 4 of 128                             151 / 112
//   4096, 8 in groups of 4 of 128 (66)                            491 / 218
//   2 x 2048, 16 in groups of 4 of 128 (136)                      278 / 182
//   8192, 6 of 64 (390); 12 in groups of 3 of 64 (260)            244 / 230, 553 / 424
//   2 x 4096 not causal, 8 in groups of 4 of 64 (132)             482 / 281
// and under the bound, with runs from half of it on: 2 x 1024 of 6 of 64 39.9 /
// 43.8, 1024 39.8 / 43.2, but 2000 and 48 65 / 58.
struct Runs {
  int64_t most;
  int least;
  float share;
  bool last_first;
};
Runs dkv_runs(int64_t Tq, int64_t Tk, int64_t B, int64_t heads, int64_t kv_heads, int64_t D,
              bool causal) {
  if (B == 0 || kv_heads == 0 || Tk == 0) return {1, 1, 0.0f, false};
  const int64_t units = tile_bound(Tk, B) * kv_heads, slots = D <= 64 ? 512 : 256;
  const double tiles = (double)Tq * (heads / kv_heads) / attn::kBN, likely = tiles * tiles / B;
  const int least = units < slots / 4 || (D > 64 && units < slots) ? 8 : 16;
  const double enough = least == 8 ? 24 : 32;
  if (likely < enough * enough || units >= (causal ? 4 : 1) * slots) return {1, 1, 0.0f, false};
  return {units < slots / 8 ? 8 : units < slots ? 4 : 2, least,
          units >= slots && 2 * units < 3 * slots ? 0.0f : (causal ? 0.5f : 1.0f) / slots,
          units >= slots};
}
}  // namespace

int64_t attention_backward_scratch(int64_t Tq, int64_t Tk, int64_t B, int64_t heads,
                                   int64_t kv_heads, int64_t D, bool causal) {
  const int64_t rows = 2 * heads * Tq, splits = dkv_runs(Tq, Tk, B, heads, kv_heads, D, causal).most;
  if (splits <= 1) return rows;
  return (rows + 63) / 64 * 64 +
         tile_bound(Tk, B) * kv_heads * splits * attn::kWaves * 64 * padded_dim(D);
}

int32_t launch_attention_backward(const AttentionBackwardProblem &p, hipStream_t s) {
  if (p.f.heads == 0 || p.f.D == 0 || p.f.B == 0) return NOVA_HIP_SUCCESS;
  attn::BwdArgs a;
  a.q = static_cast<const uint16_t *>(p.f.q.p);
  a.k = static_cast<const uint16_t *>(p.f.k.p);
  a.v = static_cast<const uint16_t *>(p.f.v.p);
  a.o = static_cast<const uint16_t *>(p.f.o.p);
  a.go = static_cast<const uint16_t *>(p.go.p);
  a.dq = static_cast<uint16_t *>(p.dq.p);
  a.dk = static_cast<uint16_t *>(p.dk.p);
  a.dv = static_cast<uint16_t *>(p.dv.p);
  a.lse = p.f.lse;
  a.slse = p.f.slse;
  a.rows = p.scratch;
  a.q_off = p.f.q_off;
  a.k_off = p.f.k_off;
  a.sq = {p.f.q.st, p.f.q.sh};
  a.sk = {p.f.k.st, p.f.k.sh};
  a.sv = {p.f.v.st, p.f.v.sh};
  a.so = {p.f.o.st, p.f.o.sh};
  a.sgo = {p.go.st, p.go.sh};
  a.sdq = {p.dq.st, p.dq.sh};
  a.sdk = {p.dk.st, p.dk.sh};
  a.sdv = {p.dv.st, p.dv.sh};
  a.Tq = (int)p.f.Tq;
  a.Tk = (int)p.f.Tk;
  a.B = (int)p.f.B;
  a.heads = (int)p.f.heads;
  a.group = (int)(p.f.heads / p.f.kv_heads);
  a.D = (int)p.f.D;
  a.tiles = 0;
  a.c = p.f.scale * attn::kLog2e;
  a.scale = p.f.scale;
  const Runs runs = dkv_runs(p.f.Tq, p.f.Tk, p.f.B, p.f.heads, p.f.kv_heads, p.f.D, p.f.causal);
  a.splits = (int)runs.most;
  a.least = runs.least;
  a.last_first = runs.last_first;
  a.share = runs.share;
  const int64_t qt = tile_bound(p.f.Tq, p.f.B), kt = tile_bound(p.f.Tk, p.f.B);
  a.partial = p.scratch + (2 * p.f.heads * p.f.Tq + 63) / 64 * 64;
  // A grid's dimension holds less than 2^32 threads.
  if (std::max(qt * p.f.heads, kt * p.f.kv_heads * a.splits) >= 1 << 24)
    return fail(NOVA_HIP_ERANGE, "attention_backward: more than 2^24 - 1 tiles");
  const char *w = "attention_backward";
  const int64_t Tq = p.f.Tq, Tk = p.f.Tk, H = p.f.heads, G = p.f.kv_heads, D = p.f.D;
  const Extent q = extent("q", p.f.q, Tq, H, D), k = extent("k", p.f.k, Tk, G, D),
               v = extent("v", p.f.v, Tk, G, D), out = extent("out", p.f.o, Tq, H, D),
               go = extent("grad_out", p.go, Tq, H, D), dq = extent("dq", p.dq, Tq, H, D),
               dk = extent("dk", p.dk, Tk, G, D), dv = extent("dv", p.dv, Tk, G, D),
               lse = {"lse", p.f.lse, 4 * Tq, {H, 1, 1}, {4 * p.f.slse, 0, 0}};
  int32_t rc;
  if ((rc = check_apart(w, dq, {q, k, v, out, go, lse, dk, dv})) ||
      (rc = check_apart(w, dk, {q, k, v, out, go, lse, dv})) ||
      (rc = check_apart(w, dv, {q, k, v, out, go, lse})))
    return rc;
  return p.f.dt == NOVA_HIP_DT_BF16
             ? attn::launch_bwd<NOVA_HIP_DT_BF16>(a, p.f.causal, qt, kt, s)
             : attn::launch_bwd<NOVA_HIP_DT_F16>(a, p.f.causal, qt, kt, s);
}

}  // namespace nova_hip

// Attention of chunks of new tokens over a paged cache: the queries of sequence
// b are the packed rows offsets[b] .. offsets[b + 1], its keys and values the
// first lengths[b] rows of its pages, the new tokens' own among them.
//
// The query heads of a group read the same keys, so a tile's rows are (token,
// head of the group) pairs: row r is token r / group, head r % group, and keys
// and values are read once for the group.  The products, the running maximum and
// sum and the LDS tiles are those of the packed forward (attention.hip).
//
// Two forms.  Chunks: four waves of 32 rows share tiles of 64 keys; bound by the products
// and the softmax between them (32 heads on 8 of 128 in bf16: a prompt of 8192 530 to 565 us,
// 0.97 to 1.04 PFLOP/s; 512 tokens over 8192 rows 88 to 91, 730 to 760 TFLOP/s; the matrix
// cores are busy for 43 % of a step of 3751 tokens).  Up to 32 rows per sequence (single
// tokens): a wave per split of the keys, tiles of 32, without a barrier; bound by HBM (32
// tokens over 1500 to 8192 rows 108 us, 5.5 TB/s; 8 over 131072 6.5).  Either cuts the keys of
// a tile of rows into pieces where there are few tiles (see work_of); a tile whose rows see
// at most one writes its result, the others' sums go to the caller's scratch, where a second
// kernel adds them in order.
//
// Up to 64 sequences a workgroup reads all lengths and takes its unit of work from them.
// With more the host provides for splits by the sizes alone: none for chunks where tiles
// times key heads are more than 3/4 of the places, so that one workgroup to a key head walks
// the longest sequence (a prompt of 4096 beside one token over 131072 rows 257 us, with 70
// single tokens more 3060), and for single tokens as many as the table's width asks for.
//
// Keys come by DMA into LDS.  Where a page holds whole loads (rows that are a
// multiple of the 4 or 8 of one instruction) its address is a scalar: a lane looks up
// each load of a tile, a tile ahead, and a buffer of the load's rows that are there
// makes the others zero.  Other page sizes: a lane looks up each row, and a load takes
// its lanes' addresses from those; rows that are not there are a row of zeros (32 heads
// on 8 of 128, pages of one row against 16: 32 single tokens over 1500 to 8192 rows 115 us
// against 107, a prompt of 8192 620 to 627 against 558 to 563; through registers 930 and
// 1180).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "attention.h"
#include "paged_work.h"
#include "wave.h"

namespace nova_hip {
namespace attn {
namespace {
using namespace paged;

// n / d for n < 2^31: the upper bits of n m, m the least number above 2^(31 + l) / d.
struct Divider {
  uint32_t d, m;
  int l;
  Divider() = default;
  __host__ explicit Divider(int64_t by) : d((uint32_t)by), l(0) {
    while (((int64_t)1 << l) < by) ++l;
    m = (uint32_t)((((uint64_t)1 << (31 + l)) / (uint64_t)by) + 1);
  }
  __device__ __forceinline__ int of(int n) const {
    return (int)(((uint64_t)(uint32_t)n * m) >> (31 + l));
  }
};

struct PagedArgs {
  const uint16_t *q, *k, *v;
  uint16_t *o;
  float *lse;  // [heads][T] with row stride slse, or null
  // Sums of splits.  Chunks: [key heads][slots] of a tile each (see sums_at).  Up to 32
  // rows: rows of D + 2, the sum, then m c and l: [key heads][slots][32], or without
  // slots [T][heads][splits]; and for each of [T][heads] its splits (0: written) and place.
  float *partial;
  int2 *rows;
  const int *off, *lens, *table;
  Rows sq, so;
  int64_t skp, skt, skh, svp, svt, svh, stb, slse;
  double per_page;  // 1 / page
  Divider group;    // query heads to a key head
  int T, B, heads, kv_heads, D, page, pages, cap;  // cap: rows of a sequence
  int tiles;          // per key head; up to 64 sequences: with their splits
  int split_tiles;    // those that may have several
  int splits, chunk;  // chunk: what `splits` cover all rows with, at least 1
  int slots, least;   // of splits found from the lengths: room for them, their least keys
  float c;            // scale log2 e
  float places;       // workgroups resident at once, to a key head
  bool causal;
};

// A row behind the last.
__device__ const __attribute__((aligned(16))) uint32_t kZeros[64] = {};

constexpr float kSlack = 8.0f;  // as in the packed forward
// So are f16 weights taken times 2^7, in both forms (the padded single-token form, without
// the slack, 2^15): one that rounds to zero is under 2^-32 of the largest in its piece, and
// 2^20 keys of such weights together under half a step of an f16 result.
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

__device__ __forceinline__ int wave_max_int(int v) {
#define NOVA_DPP_MAX(c) v = max(v, __builtin_amdgcn_mov_dpp(v, c, 0xF, 0xF, false))
  NOVA_DPP_MAX(0xB1);   // quad_perm [1,0,3,2]
  NOVA_DPP_MAX(0x4E);   // quad_perm [2,3,0,1]
  NOVA_DPP_MAX(0x141);  // row_half_mirror
  NOVA_DPP_MAX(0x140);  // row_mirror
#undef NOVA_DPP_MAX
  return max(max(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
             max(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}

__device__ __forceinline__ Seq lane_seq(const Seq &q, int l) {
  return {__builtin_amdgcn_readlane(q.s, l), __builtin_amdgcn_readlane(q.n, l),
          __builtin_amdgcn_readlane(q.len, l)};
}
// Sum of the lanes below: within the rows of 16, then over rows.
__device__ __forceinline__ int lanes_below(int v) {
  int x = v;
#define NOVA_DPP_SCAN(c, rows) x += __builtin_amdgcn_update_dpp(0, x, c, rows, 0xF, false)
  NOVA_DPP_SCAN(0x111, 0xF);  // row_shr:1
  NOVA_DPP_SCAN(0x112, 0xF);  // row_shr:2
  NOVA_DPP_SCAN(0x114, 0xF);  // row_shr:4
  NOVA_DPP_SCAN(0x118, 0xF);  // row_shr:8
  NOVA_DPP_SCAN(0x142, 0xA);  // row_bcast:15 to rows 1 and 3
  NOVA_DPP_SCAN(0x143, 0xC);  // row_bcast:31 to rows 2 and 3
#undef NOVA_DPP_SCAN
  return x - v;
}

__device__ __forceinline__ int tiles_of(const PagedArgs &a, const Seq &q) {
  return (q.n * (int)a.group.d + kBM - 1) / kBM;
}

// Up to 64 sequences, one to a lane (none in the others), read in one go by a whole
// wave; the same for every wave of a call.  The tiles of a sequence have up to n
// splits of `piece` keys; those of sequences with more than one have slots from `base`.
struct Work {
  Seq q;
  int tiles, n, piece, base;
};
__device__ __forceinline__ Work work_of(const PagedArgs &a, int BM) {
  const int lane = threadIdx.x & 63;
  Work w;
  w.q = lane < a.B ? seq_of(a, lane) : Seq{0, 0, 0};
  w.tiles = BM == kBM ? tiles_of(a, w.q) : (w.q.n > 0 ? 1 : 0);
  w.n = 1;
  w.piece = a.cap;
  w.base = 0;
  if (a.slots == 0) return w;
  const float tiles = (float)w.tiles, len = (float)w.q.len;
  const float counted = counted_keys(w.q.n, w.q.len, a.causal);
  const float all = wave_sum(tiles), mean = wave_sum(tiles * mean_keys(w.q.n, w.q.len, a.causal)) / a.places;
  const float c = piece_keys(all, mean, a.places, (float)a.least, (float)a.slots,
                             [&](float keys, bool split) __attribute__((always_inline)) {
                               const float n = splits_at(len, counted, keys);
                               return wave_sum(split && n <= 1.0f ? 0.0f : tiles * n);
                             });
  const float n = splits_at(len, counted, c);
  // No more slots than there are, whatever the rounding.
  const float mine = n > 1.0f ? tiles * n : 0.0f;
  if (!(wave_sum(mine) <= (float)a.slots)) return w;
  w.n = (int)n;
  if (n > 1.0f) w.piece = piece_of(w.q.len, n);
  w.base = lanes_below((int)mine);
  return w;
}

// A tile of rows (n group to a sequence: of kBM, or the one that has all 32) and a
// split of its keys; `slot` is its first split's.
struct Unit {
  Seq seq;
  int b, index, split, piece, slot;
};
__device__ __forceinline__ bool unit_at(const Work &w, int first, int count, int k, Unit &u) {
  const uint64_t hit = __ballot(k >= first && k < first + count);
  if (!hit) return false;
  u.b = __builtin_ctzll(hit);
  u.seq = lane_seq(w.q, u.b);
  u.piece = __builtin_amdgcn_readlane(w.piece, u.b);
  u.split = k - __builtin_amdgcn_readlane(first, u.b);
  return true;
}
// Unit t, wave-uniform; false where there is none.
//
// One tile to a sequence, and splits of like size: one behind the other.
__device__ __forceinline__ bool find_split(const Work &w, int t, Unit &u) {
  const int n = w.tiles * w.n;
  if (!unit_at(w, lanes_below(n), n, t, u)) return false;
  u.index = 0;
  u.slot = __builtin_amdgcn_readlane(w.base, u.b);
  return true;
}
// In the order of falling work, so that what runs last is short.  A sequence's tiles,
// the last first, see falling numbers of keys, one tile's tokens less each; counted in
// such steps from the longest piece's end tile j of b lies at d(b) + j.  With S(x) =
// sum over sequences of the units below x, the unit's place is the largest x with
// S(x) <= t, found bit by bit.
__device__ __forceinline__ bool find_unit(const PagedArgs &a, const Work &w, int t, Unit &u) {
  const int len = min(w.piece, w.q.len), longest = wave_max_int(w.tiles > 0 ? len : 0);
  const float behind = (float)(longest - min(len, longest)) * (float)a.group.d * (1.0f / kBM);
  const int d = (int)fminf(behind, 1e7f);
  auto below = [&](int x) __attribute__((always_inline)) {
    return wave_sum_int(w.n * min(max(x - d, 0), w.tiles));
  };
  int x = 0;
  if (a.B > 1) {
    int bit = 1;
    while (bit < (1 << 26) && below(bit) <= t) bit <<= 1;
    for (bit >>= 1; bit > 0; bit >>= 1)
      if (below(x + bit) <= t) x += bit;
    t -= below(x);  // among the units at x
  } else {
    // One sequence: (its n, of lane 0; at most 2^26 units).
    const int n = __builtin_amdgcn_readlane(w.n, 0);
    if (n > 1) x = (int)(((double)t + 0.5) / (double)n);
    else x = t;
    t -= x * n;
  }
  const int here = x >= d && x - d < w.tiles ? w.n : 0;
  if (!unit_at(w, lanes_below(here), here, t, u)) return false;
  const int index = w.tiles - 1 - (x - d);
  u.index = __builtin_amdgcn_readlane(index, u.b);
  u.slot = __builtin_amdgcn_readlane(w.base + index * w.n, u.b);
  return true;
}

// More than 64 sequences: tile t by find_tile's numbering and search, from its end.
__device__ __forceinline__ bool find_tile_of_many(const PagedArgs &a, int t, Unit &u) {
  const int lane = threadIdx.x & 63, group = (int)a.group.d;
  int lo = 0, n = a.B;
  for (;;) {
    const int step = (n + 63) / 64, i = lo + lane * step;
    const bool at = lane * step < n && min(max(a.off[i], 0), a.T) * group / kBM + i <= t;
    const int c = __builtin_popcountll(__ballot(at));
    if (c == 0) return false;
    lo += (c - 1) * step;
    n = min(step, n - (c - 1) * step);
    if (step == 1) break;
  }
  u.b = __builtin_amdgcn_readfirstlane(lo);
  u.seq = seq_of(a, u.b);
  u.index = __builtin_amdgcn_readfirstlane(t - (u.seq.s * group / kBM + u.b));
  u.slot = t * a.splits;
  return u.index >= 0 && u.index < tiles_of(a, u.seq);
}
// Their pieces: at most a.splits of them, from the lengths.
__device__ __forceinline__ int piece_of_many(const PagedArgs &a) {
  if (a.splits == 1) return a.chunk;
  float keys = 0.0f;
  for (int b = threadIdx.x & 63; b < a.B; b += 64) {
    const Seq q = seq_of(a, b);
    keys += (float)tiles_of(a, q) * mean_keys(q.n, q.len, a.causal);
  }
  const float c = 1.25f * wave_sum(keys) / a.places;
  return __builtin_amdgcn_readfirstlane(max(a.chunk, ((int)fminf(c, (float)a.cap) + 63) / 64 * 64));
}

// A tile's sums of one split as its waves hold them: [4 waves][32-column blocks][4][64
// lanes] of four values, the registers 4 g .. 4 g + 3 of a block, then m c and l of
// [4 waves][32 rows].
template <int DP>
__device__ __forceinline__ float *sums_at(const PagedArgs &a, int kh, int slot) {
  return a.partial + ((int64_t)kh * a.slots + slot) * (kBM * (DP + 2));
}

// NW waves of 32 rows each.  WHOLE: a load's rows lie in one page.
template <int DT, int DP, int NW, bool WHOLE>
__global__ __launch_bounds__(64 * NW, 2) void attention_paged_kernel(PagedArgs a) {
  constexpr int CH = kPitch<DP>, BN = NW == 1 ? 32 : 64, kTile = BN * CH * 16;
  constexpr int kRows = 64 / CH;               // rows of one DMA instruction
  constexpr int kN = BN / kRows / NW;          // instructions of a wave and tile
  __shared__ __attribute__((aligned(1024))) char sk0_[kTile], sk1_[kTile], sv0_[kTile], sv1_[kTile];
  lds_char *const sk0 = (lds_char *)sk0_, *const sk1 = (lds_char *)sk1_;
  lds_char *const sv0 = (lds_char *)sv0_, *const sv1 = (lds_char *)sv1_;
  const int lane = threadIdx.x & 63;
  const int wave = NW == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  static_assert(NW == 1 || 32 * NW == kBM, "rows of a tile");
  const int group = (int)a.group.d;
  int kh;
  Unit u;
  if (NW == 1 && !a.slots) {
    kh = blockIdx.x;
    u.b = blockIdx.y;
    u.split = blockIdx.z;
    u.seq = seq_of(a, u.b);
    u.index = u.slot = 0;
    u.piece = a.chunk;
  } else {
    int unit;
    unit_of(blockIdx.x, a.kv_heads, a.tiles, true, kh, unit);
    if (NW == 1 || a.B <= 64) {
      const Work w = work_of(a, 32 * NW);
      if (!(NW == 1 ? find_split(w, unit, u) : find_unit(a, w, unit, u))) return;
    } else {
      if (!find_tile_of_many(a, a.tiles - 1 - unit, u)) return;
      u.split = a.splits - 1 - blockIdx.y;  // first splits last: others are long tiles'
      u.piece = piece_of_many(a);
    }
  }
  const Seq seq = u.seq;
  const int b = u.b, split = u.split;
  const int row0 = u.index * 32 * NW, R = NW == 1 ? min(seq.n, 32 / group) * group : seq.n * group;
  if (R <= row0) return;
  const int vis = seq.seen(a.group.of(min(row0 + 32 * NW, R) - 1), a.causal);
  const int from = split * u.piece, to = min(vis, from + u.piece);
  if (split > 0 && from >= vis) return;
  const bool direct = vis <= u.piece;

  const int q0 = row0 + 32 * wave, qn = min(32, R - q0);  // this wave's rows, maybe none
  const int row = min(q0 + (lane & 31), R - 1), token = a.group.of(row);
  const int head = kh * group + row - token * group;
  const bool mine = (lane & 31) < qn;
  const int end = mine ? min(to, seq.seen(token, a.causal)) : 0;  // the keys this lane's row sees
  // ... and those that the wave's first and last rows see.
  const int least = __builtin_amdgcn_readlane(end, 0);
  const int most = __builtin_amdgcn_readlane(end, max(qn, 1) - 1);
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
  // A lane to each of the next tile's loads (WHOLE) or rows finds its page and row there,
  // a tile ahead of the load itself.
  constexpr int kStep = WHOLE ? kRows : 1;
  const int mark = (lane & (BN / kStep - 1)) * kStep;
  int id = 0, at = 0;
  auto look = [&](int t) __attribute__((always_inline)) {
    const int key = min(from + t * BN + mark, to - 1), pg = page_of(key);
    id = table[pg];
    at = key - pg * a.page;
  };
  if (to > from) look(0);
  // The queries are waited for here: at their use in the loop the compiler would
  // wait for every load.
  __builtin_amdgcn_s_waitcnt(0x0F70);
  auto fetch = [&](int t, lds_char *sk, lds_char *sv) __attribute__((always_inline)) {
    const int skt = (int)a.skt * 2, svt = (int)a.svt * 2;  // bytes
    const int pg = min(max(id, 0), a.pages - 1);
    uint64_t ka = reinterpret_cast<uint64_t>(kp + pg * a.skp) + (uint32_t)(at * skt);
    uint64_t va = reinterpret_cast<uint64_t>(vp + pg * a.svp) + (uint32_t)(at * svt);
    const int left = to - (from + t * BN + mark);
    if constexpr (WHOLE) {
      // Rows behind the last read zero.
      const int n = min(left, kRows);
      const int kb = max((n - 1) * skt + 2 * a.D, 0), vb = max((n - 1) * svt + 2 * a.D, 0);
      look(t + 1);
      // Ahead of the loads: a wait for it is then none for them.
      __builtin_amdgcn_sched_barrier(0);
      auto buffer = [&](uint64_t p, int bytes, int l) __attribute__((always_inline)) {
        const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)p, l);
        const uint64_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(p >> 32), l);
        return make_rsrc(reinterpret_cast<const uint16_t *>(hi << 32 | lo),
                         __builtin_amdgcn_readlane(bytes, l));
      };
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int l = i * NW + wave, r0 = l * kRows;
        const __amdgpu_buffer_rsrc_t rk = buffer(ka, kb, l), rv = buffer(va, vb, l);
        const int lr = lane / CH, ch = (lane & (CH - 1)) ^ swz<CH>(r0 + lr);
        // Single tokens: read once by the whole chip (116 us against 125 where the caches
        // keep them).
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rk, (lds_void *)(sk + r0 * CH * 16), 16,
            ch * 8 < a.D ? (uint32_t)(lr * skt + ch * 16) : kOOB, 0, 0, NW == 1 ? 2 : 0);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rv, (lds_void *)(sv + r0 * CH * 16), 16,
            ch * 8 < a.D ? (uint32_t)(lr * svt + ch * 16) : kOOB, 0, 0, NW == 1 ? 2 : 0);
      }
    } else {
      const uint64_t zeros = reinterpret_cast<uint64_t>(kZeros);
      if (left <= 0) ka = va = zeros;
      look(t + 1);
      __builtin_amdgcn_sched_barrier(0);
      auto load = [&](uint64_t p, int r, int ch, lds_char *tile) __attribute__((always_inline)) {
        const uint32_t lo = __builtin_amdgcn_ds_bpermute(4 * r, (int)(uint32_t)p);
        const uint64_t hi = (uint32_t)__builtin_amdgcn_ds_bpermute(4 * r, (int)(p >> 32));
        typedef const __attribute__((address_space(1))) char global_char;
        __builtin_amdgcn_global_load_lds(
            (global_char *)((ch * 8 < a.D ? hi << 32 | lo : zeros) + ch * 16), (lds_void *)tile, 16, 0,
            NW == 1 ? 2 : 0);
      };
#pragma unroll
      for (int i = 0; i < kN; ++i) {
        const int r0 = (i * NW + wave) * kRows, r = r0 + lane / CH, ch = (lane & (CH - 1)) ^ swz<CH>(r);
        load(ka, r, ch, sk + r0 * CH * 16);
        load(va, r, ch, sv + r0 * CH * 16);
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
        // Weights round to the operands' type, as in the packed forward: a result is 2.0e-3
        // to 2.4e-3 off in bf16 (2-norm, relative), 1.7e-3 of it by its own rounding.
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
    // but the next stage's loads have landed.  Behind the last tile empty ones are
    // fetched: with branches around the waits the compiler adds stricter ones.
    constexpr int kInFlight = 2 * kN;
    auto landed = [&]() __attribute__((always_inline)) {
      __builtin_amdgcn_s_waitcnt(0x0F70 | (kInFlight & 15) | ((kInFlight >> 4) << 14));
    };
    auto turn = [&](int t, lds_char *sk, lds_char *sv, lds_char *nk, lds_char *nv) __attribute__((always_inline)) {
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
      __builtin_amdgcn_sched_barrier(0);
      fetch(t + 1, nk, nv);
      __builtin_amdgcn_sched_barrier(0);
      landed();
      __builtin_amdgcn_sched_barrier(0);
      step(t, sk, sv);
    };
    if (nt > 0) {
      fetch(0, sk0, sv0);
      __builtin_amdgcn_sched_barrier(0);
      landed();  // what was looked up, so that the loop need not wait for it
    }
    for (int t = 0; t < nt; t += 2) {
      turn(t, sk0, sv0, sk1, sv1);
      turn(t + 1, sk1, sv1, sk0, sv0);
    }
    __builtin_amdgcn_s_waitcnt(0x0F70);  // the LDS is no longer written
  }
  l = both_sum(l);
  if (qn <= 0) return;
  if (NW == 1 && a.rows && split == 0 && lane < qn)
    a.rows[(int64_t)(seq.s + token) * a.heads + head] =
        int2{direct ? 0 : (vis - 1) / u.piece + 1, (kh * a.slots + u.slot) * 32 + lane};
  if (direct) {
    // A row that sees no key is zero, its lse -inf.
    store_row<DT, DP>(acc, l == 0.0f ? 0.0f : 1.0f / l,
                      a.o + (seq.s + token) * a.so.t + head * a.so.h, mine, a.D, lane);
    if (a.lse && lane < qn)
      a.lse[head * a.slse + seq.s + token] =
          l == 0.0f ? -INFINITY : (mc + (__log2f(l) - kUp<DT>)) * kLn2;
    return;
  }
  if constexpr (NW > 1) {
    float *const p = sums_at<DP>(a, kh, u.slot + split);
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<gemm::f32x4 *>(p + ((wave * (DP / 32) + db) * 4 + g) * 256 + lane * 4) =
            gemm::f32x4{acc[db][4 * g], acc[db][4 * g + 1], acc[db][4 * g + 2], acc[db][4 * g + 3]};
    if (lane < 32)
      *reinterpret_cast<float2 *>(p + kBM * DP + (wave * 32 + lane) * 2) = float2{mc, l};
  } else {
    if (!mine) return;
    const int64_t at = a.slots ? (int64_t)(kh * a.slots + u.slot + split) * 32 + row
                               : ((int64_t)(seq.s + token) * a.heads + head) * a.splits + split;
    float *const p = a.partial + at * (a.D + 2);
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        const int d = 32 * db + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
        if (d < a.D) *reinterpret_cast<float2 *>(p + d) = float2{acc[db][r], acc[db][r + 1]};
      }
    if (lane < 32) *reinterpret_cast<float2 *>(p + a.D) = float2{mc, l};
  }
}

// Chunks: the sums of a tile's splits.  A workgroup per tile that has any and 32
// columns, in GROUPS groups of four waves that read what the tile's waves wrote, whole
// lines of it: group g takes splits g, g + GROUPS, ..., each to the largest maximum so
// far, and the groups join in order.
template <int DT, int DP, int GROUPS>
__global__ __launch_bounds__(2 * kBM * GROUPS) void paged_join_tile_kernel(PagedArgs a) {
  __shared__ float box[GROUPS > 1 ? GROUPS - 1 : 1][4][18][GROUPS > 1 ? 64 : 1];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3;
  const int part = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
  const int kh = blockIdx.x, db = blockIdx.z, group = (int)a.group.d;
  Unit u;
  if (a.B <= 64) {
    const Work w = work_of(a, kBM);
    const int tiles = w.n > 1 ? w.tiles : 0;
    if (!unit_at(w, lanes_below(tiles), tiles, blockIdx.y, u)) return;
    u.index = u.split;
    u.slot = __builtin_amdgcn_readlane(w.base + u.index * w.n, u.b);
  } else {
    if (!find_tile_of_many(a, blockIdx.y, u)) return;
    u.piece = piece_of_many(a);
  }
  const Seq seq = u.seq;
  const int row0 = u.index * kBM, R = seq.n * group;
  const int vis = seq.seen(a.group.of(min(row0 + kBM, R) - 1), a.causal);
  if (vis <= u.piece) return;
  const int q0 = row0 + 32 * wave, qn = min(32, R - q0);
  const float *const p = sums_at<DP>(a, kh, u.slot);
  const float *const px = p + (wave * (DP / 32) + db) * 1024 + lane * 4;
  const float *const pm = p + kBM * DP + (wave * 32 + (lane & 31)) * 2;
  f32x16 acc[1] = {};
  float mx = -INFINITY, sum = 0.0f;
  // A further split's sums, or another group's.
  auto add = [&](float m, float l, auto value) __attribute__((always_inline)) {
    const float to = fmaxf(mx, m);
    const float old = mx == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mx - to);
    const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - to);
    mx = to;
    sum = __builtin_fmaf(l, f, sum * old);
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[0][r] = __builtin_fmaf(value(r), f, acc[0][r] * old);
  };
  constexpr int kAhead = 4;  // splits whose loads are on their way together
  const int n = qn > 0 ? (vis - 1) / u.piece + 1 : 0;
  for (int s0 = part; s0 < n; s0 += kAhead * GROUPS) {
    gemm::f32x4 x[kAhead][4];
    float2 ml[kAhead];
#pragma unroll
    for (int s = 0; s < kAhead; ++s) {
      const int64_t at = (int64_t)min(s0 + s * GROUPS, n - 1) * (kBM * (DP + 2));
      ml[s] = *reinterpret_cast<const float2 *>(pm + at);
#pragma unroll
      for (int g = 0; g < 4; ++g) x[s][g] = *reinterpret_cast<const gemm::f32x4 *>(px + at + g * 256);
    }
#pragma unroll
    for (int s = 0; s < kAhead; ++s) {
      // (With a branch around the rest the compiler moves the loads into it.)
      const bool there = s0 + s * GROUPS < n;
      add(there ? ml[s].x : -INFINITY, there ? ml[s].y : 0.0f,
          [&](int r) { return there ? x[s][r >> 2][r & 3] : 0.0f; });
    }
  }
  if constexpr (GROUPS > 1) {
    if (part) {
      float(*const mine)[64] = box[part - 1][wave];
#pragma unroll
      for (int r = 0; r < 16; ++r) mine[r][lane] = acc[0][r];
      mine[16][lane] = mx;
      mine[17][lane] = sum;
    }
    __syncthreads();
    if (part) return;
#pragma unroll
    for (int g = 0; g < GROUPS - 1; ++g) {
      const float(*const other)[64] = box[g][wave];
      add(other[16][lane], other[17][lane], [&](int r) { return other[r][lane]; });
    }
  }
  if (qn <= 0) return;
  const int row = min(q0 + (lane & 31), R - 1), token = a.group.of(row);
  const int head = kh * group + row - token * group;
  store_row<DT, 32>(acc, sum == 0.0f ? 0.0f : 1.0f / sum,
                    a.o + (seq.s + token) * a.so.t + head * a.so.h + 32 * db, (lane & 31) < qn,
                    a.D - 32 * db, lane);
  if (a.lse && db == 0 && lane < qn)
    a.lse[head * a.slse + seq.s + token] =
        sum == 0.0f ? -INFINITY : (mx + (__log2f(sum) - kUp<DT>)) * kLn2;
}

// Whether a token is among the first of its sequence, which a tile of 32 rows has.  By
// a whole wave.
__device__ __forceinline__ bool in_tile(const PagedArgs &a, int t) {
  const int lane = threadIdx.x & 63, most = 32 / (int)a.group.d;
  if (a.B <= 64) {
    const int s = lane < a.B ? max(a.off[lane], 0) : a.T;
    return __ballot(s <= t && t < a.off[min(lane, a.B - 1) + 1] && t - s < most) != 0;
  }
  // The sequences that end at or before t are counted out, 64 probes at a time.
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
  return lo < a.B && a.off[lo] <= t && t < a.off[lo + 1] && t - max(a.off[lo], 0) < most;
}

// A row's sums as its tile left them: its splits (0: none), the first one's place and
// the rows from one to the next.  What a.rows holds of a row that no tile had (where
// sequences overlap) is cut to the scratch.
struct Sums {
  int n;
  const float *p;
};
__device__ __forceinline__ Sums sums_of(const PagedArgs &a, int t, int head) {
  const int2 r = a.rows[(int64_t)t * a.heads + head];
  if (!a.slots)
    return {min(max(r.x, 0), a.splits),
            a.partial + ((int64_t)t * a.heads + head) * a.splits * (a.D + 2)};
  const int all = a.kv_heads * a.slots * 32, at = min(max(r.y, 0), all - 1);
  return {min(max(r.x, 0), (all - 1 - at) / 32 + 1), a.partial + (int64_t)at * (a.D + 2)};
}

// The sums of splits first, first + STEP, ... of a row (p: split 0's, `step` from one
// to the next), by a wave: to the largest maximum mx, in the splits' order.  A lane holds values
// 2 lane and 2 lane + 1; a split's maximum and sum of weights are a lane's.
struct Joined {
  float mx, sum, x0, x1;
};
template <int STEP>
__device__ __forceinline__ Joined join(const PagedArgs &a, const float *p, int64_t step, int first,
                                       int n) {
  const int lane = threadIdx.x & 63;
  Joined j = {-INFINITY, 0.0f, 0.0f, 0.0f};
  const float *v = p + min(2 * lane, a.D - 2);
  for (int i0 = first; i0 < n; i0 += 64 * STEP) {
    const int i = i0 + lane * STEP, count = min(64, (n - i0 + STEP - 1) / STEP);
    float2 ml = {-INFINITY, 0.0f};
    if (i < n) ml = *reinterpret_cast<const float2 *>(p + i * step + a.D);
    const float mx = fmaxf(j.mx, wave_max(ml.x));
    const float old = j.mx == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(j.mx - mx);
    const float f = ml.x == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml.x - mx);
    j = {mx, j.sum * old + wave_sum(ml.y * f), j.x0 * old, j.x1 * old};
    for (int k0 = 0; k0 < count; k0 += 8) {
      float2 x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        x[k] = *reinterpret_cast<const float2 *>(v + (i0 + min(k0 + k, count - 1) * STEP) * step);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const bool there = k0 + k < count;
        const float g = lane_value(f, (k0 + k) & 63);
        j.x0 = there ? __builtin_fmaf(x[k].x, g, j.x0) : j.x0;
        j.x1 = there ? __builtin_fmaf(x[k].y, g, j.x1) : j.x1;
      }
    }
  }
  return j;
}

template <int DT>
__device__ __forceinline__ void store_joined(const PagedArgs &a, int t, int head, int lane,
                                             const Joined &j) {
  const float inv = j.sum == 0.0f ? 0.0f : 1.0f / j.sum;
  if (2 * lane < a.D)
    *reinterpret_cast<uint32_t *>(a.o + t * a.so.t + head * a.so.h + 2 * lane) =
        pack<DT>(j.x0 * inv, j.x1 * inv);
  if (a.lse && lane == 0)
    a.lse[head * a.slse + t] = j.sum == 0.0f ? -INFINITY : (j.mx + (__log2f(j.sum) - kUp<DT>)) * kLn2;
}

// Up to 32 rows of a sequence: one workgroup per (token, head), its waves take every
// fourth split and join in order.
template <int DT>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedArgs a) {
  __shared__ float smax[4], ssum[4], sx[4][128];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t = blockIdx.x / a.heads, head = blockIdx.x - t * a.heads;
  const Sums s = sums_of(a, t, head);
  if (!in_tile(a, t) || s.n == 0) return;
  Joined j = join<4>(a, s.p, (a.slots ? 32 : 1) * (int64_t)(a.D + 2), wave, s.n);
  sx[wave][2 * lane] = j.x0;
  sx[wave][2 * lane + 1] = j.x1;
  if (lane == 0) {
    smax[wave] = j.mx;
    ssum[wave] = j.sum;
  }
  __syncthreads();
  if (wave) return;
  j = {fmaxf(fmaxf(smax[0], smax[1]), fmaxf(smax[2], smax[3])), 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float f = smax[w] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(smax[w] - j.mx);
    j.sum = __builtin_fmaf(ssum[w], f, j.sum);
    j.x0 = __builtin_fmaf(sx[w][2 * lane], f, j.x0);
    j.x1 = __builtin_fmaf(sx[w][2 * lane + 1], f, j.x1);
  }
  store_joined<DT>(a, t, head, lane, j);
}

template <int DT, int DP, bool WHOLE>
void launch_paged_t(const PagedArgs &a, bool narrow, hipStream_t s) {
  const unsigned units = (unsigned)(a.tiles * a.kv_heads);
  if (narrow)
    hipLaunchKernelGGL(
        (attention_paged_kernel<DT, DP, 1, WHOLE>),
        a.slots ? dim3(units) : dim3((unsigned)a.kv_heads, (unsigned)a.B, (unsigned)a.splits), dim3(64),
        0, s, a);
  else
    hipLaunchKernelGGL((attention_paged_kernel<DT, DP, 4, WHOLE>),
                       dim3(units, a.B <= 64 ? 1u : (unsigned)a.splits), dim3(256), 0, s, a);
}
template <int DT, int DP>
int32_t launch_paged_d(const PagedArgs &a, bool narrow, hipStream_t s) {
  // A load is of 8 rows up to D = 64, of 4 beyond.
  if (a.page % (64 / kPitch<DP>) == 0) launch_paged_t<DT, DP, true>(a, narrow, s);
  else launch_paged_t<DT, DP, false>(a, narrow, s);
  const int32_t rc = check_hip(hipGetLastError(), "paged_attention launch");
  if (rc || !a.partial) return rc;
  if (narrow)
    hipLaunchKernelGGL(paged_join_kernel<DT>, dim3((unsigned)(a.T * a.heads)), dim3(256), 0, s, a);
  else {
    // Groups where tiles are so few, and keys so many, that a tile may have eight splits and
    // more (one group against four, heads of 128: 16 tokens over 32768 rows 44.7 us against
    // 38.7, a step of 3751 tokens 238 against 245; 300 over 1000, heads of 64, 12.7 against 14.7).
    const dim3 grid((unsigned)a.kv_heads, (unsigned)a.split_tiles, DP / 32);
    if (a.split_tiles * 8 <= a.places && a.cap >= 8 * a.least)
      hipLaunchKernelGGL((paged_join_tile_kernel<DT, DP, 4>), grid, dim3(8 * kBM), 0, s, a);
    else
      hipLaunchKernelGGL((paged_join_tile_kernel<DT, DP, 1>), grid, dim3(2 * kBM), 0, s, a);
  }
  return check_hip(hipGetLastError(), "paged_attention join launch");
}
template <int DT>
int32_t launch_paged(const PagedArgs &a, bool narrow, hipStream_t s) {
  if (a.D <= 32) return launch_paged_d<DT, 32>(a, narrow, s);
  if (a.D <= 64) return launch_paged_d<DT, 64>(a, narrow, s);
  if (a.D <= 96) return launch_paged_d<DT, 96>(a, narrow, s);
  return launch_paged_d<DT, 128>(a, narrow, s);
}

}  // namespace
}  // namespace attn

int64_t paged_attention_scratch(int64_t T, int64_t B, int64_t heads, int64_t kv_heads, int64_t D,
                                int64_t rows, int64_t max_queries) {
  const attn::paged::Plan p = attn::paged::plan_of(T, B, heads, kv_heads, D, rows, max_queries);
  if (!p.narrow) return kv_heads * p.slots * attn::paged::kBM * ((D + 31) / 32 * 32 + 2);
  const int64_t sums = p.slots ? kv_heads * p.slots * 32 : p.splits > 1 ? T * heads * p.splits : 0;
  return sums ? sums * (D + 2) + (2 * T * heads + 3) / 4 * 4 : 0;
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
  a.group = attn::Divider(p.heads / c.kv_heads);
  a.D = (int)c.D;
  a.page = (int)c.page;
  a.pages = (int)c.pages;
  a.cap = (int)(c.width * c.page);
  const attn::paged::Plan plan = attn::paged::plan_of(p.T, c.B, p.heads, c.kv_heads, c.D, a.cap, p.max_queries);
  // Rows are counted in 32 bits, a grid's dimension holds less than 2^32 threads.
  if (p.T * p.heads >= (1LL << 31) - (1 << 20) || plan.tiles * c.kv_heads >= 1 << 24 ||
      (plan.narrow && (plan.splits > 1 || plan.slots > 0) && p.T * p.heads >= 1 << 24))
    return fail(NOVA_HIP_ERANGE, "paged_attention: %lld tokens of %lld heads in %lld sequences",
                (long long)p.T, (long long)p.heads, (long long)c.B);
  if (plan.splits > 1 || plan.slots) {
    a.rows = plan.narrow ? reinterpret_cast<int2 *>(p.partial) : nullptr;
    a.partial = p.partial + (plan.narrow ? (2 * p.T * p.heads + 3) / 4 * 4 : 0);
  }
  a.tiles = (int)plan.tiles;
  a.split_tiles = (int)(c.B <= 64 ? std::min(plan.tiles - plan.slots, plan.slots / 2) : plan.tiles);
  a.splits = (int)plan.splits;
  a.chunk = (int)plan.chunk;
  a.c = p.scale * attn::kLog2e;
  a.causal = p.causal;
  a.slots = (int)plan.slots;
  a.least = (int)plan.least;
  a.places = (float)plan.places / (float)c.kv_heads;
  return p.dt == NOVA_HIP_DT_BF16 ? attn::launch_paged<NOVA_HIP_DT_BF16>(a, plan.narrow, s)
                                  : attn::launch_paged<NOVA_HIP_DT_F16>(a, plan.narrow, s);
}

}  // namespace nova_hip

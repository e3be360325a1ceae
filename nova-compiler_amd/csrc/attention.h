// Device-side pieces shared by the attention kernels (attention.hip,
// attention_bwd.hip, attention_decode.hip): argument blocks, the search for a
// tile's sequence, operand tiles in LDS and their fragments.
//
// All of them multiply on v_mfma_f32_32x32x16 with 32 rows of one side held in
// registers for the whole loop (queries, or keys for dK and dV), as the
// instruction's COLUMNS, and the other side streamed through LDS as its rows.
// Lane l of the result then holds column l % 32 and rows
//   8 (r / 4) + 4 (l / 32) + r % 4,   r = 0 .. 15,
// so a softmax statistic of a query is one value per lane, and registers
// 8 kk .. 8 kk + 7 packed to 16 bits are, without any exchange between lanes,
// the second operand of the next product's step over 16 of those rows: its
// k slots 8 h .. 8 h + 7 (h = l / 32) stand for rows
//   16 kk + 4 h + {0, 1, 2, 3} and 16 kk + 8 + 4 h + {0, 1, 2, 3},
// which is what two transposing LDS reads of four rows each give the first
// operand.
//
// An LDS tile is [rows][16-byte chunks of 8 values], eight or sixteen chunks
// to a row, chunk c of row r at c ^ swz(r): both the 16-byte reads of
// consecutive rows and the transposing reads of four rows touch every bank
// once.
#pragma once

#include <algorithm>

#include "gemm_common.h"

namespace nova_hip {
namespace attn {

using gemm::f32x16;
using gemm::kOOB;
using gemm::make_rsrc;
using gemm::mfma_32x32x16;
using gemm::u32x2;
using gemm::u32x4;

typedef __attribute__((address_space(3))) void lds_void;
// Tiles are passed as LDS pointers: through generic ones the compiler keeps
// null checks of the conversion.
typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(3))) float lds_float;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Strides in elements.
struct Rows {
  int64_t t, h;  // token and head strides
};

// Chunks to an LDS row for a head dimension padded to DP.
template <int DP>
constexpr int kPitch = DP <= 64 ? 8 : 16;

template <int CH>
__device__ __forceinline__ int swz(int row) {
  if constexpr (CH == 16) return ((row & 3) << 2) | ((row >> 2) & 3);
  else return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
}

// Workgroup id -> (head, tile).  The hardware deals ids to the 8 XCDs in turn.
// Equal tiles: each XCD takes one run of the heads' tiles, head after head, so
// that the workgroups that read the same keys share an L2.  Tiles of falling
// work (causal): every head's first tile, then every head's second, the heads
// still divided over the XCDs where they divide evenly; with heads in turn the
// last one's largest tiles start late and run alone.  Forward / backward, us,
// heads in turn against this: 8192 tokens of 32 heads of 128 566 / 1817 against
// 535 / 1786, of 12 heads 288 / 1096 against 228 / 712.
__device__ __forceinline__ void unit_of(int id, int heads, int tiles, bool causal, int &head,
                                        int &tile) {
  const int x = id & 7, r = id >> 3;
  if (!causal) {
    const int total = heads * tiles, per = total >> 3, rem = total & 7;
    const int w = x * per + min(x, rem) + r;
    head = w / tiles;
    tile = w - head * tiles;
  } else if (heads % 8 == 0) {
    const int mine = heads >> 3;
    tile = r / mine;
    head = x * mine + r - tile * mine;
  } else {
    tile = id / heads;
    head = id - tile * heads;
  }
}

__device__ __forceinline__ int wave_sum_int(int v) {
#define NOVA_DPP_ADD(c) v += __builtin_amdgcn_mov_dpp(v, c, 0xF, 0xF, false)
  NOVA_DPP_ADD(0xB1);   // quad_perm [1,0,3,2]
  NOVA_DPP_ADD(0x4E);   // quad_perm [2,3,0,1]
  NOVA_DPP_ADD(0x141);  // row_half_mirror
  NOVA_DPP_ADD(0x140);  // row_mirror
#undef NOVA_DPP_ADD
  return (__builtin_amdgcn_readlane(v, 0) + __builtin_amdgcn_readlane(v, 16)) +
         (__builtin_amdgcn_readlane(v, 32) + __builtin_amdgcn_readlane(v, 48));
}

// A tile's place: its index among its sequence's tiles, their number, and the
// sequence's rows in the operand that is tiled and in the other one.
struct Tile {
  int index, tiles, s, e, os, oe;
};

// Tile t of the sequences' tiles of BM rows, off[0 .. B] being the sequences'
// first rows and other[0 .. B] those of the other operand; whatever they hold,
// every sequence is cut to rows inside [0, T) and [0, To).  False when there is
// no such tile.  Wave-uniform; every wave searches for itself.
//
// Up to 64 sequences, whose rows one load brings into registers: in the order of
// falling index within the sequence, the last tiles of the longest sequences
// first, which is the order of falling work of causal attention (or of rising
// index counted from the end, for keys), so that what runs last is short.  With
// S(l) = sum over sequences of max(0, tiles - l), the tiles of index l and above,
// that is the largest l with S(l) > t, found bit by bit.
//
// More: sequence b's tiles are numbered from off[b] / BM + b, which leaves it at
// least as many numbers as it has tiles and needs no sums; 64 sequences are
// probed at a time (three loads for 2^18 sequences), the last ones first.
__device__ __forceinline__ bool find_tile(const int *off, const int *other, int B, int T, int To,
                                          int BM, int t, Tile &tile) {
  const int lane = threadIdx.x & 63;
  auto rows_of = [&](const int *o, int n, int b, int &s, int &e) __attribute__((always_inline)) {
    s = e = 0;
    if (b < B) {
      s = min(max(o[b], 0), n);
      e = max(s, min(max(o[b + 1], 0), n));
    }
  };
  int s0, e0, os0, oe0, l;
  if (B <= 64) {
    rows_of(off, T, lane, s0, e0);
    rows_of(other, To, lane, os0, oe0);
    const int n = (e0 - s0 + BM - 1) / BM;
    auto above = [&](int k) __attribute__((always_inline)) { return wave_sum_int(max(0, n - k)); };
    if (above(0) <= t) return false;
    int level = 0, bit = 1;
    while (bit < (1 << 25) && above(bit) > t) bit <<= 1;
    for (bit >>= 1; bit > 0; bit >>= 1)
      if (above(level + bit) > t) level += bit;
    const int k = t - above(level + 1);  // among the sequences with a tile of that index
    const uint64_t has = __ballot(n > level);
    const int rank = __builtin_amdgcn_mbcnt_hi((uint32_t)(has >> 32),
                                               __builtin_amdgcn_mbcnt_lo((uint32_t)has, 0));
    const uint64_t hit = __ballot(n > level && rank == k);
    if (!hit) return false;
    l = __builtin_ctzll(hit);
    tile.index = level;
    tile.tiles = __builtin_amdgcn_readlane(n, l);
  } else {
    t = T / BM + B - 1 - t;
    int lo = 0, n = B;
    for (;;) {
      const int step = (n + 63) / 64, b = lo + lane * step;
      const bool at = lane * step < n && min(max(off[b], 0), T) / BM + b <= t;
      const int c = __builtin_popcountll(__ballot(at));
      if (c == 0) return false;
      lo += (c - 1) * step;
      n = min(step, n - (c - 1) * step);
      if (step == 1) break;
    }
    rows_of(off, T, lo, s0, e0);
    rows_of(other, To, lo, os0, oe0);
    l = 0;
    tile.index = t - (s0 / BM + lo);
    tile.tiles = (e0 - s0 + BM - 1) / BM;
    if (tile.index < 0 || tile.index >= tile.tiles) return false;
  }
  tile.index = __builtin_amdgcn_readfirstlane(tile.index);
  tile.tiles = __builtin_amdgcn_readfirstlane(tile.tiles);
  tile.s = __builtin_amdgcn_readlane(s0, l);
  tile.e = __builtin_amdgcn_readlane(e0, l);
  tile.os = __builtin_amdgcn_readlane(os0, l);
  tile.oe = __builtin_amdgcn_readlane(oe0, l);
  return true;
}

// The tiles find_tile may give: whole ones and, for each sequence, at most one
// that is not.
inline int64_t tile_bound(int64_t T, int64_t B, int64_t BM) {
  return B <= 64 ? std::min(T, T / BM + B) : T / BM + B;
}

// Loads of one LDS tile of ROWS rows by NW waves: per thread, the byte offset
// from the tile's first row of each 16-byte chunk it fetches.  A DMA
// instruction writes 64 lanes x 16 bytes in a row, so the swizzle is applied
// by choosing the chunk; chunks past the head dimension read zero.
template <int ROWS, int CH, int NW>
struct TileLoad {
  static constexpr int kN = ROWS * CH / 64 / NW;
  static constexpr int kStep = 64 * NW / CH;  // rows from one of a thread's chunks to its next
  static_assert(ROWS * CH % (64 * NW) == 0 && kStep % 16 == 0, "whole rounds, one swizzle");
  uint32_t off;   // of the thread's first chunk, or kOOB
  uint32_t step;  // bytes to the next one

  // By threads 0 .. 64 NW - 1 of each group of that many.
  __device__ __forceinline__ void init(int64_t stride, int D) {
    const int slot = threadIdx.x % (64 * NW), row = slot / CH, c = (slot & (CH - 1)) ^ swz<CH>(row);
    off = c * 8 < D ? (uint32_t)(row * stride + c * 8) * 2u : kOOB;
    step = (uint32_t)(kStep * stride) * 2u;
  }
  // Rows [0, rows) at p to the tile; rows behind them read zero.
  __device__ __forceinline__ void load(const uint16_t *p, int64_t stride, int rows, int D,
                                       lds_char *tile) const {
    const int n = min(rows, ROWS);
    const uint32_t bytes = n > 0 ? ((uint32_t)(n - 1) * (uint32_t)stride + D) * 2u : 0u;
    const __amdgpu_buffer_rsrc_t rs = make_rsrc(p, bytes);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % NW;
#pragma unroll
    for (int i = 0; i < kN; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rs, (lds_void *)(tile + (i * NW + wave) * 1024), 16, off + (uint32_t)i * step, 0, 0, 0);
  }
};

// Byte offset of a lane's 16-byte read of rows [r0, r0 + 32), k step s.
template <int CH>
__device__ __forceinline__ uint32_t row_frag(int r0, int s, int lane) {
  const int row = r0 + (lane & 31);
  return (uint32_t)(row * CH + ((2 * s + (lane >> 5)) ^ swz<CH>(row))) * 16u;
}
__device__ __forceinline__ u32x4 read_row_frag(const lds_char *tile, uint32_t off) {
  typedef __attribute__((address_space(3))) const u32x4 lds_u32x4;
  return *(lds_u32x4 *)(tile + off);
}

typedef short i16x4 __attribute__((ext_vector_type(4)));
// The transposed fragment: columns [d0, d0 + 32) as the instruction's rows,
// LDS rows r0 + 16 kk + .. as its k slots in the order given above.
template <int CH>
__device__ __forceinline__ uint32_t col_frag(int r, int d0, int lane) {
  const int g = lane >> 4, p = lane & 15;
  const int row = r + 4 * (g >> 1) + (p >> 2), d = d0 + 16 * (g & 1) + 4 * (p & 3);
  return (uint32_t)((row * CH + ((d >> 3) ^ swz<CH>(row))) * 8 + (d & 7)) * 2u;
}
__device__ __forceinline__ u32x2 read_tr(const lds_char *p) {
  typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4 *)p));
}
template <int CH>
__device__ __forceinline__ u32x4 read_col_frag(const lds_char *tile, int r0, int d0, int lane) {
  const u32x2 lo = read_tr(tile + col_frag<CH>(r0, d0, lane));
  const u32x2 hi = read_tr(tile + col_frag<CH>(r0 + 8, d0, lane));
  return u32x4{lo[0], lo[1], hi[0], hi[1]};
}

// Inside a wave-uniform branch around masks: an empty statement with a side
// effect keeps the compiler from turning the branch into selects, which every
// tile would pay for.
__device__ __forceinline__ void keep_branch() { asm volatile(""); }

template <int DT>
__device__ __forceinline__ uint32_t pack(float a, float b) {
  return DT == NOVA_HIP_DT_BF16 ? gemm::pack_bf16(a, b) : gemm::pack_f16(a, b);
}
// Registers 8 kk .. 8 kk + 7 of a result tile as the next product's operand.
template <int DT>
__device__ __forceinline__ u32x4 pack_frag(const f32x16 &x, int kk) {
  u32x4 f;
#pragma unroll
  for (int j = 0; j < 4; ++j) f[j] = pack<DT>(x[8 * kk + 2 * j], x[8 * kk + 2 * j + 1]);
  return f;
}

// The 32 rows at p (row l % 32 of them this lane's) as the instruction's
// columns: 8 values at d = 16 s + 8 (l / 32).  Rows behind `rows` and values
// behind D are zero.
template <int DP>
__device__ __forceinline__ void load_cols(u32x4 (&f)[DP / 16], const uint16_t *p, int64_t stride,
                                          int rows, int D, int lane) {
  const int n = min(rows, 32);
  const uint32_t bytes = n > 0 ? (uint32_t)(((n - 1) * stride + D) * 2) : 0u;
  const __amdgpu_buffer_rsrc_t rs = make_rsrc(p, bytes);
  const uint32_t row = (uint32_t)((lane & 31) * stride) * 2u;
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    const int d = 16 * s + 8 * (lane >> 5);
    f[s] = __builtin_bit_cast(
        u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, d < D ? row + (uint32_t)d * 2u : kOOB, 0, 0));
  }
}

// max / sum over a lane and its partner 32 lanes away (the other rows of the
// same column).
__device__ __forceinline__ float both_max(float v) { return fmaxf(v, __shfl_xor(v, 32)); }
__device__ __forceinline__ float both_sum(float v) { return v + __shfl_xor(v, 32); }

// A wave's transposed result [DP columns d][32 rows], times `mul` of the
// lane's row, to 16-bit rows at p: row l % 32 < rows.  Lane halves trade 8-byte
// pieces so that each lane stores 16 bytes.
template <int DT, int DP>
__device__ __forceinline__ void store_rows(const f32x16 (&acc)[DP / 32], float mul, uint16_t *p,
                                           int64_t stride, int rows, int D, int lane) {
  uint16_t *dst = p + (lane & 31) * stride;
  const bool ok = (lane & 31) < rows;
#pragma unroll
  for (int b = 0; b < DP / 32; ++b)
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      uint32_t x[2], y[2];  // d = 32 b + 8 i + 4 h + .., and 8 on
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        x[j] = pack<DT>(acc[b][4 * i + 2 * j] * mul, acc[b][4 * i + 2 * j + 1] * mul);
        y[j] = pack<DT>(acc[b][4 * i + 4 + 2 * j] * mul, acc[b][4 * i + 5 + 2 * j] * mul);
        const auto sw = __builtin_amdgcn_permlane32_swap(x[j], y[j], false, false);
        x[j] = sw[0];
        y[j] = sw[1];
      }
      const int d = 32 * b + 8 * (i + (lane >> 5));
      if (ok && d < D) *reinterpret_cast<u32x4 *>(dst + d) = u32x4{x[0], x[1], y[0], y[1]};
    }
}

}  // namespace attn
}  // namespace nova_hip

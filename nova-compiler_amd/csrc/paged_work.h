// How the work of a paged attention call is cut: the form, grid and scratch from the
// sizes (plan_of, on the host), the keys of a piece from the lengths (piece_keys, in
// every workgroup).  Plain C++: a host compiler takes it too.
#pragma once
#include <algorithm>
#include <cmath>
#include <cstdint>

#ifdef __HIPCC__
#define NOVA_BOTH __host__ __device__ __forceinline__
#else
#define NOVA_BOTH inline
#endif

namespace nova_hip {
namespace attn {
namespace paged {

constexpr int kBM = 128;  // (token, head of the group) rows of a chunk's tile

// The work is cut so that it fills the chip's places for workgroups and no place is
// left with a long remainder.  With fewer tiles than places, a sequence's keys into as
// many splits as fill the places once; with more, only where its tiles see kLong times
// the keys that a place has in the mean (one token over a long cache among prompts).  20
// drawn steps of 1.05 to 4 tiles to a place, heads of 64 and 128, at 1.0 / 1.3 / 1.6 / 2.0
// take 2.3 / 1.5 / 2.5 / 7.9 % longer than the best of the four in the mean, 18 / 17 / 12 /
// 29 % at most; with what counted_keys leaves whole 1.6 against 2.0: 4 % less in the mean, 19 %
// less to 8 % more.  A step of 3751 tokens 236 us at either, a prompt of 4096 beside one token
// over 131072 rows 255 against 304.
constexpr float kLong = 1.6f;
// Filling the places once ends with the longest piece.  A causal prompt alone, whose tiles
// see half of it in the mean, finds its tiles whole at less than 3 times that.
constexpr float kFill = 3.0f;

NOVA_BOTH float reciprocal(float x) {
#ifdef __HIP_DEVICE_COMPILE__
  return __builtin_amdgcn_rcpf(x);
#else
  return 1.0f / x;
#endif
}

// Keys that the tiles of a sequence of n new tokens and len rows see in the mean, or more.
NOVA_BOTH float mean_keys(int n, int len, bool causal) {
  return causal ? fmaxf(0.5f * (float)len, (float)len - 0.5f * (float)n) : (float)len;
}

// What counts of them against a piece, at least 3/4 of the rows: the last tiles of a causal
// prompt see all of it, but run beside its first ones, which leave them the CU.  A prompt
// alone, or several of a length, are so never cut where tiles are as many as places (8192
// tokens of 12 heads of 64: 153 us, counted in full, and cut, 168).
NOVA_BOTH float counted_keys(int n, int len, bool causal) {
  return fmaxf(mean_keys(n, len, causal), 0.75f * (float)len);
}

// Splits at c keys to a piece of a sequence of len rows, `counted` of them, and the rows of a
// piece: what the quotient is off by is less than the margin, so that n of them hold it.
NOVA_BOTH float splits_at(float len, float counted, float c) {
  return counted > c ? fmaxf(1.0f, ceilf(len * reciprocal(c))) : 1.0f;
}
NOVA_BOTH int piece_of(int len, float n) {
  return ((int)((float)len * reciprocal(n)) + 2 + (len >> 20) + 63) / 64 * 64;
}

// Keys of a piece, `least` or more, of `all` tiles that see `mean` times `places` keys;
// units(c, split) counts the units at c keys to a piece, or only those of sequences that
// are split then, for which there is room.  The search for what fills the places may end a
// few units above them; where only pieces past kFill times its start would fill them, the
// tiles are cut as where there are more.  Room is then found by longer pieces: the units of
// split sequences are sum tiles ceil(len / c) < 2 sum tiles len / c, and a mean is half of
// len or more, so they are less than 4 places mean / c.  That is the places, the least room
// there is, at 4 times the mean.
// (13 chunks of 128 tokens over 8192 rows beside one token over 131072, 16 heads in groups
// of 4 of 128: 208 us, 3090 where a batch whose search ends above its room is not split.)
template <typename Units>
NOVA_BOTH float piece_keys(float all, float mean, float places, float least, float room, Units units) {
  float c = fmaxf(mean, 1.0f);
  const float end = all < places ? kFill * c : 0.0f;
  for (int i = 0; i < 8 && c <= end; ++i) {
    const float n = units(c, false);
    if (n <= places) return fmaxf(c, least);
    c *= fmaxf(1.02f, n * reciprocal(places));
  }
  c = fmaxf(c > end ? kLong * mean : c, least);
  for (int i = 0; i < 32 && units(c, true) > room; ++i) c *= 1.05f;
  return c;
}

// The form of a call, its tiles of rows per key head (up to 64 sequences: with their
// splits), its splits and slots.
struct Plan {
  bool narrow;
  int64_t tiles, chunk, splits, slots, least, places;
};
inline Plan plan_of(int64_t T, int64_t B, int64_t heads, int64_t kv_heads, int64_t D, int64_t rows,
                    int64_t max_queries) {
  Plan p = {};
  const int64_t group = heads / kv_heads;
  // Single tokens in the chunks' form: those 32 128 us, one over 8192 rows 20 against 15.
  p.narrow = max_queries * group <= 32 && B <= 0xffff;
  p.chunk = std::max<int64_t>(rows, 1);
  // Workgroups resident at once, by LDS (a wave's 32 or 16 KB) and registers; single
  // tokens: as many as it takes to fill the memory's pipes (512 / 768 / 1024: 32 tokens over
  // 1500 to 8192 rows 123 / 116 / 116 us, 8 over 8192 55 / 52 / 56; chunks, 256 / 512 / 768:
  // 512 tokens over 8192 rows 105 / 90 / 100).  Least keys of a piece of 128 instead of 256
  // and 32 instead of 64: within 1 us either way.
  p.places = p.narrow ? (D <= 64 ? 1536 : 768) : (D <= 64 ? 768 : 512);
  p.least = p.narrow ? 64 : 256;
  const int64_t most = (rows + p.least - 1) / p.least, mine = (p.places + kv_heads - 1) / kv_heads;
  // For the units of split sequences (see piece_keys): the places, or twice those where
  // there may be more tiles than places.
  auto room = [&](int64_t tiles) { return std::min(tiles * most, tiles < mine ? mine : 2 * mine); };
  if (p.narrow && B <= 64 && B * kv_heads * most > p.places) {
    p.slots = room(B);
    p.tiles = B + p.slots;
  } else if (p.narrow) {
    // As for the padded cache (attention_decode.hip).
    const int64_t all = B * rows * kv_heads;
    const int64_t keys = std::max(std::min<int64_t>(512, all / 2048), std::min<int64_t>(2048, all / 8192));
    p.chunk = std::max<int64_t>(64, (std::max(keys, rows / 32768) + 63) / 64 * 64);
  } else if (B <= 64) {
    p.tiles = std::min(T * group, T * group / kBM + B);
    if (most > 1) p.slots = room(p.tiles);
    p.tiles += p.slots;
  } else {
    p.tiles = T * group / kBM + B;
    const int64_t splits =
        std::max<int64_t>(1, std::min(3 * p.places / (2 * p.tiles * kv_heads), rows / 512));
    p.chunk = std::max<int64_t>(64, ((rows + splits - 1) / splits + 63) / 64 * 64);
  }
  p.splits = std::max<int64_t>(1, (rows + p.chunk - 1) / p.chunk);
  if (!p.narrow && p.splits > 1) p.slots = p.tiles * p.splits;
  return p;
}

}  // namespace paged
}  // namespace attn
}  // namespace nova_hip

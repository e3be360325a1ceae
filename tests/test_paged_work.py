"""How a paged attention call's keys are cut (paged_work.h), compiled for the host:
for batches of up to 64 sequences no split is lost, and no piece is much longer than
what a place for a workgroup has in the mean."""
import ctypes
import os
import random
import subprocess

import pytest

from conftest import PKG

SOURCE = r"""
#include "csrc/paged_work.h"
using namespace nova_hip::attn::paged;
extern "C" void cut(long T, int B, const int *n, const int *len, long heads, long kv_heads, long D, long rows,
                    long most, int causal, long *sizes, float *found, int *splits, int *piece) {
  const Plan p = plan_of(T, B, heads, kv_heads, D, rows, most);
  const int group = (int)(heads / kv_heads);
  const float places = (float)p.places / (float)kv_heads;
  float all = 0.0f, keys = 0.0f;
  auto tiles = [&](int b) { return p.narrow ? (float)(n[b] > 0) : (float)((n[b] * group + kBM - 1) / kBM); };
  for (int b = 0; b < B; ++b) all += tiles(b), keys += tiles(b) * mean_keys(n[b], len[b], causal != 0);
  auto splits_of = [&](int b, float c) {
    return splits_at((float)len[b], counted_keys(n[b], len[b], causal != 0), c);
  };
  auto units = [&](float c, bool split) {
    float sum = 0.0f;
    for (int b = 0; b < B; ++b) {
      const float k = splits_of(b, c);
      sum += split && k <= 1.0f ? 0.0f : tiles(b) * k;
    }
    return sum;
  };
  const float c = piece_keys(all, keys / places, places, (float)p.least, (float)p.slots, units);
  sizes[0] = p.narrow, sizes[1] = p.tiles, sizes[2] = p.slots, sizes[3] = p.least;
  found[0] = units(c, false), found[1] = units(c, true), found[2] = keys / places;
  for (int b = 0; b < B; ++b) {
    const float k = splits_of(b, c);
    splits[b] = (int)k;
    piece[b] = k > 1.0f ? piece_of(len[b], k) : len[b];
  }
}
"""


@pytest.fixture(scope="module")
def cut(tmp_path_factory):
    d = tmp_path_factory.mktemp("work")
    (d / "work.cpp").write_text(SOURCE)
    so = str(d / "work.so")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I" + PKG,
                    str(d / "work.cpp"), "-o", so], check=True)
    lib = ctypes.CDLL(so)

    def call(new, lens, heads, kv_heads, D, causal=True):
        """Checks what every cut has to hold; (longest piece, a place's mean, units)."""
        B, L = len(new), ctypes.c_long
        ints, size = ctypes.c_int * B, (L * 4)()
        found, splits, piece = (ctypes.c_float * 3)(), ints(), ints()
        lib.cut(L(sum(new)), B, ints(*new), ints(*lens), L(heads), L(kv_heads), L(D), L(max(lens)), L(max(new)),
                int(causal), size, found, splits, piece)
        narrow, tiles, slots, least = size
        if not slots:
            return None
        units, split, mean = found
        what = (new, lens, heads, kv_heads, D, causal)
        assert split <= slots and units <= tiles, what     # the splits have their room, the units their workgroup
        for k, p, n in zip(splits, piece, lens):
            assert k * p >= n and (k == 1 or p % 64 == 0), what
        longest = max(p for p, n in zip(piece, new) if n)
        # Up to 4 times the mean where room is short, in steps of 5 %, rounded to 64.
        assert longest <= 4.2 * max(mean, least) + 64 + 2, (longest, mean, what)
        return longest, mean, units

    return call


@pytest.mark.parametrize("kv_heads,group", [(1, 1), (1, 4), (2, 1), (4, 4), (8, 4), (6, 1)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new", [1, 128])
def test_equal_lengths_and_one_long_sequence(cut, new, D, kv_heads, group):
    """Lengths that fill the places all at once only at one piece size, beside a long
    one: the longest piece stays near the mean, however many sequences there are."""
    for count in range(1, 64):
        for rows in (1000, 8192):
            for long in (2 * rows, 131072):
                cut([new] * count + [1], [rows] * count + [long], kv_heads * group, kv_heads, D)


def test_batches_that_missed_their_room(cut):
    longest, mean, _ = cut([128] * 13 + [1], [8192] * 13 + [131072], 16, 4, 128)
    assert longest <= 1.5 * mean
    longest, mean, _ = cut([1] * 64, [8192] * 63 + [16384], 2, 2, 128)
    assert longest <= 1.5 * mean
    # Nearly as many tiles as places: the long one is cut all the same.
    longest, mean, _ = cut([32] * 60 + [1], [1000] * 60 + [131072], 32, 8, 128)
    assert longest <= 2.0 * mean


def test_a_long_sequence_among_more_tiles_than_places(cut):
    """No piece past 1.6 times what a place has in the mean, and its rounding."""
    for new, lens, heads, kv_heads in (([4096, 1], [4096, 131072], 32, 8), ([2048, 2048, 64], [2048, 2048, 16384], 32, 8),
                                       ([8192] * 3 + [1], [8192] * 3 + [65536], 12, 12)):
        longest, mean, _ = cut(new, lens, heads, kv_heads, 128)
        assert longest <= 1.6 * mean + 64 + 2


@pytest.mark.parametrize("heads,kv_heads,D,places", [(32, 8, 128, 64), (12, 12, 64, 64), (6, 6, 64, 128),
                                                     (64, 8, 128, 64), (9, 3, 80, 171)])
def test_plain_prompts_stay_whole(cut, heads, kv_heads, D, places):
    """Prompts of one length and as many tiles as places, or more: no unit but their tiles."""
    for count in (1, 2, 3, 5):
        for more in range(3, 400, 7):
            tokens = ((-(-places // count) - 1) * 128 + more) // (heads // kv_heads) + 1
            tiles = count * -(-tokens * (heads // kv_heads) // 128)
            assert tiles >= places
            found = cut([tokens] * count, [tokens] * count, heads, kv_heads, D)
            assert found is None or found[2] == tiles  # (None: no room for splits at all)


@pytest.mark.parametrize("seed", range(8))
def test_any_batch(cut, seed):
    rng = random.Random(seed)
    for _ in range(400):
        kv_heads = rng.choice([1, 2, 3, 4, 6, 8, 16])
        B, most = rng.randint(1, 64), rng.choice([1, 1, 7, 300, 3000])
        base = rng.choice([1, 60, 700, 5000, 40000, 1 << 20])
        new = [rng.choice([0, 1, 1, rng.randint(1, most)]) for _ in range(B)]
        lens = [max(n, rng.choice([0, base, rng.randint(1, base)])) for n in new]
        if max(new):
            cut(new, lens, kv_heads * rng.choice([1, 2, 4, 8]), kv_heads, rng.choice([32, 64, 128]),
                rng.random() < 0.8)

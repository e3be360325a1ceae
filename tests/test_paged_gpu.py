"""The paged cache: where new tokens' keys and values go, and the attention over
it against its definition in 64 bits (tolerances: test_attention_gpu.py,
test_positions_gpu.py)."""
import pytest
import torch

import nova_hip as nh
from test_attention_gpu import BF, HF, check, offsets
from test_positions_gpu import freqs_of, near, turned

pytestmark = pytest.mark.gpu
NAN = float("nan")


class Cache:
    """Pages in a random order; rows that no sequence has hold NaN, entries of the
    table that no sequence needs point outside the pages."""

    def __init__(self, dev, lens, G, D, page, dt, order="psgd", width=None, seed=0, spare=2):
        g = torch.Generator(device=dev).manual_seed(seed)
        need = [-(-n // page) for n in lens]
        pool = sum(need) + spare
        self.page, self.lens = page, lens
        if order == "psgd":
            self.k, self.v = (torch.full((pool, page, G, D), NAN, dtype=dt, device=dev) for _ in range(2))
        elif order == "pgsd":
            self.k, self.v = (torch.full((pool, G, page, D), NAN, dtype=dt, device=dev).transpose(1, 2)
                              for _ in range(2))
        else:  # keys and values of a page in one buffer, heads outermost
            kv = torch.full((G, pool, 2, page, D), NAN, dtype=dt, device=dev).permute(1, 2, 3, 0, 4)
            self.k, self.v = kv[:, 0], kv[:, 1]
        width = max(need + [1]) + 1 if width is None else width
        self.table = torch.full((len(lens), width), 1 << 30, dtype=torch.int32, device=dev)
        self.table[:, 1::2] = -7
        ids = torch.randperm(pool, generator=g, device=dev).int()
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = ids[at:at + n]
            at += n
        self.packed = [torch.randn(sum(lens), G, D, generator=g, device=dev).to(dt) for _ in range(2)]
        at = 0
        for b, n in enumerate(lens):
            pos = torch.arange(n, device=dev)
            where = (self.table[b].long()[pos // page], pos % page)
            self.k[where], self.v[where] = self.packed[0][at:at + n], self.packed[1][at:at + n]
            at += n
        self.lengths = torch.tensor(lens, dtype=torch.int32, device=dev)


def run(dev, seqs, H, G, D, dt=BF, page=16, causal=True, order="psgd", width=None, hint=True, pad=0, seed=0,
        scale=None):
    """seqs: (new tokens, rows) of each sequence."""
    new, lens = [n for n, _ in seqs], [r for _, r in seqs]
    c = Cache(dev, lens, G, D, page, dt, order, width, seed)
    g = torch.Generator(device=dev).manual_seed(seed + 1)
    T = sum(new)
    q = torch.randn(T + pad, H, D, generator=g, device=dev).to(dt)
    q[T:] = NAN
    out = torch.full(q.shape, 7.0, dtype=dt, device=dev)
    lse = torch.full((H, T + pad), 7.0, device=dev)
    off = offsets(new, dev)
    scale = D ** -0.5 if scale is None else scale
    nh.paged_attention(q, c.k, c.v, off, c.lengths, c.table, causal=causal, scale=scale, out=out, lse=lse,
                       max_queries=max(new + [1]) if hint else None)
    what = (seqs if len(seqs) < 20 else len(seqs), H, G, D, dt, page, causal, order, hint)
    assert (out[T:] == 7.0).all() and (lse[:, T:] == 7.0).all(), what
    check(out, lse, q, c.packed[0], c.packed[1], new, lens, causal, scale, what)
    return q, c, off, out, lse


SINGLE = [(1, 97), (1, 1), (1, 64), (1, 130)]
CHUNKS = [(5, 97), (64, 64), (33, 300), (1, 130), (130, 131), (0, 50)]


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("D", [8, 32, 40, 64, 80, 96, 120, 128])
@pytest.mark.parametrize("seqs", [SINGLE, CHUNKS])
def test_head_dims(cuda, seqs, D, dt):
    run(cuda, seqs, 8, 2, D, dt)


@pytest.mark.parametrize("page", [1, 2, 4, 5, 8, 12, 16, 24, 31, 32, 48, 64, 100, 128, 256, 1000])
@pytest.mark.parametrize("seqs", [SINGLE, CHUNKS])
@pytest.mark.parametrize("D", [64, 128])
def test_page_sizes(cuda, seqs, page, D):
    run(cuda, seqs, 4, 2, D, page=page)


@pytest.mark.parametrize("order", ["psgd", "pgsd", "gp2sd"])
@pytest.mark.parametrize("H,G", [(1, 1), (6, 6), (7, 1), (32, 8), (33, 1), (71, 1), (64, 32), (140, 1), (10, 2)])
@pytest.mark.parametrize("hint", [False, True])
def test_orders_and_shared_heads(cuda, H, G, order, hint):
    run(cuda, [(1, 33), (1, 200), (1, 1)], H, G, 64, order=order, hint=hint)
    run(cuda, [(3, 33), (70, 200), (2, 1)], H, G, 64, order=order, hint=hint)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("seqs", [
    [(1, 0)], [(3, 0), (2, 5)], [(9, 4), (4, 4), (1, 1)],   # more queries than rows: empty rows
    [(0, 0), (0, 9), (1, 9)], [(300, 100)], [(129, 128), (128, 129)], [(1, 2000)], [(31, 2000), (2, 7)]])
def test_empty_rows_and_edges(cuda, seqs, causal):
    for hint in (False, True):
        run(cuda, seqs, 4, 2, 64, causal=causal, hint=hint, pad=3)


@pytest.mark.parametrize("rows", [63, 64, 65, 511, 512, 513, 1000, 3001])
@pytest.mark.parametrize("new", [1, 2, 20])
def test_splits(cuda, rows, new):
    run(cuda, [(new, rows), (1, rows // 2), (new, rows - 1)], 8, 2, 128, HF)
    run(cuda, [(new, rows)], 4, 4, 64, page=8, width=rows // 8 + 200)  # a table far wider than the rows


def test_many_splits_and_sequences(cuda):
    run(cuda, [(1, 40000), (1, 3)], 4, 1, 64, page=64)
    run(cuda, [(17, 30000)], 4, 1, 64, page=32)
    run(cuda, [(1, 700), (1, 5), (1, 90)] * 40, 8, 2, 64)
    run(cuda, [(1, 70), (3, 5), (0, 4), (40, 90)] * 40, 8, 2, 64)
    run(cuda, [(i % 3, 1 + i % 50) for i in range(5000)], 2, 1, 32, page=16, hint=False)


def test_large_chunks(cuda):
    run(cuda, [(2048, 2048), (1024, 3000), (1, 4000)], 8, 2, 128, page=64, order="pgsd")
    run(cuda, [(1500, 1700)], 6, 6, 64, HF, page=48, causal=False)
    run(cuda, [(700, 1700)], 6, 6, 96, HF, page=24)


def test_lengths_and_entries_out_of_range(cuda):
    """Lengths are cut to the table, entries to the pages: every result is one of
    rows that are there."""
    q, c, off, out, lse = run(cuda, [(2, 40), (1, 16), (3, 60)], 4, 2, 64, page=16, width=4)
    long = torch.tensor([-5, 10 ** 9, 2 ** 31 - 1], dtype=torch.int32, device=cuda)
    c.k.nan_to_num_(0.5)
    c.v.nan_to_num_(0.5)
    for hint in (None, 3):
        got = nh.paged_attention(q, c.k, c.v, off, long, c.table, max_queries=hint)
        assert (got[:2] == 0).all()
        t = c.table.long().clamp(0, len(c.k) - 1)
        kp, vp = (x[t[b]].flatten(0, 1) for b in (1, 2) for x in (c.k, c.v)), None
        k1, v1, k2, v2 = kp
        check(got[2:], None, q[2:], torch.cat([k1, k2]), torch.cat([v1, v2]), [1, 3], [64, 64], True, 64 ** -0.5)
    # No pages, no table: rows of zeros.
    assert (nh.paged_attention(q, c.k[:0], c.v[:0], off, c.lengths, c.table) == 0).all()
    assert (nh.paged_attention(q, c.k, c.v, off, c.lengths, c.table[:, :0]) == 0).all()
    # Offsets past the tokens are cut, those that fall make empty sequences.
    bad = torch.tensor([4, 2, 900, 3], dtype=torch.int32, device=cuda)
    got = nh.paged_attention(q, c.k, c.v, bad, c.lengths, c.table, out=torch.zeros_like(q))
    assert torch.isfinite(got).all()


def test_a_hint_leaves_out_no_token_it_counts(cuda):
    """Two new tokens of each sequence with max_queries 2 to 9 and unknown: the
    same rows, whichever form takes them."""
    q, c, off, out, _ = run(cuda, [(2, 100), (2, 700), (1, 3)], 8, 2, 128)
    for hint in (2, 3, 8, 9, None):
        got = nh.paged_attention(q, c.k, c.v, off, c.lengths, c.table, max_queries=hint)
        assert (got.double() - out.double()).abs().max() <= 2.0 ** -6  # two roundings of values below 4


@pytest.mark.parametrize("new", [1, 30])
def test_nan_and_masked_places(cuda, new):
    """A NaN query reaches its own rows alone; NaN in the rows of other sequences
    none; infinities of a key that only later tokens see stay with those more than
    127 rows behind it unseen."""
    q, c, off, out, lse = run(cuda, [(new, 300), (new, 200)], 4, 2, 64)
    q[0, 1] = NAN
    again, l2 = torch.empty_like(out), torch.empty_like(lse)
    nh.paged_attention(q, c.k, c.v, off, c.lengths, c.table, out=again, lse=l2, max_queries=new)
    assert torch.isnan(again[0, 1]).all() and torch.isnan(l2[1, 0])
    bad = torch.zeros(out.shape[:2], dtype=torch.bool, device=cuda)
    bad[0, 1] = True
    assert torch.equal(again[~bad], out[~bad]) and torch.equal(l2.t()[~bad], lse.t()[~bad])


def test_keys_of_minus_infinity(cuda):
    """A row whose visible scores are all -inf is zero, its lse -inf."""
    q, c, off, out, lse = run(cuda, [(1, 70), (40, 70)], 4, 2, 64)
    q.fill_(1.0)
    c.k.fill_(0.0)
    c.k[..., 0] = -float("inf")
    for hint in (None, 40):
        got = nh.paged_attention(q, c.k, c.v.nan_to_num(0.0), off, c.lengths, c.table, lse=lse, max_queries=hint)
        assert (got == 0).all() and torch.isinf(lse).all() and (lse < 0).all()


@pytest.mark.parametrize("new", [1, 40])
def test_places_past_32_bits(cuda, new):
    """Pages more than 2^32 bytes apart, and a pool's head beyond 2^32."""
    P, D, far = 16, 64, (1 << 31) + 4096
    flat = torch.empty(far + 3 * P * D, dtype=BF, device=cuda)
    k = flat.as_strided((2, P, 2, D), (far, D, P * D, 1))
    g = torch.Generator(device=cuda).manual_seed(1)
    k.copy_(torch.randn(2, P, 2, D, generator=g, device=cuda).to(BF))
    table = torch.tensor([[1, 0]], dtype=torch.int32, device=cuda)
    q = torch.randn(new, 4, D, generator=g, device=cuda).to(BF)
    n = torch.tensor([29], dtype=torch.int32, device=cuda)
    out = nh.paged_attention(q, k, k, offsets([new], cuda), n, table, max_queries=new)
    rows = torch.cat([k[1], k[0]])[:29]
    check(out, None, q, rows, rows, [new], [29], True, D ** -0.5)


# ---- append -------------------------------------------------------------------------------

@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("D,R", [(64, 64), (128, 128), (80, 32), (40, 40), (8, 8), (256, 128), (64, None)])
def test_append(cuda, D, R, dt, interleaved):
    append_case(cuda, [(1, 1), (1, 700), (30, 40), (0, 9), (5, 5), (17, 64)], 6, 2, D, R, dt, interleaved)


@pytest.mark.parametrize("order", ["psgd", "pgsd", "gp2sd"])
@pytest.mark.parametrize("page", [1, 5, 16, 64, 1000])
def test_append_pages_and_orders(cuda, page, order):
    append_case(cuda, [(1, 700), (30, 1040), (2, 2)], 4, 2, 64, 64, BF, False, page, order)


@pytest.mark.parametrize("seqs", [[(1, 1 + i % 40) for i in range(300)], [(3000, 3000), (1, 9), (2000, 2500)],
                                  [(i % 3, 2 + i % 50) for i in range(5000)], [(0, 3)] * 70 + [(4, 9)]])
def test_append_many(cuda, seqs):
    append_case(cuda, seqs, 3, 1, 64, 64, BF, False)


def append_case(dev, seqs, H, G, D, R, dt, interleaved, page=16, order="psgd"):
    new, lens = [n for n, _ in seqs], [r for _, r in seqs]
    c = Cache(dev, lens, G, D, page, dt, order)
    kp, vp = c.k.clone(), c.v.clone()
    g = torch.Generator(device=dev).manual_seed(3)
    T, pad = sum(new), 2
    qkv = torch.randn(T + pad, H + 2 * G, D, generator=g, device=dev).to(dt)
    q, k, v = qkv[:, :H], qkv[:, H:H + G], qkv[:, H + G:]
    f = None if R is None else freqs_of(R, dev)
    off = offsets(new, dev)
    q_out = torch.full((T + pad, H, D), 7.0, dtype=dt, device=dev)
    nh.paged_append(k, v, c.k, c.v, off, c.lengths, c.table, freqs=f, interleaved=interleaved, scale=1.5, q=q,
                    q_out=q_out)
    assert (q_out[T:] == 7.0).all()
    pos = torch.cat([torch.arange(r - n, r, device=dev) for n, r in seqs])
    seq = torch.repeat_interleave(torch.arange(len(seqs), device=dev), torch.tensor(new, device=dev))
    where = (c.table.long()[seq, pos // page], pos % page)
    assert torch.equal(c.v[where], v[:T])
    for got, x in ((q_out[:T], q[:T]), (c.k[where], k[:T])):
        if f is None:
            assert torch.equal(got, x)
        else:
            want, amp = turned(x.double(), pos, f, interleaved, 1.5)
            near(got, want, amp, 2.0 ** -21)
    for a, b in ((c.k, kp), (c.v, vp)):  # every other row as it was, NaN included
        a[where] = 0.0
        b[where] = 0.0
        assert torch.equal(torch.nan_to_num(a, 9.0), torch.nan_to_num(b, 9.0))
    if f is not None:
        # The rotation on the way is the rotation of its own call.
        assert torch.equal(q_out[:T], nh.rotary(q[:T], pos.int(), f, interleaved=interleaved, scale=1.5))


def test_append_stores_nothing_outside(cuda):
    """Negative positions, positions beyond the table, pages that are none and
    tokens of no sequence."""
    c = Cache(cuda, [16, 16, 16, 16], 2, 64, 16, BF, width=1)
    c.table[2, 0], c.table[3, 0] = -1, len(c.k)
    kp, vp = c.k.clone(), c.v.clone()
    x = torch.ones(12, 2, 64, dtype=BF, device=cuda)
    lens = torch.tensor([1, 17, 16, 16], dtype=torch.int32, device=cuda)
    off = torch.tensor([2, 4, 5, 7, 9], dtype=torch.int32, device=cuda)
    q = torch.full((12, 2, 64), 3.0, dtype=BF, device=cuda)
    nh.paged_append(x, x, c.k, c.v, off, lens, c.table, q=q, q_out=q)
    row = c.table[0, 0].long()
    assert (c.k[row, 0] == 1).all() and (c.v[row, 0] == 1).all()  # token 3, at position 0
    c.k[row, 0], c.v[row, 0] = kp[row, 0], vp[row, 0]
    for a, b in ((c.k, kp), (c.v, vp)):
        assert torch.equal(torch.nan_to_num(a, 9.0), torch.nan_to_num(b, 9.0))
    # No pages at all: only q.
    nh.paged_append(x, x, c.k[:0], c.v[:0], off, lens, c.table, q=q, q_out=q)
    assert (q == 3.0).all()


def test_tokens_beyond_the_hint_are_left_out(cuda):
    """Seven new tokens where the call is told of one: the first ones that a tile
    of 32 rows holds are computed, the others' rows stay, whatever the splits."""
    for rows in (60, 3000):
        q, c, off, out, lse = run(cuda, [(7, rows), (1, rows)], 20, 2, 64)  # 10 heads to a key head
        got, l2 = torch.full_like(out, 5.0), torch.full_like(lse, 5.0)
        nh.paged_attention(q, c.k, c.v, off, c.lengths, c.table, out=got, lse=l2, max_queries=1)
        near = (got.double() - out.double()).abs() <= 2.0 ** -6
        assert near[:3].all() and near[7:].all() and (l2[:, :3] - lse[:, :3]).abs().max() < 1e-4
        assert (got[3:7] == 5.0).all() and (l2[:, 3:7] == 5.0).all()


@pytest.mark.parametrize("page", [5, 16])
@pytest.mark.parametrize("D", [64, 128])
def test_chunks_of_many_long_sequences(cuda, D, page):
    """More sequences than a wave has lanes, of few tokens over several splits."""
    seqs = [((0, 5, 1, 7)[i % 4], (2000, 1, 700, 1030, 0, 1500)[i % 6]) for i in range(70)]
    for causal in (False, True):
        run(cuda, seqs, 8, 1, D, page=page, causal=causal, pad=2)


@pytest.mark.parametrize("new", [1, 40])
def test_sequences_share_pages(cuda, new):
    """The same pages in two tables, and the same page twice in one."""
    lens = [70, 70, 70]
    c = Cache(cuda, lens, 2, 64, 16, BF)
    c.table[1] = c.table[0]
    c.table[2, 1] = c.table[2, 0]
    k, v = (p.clone() for p in c.packed)
    for x in (k, v):
        x[70:140] = x[:70]
        x[156:172] = x[140:156]
    q = torch.randn(3 * new, 4, 64, device=cuda).to(BF)
    out, lse = torch.empty_like(q), torch.empty(4, 3 * new, device=cuda)
    nh.paged_attention(q, c.k, c.v, offsets([new] * 3, cuda), c.lengths, c.table, out=out, lse=lse)
    check(out, lse, q, k, v, [new] * 3, lens, True, 64 ** -0.5, new)


@pytest.mark.parametrize("count", [3, 90])
def test_offsets_that_overlap(cuda, count):
    """Whatever the offsets hold, only the tokens' rows are written, and sequences
    that are sound and alone with their tokens have their result."""
    seqs = [(1, 900)] + [(60, 900)] * 2 + [(3, 20)] * (count - 3)
    q, c, off, out, _ = run(cuda, seqs, 8, 2, 64)
    T = len(q)
    wide = torch.full((T + 9, 8, 64), 7.0, dtype=BF, device=cuda)
    bad = off.clone()
    bad[2] = 2 ** 31 - 1  # sequence 1 has all tokens from its first, sequence 2 none
    bad[3] = 1
    for lens in (c.lengths, c.lengths - 10 ** 9, c.lengths + 10 ** 9):
        nh.paged_attention(q, c.k, c.v, bad, lens, c.table, out=wide[:T])
        assert (wide[T:] == 7.0).all()
    nh.paged_attention(q, c.k, c.v, bad, c.lengths, c.table, out=wide[:T])
    assert (wide[:1].double() - out[:1].double()).abs().max() <= 2.0 ** -6

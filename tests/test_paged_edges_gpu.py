"""Paged attention where batches and contents are unusual: lengths whose pieces are
searched for long, infinities and NaN in masked places, sequences that overlap, the
same call twice; and the gradients of a training step with positions, closely."""
import math

import pytest
import torch

import nova_hip as nh
from test_attention_gpu import BF, HF
from test_paged_gpu import run
from test_paged_step_gpu import D, G, H, LENS, split, train, training_state

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("seqs,H,G", [
    ([(128, 2048)] * 13 + [(1, 32768)], 16, 4), ([(1, 2048)] * 63 + [(1, 4096)], 2, 2),
    ([(32, 1000)] * 60 + [(1, 40000)], 32, 8), ([(2, 700)] * 40 + [(1, 30000)], 8, 4)])
def test_equal_lengths_and_one_long_sequence(cuda, seqs, H, G):
    run(cuda, seqs, H, G, 128, page=64)


def place(c, b, row):
    return int(c.table[b, row // c.page]), row % c.page


@pytest.mark.parametrize("bad", [NAN, INF])
@pytest.mark.parametrize("new,hint", [(300, None), (8, 8)])
def test_masked_rows_that_are_not_finite(cuda, new, hint, bad):
    """One row of a chunk's keys, then of its values.  Keys: tokens ahead of it keep
    their bits, those from it on, in the heads that read it, are NaN.  Values: tokens
    128 and more ahead of it keep their bits, nearer ones take 0 times it; no
    log-sum-exp changes.  Other sequences, and other heads, never do."""
    rows, at, heads = 500, new - 3, slice(2, 4)  # of key head 1 of 2
    q, c, off, out, lse = run(cuda, [(new, rows), (new, 90 + new)], 4, 2, 64)
    again = lambda: (lambda o, l: (nh.paged_attention(q, c.k, c.v, off, c.lengths, c.table, out=o, lse=l,
                                                      max_queries=hint), l))(torch.empty_like(out),
                                                                             torch.empty_like(lse))
    out, lse = again()
    where = place(c, 0, rows - new + at)
    for pages, ahead in ((c.k, at), (c.v, max(at - 127, 0))):
        row = pages[where][1].clone()
        pages[where][1] = bad
        got, l2 = again()
        pages[where][1] = row
        assert torch.equal(got[new:], out[new:]) and torch.equal(l2[:, new:], lse[:, new:])
        assert torch.equal(got[:new, :2], out[:new, :2]) and torch.equal(l2[:2], lse[:2])
        assert torch.equal(got[:ahead], out[:ahead])
        seen = got[at:new, heads]
        if pages is c.k:
            assert torch.equal(l2[:, :at], lse[:, :at])
            # (An infinite score may be either infinity; -inf alone has weight 0.)
            assert torch.isnan(seen).all() if math.isnan(bad) else not torch.equal(seen, out[at:new, heads])
        else:
            assert torch.equal(l2, lse) and not torch.isfinite(seen).any()
    got, l2 = again()
    assert torch.equal(got, out) and torch.equal(l2, lse)


@pytest.mark.parametrize("count", [3, 40, 90])
def test_overlapping_offsets_of_single_tokens(cuda, count):
    """As for chunks: only the tokens' rows are written, a sequence alone with its token
    has its result, and a sound call after it the same bits as before."""
    q, c, off, out, _ = run(cuda, [(1, 3000)] + [(1, 2500)] * 2 + [(1, 20)] * (count - 3), 8, 2, 64)
    T = len(q)
    wide = torch.full((T + 9, 8, 64), 7.0, dtype=BF, device=cuda)
    bad = off.clone()
    bad[2] = 2 ** 31 - 1  # sequence 1 has all tokens from its first, sequence 2 none
    bad[3] = 1
    down = off.flip(0).contiguous()
    for o in (bad, down, off - 2, off + count // 2):
        for lens in (c.lengths - 10 ** 9, c.lengths + 10 ** 9, c.lengths):
            for hint in (1, 3):
                nh.paged_attention(q, c.k, c.v, o, lens, c.table, out=wide[:T], max_queries=hint)
                assert (wide[T:] == 7.0).all()
    nh.paged_attention(q, c.k, c.v, bad, c.lengths, c.table, out=wide[:T], max_queries=1)
    assert (wide[:1].double() - out[:1].double()).abs().max() <= 2.0 ** -6  # two roundings of values below 4
    assert torch.equal(nh.paged_attention(q, c.k, c.v, off, c.lengths, c.table, max_queries=1), out)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("seqs", [[(1, 1000)], [(1, 1500 + 211 * i) for i in range(32)],
                                  [(2048, 2048), (512, 4000), (37, 37), (1, 3000)],
                                  [(1, 700), (1, 5), (30, 90)] * 30])
def test_the_same_bits_every_time(cuda, seqs, dt):
    q, c, off, out, lse = run(cuda, seqs, 8, 2, 128, dt)
    for _ in range(5):
        o, l = torch.empty_like(out), torch.empty_like(lse)
        nh.paged_attention(q, c.k, c.v, off, c.lengths, c.table, out=o, lse=l, max_queries=max(n for n, _ in seqs))
        assert torch.equal(o, out) and torch.equal(l, lse)


@pytest.mark.parametrize("seed", [0, 1, 2])
def test_gradients_of_a_training_step_closely(cuda, seed):
    """Against autograd in 64 bits.  A rounding to bf16 is off by u = 2^-8 of a value at
    most, evenly up to that: u / sqrt 3 in the 2-norm.  The eight on the way (qkv, q and
    k, weights, out, weights and dS, dq and dk, again, the result) are independent, each
    with a gain of four at most (dP - delta is a difference of terms up to four times its
    size): sqrt(8) 4 u / sqrt 3 = 0.026 of a gradient."""
    st = training_state(cuda, seed)
    r = train(st)
    p = {n: st[n].double().requires_grad_() for n in ("w", "wq", "wk")}
    qkv = st["x"].double() @ p["w"] + st["b"].double()
    q, k, v = split(qkv)
    t = st["pos"].double()[:, None, None] * st["f"].double()

    def placed(x, w):
        y = torch.nn.functional.normalize(x, dim=-1, eps=0.0) * D ** 0.5  # (eps of the norm: 1e-6 of values of 1)
        a, b = (y * w).tensor_split(2, -1)
        z = torch.complex(a, b) * torch.polar(torch.ones_like(t), t)
        return torch.cat([z.real, z.imag], -1)

    q, k = placed(q, p["wq"]), placed(k, p["wk"])
    loss, a = 0.0, 0
    for n in LENS:
        later = torch.ones(n, n, dtype=torch.bool, device=cuda).triu(1)
        for h in range(H):
            s = torch.mm(q[a:a + n, h], k[a:a + n, h * G // H].t()) * D ** -0.5
            o = torch.mm(s.masked_fill(later, -INF).softmax(1), v[a:a + n, h * G // H])
            loss = loss + (o * st["do"][a:a + n, h].double()).sum()
        a += n
    want = torch.autograd.grad(loss, [*p.values(), qkv])
    for got, w in zip((r["dw"], r["dwq"], r["dwk"], r["dqkv"].view(len(qkv), -1)), want):
        rel = ((got.double() - w).norm() / w.norm()).item()
        assert rel <= 8 ** 0.5 * 4 * 2.0 ** -8 / 3 ** 0.5, (tuple(w.shape), rel)

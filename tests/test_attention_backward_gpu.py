"""attention_backward on the GPU against its formula in 64 bits, and against
differences of the forward.

Tolerances, u = finfo(dtype).eps / 2.  P and dS round once to dtype for the
products and each gradient once at the end: u times the sums of absolute
products, and u |result|.  f32 scores and dP are sums of exact products; scores
below 64 and D <= 128 keep P within 4e-5 of itself, dP and delta within 1e-5 of
their absolute sums.  In f16 a dS under 2^-14 rounds by 2^-25 at most."""
import math

import pytest
import torch

import nova_hip as nh
from test_attention_gpu import BF, F64, HF, make, offsets

pytestmark = pytest.mark.gpu


def reference(go, q, k, v, o, lse, qlens, klens, causal, scale):
    """(dq, dk, dv) and, for each, the bound of its error without u |result|."""
    H, G, dev = q.shape[1], k.shape[1], q.device
    u = torch.finfo(q.dtype).eps / 2
    tiny = 2.0 ** -25 if q.dtype == HF else 0.0
    res = [torch.zeros(t.shape, dtype=F64, device=dev) for t in (q, k, k)]
    tol = [torch.zeros_like(r) for r in res]
    a = c = 0
    for n, m in zip(qlens, klens):
        keep = torch.ones(n, m, dtype=torch.bool, device=dev)
        if causal:
            keep = keep.tril(m - n)
        for h in range(H if n and m else 0):
            g = h * G // H
            Q, GO, O = (t[a:a + n, h].double() for t in (q, go, o))
            K, V = k[c:c + m, g].double(), v[c:c + m, g].double()
            s = torch.mm(Q, K.t().contiguous()) * scale
            p = torch.where(keep, torch.exp(s - lse[h, a:a + n].double()[:, None]), torch.zeros_like(s))
            dp = torch.mm(GO, V.t().contiguous())
            ds = p * (dp - (GO * O).sum(1)[:, None])
            slack = p * (torch.mm(GO.abs(), V.t().abs().contiguous()) + (GO * O).abs().sum(1)[:, None])
            ds_err = (u * 1.01 + 4e-5) * ds.abs() + 1e-5 * slack + tiny * keep
            p_err = (u * 1.01 + 4e-5) * p + (tiny / 256) * keep
            sl, kl = slice(a, a + n), slice(c, c + m)
            res[0][sl, h] = torch.mm(ds, K) * scale
            tol[0][sl, h] = torch.mm(ds_err, K.abs()) * scale
            res[1][kl, g] += torch.mm(ds.t().contiguous(), Q) * scale
            tol[1][kl, g] += torch.mm(ds_err.t().contiguous(), Q.abs()) * scale
            res[2][kl, g] += torch.mm(p.t().contiguous(), GO)
            tol[2][kl, g] += torch.mm(p_err.t().contiguous(), GO.abs())
        a, c = a + n, c + m
    return res, tol


def run(dev, qlens, klens, H, G, D, dt, causal, layout="thd", seed=0, pad=0):
    q, k, v = make(dev, qlens, klens, H, G, D, dt, seed, layout, pad)
    g = torch.Generator(device=dev).manual_seed(seed + 1)
    go = torch.randn(q.shape, generator=g, device=dev).to(dt)
    Tq, Tk = sum(qlens), sum(klens)
    go[Tq:] = float("nan")
    if layout == "htd":
        go = go.transpose(0, 1).contiguous().transpose(0, 1)
    scale = D ** -0.5
    qo, ko = offsets(qlens, dev), offsets(klens, dev)
    o, lse = nh.attention(q, k, v, qo, ko, causal=causal)
    grads = [torch.full(t.shape, 7.0, dtype=dt, device=dev) for t in (q, k, v)]
    nh.attention_backward(go, q, k, v, o, lse, qo, ko, causal=causal, dq=grads[0], dk=grads[1],
                          dv=grads[2])
    want, tol = reference(go, q, k, v, o, lse, qlens, klens, causal, scale)
    u = torch.finfo(dt).eps / 2
    for name, got, w, t, T in zip(("dq", "dk", "dv"), grads, want, tol, (Tq, Tk, Tk)):
        assert (got[T:] == 7.0).all(), name  # rows behind the last sequence
        err = (got.double() - w).abs()[:T]
        assert not torch.isnan(err).any(), name
        bound = t[:T] * 1.01 + u * w[:T].abs() * 1.01 + 2.0 ** -25 * (dt == HF) + 1e-30
        worst = (err - bound).max().item() if err.numel() else 0.0
        assert worst <= 0, (name, worst, err.max().item(), qlens, klens, H, G, D, dt, causal, layout)
    return q, k, v, go, grads


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D", [8, 32, 40, 64, 80, 96, 128])
def test_head_dims(cuda, dt, causal, D):
    run(cuda, [197, 33], [197, 33], 4, 2, D, dt, causal)


@pytest.mark.parametrize("n", [1, 2, 31, 33, 63, 64, 65, 127, 129, 257, 600])
@pytest.mark.parametrize("causal", [False, True])
def test_lengths(cuda, n, causal):
    run(cuda, [n], [n], 2, 1, 64, BF, causal)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("qlens,klens", [
    ([5, 0, 130, 1], [77, 3, 130, 200]),
    ([40, 3, 0], [0, 70, 0]),
    ([200, 64], [70, 1]),
    ([1] * 70 + [65] + [0] * 70 + [2], [64] * 70 + [65] + [0] * 70 + [1]),
])
def test_uneven_and_empty_sequences(cuda, qlens, klens, D):
    for causal in (False, True):
        run(cuda, qlens, klens, 4, 2, D, BF, causal, pad=3)


@pytest.mark.parametrize("layout", ["thd", "htd", "fused"])
@pytest.mark.parametrize("H,G", [(1, 1), (8, 1), (9, 3), (32, 8)])
def test_layouts_and_shared_heads(cuda, layout, H, G):
    run(cuda, [150, 70, 3], [150, 70, 3], H, G, 64, HF, True, layout, pad=5 if layout != "fused" else 0)


def test_long_sequence(cuda):
    run(cuda, [2500], [4001], 2, 1, 128, BF, True)
    run(cuda, [4001], [4001], 1, 1, 64, HF, False)


def test_same_bits_on_every_run(cuda):
    first = run(cuda, [300, 200], [300, 200], 8, 2, 128, BF, True)[4]
    for _ in range(3):
        again = run(cuda, [300, 200], [300, 200], 8, 2, 128, BF, True)[4]
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_against_differences_of_the_forward(cuda):
    """d loss / d x along a random direction by central differences of the
    64-bit forward, loss = sum(out * grad_out).  The step's error is of order
    h^2; the gradients' own roundings, independent from element to element, give
    u |x'| |direction| each, within six standard deviations."""
    lens, H, G, D = [50, 21], 4, 2, 64
    q, k, v, go, grads = run(cuda, lens, lens, H, G, D, BF, True)

    def loss(q, k, v):
        total, a = 0.0, 0
        for n in lens:
            keep = torch.ones(n, n, dtype=torch.bool, device=cuda).tril()
            for h in range(H):
                s = torch.mm(q[a:a + n, h], k[a:a + n, h * G // H].t().contiguous()) * D ** -0.5
                p = torch.softmax(s.masked_fill(~keep, -math.inf), 1)
                total = total + (torch.mm(p, v[a:a + n, h * G // H]) * go[a:a + n, h].double()).sum()
            a += n
        return total

    x = [t.double() for t in (q, k, v)]
    gen = torch.Generator(device=cuda).manual_seed(9)
    for i in range(3):
        d = torch.randn(x[i].shape, generator=gen, device=cuda, dtype=F64)
        step = 1e-4
        hi, lo = list(x), list(x)
        hi[i], lo[i] = x[i] + step * d, x[i] - step * d
        numeric = ((loss(*hi) - loss(*lo)) / (2 * step)).item()
        ours = (grads[i].double() * d).sum().item()
        u = 2.0 ** -8
        # Rounded weights and dS: their sums err by at most the same again.
        noise = 6 * 2 * u * ((grads[i].double() * d) ** 2).sum().sqrt().item() + 6 * u * d.norm().item()
        assert abs(ours - numeric) <= noise + 1e-6 * abs(numeric), (i, ours, numeric, noise)


@pytest.mark.parametrize("B", [64, 65, 200])
def test_many_sequences(cuda, B):
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, 4, (B,), generator=g).tolist()
    for i, n in ((0, 150), (B // 2, 130), (B - 1, 129)):
        lens[i] = n
    run(cuda, lens, lens, 4, 2, 64, BF, True, pad=2)


def test_split_runs_of_queries(cuda):
    """Few tiles of keys under many queries are split into runs whose sums are
    joined: head groups, ragged and empty ends among them."""
    assert nh.lib().nova_hip_attention_backward_scratch(1500, 700, 2, 4, 1, 64, 1) > 2 * 4 * 1500
    run(cuda, [1300, 200], [500, 200], 4, 1, 64, BF, True, pad=1)
    run(cuda, [1300, 200], [500, 200], 4, 1, 128, HF, False)
    run(cuda, [1100], [1100], 2, 2, 128, BF, True)


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
def test_keys_shared_by_two_groups_of_waves(cuda, dt, D):
    """Few tiles of long sequences: two groups of waves take a tile's keys in
    turn.  Odd and even numbers of tiles, one tile alone, none at all."""
    run(cuda, [700, 65, 1, 200], [2600, 64, 0, 129], 2, 1, D, dt, True)
    run(cuda, [33, 90], [1281, 1], 4, 2, D, dt, False, pad=1)


def test_many_runs_of_queries(cuda):
    """Eight runs to a tile of keys, some of them of masked tiles alone, and a
    sequence with fewer tiles of queries than runs."""
    need = nh.lib().nova_hip_attention_backward_scratch(2100, 300, 2, 8, 1, 128, 1)
    assert need >= 2 * 8 * 2100 + 4 * 8 * 4 * 64 * 128
    run(cuda, [2000, 100], [200, 100], 8, 1, 128, BF, True)
    run(cuda, [2000, 3], [200, 100], 8, 1, 64, HF, True)


@pytest.mark.parametrize("D", [64, 128])
def test_runs_of_the_long_sequences_alone(cuda, D):
    """Batches whose long sequences' tiles are split and whose short ones' are
    not, with empty sequences and more queries than keys among them."""
    lens = [3, 2500, 0, 70, 129, 1]
    run(cuda, lens, lens, 6, 2, D, BF, True, pad=2)
    run(cuda, [2600, 64, 1], [200, 64, 30], 4, 1, D, HF, True)
    run(cuda, [2600, 64, 1], [200, 64, 30], 4, 1, D, BF, False)
    lens = [1300] + [40] * 30 + [900] + [33] * 40  # beyond 64 sequences
    run(cuda, lens, lens, 8, 1, D, BF, True)


def test_two_runs_last_ones_first(cuda):
    """More tiles of keys than the chip takes at once."""
    H, lens = 16, [3300, 40, 65, 700]
    need = nh.lib().nova_hip_attention_backward_scratch(sum(lens), sum(lens), len(lens), H, H, 128, 1)
    tiles = sum(lens) // 128 + len(lens)
    assert need >= 2 * H * sum(lens) + 2 * H * tiles * 4 * 64 * 128
    run(cuda, lens, lens, H, H, 128, BF, True)


def test_runs_in_a_captured_graph(cuda):
    """Split and joined runs replayed with new inputs, eager calls of other
    shapes between the replays: the same bits as eager calls."""
    lens, H, G, D = [2000, 300, 5], 4, 1, 128
    q, k, v = make(cuda, lens, lens, H, G, D, BF, 0, "thd", 0)
    off = offsets(lens, cuda)
    go = torch.randn(q.shape, device=cuda).to(BF)
    o, lse = nh.attention(q, k, v, off, off)
    dq, dk, dv = (torch.empty_like(t) for t in (q, k, v))
    nh.attention_backward(go, q, k, v, o, lse, off, off, dq=dq, dk=dk, dv=dv)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        nh.attention(q, k, v, off, off, out=o, lse=lse)
        nh.attention_backward(go, q, k, v, o, lse, off, off, dq=dq, dk=dk, dv=dv)
    gen = torch.Generator(device=cuda).manual_seed(3)
    for _ in range(4):
        for t in (q, k, v, go):
            t.copy_(torch.randn(t.shape, generator=gen, device=cuda))
        for t in (dq, dk, dv):
            t.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        run(cuda, [130, 70], [130, 70], 8, 1, 64, BF, True)
        o2, lse2 = nh.attention(q, k, v, off, off)
        want = nh.attention_backward(go, q, k, v, o2, lse2, off, off)
        assert all(torch.equal(a, b) for a, b in zip((dq, dk, dv), want))


def scaled(dev, qlens, klens, H, G, D, dt, causal, grad, q_up=1.0, k_up=1.0, v_up=1.0, rows=None):
    """(grads, reference, bounds) with grad_out of size `grad` and q, k, v of the
    given sizes (their products kept where scores are of size 1).  dS rounds by u
    of itself and in f16, where a column of the product with it (a query's row for
    dQ, a key's for dK) has a factor that keeps its largest value above 2^5, by
    2^-25 of 2^-5 of that."""
    q, k, v = make(dev, qlens, klens, H, G, D, dt)
    q, k, v = ((x.float() * up).to(dt) for x, up in ((q, q_up), (k, k_up), (v, v_up)))
    g = torch.Generator(device=dev).manual_seed(5)
    go = torch.randn(q.shape, generator=g, device=dev) * grad
    if rows is not None:
        go *= rows[:, None, None]
    go = go.to(dt)
    scale = D ** -0.5 / (q_up * k_up)
    qo, ko = offsets(qlens, dev), offsets(klens, dev)
    o, lse = nh.attention(q, k, v, qo, ko, causal=causal, scale=scale)
    got = nh.attention_backward(go, q, k, v, o, lse, qo, ko, causal=causal, scale=scale)
    u = torch.finfo(dt).eps / 2
    want = [torch.zeros(t.shape, dtype=F64, device=dev) for t in (q, k, k)]
    tol = [torch.zeros_like(w) for w in want]
    a = c = 0
    for n, m in zip(qlens, klens):
        keep = torch.ones(n, m, dtype=torch.bool, device=dev)
        if causal:
            keep = keep.tril(m - n)
        sl, kl = slice(a, a + n), slice(c, c + m)
        for j in range(G):
            K, V = k[c:c + m, j].double(), v[c:c + m, j].double()
            heads = []
            for h in range(j * H // G, (j + 1) * H // G):
                Q, GO, O = (t[a:a + n, h].double() for t in (q, go, o))
                s = torch.mm(Q, K.t().contiguous()) * scale
                p = torch.where(keep, torch.exp(s - lse[h, a:a + n].double()[:, None]), torch.zeros_like(s))
                delta = (GO * O).sum(1)[:, None]
                ds = p * (torch.mm(GO, V.t().contiguous()) - delta)
                slack = p * (torch.mm(GO.abs(), V.t().abs().contiguous()) + (GO * O).abs().sum(1)[:, None])
                heads.append((h, Q, GO, p, ds, (u * 1.01 + 4e-5) * ds.abs() + 1e-5 * slack,
                              2.0 ** -30 * (ds.abs() + 1e-5 * slack) * (dt == HF)))
            # A key's factor is common to the heads of its group.
            least = torch.stack([x[6].amax(0, keepdim=True) for x in heads]).amax(0)
            for h, Q, GO, p, ds, err, tiny in heads:
                row, col = err + tiny.amax(1, keepdim=True) * keep, err + least * keep
                want[0][sl, h] = torch.mm(ds, K) * scale
                tol[0][sl, h] = torch.mm(row, K.abs()) * scale
                want[1][kl, j] += torch.mm(ds.t().contiguous(), Q) * scale
                tol[1][kl, j] += torch.mm(col.t().contiguous(), Q.abs()) * scale
                want[2][kl, j] += torch.mm(p.t().contiguous(), GO)
                tol[2][kl, j] += torch.mm(((u * 1.01 + 4e-5) * p + 2.0 ** -33 * keep * (dt == HF)).t().contiguous(),
                                          GO.abs())
        a, c = a + n, c + m
    for name, x, w, t in zip(("dq", "dk", "dv"), got, want, tol):
        bound = t * 1.01 + u * w.abs() * 1.01 + 2.0 ** -25 * (dt == HF) + 1e-30
        # Beyond the type's largest value there is no bound to hold.
        fits = w.abs() + t < 0.99 * torch.finfo(dt).max
        err = (x.double() - w).abs()
        assert (err <= bound)[fits].all(), (name, (err - bound)[fits].max().item(), w.abs().max().item())
        assert torch.isfinite(x[fits]).all(), name
    return got, want


@pytest.mark.parametrize("D", [64, 80, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dt", [BF, HF])
def test_small_gradients(cuda, dt, causal, D):
    """grad_out as a mean over thousands of tokens leaves it: dS lies under f16's
    least number where dQ and dK, products with large K and Q, do not."""
    for grad in (2.0 ** -10, 2.0 ** -16, 2.0 ** -20):
        got, want = scaled(cuda, [700, 130], [700, 130], 4, 2, D, dt, causal, grad, k_up=64.0, q_up=1 / 64)
        assert want[0].abs().max() > 2.0 ** -17
        got, want = scaled(cuda, [700, 130], [700, 130], 4, 2, D, dt, causal, grad, q_up=64.0, k_up=1 / 64)
        assert want[1].abs().max() > 2.0 ** -17


@pytest.mark.parametrize("D", [64, 128])
def test_large_gradients(cuda, D):
    """grad_out and values whose dS passes f16's largest number (a loss scale) where
    dQ (small K) or dK (small Q) does not."""
    for i, up in ((0, 64.0), (1, 1 / 64)):
        got, want = scaled(cuda, [300, 40], [300, 40], 4, 2, D, HF, True, 256.0, v_up=256.0, q_up=up, k_up=1 / up)
        assert 100.0 < want[i].abs().max() < 60000.0


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("shape", [([900], [900]), ([1300, 200], [500, 200]), ([700, 65], [2600, 64])])
def test_gradients_of_rows_of_all_sizes(cuda, shape, D):
    """Rows of grad_out from 2^-20 to 2^4, the small ones first, last and in turn:
    the factors of keys fall on the way, in runs of queries and in two groups of
    waves as well."""
    n = sum(shape[0])
    for rows in (torch.linspace(-20, 4, n), torch.linspace(4, -20, n),
                 torch.where(torch.arange(n) % 97 == 0, 4.0, -20.0)):
        scaled(cuda, *shape, 4, 1, D, HF, True, 1.0, k_up=8.0, q_up=1 / 8, rows=(2.0 ** rows).to(cuda))


def runs_scratch(lens, H, G, D, causal=True):
    """Floats of scratch beyond the rows' constants, over those of one run of all
    tiles of keys: the most runs a tile may have."""
    T = sum(lens)
    need = nh.lib().nova_hip_attention_backward_scratch(T, T, len(lens), H, G, D, causal)
    tiles = (T // 128 + len(lens)) * G
    return tiles, (need - (2 * H * T + 63) // 64 * 64) // (tiles * 4 * 64 * D)


@pytest.mark.parametrize("D,H,G,lens", [
    (128, 12, 12, [2500, 597]),  # every tile halved: just more than 256 tiles ...
    (128, 26, 13, [2400, 130]),  # (heads in groups)
    (64, 24, 24, [2500, 597]),   # ... or 512 at D <= 64
    (64, 32, 32, [3300, 40, 65, 700]),    # two runs of the long tiles, the last ones first
    (128, 16, 16, [4200, 40, 65, 700]),
])
def test_more_tiles_than_the_chip_takes_at_once(cuda, D, H, G, lens):
    tiles, most = runs_scratch(lens, H, G, D)
    slots = 512 if D <= 64 else 256
    assert most == 2 and slots <= tiles < 4 * slots, (tiles, most)
    assert (2 * tiles < 3 * slots) == (lens[0] in (2400, 2500)), tiles
    run(cuda, lens, lens, H, G, D, BF, True, pad=1)


@pytest.mark.parametrize("D,H,lens", [(64, 6, [1024] * 8), (64, 6, [2048] * 4), (128, 3, [1024] * 8)])
@pytest.mark.parametrize("causal", [True, False])
def test_equal_sequences(cuda, D, H, lens, causal):
    """Batches that may be split by their tokens, of which the device splits few
    tiles or none."""
    assert runs_scratch(lens, H, H, D, causal)[1] > 1
    run(cuda, lens, lens, H, H, D, HF, causal)

"""Attention of packed sequences on the GPU against its definition in 64 bits.

Tolerances, with u = finfo(dtype).eps / 2 and A = sum_j p_j |v_j| for an output
row: the weights round once to dtype (u A, and in f16 2^-25 per weight below
2^-14, as the largest is at least 1), the result once (u |o|).  Scores are f32
sums of exact products; with D <= 128 unit-normal values they are off by less
than 1e-5, which moves a weight by that much of itself: 4e-5 A covers them, the
exponential, the sum and the division."""
import math

import pytest
import torch

import nova_hip as nh

pytestmark = pytest.mark.gpu
F64 = torch.float64
BF, HF = torch.bfloat16, torch.float16


def offsets(lens, dev, first=0):
    o = [first]
    for n in lens:
        o.append(o[-1] + n)
    return torch.tensor(o, dtype=torch.int32, device=dev)


def make(dev, qlens, klens, H, G, D, dt, seed=0, layout="thd", pad=0):
    """q, k, v: packed rows, `pad` rows of NaN behind the last sequence."""
    g = torch.Generator(device=dev).manual_seed(seed)
    Tq, Tk = sum(qlens), sum(klens)

    def one(T, heads):
        x = torch.randn(T + pad, heads, D, generator=g, device=dev).to(dt)
        if pad:
            x[T:] = float("nan")
        if layout == "htd":
            x = x.transpose(0, 1).contiguous().transpose(0, 1)
        return x

    if layout == "fused":
        qkv = torch.randn(Tq + pad, H + 2 * G, D, generator=g, device=dev).to(dt)
        if pad:
            qkv[Tq:] = float("nan")
        return qkv[:, :H], qkv[:, H:H + G], qkv[:, H + G:]
    return one(Tq, H), one(Tk, G), one(Tk, G)


def reference(q, k, v, qlens, klens, causal, scale):
    """out, lse, sum p|v|, sum of visible |v|, all [.., heads] in 64 bits."""
    Tq, H, D = q.shape
    G = k.shape[1]
    dev = q.device
    out = torch.zeros(Tq, H, D, dtype=F64, device=dev)
    amp, vis = torch.zeros_like(out), torch.zeros_like(out)
    lse = torch.full((H, Tq), -math.inf, dtype=F64, device=dev)
    a = c = 0
    for n, m in zip(qlens, klens):
        keep = torch.ones(n, m, dtype=torch.bool, device=dev)
        if causal:
            keep = keep.tril(m - n)
        some = keep.any(1)
        for h in range(H):
            kh, vh = k[c:c + m, h * G // H].double(), v[c:c + m, h * G // H].double()
            s = (torch.mm(q[a:a + n, h].double(), kh.t().contiguous()) * scale).masked_fill(~keep, -math.inf)
            p = torch.where(some[:, None], torch.softmax(s, 1), torch.zeros_like(s)) if m else s
            # A masked weight takes no part, whatever stands in v.
            clean = torch.nan_to_num(vh, 0.0, 0.0, 0.0)
            out[a:a + n, h] = torch.mm(p, clean)
            amp[a:a + n, h] = torch.mm(p, clean.abs())
            vis[a:a + n, h] = torch.mm(keep.double(), clean.abs())
            lse[h, a:a + n] = torch.logsumexp(s, 1) if m else -math.inf
        a, c = a + n, c + m
    return out, lse, amp, vis


def check(out, lse, q, k, v, qlens, klens, causal, scale, what=""):
    want, wlse, amp, vis = reference(q, k, v, qlens, klens, causal, scale)
    T = sum(qlens)
    u = torch.finfo(q.dtype).eps / 2
    tol = u * (amp + want.abs()) * 1.01 + 4e-5 * amp + (2.0 ** -25 * vis if q.dtype == HF else 0.0)
    tol = tol + torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps  # subnormal results
    err = (out.double() - want).abs()[:T]
    assert not torch.isnan(err).any(), what
    worst = (err - tol[:T]).max().item() if err.numel() else 0.0
    assert worst <= 0, (what, worst, err.max().item())
    if lse is not None:
        empty = torch.isinf(wlse[:, :T])
        assert torch.equal(torch.isinf(lse[:, :T]), empty), what
        d = (lse[:, :T].double() - wlse[:, :T]).masked_fill(empty, 0.0).abs()
        assert d.numel() == 0 or d.max().item() <= 4e-5, (what, d.max().item())


def run(dev, qlens, klens, H, G, D, dt, causal, layout="thd", seed=0, scale=None, pad=0):
    q, k, v = make(dev, qlens, klens, H, G, D, dt, seed, layout, pad)
    scale = D ** -0.5 if scale is None else scale
    out = torch.full(q.shape, 7.0, dtype=dt, device=dev)
    lse = torch.full((H, q.shape[0]), 7.0, device=dev)
    nh.attention(q, k, v, offsets(qlens, dev), offsets(klens, dev), causal=causal, scale=scale,
                 out=out, lse=lse)
    T = sum(qlens)
    assert (out[T:] == 7.0).all() and (lse[:, T:] == 7.0).all()  # rows behind the last sequence
    check(out, lse, q, k, v, qlens, klens, causal, scale, (qlens, klens, H, G, D, dt, causal, layout))
    return out


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("D", [8, 32, 40, 64, 80, 96, 120, 128])
def test_head_dims(cuda, dt, causal, D):
    run(cuda, [197, 33], [197, 33], 4, 2, D, dt, causal)


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 1000])
@pytest.mark.parametrize("causal", [False, True])
def test_lengths(cuda, n, causal):
    run(cuda, [n], [n], 2, 1, 64, BF, causal)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("qlens,klens", [
    ([5, 0, 130, 1], [77, 3, 130, 200]),    # more keys than queries, an empty query part
    ([40, 3, 0], [0, 70, 0]),               # no keys; nothing at all
    ([200, 64], [70, 1]),                   # causal: the first queries see no key
    ([1] * 70 + [65] + [0] * 70 + [2], [64] * 70 + [65] + [0] * 70 + [1]),
])
def test_uneven_and_empty_sequences(cuda, qlens, klens, D):
    for causal in (False, True):
        run(cuda, qlens, klens, 4, 2, D, BF, causal, pad=3)


@pytest.mark.parametrize("layout", ["thd", "htd", "fused"])
@pytest.mark.parametrize("H,G", [(1, 1), (8, 1), (6, 6), (9, 3), (32, 8)])
def test_layouts_and_shared_heads(cuda, layout, H, G):
    run(cuda, [150, 70, 3], [150, 70, 3], H, G, 64, HF, True, layout, pad=5 if layout != "fused" else 0)


@pytest.mark.parametrize("scale", [1e-3, 0.125, 1.0])
def test_scales(cuda, scale):
    # Scores of scale 1 reach +-40: the running maximum moves and the sums are
    # rescaled.  |s| <= 64 carries 64 * 128 * 2^-24 of rounding at most, but the
    # f32 sum's is far below its bound; 4e-5 still holds as 2^-24 * 64 * 8.
    run(cuda, [300], [300], 2, 2, 64, BF, True, scale=scale)


def test_growing_scores_move_the_maximum(cuda):
    """Keys ordered so that each tile's scores are far above the last one's."""
    n, D = 512, 64
    q = torch.ones(n, 1, D, device=cuda, dtype=BF)
    k = (torch.arange(n, device=cuda)[:, None, None] / 8.0 * torch.ones(1, 1, D, device=cuda)).to(BF)
    v = torch.randn(n, 1, D, device=cuda).to(BF)
    for flip in (False, True):
        kk = k.flip(0).contiguous() if flip else k
        out, lse = nh.attention(q, kk, v, offsets([n], cuda), offsets([n], cuda), causal=False,
                                scale=0.125)
        # Scores are exact multiples of 1/8 up to 2^9; lse rounds at 2^-15 there.
        want, wlse, amp, _ = reference(q, kk, v, [n], [n], False, 0.125)
        u = 2.0 ** -8
        assert ((out.double() - want).abs() <= u * (amp + want.abs()) * 1.01 + 4e-4 * amp).all()
        assert ((lse.double() - wlse).abs() <= 2.0 ** -13).all()


def test_rows_of_other_sequences_do_not_leak(cuda):
    """A sequence between two that hold NaN and infinity."""
    lens = [37, 70, 50]
    q, k, v = make(cuda, lens, lens, 2, 2, 64, BF)
    for t in (q, k, v):
        t[:37] = float("nan")
        t[107:] = float("inf")
    out, lse = nh.attention(q, k, v, offsets(lens, cuda), offsets(lens, cuda), causal=False)
    sl = slice(37, 107)
    check(out[sl], lse[:, sl], q[sl], k[sl], v[sl], [70], [70], False, 0.125)


def test_long_sequence(cuda):
    run(cuda, [2500], [4001], 2, 1, 128, BF, True)


@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_keys_shared_by_two_groups_of_waves(cuda, D, causal):
    """Few tiles of queries over long keys: odd numbers of tiles of keys, rows
    that see none, sequences without any."""
    run(cuda, [1000, 0, 70, 5], [1500, 700, 3, 1], 2, 1, D, HF, causal, pad=1)
    run(cuda, [900], [577], 3, 3, D, BF, causal)


def test_long_sequences_of_many_heads(cuda):
    run(cuda, [700, 600], [700, 600], 64, 8, 64, BF, True, "fused")
    run(cuda, [700, 600], [700, 600], 64, 64, 128, BF, False)


def test_no_keys_or_no_queries_at_all(cuda):
    for qlens, klens in (([5, 3], [0, 0]), ([0, 0], [4, 70])):
        q, k, v = make(cuda, qlens, klens, 2, 1, 64, BF)
        qo, ko = offsets(qlens, cuda), offsets(klens, cuda)
        out, lse = nh.attention(q, k, v, qo, ko)
        assert (out == 0).all() and torch.isinf(lse).all()
        dq, dk, dv = nh.attention_backward(q, q, k, v, out, lse, qo, ko)
        assert all((t == 0).all() for t in (dq, dk, dv))
        assert dq.shape == q.shape and dk.shape == k.shape


def test_strides_far_apart(cuda):
    """Rows 2^22 elements apart (8 MB), the largest stride's half: offsets inside
    a tile of 64 or 128 rows stay in range; heads past 2^32 bytes."""
    n, D, step = 130, 64, 1 << 22
    flat = torch.empty(n * step + (1 << 31) + 4096, dtype=BF, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(1)

    def view(T, heads):
        x = flat.as_strided((T, heads, D), (step, (1 << 31) // 2 + 64, 1))
        for h in range(heads):
            x[:, h] = torch.randn(T, D, generator=g, device=cuda).to(BF)
        return x

    k = view(n, 2)
    q = torch.randn(n, 2, D, generator=g, device=cuda).to(BF)
    off = offsets([n], cuda)
    out, lse = nh.attention(q, k, k, off, off)
    check(out, lse, q, k, k, [n], [n], True, 0.125)
    a = nh.attention_backward(q, q, k, k, out, lse, off, off)
    kc = k.contiguous()
    b = nh.attention_backward(q, q, kc, kc, out, lse, off, off)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("B", [63, 64, 65, 128, 200, 4100])
def test_many_sequences(cuda, B):
    """Around the 64 sequences that are searched in registers, and far beyond:
    lengths 0 to 3 and a few long ones, first, last and in the middle."""
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, 4, (B,), generator=g).tolist()
    for i, n in ((0, 150), (B // 2, 130), (B - 1, 129)):
        lens[i] = n
    if B < 1000:
        for causal in (False, True):
            run(cuda, lens, lens, 2, 1, 64, BF, causal, pad=2)
        return
    # The reference takes a loop turn per sequence: whole sequences of one batch
    # against the same ones alone.
    q, k, v = make(cuda, lens, lens, 2, 1, 64, BF)
    out, lse = nh.attention(q, k, v, offsets(lens, cuda), offsets(lens, cuda))
    start = [0]
    for n in lens:
        start.append(start[-1] + n)
    for i in (0, 1, 2, 63, 64, 65, B // 2, B - 2, B - 1):
        sl = slice(start[i], start[i + 1])
        check(out[sl], lse[:, sl], q[sl], k[sl], v[sl], [lens[i]], [lens[i]], True, 0.125, i)
    one = offsets([1] * B, cuda)
    q1, k1, v1 = make(cuda, [1] * B, [1] * B, 2, 1, 64, BF)
    out, _ = nh.attention(q1, k1, v1, one, one)  # a row that sees itself alone is its value
    assert torch.equal(out, v1.expand(B, 2, 64))


@pytest.mark.parametrize("bad", [[5, 2 ** 31 - 1, -7, 40], [-9, 20, 10, 10 ** 9], [60, 0, 60, 0],
                                 [0] + [60, 0] * 40])
def test_offsets_outside_the_operands(cuda, bad):
    """Sequences are cut to the operands' rows: nothing else is read or written."""
    H, G, D, T = 2, 1, 64, 60
    guard = 64
    q = torch.randn(T + 2 * guard, H, D, device=cuda).to(BF)
    kv = torch.randn(T + 2 * guard, G, D, device=cuda).to(BF)
    out = torch.full_like(q, 7.0)
    off = torch.tensor(bad, dtype=torch.int32, device=cuda)
    mid = slice(guard, guard + T)
    lse = torch.full((H, T), 7.0, device=cuda)
    nh.attention(q[mid], kv[mid], kv[mid], off, off, out=out[mid], lse=lse)
    d = [torch.full_like(t, 7.0) for t in (q, kv, kv)]
    nh.attention_backward(q[mid], q[mid], kv[mid], kv[mid], out[mid], lse, off, off, dq=d[0][mid],
                          dk=d[1][mid], dv=d[2][mid])
    torch.cuda.synchronize()
    for t in [out] + d:
        assert (t[:guard] == 7.0).all() and (t[guard + T:] == 7.0).all()


@pytest.mark.parametrize("form", ["prompt", "causal", "two groups", "single token", "long cache"])
@pytest.mark.parametrize("dt", [BF, HF])
def test_many_small_weights_behind_a_large_one(cuda, dt, form):
    """One key's score 17.5 above those of n - 1 others, whose weights of e^-17.5 =
    2^-25.2 lie under half of f16's least number and whose values alone differ from
    zero.  A weight rounds by u of itself or, in f16, by 2^-32 at most (n - 1
    times), the result by u; scores are exact and exponentials within 4e-5.  A row's
    sum is added up by two lanes, n / 2 f32 additions each (long cache: in parts of
    at most 2048 keys): 2^-25 of it for each of n, here SUM."""
    SUM = 2.0 ** -25 * 4096
    n = 70000 if form == "long cache" else 1000 if form == "single token" else 4095
    D, rows = 64, 1 if form in ("single token", "long cache") else 300 if form == "two groups" else 3000
    heads = 2 if form == "two groups" else 32  # few tiles: two groups of waves share the keys
    q = torch.zeros(rows, heads, D, dtype=dt, device=cuda)
    q[:, :, 0] = 17.5
    k = torch.zeros(n, 1, D, dtype=dt, device=cuda)
    v = torch.full((n, 1, D), 1000.0, dtype=dt, device=cuda)
    k[7, 0, 0], v[7] = 1.0, 0.0
    if rows == 1:
        lse = torch.empty(1, heads, device=cuda)
        out = nh.attention_decode(q, k[None], v[None], torch.tensor([n], dtype=torch.int32, device=cuda),
                                  scale=1.0, lse=lse)
        lse = lse.t()
    else:
        out, lse = nh.attention(q, k, v, offsets([rows], cuda), offsets([n], cuda), scale=1.0,
                                causal=form == "causal")
    # Causal: query i sees n - rows + i + 1 keys, the seventh among them.
    seen = torch.full((rows,), float(n), dtype=F64, device=cuda)
    if form == "causal":
        seen = torch.arange(n - rows + 1, n + 1, device=cuda, dtype=F64)
    w = math.exp(-17.5)
    total = 1.0 + (seen - 1) * w
    want = 1000.0 * (seen - 1) * w / total
    u = torch.finfo(dt).eps / 2
    tol = 2 * u * want * 1.01 + (4e-5 + SUM) * want + (1000.0 * 2.0 ** -32 * (seen - 1) if dt == HF else 0.0)
    err = (out.double() - want[:, None, None]).abs()
    assert (err <= tol[:, None, None]).all(), (err.max().item(), want.max().item(), tol.max().item())
    d = (lse.double() - (17.5 + torch.log(total))[None]).abs().max().item()
    assert d <= 4e-5 + SUM, d

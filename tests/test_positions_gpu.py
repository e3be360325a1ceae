"""Rotary positions and the norm of query and key heads, with its backward pass,
against their formulas in 64 bits.

Tolerances, u = finfo(dtype).eps / 2 for the one rounding of a result.  In f32: a
sine or cosine is off by two units of its last place, 2^-23, the two products and
their sum by 3 2^-24 of |a| + |b|: 2^-21 (|a| + |b|) covers a rotated value.  The
norm's sum of up to 256 squares, taken in 32 terms per lane and a tree of five, is
off by 37 2^-24 of itself and half as much through the root, the root by two units,
the products by three: 2^-19 with the rotation.  Backward, the two sums and the
difference: 2^-18 of r (|t| + |x| r^2 mean |t x|).  A weight's gradient sums its
rows in at most 300 steps: 2^-15 of sum |g x r|."""
import pytest
import torch

import nova_hip as nh

pytestmark = pytest.mark.gpu
F64, F32, BF, HF = torch.float64, torch.float32, torch.bfloat16, torch.float16
DTYPES = [F32, BF, HF]


def freqs_of(R, dev, base=10000.0):
    return (base ** (-torch.arange(0, R, 2, dtype=F64) / max(R, 1))).float().to(dev)


def pairs(x, R, interleaved):
    if interleaved:
        return x[..., 0:R:2], x[..., 1:R:2]
    return x[..., :R // 2], x[..., R // 2:R]


def turned(x, pos, freqs, interleaved, scale=1.0, inverse=False):
    """(rotated, |a| + |b| of each value) in 64 bits."""
    R = 2 * len(freqs)
    y, amp = x.clone(), x.abs()
    t = pos.double()[:, None, None] * freqs.double() * (-1.0 if inverse else 1.0)
    a, b = (v.clone() for v in pairs(x, R, interleaved))
    ya, yb = pairs(y, R, interleaved)
    ya.copy_(scale * (a * t.cos() - b * t.sin()))
    yb.copy_(scale * (b * t.cos() + a * t.sin()))
    for v in pairs(amp, R, interleaved):
        v.copy_(abs(scale) * (a.abs() + b.abs()))
    return y, amp


def near(got, want, amp, rel, what=""):
    f = torch.finfo(got.dtype)
    tol = f.eps / 2 * want.abs() * 1.01 + rel * amp * 1.01 + f.smallest_normal * f.eps
    err = (got.double() - want).abs()
    assert not torch.isnan(err).any(), what
    assert err.numel() == 0 or (err - tol).max().item() <= 0, (what, (err - tol).max().item(), err.max().item())


def make(dev, T, H, D, dt, seed=0, layout="thd"):
    g = torch.Generator(device=dev).manual_seed(seed)
    if layout == "fused":
        return torch.randn(T, H + 5, D, generator=g, device=dev).to(dt)[:, 2:2 + H]
    if layout == "htd":
        return torch.randn(H, T, D, generator=g, device=dev).to(dt).transpose(0, 1)
    return torch.randn(T, H, D, generator=g, device=dev).to(dt)


def places(dev, T, seed=0, far=100000):
    g = torch.Generator(device=dev).manual_seed(seed + 77)
    return torch.randint(-far, far, (T,), generator=g, device=dev, dtype=torch.int32)


# D, rotated values: whole heads, parts, halves that are no multiple of 8, none.
SHAPES = [(8, 8), (8, 0), (16, 8), (32, 32), (40, 40), (64, 16), (80, 32), (80, 80), (96, 48), (104, 24),
          (120, 104), (128, 128), (128, 8), (192, 64), (256, 256), (256, 8), (248, 248)]


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("D,R", SHAPES)
def test_rotary(cuda, D, R, dt, interleaved):
    T, H = 37, 5
    x, pos, f = make(cuda, T, H, D, dt), places(cuda, T), freqs_of(R, cuda)
    for inverse, scale in ((False, 1.0), (True, 0.75)):
        want, amp = turned(x.double(), pos, f, interleaved, scale, inverse)
        y = nh.rotary(x, pos, f, interleaved=interleaved, inverse=inverse, scale=scale)
        near(y, want, amp, 2.0 ** -21, (D, R, dt, interleaved, inverse))
        assert torch.equal(y[..., R:], x[..., R:])  # what is not rotated keeps its bits


@pytest.mark.parametrize("layout", ["thd", "fused", "htd"])
@pytest.mark.parametrize("T,H", [(1, 1), (1, 71), (3, 300), (1023, 2), (1024, 1), (2049, 3), (9001, 2), (5000, 7)])
def test_rotary_sizes_and_layouts(cuda, T, H, layout):
    x, pos, f = make(cuda, T, H, 64, BF, T, layout), places(cuda, T, T), freqs_of(64, cuda)
    want, amp = turned(x.double(), pos, f, False)
    near(nh.rotary(x, pos, f), want, amp, 2.0 ** -21)
    out = make(cuda, T, H, 64, BF, 1, layout)
    nh.rotary(x, pos, f, out=out)
    near(out, want, amp, 2.0 ** -21)
    nh.rotary(x, pos, f, out=x)  # in place
    assert torch.equal(x, out)


def test_rotary_far_positions_and_what_stays(cuda):
    """Positions up to the ends of i32; infinities and NaN outside the rotated
    values stay where they are, others reach their own pair alone."""
    ends = [0, 1, -1, 2 ** 31 - 1, -2 ** 31, 16777217, 1 << 20, 99999999]
    pos = torch.tensor(ends, dtype=torch.int32, device=cuda)
    f = torch.tensor([1.0, 0.731, 2.5, 1e-4], device=cuda)
    x = make(cuda, len(ends), 3, 16, F32)
    for inter in (False, True):
        want, amp = turned(x.double(), pos, f, inter)
        # 2^31 turns' product with 1 / 2 pi is off by 2^-52 of itself: 2^-21 of an angle.
        near(nh.rotary(x, pos, f, interleaved=inter), want, amp, 2.0 ** -20)
    y = x.clone()
    y[2, 1, 9], y[2, 1, 12], y[3, 0, 5] = float("inf"), float("nan"), float("nan")
    got, want = nh.rotary(y, pos, f), nh.rotary(x, pos, f)
    bad = torch.isnan(got) | torch.isinf(got)
    expect = torch.zeros_like(bad)
    expect[2, 1, 9] = expect[2, 1, 12] = expect[3, 0, 5] = expect[3, 0, 1] = True
    assert torch.equal(bad, expect) and torch.equal(got[~bad], want[~bad])


def test_rotary_strides_past_32_bits(cuda):
    far = (1 << 31) + 1024  # elements between two heads
    flat = torch.empty(far + 4096, dtype=BF, device=cuda)
    x = flat.as_strided((9, 2, 64), (64, far, 1))
    x.copy_(make(cuda, 9, 2, 64, BF))
    pos, f = places(cuda, 9), freqs_of(64, cuda)
    want = nh.rotary(x.contiguous(), pos, f)
    assert torch.equal(nh.rotary(x, pos, f, out=x), want)


def test_rotary_empty(cuda):
    f = freqs_of(64, cuda)
    none = torch.empty(0, dtype=torch.int32, device=cuda)
    assert nh.rotary(make(cuda, 0, 3, 64, BF), none, f).shape == (0, 3, 64)
    assert nh.rotary(make(cuda, 4, 0, 64, BF), places(cuda, 4), f).shape == (4, 0, 64)


@pytest.mark.parametrize("dim,base,factor,original,low,high", [
    (128, 10000.0, 1.0, 0, 1.0, 32.0), (64, 500000.0, 8.0, 8192, 1.0, 4.0), (80, 10000.0, 4.0, 0, 1.0, 32.0),
    (8, 1e6, 16.0, 4096, 0.5, 100.0), (256, 10000.0, 0.5, 2048, 1.0, 32.0)])
def test_frequencies(cuda, dim, base, factor, original, low, high):
    got = nh.rotary_frequencies(dim, base, factor=factor, original=original, low=low, high=high)
    f = base ** (-torch.arange(0, dim, 2, dtype=F64) / dim)
    keep = ((original * f / (2 * torch.pi) - low) / (high - low)).clamp(0, 1) if original else 0.0
    want = f * (keep + (1 - keep) / factor)
    # 64 bits throughout, the logarithm of 10^6 times 2^-52 in the power: one rounding.
    assert ((got.double().cpu() - want).abs() <= 2.0 ** -24 * 1.001 * want).all()


def normed(x, w, eps):
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    return x * r * w, r


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("D,R", SHAPES)
def test_norm_and_backward(cuda, D, R, dt, interleaved):
    norm_case(cuda, 41, 6, 3, D, R, dt, interleaved, weight=dt)


@pytest.mark.parametrize("T,H,G,D", [(1023, 70, 3, 256), (1100, 40, 8, 256), (1500, 33, 1, 96), (2500, 5, 0, 8),
                                     (8300, 17, 4, 64), (1024, 1, 1, 248), (1, 600, 1, 128)])
def test_norm_of_many_heads(cuda, T, H, G, D):
    """Workgroups of every shape: more rows to a token than threads, and fewer."""
    norm_case(cuda, T, H, G, D, D, BF, False)
    norm_case(cuda, min(T, 1500), H, G, D, 8, F32, True, layout="htd")


@pytest.mark.parametrize("T,H,G", [(12001, 2, 1), (25000, 0, 1), (4095, 1, 1), (4097, 2, 3), (20007, 1, 0)])
def test_norm_of_many_tokens(cuda, T, H, G):
    """Runs of up to eight tokens, several to a workgroup of the backward pass."""
    norm_case(cuda, T, H, G, 40, 24, HF, True)


@pytest.mark.parametrize("layout", ["thd", "fused", "htd"])
@pytest.mark.parametrize("T,H,G", [(1, 1, 1), (1, 40, 8), (7, 0, 2), (7, 3, 0), (1024, 2, 1), (2500, 12, 12),
                                   (9001, 3, 1), (1, 300, 7)])
def test_norm_sizes_and_layouts(cuda, T, H, G, layout):
    norm_case(cuda, T, H, G, 64, 64, BF, False, layout=layout, weight=F32)


def norm_case(dev, T, H, G, D, R, dt, interleaved, layout="thd", weight=F32, scale=1.25, eps=1e-5):
    q, k = make(dev, T, H, D, dt, 1, layout), make(dev, T, G, D, dt, 2, layout)
    gq, gk = make(dev, T, H, D, dt, 3, layout), make(dev, T, G, D, dt, 4, layout)
    g = torch.Generator(device=dev).manual_seed(5)
    wq, wk = ((1 + 0.3 * torch.randn(D, generator=g, device=dev)).to(weight) for _ in range(2))
    pos, f = places(dev, T), freqs_of(R, dev)
    kw = dict(eps=eps, interleaved=interleaved, scale=scale)
    y = nh.qk_norm_rotary(q, k, wq, wk, pos, f, **kw)
    for got, x, w in zip(y, (q, k), (wq, wk)):
        want, amp = turned(normed(x.double(), w.double(), eps)[0], pos, f, interleaved, scale)
        near(got, want, amp, 2.0 ** -19, ("forward", T, D, R, dt))
    back = nh.qk_norm_rotary_backward(gq, gk, q, k, wq, wk, pos, f, **kw)
    again = nh.qk_norm_rotary_backward(gq, gk, q, k, wq, wk, pos, f, **kw)
    assert all(torch.equal(a, b) for a, b in zip(back, again))  # a fixed order of sums
    for dx, dw, grad, x, w in zip(back[:2], back[2:], (gq, gk), (q, k), (wq, wk)):
        xd, wd = x.double().requires_grad_(), w.double().requires_grad_()
        # The rotation is linear: its transpose is the inverse.
        up, amp = turned(grad.double(), pos, f, interleaved, scale, inverse=True)
        n, r = normed(xd, wd, eps)
        want, want_w = torch.autograd.grad(n, (xd, wd), up)
        r, xa = r.detach(), x.double().abs()
        ta = amp * wd.detach().abs()
        near(dx, want, r * (ta + xa * r * r * (ta * xa).mean(-1, keepdim=True)), 2.0 ** -18,
             ("dx", T, D, R, dt))
        near(dw, want_w, (amp * xa * r).sum((0, 1)), 2.0 ** -15, ("dw", T, D, R, dt))


@pytest.mark.parametrize("D,R,interleaved", [(64, 32, False), (40, 40, True), (128, 128, False)])
def test_backward_against_differences(cuda, D, R, interleaved):
    """Along random directions, f32: the difference quotient of the call itself.
    With step h = 2^-6 its error is h^2 / 6 times a third derivative of order one
    and, from rounding, 2^-21 sqrt(count) / h: both under 2^-9 of the slope's
    scale, the norm of the gradient times that of the direction (one)."""
    T, H, G, h = 5, 3, 2, 2.0 ** -6
    q, k = make(cuda, T, H, D, F32, 1), make(cuda, T, G, D, F32, 2)
    gq, gk = make(cuda, T, H, D, F32, 3), make(cuda, T, G, D, F32, 4)
    wq, wk = torch.full((D,), 1.2, device=cuda), torch.full((D,), 0.8, device=cuda)
    pos, f = places(cuda, T), freqs_of(R, cuda)
    grads = nh.qk_norm_rotary_backward(gq, gk, q, k, wq, wk, pos, f, interleaved=interleaved)

    def value(*a):
        yq, yk = nh.qk_norm_rotary(*a, pos, f, interleaved=interleaved)
        return (yq.double() * gq.double()).sum() + (yk.double() * gk.double()).sum()

    g = torch.Generator(device=cuda).manual_seed(9)
    at = [q, k, wq, wk]
    for i, grad in enumerate(grads):
        d = torch.randn(at[i].shape, generator=g, device=cuda)
        d /= d.norm()
        plus, minus = list(at), list(at)
        plus[i], minus[i] = at[i] + h * d, at[i] - h * d
        slope = (value(*plus) - value(*minus)) / (2 * h)
        want = (grad.double() * d.double()).sum()
        assert abs(slope - want).item() <= 2.0 ** -9 * grad.double().norm().item(), (i, slope, want)


def test_norm_alone_rows_of_zeros_and_in_place(cuda):
    q, k = make(cuda, 33, 4, 96, BF), make(cuda, 33, 2, 96, BF, 1)
    q[3] = 0.0
    w = torch.ones(96, device=cuda)
    yq, yk = nh.qk_norm_rotary(q, k, w, w)
    want, _ = normed(q.double(), w.double(), 1e-6)
    near(yq, want, want.abs(), 2.0 ** -19)
    assert (yq[3] == 0).all()
    gq, gk = make(cuda, 33, 4, 96, BF, 2), make(cuda, 33, 2, 96, BF, 3)
    back = nh.qk_norm_rotary_backward(gq, gk, q, k, w, w)
    assert torch.isfinite(back[0]).all()
    a, b = q.clone(), gk.clone()
    into = nh.qk_norm_rotary_backward(gq, b, a, k, w, w, dq=a, dk=b)  # over q, over grad_k
    assert all(torch.equal(x, y) for x, y in zip(into, back))
    nh.qk_norm_rotary(q, k, w, w, q_out=q, k_out=k)
    assert torch.equal(q, yq) and torch.equal(k, yk)


def test_nothing_to_sum(cuda):
    e = torch.empty(0, 3, 64, dtype=BF, device=cuda)
    w = torch.ones(64, device=cuda)
    dq, dk, dwq, dwk = nh.qk_norm_rotary_backward(e, e, e, e, w, w)
    assert dq.shape == e.shape and (dwq == 0).all() and (dwk == 0).all()

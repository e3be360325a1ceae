"""token_logp, policy_loss and preference_loss on the GPU against their
definitions in 64 bits.

Tolerances.  A row's sum of exponentials is f32, at most 100 sequential and tree
additions of terms each within 2^-23 (1 + 1.5 |x - max|) of their value: 8e-6 of
the sum; its logarithm and the label's distance to the maximum round at 2^-24 of
their size.  So a log-probability is within
  LP = 8e-6 + 2^-23 (|x_y - max| + |lp|),
a softmax value p within 2e-5 p (for |x - max| < 40), a ratio within LP of
itself (and 2 ulp of expf).  Gradients round once to the logits' type."""
import math

import pytest
import torch

import nova_hip as nh

pytestmark = pytest.mark.gpu
F64 = torch.float64
F32, BF, HF = torch.float32, torch.bfloat16, torch.float16
SIZES = [1, 2, 3, 7, 8, 63, 64, 255, 1000, 1023, 1024, 1025, 2048, 2049, 4095, 5000, 8192, 8193,
         10034, 16384, 16385, 32000, 32768, 32769, 50257, 50304]


def make(dev, R, C, dt, seed=0, pad=0, masked=0.3):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.full((R, C + pad), float("nan"), dtype=dt, device=dev)[:, :C]
    x.copy_((2 * torch.randn(R, C, generator=g, device=dev)).to(dt))
    y = torch.randint(0, C, (R,), generator=g, device=dev, dtype=torch.int32)
    if masked:
        y[torch.rand(R, generator=g, device=dev) < masked] = -1
    return x, y, g


def rows64(x, y):
    """lp, p, max distance of the label, valid, in 64 bits."""
    ok = y >= 0
    z = torch.log_softmax(x.double(), 1)
    at = y.clamp(min=0).long()[:, None]
    lp = torch.where(ok, z.gather(1, at)[:, 0], torch.zeros_like(z[:, 0]))
    dist = (x.double().amax(1) - x.double().gather(1, at)[:, 0])
    return lp, z.exp(), dist, ok


def lp_tol(lp, dist):
    return 8e-6 + 2.0 ** -23 * (dist + lp.abs())


def check_grad(got, slope, slope_err, p, y, ok, scale=1.0):
    """got = scale * slope (onehot - p) in rows with a label, zero elsewhere."""
    one = torch.zeros_like(p)
    one.scatter_(1, y.clamp(min=0).long()[:, None], 1.0)
    want = scale * slope[:, None] * (one - p) * ok[:, None]
    u = torch.finfo(got.dtype).eps / 2
    tol = u * want.abs() + abs(scale) * (slope.abs()[:, None] * (2e-5 * p + 2.0 ** -23 * one)
                                         + slope_err[:, None] * (one + p)) * ok[:, None]
    tol = tol * 1.01 + (2.0 ** -25 if got.dtype == HF else 1e-38)
    err = (got.double() - want).abs()
    assert not torch.isnan(err).any()
    assert (err <= tol).all(), ((err - tol).max().item(), err.max().item())
    assert (got[~ok] == 0).all()


@pytest.mark.parametrize("dt", [F32, BF, HF])
@pytest.mark.parametrize("C", SIZES)
def test_token_logp(cuda, dt, C):
    for R, pad in ((1, 0), (13, 0), (6, 5)):
        x, y, _ = make(cuda, R, C, dt, seed=C, pad=pad)
        lse = torch.full((R,), 7.0, device=cuda)
        got = nh.token_logp(x, y, lse=lse)
        lp, _, dist, ok = rows64(x, y)
        assert ((got.double() - lp).abs() <= lp_tol(lp, dist)).all()
        want = torch.where(ok, torch.logsumexp(x.double(), 1), torch.zeros_like(lp))
        assert ((lse.double() - want).abs() <= 8e-6 + 2.0 ** -23 * want.abs()).all()


@pytest.mark.parametrize("dt", [F32, BF, HF])
@pytest.mark.parametrize("C", [51201, 102401, 151936])
def test_rows_beyond_the_registers(cuda, dt, C):
    policy(cuda, 5, C, dt, kl=0.1)
    x, y, _ = make(cuda, 4, C, dt)
    lp, _, dist, _ = rows64(x, y)
    assert ((nh.token_logp(x, y).double() - lp).abs() <= lp_tol(lp, dist)).all()


def test_labels_out_of_range_and_masked_rows_are_not_read(cuda):
    x, y, _ = make(cuda, 6, 1000, F32, masked=0)
    y[:] = torch.tensor([-1, 5, 1000, -7, 2 ** 31 - 1, 999], dtype=torch.int32)
    x[0], x[3] = float("nan"), float("inf")
    lp = nh.token_logp(x, y)
    assert torch.isnan(lp).tolist() == [False, False, True, False, True, False]
    assert lp[0] == 0 and lp[3] == 0
    one = torch.ones(6, device=cuda)
    w = one.clone()
    w[4] = 0.0  # weight 0: no part either
    y[2] = 7
    loss, logp, grad = nh.policy_loss(x, y, torch.zeros_like(one), one, w)
    assert torch.isfinite(loss).all() and torch.isfinite(grad).all() and logp[4] == 0
    assert (grad[[0, 3, 4]] == 0).all()
    y[1] = 1000
    loss, logp, grad = nh.policy_loss(x, y, torch.zeros_like(one), one, w)
    assert torch.isnan(loss).all() and torch.isnan(grad[1]).all() and torch.isfinite(grad[2]).all()


@pytest.mark.parametrize("dt", [F32, BF, HF])
def test_infinite_logits(cuda, dt):
    """-inf is a class that cannot occur; a row of nothing else has no
    distribution (NaN), as has one with +inf or NaN."""
    for C in (100, 3000, 60000, 110000):
        x, y, _ = make(cuda, 5, C, dt, masked=0)
        y[:] = 3
        x[0, 10:60] = float("-inf")
        x[1] = float("-inf")
        x[2, 0] = float("nan")
        x[3, C - 1] = float("inf")
        x[4, 3] = float("-inf")
        lp = nh.token_logp(x, y)
        want, _, dist, _ = rows64(x[:1], y[:1])
        assert ((lp[0].double() - want[0]).abs() <= lp_tol(want, dist)[0])
        assert torch.isnan(lp[1:4]).all() and lp[4] == float("-inf")


def policy(dev, R, C, dt, kl=0.0, seed=0, pad=0, clip=(0.2, 0.3), scale=1.0, big=0.3):
    x, y, g = make(dev, R, C, dt, seed, pad)
    lp, p, dist, ok = rows64(x, y)
    step = big * torch.randn(R, generator=g, device=dev, dtype=F64)
    for edge in (math.log(1 - clip[0]), math.log(1 + clip[1])):  # off the kinks
        step = torch.where((step - edge).abs() < 1e-3, torch.full_like(step, edge + 2e-3), step)
    old = (lp - step).float()
    ref = (lp + 0.2 * torch.randn(R, generator=g, device=dev, dtype=F64)).float() if kl else None
    adv = torch.randn(R, generator=g, device=dev)
    w = torch.rand(R, generator=g, device=dev) / R
    grad = torch.full((R, C + pad), 7.0, dtype=dt, device=dev)
    row_loss = torch.empty(R, device=dev)
    loss, logp, _ = nh.policy_loss(x, y, old, adv, w, ref_logp=ref, clip=clip, kl_coef=kl,
                                   grad_scale=scale, grad=grad[:, :C], row_loss=row_loss)
    assert (grad[:, C:] == 7.0).all()
    tol = lp_tol(lp, dist)
    assert ((logp.double() - lp).abs() <= tol).all()
    A, W = adv.double(), w.double() * ok
    ratio = torch.exp(lp - old.double())
    plain, clipped = ratio * A, ratio.clamp(1 - clip[0], 1 + clip[1]) * A
    per, slope = -torch.minimum(plain, clipped), torch.where(plain <= clipped, -plain, torch.zeros_like(plain))
    rel = (tol + 1e-6) * 1.01
    err = rel * plain.abs() + 2.0 ** -23 * clipped.abs()
    if kl:
        d = ref.double() - lp
        per = per + kl * (torch.expm1(d) - d)
        slope = slope - kl * torch.expm1(d)
        err = err + kl * (rel * (d.exp() + 1) + 1e-6 * d.abs())
    err = W * (err + 2.0 ** -22 * per.abs())
    assert ((row_loss.double() - W * per).abs() <= err + 1e-38).all()
    assert abs(loss.double().item() - (W * per).sum().item()) <= err.sum().item() + 2.0 ** -23 * abs(loss.item())
    check_grad(grad[:, :C], slope * W, err + 2.0 ** -22 * (slope * W).abs(), p, y, ok, scale)
    return loss, logp, grad


@pytest.mark.parametrize("dt", [F32, BF, HF])
@pytest.mark.parametrize("C", SIZES)
def test_policy_sizes(cuda, dt, C):
    policy(cuda, 9, C, dt, kl=0.05, seed=C)
    policy(cuda, 4, C, dt, pad=3, seed=C, scale=256.0)


@pytest.mark.parametrize("kl", [0.0, 0.3])
@pytest.mark.parametrize("clip", [(0.2, 0.2), (0.0, 0.0), (1.0, 5.0)])
def test_policy_clips(cuda, kl, clip):
    if clip == (0.0, 0.0):
        # Everything is outside or on the clip; on it both sides are equal.
        x, y, g = make(cuda, 50, 500, F32, masked=0)
        lp = nh.token_logp(x, y)
        adv = torch.randn(50, generator=g, device=cuda)
        w = torch.full((50,), 0.02, device=cuda)
        loss, logp, grad = nh.policy_loss(x, y, lp, adv, w, clip=clip)
        _, p, _, ok = rows64(x, y)
        assert torch.equal(logp, lp)  # ratio exactly 1: the first side's gradient
        check_grad(grad, -adv.double() * 0.02, 1e-6 * adv.double().abs(), p, y, ok)
    else:
        policy(cuda, 300, 700, F32, kl=kl, clip=clip, big=0.6) if clip[0] < 1 else \
            policy_wide(cuda, kl, clip)


def policy_wide(dev, kl, clip):
    x, y, g = make(dev, 40, 300, F32, masked=0)
    lp = nh.token_logp(x, y)
    adv, w = torch.randn(40, generator=g, device=dev), torch.ones(40, device=dev)
    a = nh.policy_loss(x, y, lp - 0.5, adv, w, ref_logp=lp, kl_coef=kl, clip=clip)
    ratio = math.exp(0.5)
    want = -(ratio * adv.double()).sum() + 40 * kl * 0.0
    assert abs(a[0].item() - want.item()) <= 1e-4 * adv.abs().sum().item()


def test_policy_empty_and_all_masked(cuda):
    f = lambda *s: torch.zeros(*s, device=cuda)
    loss, logp, grad = nh.policy_loss(f(0, 10), f(0).int(), f(0), f(0), f(0))
    assert loss.item() == 0 and grad.shape == (0, 10)
    x, y, _ = make(cuda, 5, 100, BF, masked=0)
    loss, logp, grad = nh.policy_loss(x, torch.full_like(y, -1), f(5), f(5), f(5) + 1)
    assert loss.item() == 0 and (grad == 0).all() and (logp == 0).all()


def test_policy_without_a_gradient(cuda):
    x, y, _ = make(cuda, 20, 3000, BF)
    one = torch.ones(20, device=cuda)
    a = nh.policy_loss(x, y, -one, one, one)
    b = nh.policy_loss(x, y, -one, one, one, want_grad=False)
    assert b[2] is None and torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def preference(dev, lens, C, dt, seed=0, pad=0, first=0, behind=0, beta=0.1, eps=0.05, spread=8.0,
               scale=1.0):
    T = first + sum(lens)
    R = T + behind
    x, y, g = make(dev, R, C, dt, seed, pad)
    o = [first]
    for n in lens:
        o.append(o[-1] + n)
    off = torch.tensor(o, dtype=torch.int32, device=dev)
    lp, p, dist, ok = rows64(x, y)
    seq = torch.stack([lp[a:b].sum() for a, b in zip(o[:-1], o[1:])])
    ref = (seq + spread * torch.randn(len(lens), generator=g, device=dev, dtype=F64)).float()
    grad = torch.full((R, C + pad), 7.0, dtype=dt, device=dev)
    pair = torch.empty(len(lens) // 2, device=dev)
    token = torch.empty(3, R, device=dev)
    loss, got_seq, _ = nh.preference_loss(x, y, off, ref, beta=beta, smoothing=eps, grad_scale=scale,
                                          grad=grad[:, :C], pair_loss=pair, token=token)
    assert (grad[:, C:] == 7.0).all()
    tol = lp_tol(lp, dist) * ok
    seq_tol = torch.stack([tol[a:b].sum() for a, b in zip(o[:-1], o[1:])])
    assert ((got_seq.double() - seq).abs() <= seq_tol + 2.0 ** -24 * seq.abs()).all()
    r = seq - ref.double()
    h = beta * (r[0::2] - r[1::2])
    herr = abs(beta) * (seq_tol[0::2] + seq_tol[1::2]) + 1e-7 * h.abs()  # f32 beta
    logsig = torch.nn.functional.logsigmoid
    want = -((1 - eps) * logsig(h) + eps * logsig(-h))
    assert ((pair.double() - want).abs() <= herr + 2.0 ** -23 * want + 1e-7).all()
    assert abs(loss.item() - want.mean().item()) <= herr.mean().item() + 2e-7 * (1 + want.mean().item())
    P = len(lens) // 2
    s = beta * (eps * torch.sigmoid(h) - (1 - eps) * torch.sigmoid(-h)) / P
    serr = abs(beta) / P * (herr / 4 + 1e-7) + 2e-7 * s.abs()
    slope, err, inside = torch.zeros_like(lp), torch.zeros_like(lp), torch.zeros_like(ok)
    for i, (a, b) in enumerate(zip(o[:-1], o[1:])):
        slope[a:b] = s[i // 2] * (1 if i % 2 == 0 else -1)
        err[a:b] = serr[i // 2]
        inside[a:b] = True
    # p comes from the stored lse: its error adds to p's.
    check_grad(grad[:, :C], slope, err + slope.abs() * 2e-5, p, y, ok & inside, scale)
    assert ((token[2].double() - scale * slope).abs() <= abs(scale) * err + 2e-7 * slope.abs() * abs(scale)).all()
    return loss, grad


@pytest.mark.parametrize("dt", [F32, BF, HF])
@pytest.mark.parametrize("C", [1, 7, 64, 1000, 1025, 2049, 5000, 10034, 32000, 50257, 110001])
def test_preference_sizes(cuda, dt, C):
    preference(cuda, [5, 7], C, dt, seed=C)
    preference(cuda, [1, 4, 3, 2], C, dt, seed=C, pad=5, first=2, behind=3, scale=64.0)


@pytest.mark.parametrize("lens", [[0, 0], [0, 5], [300, 0, 1, 700], [1] * 200])
def test_preference_lengths(cuda, lens):
    preference(cuda, lens, 300, F32, behind=1)


@pytest.mark.parametrize("beta,eps,spread", [(0.5, 0.0, 0.0), (0.1, 0.5, 5.0), (2.0, 0.0, 40.0), (0.01, 1.0, 1.0)])
def test_preference_parameters(cuda, beta, eps, spread):
    preference(cuda, [50, 60, 20, 33], 400, F32, beta=beta, eps=eps, spread=spread)


def test_gradients_against_differences(cuda):
    """Central differences of the 64-bit losses along random directions."""
    x, y, g = make(cuda, 12, 50, F32)
    off = torch.tensor([0, 5, 12], dtype=torch.int32, device=cuda)
    ref = torch.tensor([-9.0, -12.0], device=cuda)
    lp0 = rows64(x, y)[0]
    old = (lp0 - 0.05).float()
    adv, w = torch.randn(12, generator=g, device=cuda), torch.rand(12, generator=g, device=cuda)

    def pref(z):
        lp = rows64(z, y)[0]
        h = 0.3 * ((lp[:5].sum() - ref[0].double()) - (lp[5:].sum() - ref[1].double()))
        return -torch.nn.functional.logsigmoid(h)

    def pol(z):
        lp = rows64(z, y)[0]
        r = torch.exp(lp - old.double())
        d = old.double() - lp
        per = -torch.minimum(r * adv.double(), r.clamp(0.8, 1.2) * adv.double()) + 0.1 * (d.exp() - d - 1)
        return (per * w.double() * (y >= 0)).sum()

    grads = (nh.preference_loss(x, y, off, ref, beta=0.3)[2],
             nh.policy_loss(x, y, old, adv, w, ref_logp=old, kl_coef=0.1)[2])
    d = torch.randn(x.shape, generator=g, device=cuda, dtype=F64)
    for fn, grad in zip((pref, pol), grads):
        h = 1e-5
        num = ((fn(x.double() + h * d) - fn(x.double() - h * d)) / (2 * h)).item()
        ours = (grad.double() * d).sum().item()
        scale = (grad.double() * d).abs().sum().item()
        # f32 gradients: 3e-5 of each term; the difference: h^2 and 64-bit noise / h.
        assert abs(ours - num) <= 3e-5 * scale + 1e-8, (ours, num)


def test_rows_far_apart(cuda):
    """Rows 2^31 elements apart: a row's offset passes 32 bits in elements and
    bytes, in the logits and in the gradient."""
    C, step = 3000, 1 << 31
    flat = torch.empty(2 * step + C, dtype=BF, device=cuda)
    far = flat.as_strided((3, C), (step, 1))
    x, y, g = make(cuda, 3, C, BF, masked=0)
    one = torch.ones(3, device=cuda)
    lp = nh.token_logp(x, y)
    want = nh.policy_loss(x, y, lp - 0.1, one, one)
    off = torch.tensor([0, 1, 3], dtype=torch.int32, device=cuda)
    pref = nh.preference_loss(x, y, off, one[:2])
    far.copy_(x)
    assert torch.equal(nh.token_logp(far, y), lp)
    assert all(torch.equal(a, b) for a, b in zip(nh.policy_loss(far, y, lp - 0.1, one, one), want))
    assert all(torch.equal(a, b) for a, b in zip(nh.preference_loss(far, y, off, one[:2]), pref))
    nh.policy_loss(x, y, lp - 0.1, one, one, grad=far)
    assert torch.equal(far, want[2])
    nh.preference_loss(x, y, off, one[:2], grad=far)
    assert torch.equal(far, pref[2])


@pytest.mark.parametrize("C", [100, 5000, 50304, 60000])
@pytest.mark.parametrize("shift", [8192.0, -8192.0])
def test_logits_far_from_zero(cuda, C, shift):
    """Logits that are multiples of 2^-9 keep their exact differences 8192 away
    from zero, so log-probabilities and gradients keep the bounds of the logits
    around zero: |x - x_y| and |lp| stay under 40, and 2^-23 of those within the
    2e-5 the bounds leave to a softmax value.  (The lse itself rounds by 2^-11.)"""
    x, y, _ = make(cuda, 12, C, F32, seed=C)
    x = (x * 512).round() / 512
    y[0], y[7] = 3, C - 1  # a label in each sequence
    lp, p, dist, ok = rows64(x, y)
    assert dist.max() < 20 and lp.abs().max() < 40
    far = x + shift
    assert torch.equal(far - shift, x)
    assert ((nh.token_logp(far, y).double() - lp).abs() <= lp_tol(lp, dist) * ok).all()
    off = torch.tensor([0, 6, 12], dtype=torch.int32, device=cuda)
    ref = torch.stack([lp[:6].sum(), lp[6:].sum()]).float()
    token = torch.empty(3, 12, device=cuda)
    _, _, grad = nh.preference_loss(far, y, off, ref, token=token)
    slope = token[2].double()
    check_grad(grad, slope, slope.abs() * 2e-5, p, y, ok)
    one = torch.ones(12, device=cuda)
    _, _, grad = nh.policy_loss(far, y, lp.float(), one, one)
    check_grad(grad, -torch.ones_like(lp), lp_tol(lp, dist) + 2.0 ** -24 * lp.abs() + 2.0 ** -22, p, y, ok)


@pytest.mark.parametrize("C", [300, 5000, 32000, 50304, 60000, 120000])
@pytest.mark.parametrize("dt", [F32, BF])
def test_results_written_over_the_inputs(cuda, dt, C):
    """logp over old_logp, ref_logp or advantage, row_loss over weight, seq_logp
    over the sequences' ref_logp: the bits of separate memory."""
    R = 700
    x, y, g = make(cuda, R, C, dt, masked=0.2)
    old = nh.token_logp(x, y) - 0.1 * torch.randn(R, generator=g, device=cuda)
    ref, adv, w = old + 0.05, torch.randn(R, generator=g, device=cuda), torch.rand(R, generator=g, device=cuda)
    row = torch.empty(R, device=cuda)
    call = lambda o, f, a, v, **k: nh.policy_loss(x, y, o, a, v, ref_logp=f, kl_coef=0.1, **k)
    want = call(old, ref, adv, w, row_loss=row)
    for i in range(3):
        ins = [t.clone() for t in (old, ref, adv, w)]
        got = call(*ins, logp=ins[i], row_loss=ins[3])
        assert torch.equal(ins[i], want[1]) and torch.equal(ins[3], row)
        assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])
    off = torch.tensor([0, 100, 350, 420, 700], dtype=torch.int32, device=cuda)
    ref = torch.randn(4, generator=g, device=cuda) * 10 - 900
    want = nh.preference_loss(x, y, off, ref)
    got = nh.preference_loss(x, y, off, ref, seq_logp=ref)
    assert torch.equal(ref, want[1]) and torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])


@pytest.mark.parametrize("C", [300, 5000, 50304, 110001])
@pytest.mark.parametrize("dt", [F32, BF])
def test_rows_of_weight_zero(cuda, dt, C):
    """Their log-probability is the label's, so that it can be the next step's
    old_logp (within LP of the module's docstring: calls with and without a
    gradient give a row different numbers of threads and so add it up in different
    orders, each within LP); they add no loss and have a zero gradient, even where
    their logits or ratio are infinite or NaN; the other rows are what they were."""
    x, y, g = make(cuda, 12, C, dt, masked=0)
    y[3] = -1
    x[5, 7], x[6, 0] = float("nan"), float("inf")
    old = torch.zeros(12, device=cuda)
    old[7] = -1e30
    adv, w = torch.randn(12, generator=g, device=cuda), torch.rand(12, generator=g, device=cuda) + 0.1
    none = torch.tensor([1, 3, 5, 6, 7], device=cuda)
    w[none] = 0.0
    row = torch.full((12,), 7.0, device=cuda)
    loss, logp, grad = nh.policy_loss(x, y, old, adv, w, ref_logp=old, kl_coef=0.1, row_loss=row)
    want, _, dist, _ = rows64(x, y)
    assert torch.isnan(logp[[5, 6]]).all() and torch.isnan(want[[5, 6]]).all()
    fine = torch.tensor([i for i in range(12) if i not in (5, 6)], device=cuda)
    assert ((logp.double() - want).abs() <= lp_tol(want, dist))[fine].all()
    assert logp[1] < 0 and logp[3] == 0
    assert (row[none] == 0).all() and (grad[none] == 0).all() and torch.isfinite(loss).all()
    rest = torch.tensor([i for i in range(12) if i not in none.tolist()], device=cuda)
    a = nh.policy_loss(x[rest], y[rest], old[rest], adv[rest], w[rest], ref_logp=old[rest], kl_coef=0.1)
    assert torch.equal(grad[rest], a[2]) and torch.equal(logp[rest], a[1])
    assert abs(loss.item() - a[0].item()) <= 2.0 ** -23 * abs(a[0].item())


@pytest.mark.parametrize("kl", [0.0, 0.3, -0.2])
@pytest.mark.parametrize("dt", [F32, BF])
def test_policy_wide_clip_with_a_kl_term(cuda, dt, kl):
    """clip (1, 5): the ratio in [0, 6], so only ratios above 6 are clipped; the
    loss, its rows and the gradient with a reference that differs from logp."""
    R, C, lo, hi, scale = 60, 700, 1.0, 5.0, 4.0
    x, y, g = make(cuda, R, C, dt, seed=5)
    lp, p, dist, ok = rows64(x, y)
    step = torch.linspace(-3.0, 3.0, R, device=cuda, dtype=F64)  # no step within 0.01 of log 6
    assert (step - math.log(1 + hi)).abs().min() > 0.01
    old, ref = (lp - step).float(), (lp + 0.7 * torch.randn(R, generator=g, device=cuda, dtype=F64)).float()
    adv, w = torch.randn(R, generator=g, device=cuda), torch.rand(R, generator=g, device=cuda)
    row = torch.empty(R, device=cuda)
    loss, logp, grad = nh.policy_loss(x, y, old, adv, w, ref_logp=ref, kl_coef=kl, clip=(lo, hi),
                                      grad_scale=scale, row_loss=row)
    tol = lp_tol(lp, dist)
    assert ((logp.double() - lp).abs() <= tol).all()
    A, W, k = adv.double(), w.double() * ok, float(torch.tensor(kl, dtype=F32))
    ratio = torch.exp(lp - old.double())
    plain, clipped, d = ratio * A, ratio.clamp(1 - lo, 1 + hi) * A, ref.double() - lp
    per = -torch.minimum(plain, clipped) + k * (torch.expm1(d) - d)
    slope = torch.where(plain <= clipped, -plain, torch.zeros_like(plain)) - k * torch.expm1(d)
    # A ratio is off by lp's error and expf's 2 ulp, a clipped one by nothing; the
    # KL term by lp's error times its slope (d.exp() + 1) and a few ulp.
    rel = (tol + 1e-6) * 1.01
    err = rel * plain.abs() + 2.0 ** -23 * clipped.abs() + abs(k) * (rel * (d.exp() + 1) + 1e-6 * d.abs())
    err = W * (err + 2.0 ** -22 * per.abs())
    assert ((row.double() - W * per).abs() <= err + 1e-38).all()
    assert abs(loss.item() - (W * per).sum().item()) <= err.sum().item() + 2.0 ** -23 * abs(loss.item())
    check_grad(grad, slope * W, err + 2.0 ** -22 * (slope * W).abs(), p, y, ok, scale)

"""Single-token attention over a padded cache against its definition in 64
bits (tolerances: test_attention_gpu.py)."""
import pytest
import torch

import nova_hip as nh
from test_attention_gpu import BF, HF, check

pytestmark = pytest.mark.gpu


def run(dev, lens, S, H, G, D, dt, order="bshd", seed=0, scale=None):
    g = torch.Generator(device=dev).manual_seed(seed)
    B = len(lens)
    q = torch.randn(B, H, D, generator=g, device=dev).to(dt)
    if order == "bshd":
        k, v = (torch.randn(B, S, G, D, generator=g, device=dev).to(dt) for _ in range(2))
    elif order == "bhsd":
        k, v = (torch.randn(B, G, S, D, generator=g, device=dev).to(dt).transpose(1, 2) for _ in range(2))
    else:  # keys and values of a row side by side, sequences innermost but one
        kv = torch.randn(S, B, G, 2, D, generator=g, device=dev).to(dt).transpose(0, 1)
        k, v = kv[..., 0, :], kv[..., 1, :]
    cut = [min(max(n, 0), S) for n in lens]
    for b, n in enumerate(cut):  # rows behind a length are not read
        k[b, n:] = float("nan")
        v[b, n:] = float("nan")
    length = torch.tensor(lens, dtype=torch.int32, device=dev)
    lse = torch.full((B, H), 7.0, device=dev)
    out = nh.attention_decode(q, k, v, length, lse=lse, scale=scale)
    kp = torch.cat([k[b, :n] for b, n in enumerate(cut)])
    vp = torch.cat([v[b, :n] for b, n in enumerate(cut)])
    check(out, lse.t(), q, kp, vp, [1] * B, cut, False, D ** -0.5 if scale is None else scale,
          (lens, S, H, G, D, dt, order))
    return q, k, v, length, out


@pytest.mark.parametrize("dt", [BF, HF])
@pytest.mark.parametrize("D", [8, 32, 40, 64, 80, 96, 120, 128])
def test_head_dims(cuda, dt, D):
    run(cuda, [97, 1, 64, 130], 130, 8, 2, D, dt)


@pytest.mark.parametrize("order", ["bshd", "bhsd", "mixed"])
@pytest.mark.parametrize("H,G", [(1, 1), (6, 6), (7, 1), (32, 8), (48, 1), (71, 1), (64, 32)])
def test_orders_and_shared_heads(cuda, order, H, G):
    run(cuda, [33, 200, 1], 200, H, G, 64, BF, order)


@pytest.mark.parametrize("S", [1, 31, 32, 33, 63, 64, 65, 128, 129, 1000, 1023, 1024, 1025, 1100, 3001])
@pytest.mark.parametrize("D", [64, 128])
def test_cache_sizes(cuda, S, D):
    run(cuda, [S, 1, S // 2, 0, S - 1], S, 4, 2, D, BF)


@pytest.mark.parametrize("D", [32, 40, 64, 80, 96, 128])
def test_head_dims_of_a_long_cache(cuda, D):
    run(cuda, [1500, 1, 64, 130, 1437], 1500, 8, 2, D, HF)
    run(cuda, [1500, 700], 1500, 35, 1, D, BF, "bhsd")  # more heads than one block of 32


@pytest.mark.parametrize("S", [40, 300, 1024, 1025, 3001])  # one launch up to 1024 rows, two beyond
@pytest.mark.parametrize("dt,D", [(BF, 64), (HF, 128)])
def test_nan_scores_reach_the_lse(cuda, S, dt, D):
    """A NaN query, and NaN in all keys that one wave of the joined form or one
    split takes: result and log-sum-exp are both NaN there, whatever the cache's
    size, and those of the other heads and sequences what they were."""
    g = torch.Generator(device=cuda).manual_seed(S)
    q = torch.randn(3, 4, D, generator=g, device=cuda).to(dt)
    k, v = (torch.randn(3, S, 2, D, generator=g, device=cuda).to(dt) for _ in range(2))
    n = torch.tensor([S, S - 1, S // 2], dtype=torch.int32, device=cuda)
    lse, want = torch.empty(3, 4, device=cuda), torch.empty(3, 4, device=cuda)
    plain = nh.attention_decode(q, k, v, n, lse=want)
    q[0, 1] = float("nan")
    k[1, 32:, 1] = float("nan")
    out = nh.attention_decode(q, k, v, n, lse=lse)
    bad = torch.zeros(3, 4, dtype=torch.bool, device=cuda)
    bad[0, 1] = bad[1, 2] = bad[1, 3] = True
    assert torch.isnan(lse[bad]).all() and torch.isnan(out[bad]).all()
    assert torch.equal(lse[~bad], want[~bad]) and torch.equal(out[~bad], plain[~bad])


def test_lengths_zero_and_out_of_range(cuda):
    q, k, v, length, out = run(cuda, [0, 300, -5, 70], 64, 4, 2, 64, BF)
    assert (out[0] == 0).all() and (out[2] == 0).all()
    # An empty cache: rows of zeros.
    out = nh.attention_decode(q, k[:, :0], v[:, :0], length)
    assert (out == 0).all()


def test_many_splits(cuda):
    run(cuda, [40000, 3], 40000, 4, 1, 64, BF)
    run(cuda, [8192, 1500, 5000, 77, 0, 8191] * 4, 8192, 32, 8, 128, HF, "bhsd")


def test_offsets_past_32_bits(cuda):
    """A head's rows lie more than 2^32 bytes behind the other's, a sequence's
    more than 2^33 behind the first one's."""
    n, D = 1000, 128
    head = (1 << 31) + 4096 * 8  # elements of 2 bytes
    flat = torch.empty(3 * head + n * D, dtype=BF, device=cuda)
    k = flat.as_strided((2, n, 2, D), (2 * head, D, head, 1))
    g = torch.Generator(device=cuda).manual_seed(3)
    for b in range(2):
        for h in range(2):
            k[b, :, h] = torch.randn(n, D, generator=g, device=cuda).to(BF)
    q = torch.randn(2, 4, D, generator=g, device=cuda).to(BF)
    length = torch.tensor([n, n - 1], dtype=torch.int32, device=cuda)
    lse = torch.empty(2, 4, device=cuda)
    out = nh.attention_decode(q, k, k, length, lse=lse)
    kp = torch.cat([k[0], k[1, :n - 1]])
    check(out, lse.t(), q, kp, kp, [1, 1], [n, n - 1], False, D ** -0.5)


def test_agrees_with_the_prompt_form(cuda):
    """The last row of a causal prompt is a decode step over its keys."""
    n, H, G, D = 333, 8, 2, 64
    g = torch.Generator(device=cuda).manual_seed(4)
    q = torch.randn(n, H, D, generator=g, device=cuda).to(BF)
    k, v = (torch.randn(n, G, D, generator=g, device=cuda).to(BF) for _ in range(2))
    off = torch.tensor([0, n], dtype=torch.int32, device=cuda)
    out, lse = nh.attention(q, k, v, off, off)
    one = nh.attention_decode(q[-1:], k[None], v[None], torch.tensor([n], dtype=torch.int32, device=cuda))
    # Both within their own bound of the same value: u (A + |o|) each.
    assert ((one[0].double() - out[-1].double()).abs() <= 4 * 2.0 ** -8 * v.double().abs().max()).all()

"""The attention and token-loss calls as a training step uses them, one behind
the other with nova.linear and its backward over packed sequences; the same
calls captured into graphs, on several streams and from several threads."""
import math
import threading

import pytest
import torch

import nova_hip as nh
from test_attention_gpu import check as check_attention
from test_attention_gpu import offsets

pytestmark = pytest.mark.gpu
F64, BF = torch.float64, torch.bfloat16
LENS, H, G, D, W, V = [70, 41, 130, 97], 4, 2, 64, 96, 211


def make(dev, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    T = sum(LENS)
    n = lambda *s, std=1.0: (std * torch.randn(*s, generator=g, device=dev)).to(BF)
    st = dict(x=n(T, W), wq=n(W, (H + 2 * G) * D, std=W ** -0.5), bq=n((H + 2 * G) * D, std=0.1),
              wo=n(H * D, V, std=2 * (H * D) ** -0.5), bo=n(V, std=0.1))
    st["y"] = torch.randint(0, V, (T,), generator=g, device=dev, dtype=torch.int32)
    st["y"][::5] = -1
    st["ref"] = 0.3 * torch.randn(4, generator=g, device=dev)
    st["off"] = offsets(LENS, dev)
    return st


def step(st, loss="preference"):
    """Forward, loss and the gradients of both weights; every intermediate."""
    T = st["x"].shape[0]
    r = {}
    r["qkv"] = nh.linear(st["x"], st["wq"], st["bq"])
    qkv = r["qkv"].view(T, H + 2 * G, D)
    q, k, v = qkv[:, :H], qkv[:, H:H + G], qkv[:, H + G:]
    r["o"], r["lse"] = nh.attention(q, k, v, st["off"], st["off"])
    o2 = r["o"].view(T, H * D)
    r["logits"] = nh.linear(o2, st["wo"], st["bo"])
    if loss == "preference":
        r["loss"], r["seq"], r["dlogits"] = nh.preference_loss(r["logits"], st["y"], st["off"], st["ref"],
                                                               beta=0.02)
    else:
        old = st["ref"].repeat_interleave(st["off"].diff().long(), output_size=T) - 5.0
        w = torch.full((T,), 1.0 / T, device=old.device)
        r["loss"], r["logp"], r["dlogits"] = nh.policy_loss(r["logits"], st["y"], old, old.sin(), w,
                                                            ref_logp=old, kl_coef=0.01)
    # (grad_bias holds the library's workspace of the stream.)
    do, r["dwo"], _ = nh.linear_backward(r["dlogits"], o2, st["wo"], out_dtype=BF,
                                         want=(True, True, False))
    r["do"] = do.view(T, H, D)
    r["dqkv"] = torch.empty_like(qkv)
    d = r["dqkv"]
    nh.attention_backward(r["do"], q, k, v, r["o"], r["lse"], st["off"], st["off"], dq=d[:, :H],
                          dk=d[:, H:H + G], dv=d[:, H + G:])
    _, r["dwq"], _ = nh.linear_backward(d.view(T, -1), st["x"], st["wq"], out_dtype=BF,
                                        want=(False, True, False))
    return r


def test_a_step_and_its_gradients(cuda):
    """Against autograd in 64 bits through the whole step.  Nine roundings to
    bf16 lie on the way to the last gradient (qkv, weights, out, logits,
    dlogits, do, weights and dS, dqkv, the result), each of relative size 2^-8 at
    most; dP - delta is a difference of terms up to about four times its size."""
    st = make(cuda)
    r = step(st)
    qkv = r["qkv"].view(-1, H + 2 * G, D)
    check_attention(r["o"], r["lse"], qkv[:, :H], qkv[:, H:H + G], qkv[:, H + G:], LENS, LENS, True,
                    D ** -0.5, "in the step")
    p = {k: st[k].double().requires_grad_() for k in ("wq", "wo")}
    qkv = (st["x"].double() @ p["wq"] + st["bq"].double()).view(-1, H + 2 * G, D)
    outs, a = [], 0
    for n in LENS:
        rows = []
        for h in range(H):
            s = torch.mm(qkv[a:a + n, h], qkv[a:a + n, H + h * G // H].t()) * D ** -0.5
            keep = torch.ones(n, n, dtype=torch.bool, device=cuda).tril()
            rows.append(torch.mm(torch.softmax(s.masked_fill(~keep, -math.inf), 1),
                                 qkv[a:a + n, H + G + h * G // H]))
        outs.append(torch.stack(rows, 1))
        a += n
    logits = torch.cat(outs).reshape(-1, H * D) @ p["wo"] + st["bo"].double()
    lp = torch.log_softmax(logits, 1).gather(1, st["y"].clamp(min=0).long()[:, None])[:, 0]
    lp = lp * (st["y"] >= 0)
    seq = torch.stack([t.sum() for t in lp.split(LENS)]) - st["ref"].double()
    loss = -torch.nn.functional.logsigmoid(0.02 * (seq[0::2] - seq[1::2])).mean()
    dwq, dwo = torch.autograd.grad(loss, (p["wq"], p["wo"]))
    u = 2.0 ** -8
    assert abs(r["loss"].item() - loss.item()) <= 4 * u * abs(loss.item())
    for got, want, n in ((r["dwo"], dwo, 5), (r["dwq"], dwq, 9 * 4)):
        rel = ((got.double() - want).norm() / want.norm()).item()
        assert rel <= n * u, (rel, n * u)


def equal(a, b):
    assert a.keys() == b.keys()
    for k in a:
        assert torch.equal(a[k], b[k]), k


@pytest.mark.parametrize("loss", ["preference", "policy"])
def test_two_graphs_of_one_stream_replayed_on_two(cuda, loss):
    """Captured on one stream and replayed side by side on two: the calls hold
    no workspace of the library's, so the graphs share nothing."""
    sts = [make(cuda, 1), make(cuda, 2)]
    side = torch.cuda.Stream()
    graphs, results = [], []
    with torch.cuda.stream(side):
        for st in sts:
            step(st, loss)
    torch.cuda.synchronize()
    for st in sts:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            results.append(step(st, loss))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for trial in range(3):
        fresh = [make(cuda, 10 * trial + i) for i in range(2)]
        for st, f in zip(sts, fresh):
            for k in st:
                st[k].copy_(f[k])
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for st, r in zip(sts, results):
            equal({k: v.clone() for k, v in r.items()}, step(st, loss))
            torch.cuda.synchronize()


def test_decode_in_a_graph_while_lengths_grow(cuda):
    B, S = 3, 700
    g = torch.Generator(device=cuda).manual_seed(0)
    k, v = (torch.randn(B, S, G, D, generator=g, device=cuda).to(BF) for _ in range(2))
    q = torch.randn(B, H, D, generator=g, device=cuda).to(BF)
    n = torch.tensor([1, 300, 640], dtype=torch.int32, device=cuda)
    nh.attention_decode(q, k, v, n)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = nh.attention_decode(q, k, v, n)
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, nh.attention_decode(q, k, v, n))
        q.copy_(torch.randn(B, H, D, generator=g, device=cuda))
        n += 13
    n.fill_(0)
    graph.replay()
    torch.cuda.synchronize()
    assert (out == 0).all()


def test_threads_on_own_and_on_one_stream(cuda):
    sts = [make(cuda, s) for s in range(4)]
    want = [{k: v.clone() for k, v in step(st).items()} for st in sts]
    torch.cuda.synchronize()
    one = torch.cuda.Stream()
    for shared in (False, True):
        got, errors = [None] * 4, []

        def work(i):
            try:
                with torch.cuda.stream(one if shared else torch.cuda.Stream()):
                    for _ in range(5):
                        got[i] = step(sts[i])
                    torch.cuda.current_stream().synchronize()
            except Exception as e:  # reported below, in the test's thread
                errors.append(e)

        ts = [threading.Thread(target=work, args=(i,)) for i in range(4)]
        for t in ts:
            t.start()
        for t in ts:
            t.join()
        assert not errors, errors
        for a, b in zip(got, want):
            equal(a, b)


def test_inputs_made_on_another_stream(cuda):
    """The call runs on torch's current stream: work queued there before it is
    seen, whatever stream the tensors come from."""
    st = make(cuda)
    want = step(st)["o"].clone()
    keep = st["x"].clone()
    st["x"].zero_()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        torch.cuda._sleep(2_000_000)
        st["x"].copy_(keep)
        got = step(st)["o"]
    s.synchronize()
    assert torch.equal(got, want)


def test_every_loss_twice_gives_the_same_bits(cuda):
    st = make(cuda, 3)
    for loss in ("preference", "policy"):
        equal(step(st, loss), step(st, loss))

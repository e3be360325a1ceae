"""Positions, norms, the paged cache and its attention as a server and a training
step call them, one behind the other with nova.linear; the same calls captured
into graphs, on several streams and from several threads."""
import math
import threading

import pytest
import torch

import nova_hip as nh
from test_attention_gpu import check as check_attention
from test_attention_gpu import offsets

pytestmark = pytest.mark.gpu
F64, BF = torch.float64, torch.bfloat16
H, G, D, W, PAGE = 4, 2, 64, 96, 16


def weights(dev, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    n = lambda *s, std=1.0: (std * torch.randn(*s, generator=g, device=dev)).to(BF)
    return dict(w=n(W, (H + 2 * G) * D, std=W ** -0.5), b=n((H + 2 * G) * D, std=0.1),
                wq=1 + 0.2 * n(D), wk=1 + 0.2 * n(D), f=nh.rotary_frequencies(D, factor=4.0, original=64))


def split(qkv):
    qkv = qkv.view(-1, H + 2 * G, D)
    return qkv[:, :H], qkv[:, H:H + G], qkv[:, H + G:]


def serve(m, x, pages, off, lens, table, most):
    """One step of a server: projection, norms, cache, attention."""
    q, k, v = split(nh.linear(x, m["w"], m["b"]))
    nh.qk_norm_rotary(q, k, m["wq"], m["wk"], q_out=q, k_out=k)
    nh.paged_append(k, v, pages[0], pages[1], off, lens, table, freqs=m["f"], q=q, q_out=q)
    return nh.paged_attention(q, pages[0], pages[1], off, lens, table, max_queries=most)


def test_prompts_then_tokens_against_packed_attention(cuda):
    """Three prompts in one step, then chunks and single tokens: every step's rows
    are those of the packed attention over all tokens so far."""
    m = weights(cuda)
    steps = [[37, 1, 70], [1, 1, 1], [5, 0, 40], [1, 30, 0], [1, 1, 1]]
    g = torch.Generator(device=cuda).manual_seed(1)
    pages = [torch.zeros(40, PAGE, G, D, dtype=BF, device=cuda) for _ in range(2)]
    table = torch.randperm(40, generator=g, device=cuda).int()[:36].view(3, 12)
    xs, have = [[] for _ in range(3)], [0, 0, 0]
    for new in steps:
        x = torch.randn(sum(new), W, generator=g, device=cuda).to(BF)
        for b, part in enumerate(x.split(new)):
            xs[b].append(part)
            have[b] += new[b]
        lens = torch.tensor(have, dtype=torch.int32, device=cuda)
        out = serve(m, x, pages, offsets(new, cuda), lens, table, max(new))
        # All tokens at once, by the calls of a training step.
        pos = torch.cat([torch.arange(n, device=cuda) for n in have]).int()
        q, k, v = split(nh.linear(torch.cat([torch.cat(p) for p in xs]), m["w"], m["b"]))
        nh.qk_norm_rotary(q, k, m["wq"], m["wk"], q_out=q, k_out=k)
        q, k = nh.rotary(q, pos, m["f"]), nh.rotary(k, pos, m["f"])
        last = torch.cat([torch.arange(e - n, e, device=cuda)
                          for n, e in zip(new, torch.tensor(have).cumsum(0).tolist())])
        check_attention(out, None, q[last], k, v, new, have, True, D ** -0.5, new)


LENS = [70, 41, 130]


def train(st):
    """Attention block of a training step and its gradients."""
    T = sum(LENS)
    r = {"qkv": nh.linear(st["x"], st["w"], st["b"])}
    q, k, v = split(r["qkv"])
    r["q"], r["k"] = nh.qk_norm_rotary(q, k, st["wq"], st["wk"], st["pos"], st["f"])
    r["o"], r["lse"] = nh.attention(r["q"], r["k"], v, st["off"], st["off"])
    d = r["dqkv"] = torch.empty_like(r["qkv"])
    dq, dk, dv = split(d)
    nh.attention_backward(st["do"], r["q"], r["k"], v, r["o"], r["lse"], st["off"], st["off"], dq=dq, dk=dk, dv=dv)
    _, _, r["dwq"], r["dwk"] = nh.qk_norm_rotary_backward(dq, dk, q, k, st["wq"], st["wk"], st["pos"], st["f"],
                                                          dq=dq, dk=dk)
    _, r["dw"], _ = nh.linear_backward(d.view(T, -1), st["x"], st["w"], out_dtype=BF, want=(False, True, False))
    return r


def training_state(dev, seed=0):
    st = weights(dev, seed)
    g = torch.Generator(device=dev).manual_seed(seed + 5)
    T = sum(LENS)
    st.update(x=torch.randn(T, W, generator=g, device=dev).to(BF), off=offsets(LENS, dev),
              do=torch.randn(T, H, D, generator=g, device=dev).to(BF),
              pos=torch.cat([torch.arange(n, device=dev) for n in LENS]).int())
    return st


def test_a_training_step_and_its_gradients(cuda):
    """Against autograd in 64 bits.  Eight roundings to bf16 lie on the way (qkv,
    q and k, weights, out, weights and dS, dq and dk, again, the result), each of
    relative size 2^-8 at most; dP - delta is a difference of terms up to four
    times its size."""
    st = training_state(cuda)
    r = train(st)
    p = {n: st[n].double().requires_grad_() for n in ("w", "wq", "wk")}
    q, k, v = split(st["x"].double() @ p["w"] + st["b"].double())
    t = st["pos"].double()[:, None, None] * st["f"].double()

    def placed(x, w):
        y = x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w
        a, b = y.chunk(2, -1)
        return torch.cat([a * t.cos() - b * t.sin(), b * t.cos() + a * t.sin()], -1)

    q, k = placed(q, p["wq"]), placed(k, p["wk"])
    loss, a = 0.0, 0
    for n in LENS:
        keep = torch.ones(n, n, dtype=torch.bool, device=cuda).tril()
        for h in range(H):
            s = torch.mm(q[a:a + n, h], k[a:a + n, h * G // H].t()) * D ** -0.5
            o = torch.mm(torch.softmax(s.masked_fill(~keep, -math.inf), 1), v[a:a + n, h * G // H])
            loss = loss + (o * st["do"][a:a + n, h].double()).sum()
        a += n
    want = torch.autograd.grad(loss, list(p.values()))
    for name, w in zip(("dw", "dwq", "dwk"), want):
        rel = ((r[name].double() - w).norm() / w.norm()).item()
        assert rel <= 8 * 4 * 2.0 ** -8, (name, rel)


def equal(a, b):
    for k in a:
        assert torch.equal(a[k], b[k]), k


def served(st):
    """A server's step on fresh pages, as a dict of everything it writes."""
    out = serve(st, st["x"], st["pages"], st["offs"], st["lens"], st["table"], max(st["new"]))
    return {"out": out, "k": st["pages"][0], "v": st["pages"][1]}


def server_state(dev, seed, new=(3, 1, 40), rows=(900, 2000, 40)):
    st = weights(dev, seed)
    g = torch.Generator(device=dev).manual_seed(seed + 9)
    n = sum(-(-r // PAGE) for r in rows)
    width = max(-(-r // PAGE) for r in rows)
    st["new"] = new
    st["x"] = torch.randn(sum(new), W, generator=g, device=dev).to(BF)
    st["pages"] = [torch.randn(n, PAGE, G, D, generator=g, device=dev).to(BF) for _ in range(2)]
    st["table"] = torch.zeros(len(rows), width, dtype=torch.int32, device=dev)
    at = 0
    for b, r in enumerate(rows):
        c = -(-r // PAGE)
        st["table"][b, :c] = torch.arange(at, at + c, device=dev)
        at += c
    st["offs"] = offsets(list(new), dev)
    st["lens"] = torch.tensor(rows, dtype=torch.int32, device=dev)
    return st


@pytest.mark.parametrize("step,make,fresh", [
    (train, training_state, "x"), (served, server_state, "x"),
    (served, lambda dev, seed: server_state(dev, seed, (1, 1, 1)), "x")])
def test_two_graphs_replayed_with_new_inputs(cuda, step, make, fresh):
    """Captured on one stream, replayed side by side on two, several times with new
    inputs and eager work between: every replay is the eager result."""
    sts, side = [make(cuda, 1), make(cuda, 2)], torch.cuda.Stream()
    with torch.cuda.stream(side):
        for st in sts:
            step(st)
    torch.cuda.synchronize()
    graphs, results = [], []
    for st in sts:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            results.append(step(st))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for turn in range(4):
        for i, st in enumerate(sts):
            g = torch.Generator(device=cuda).manual_seed(100 * turn + i)
            st[fresh].copy_(torch.randn(st[fresh].shape, generator=g, device=cuda))
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        got = [{k: v.clone() for k, v in r.items()} for r in results]
        for g, st in zip(got, sts):
            equal(g, step(st))
        torch.cuda.synchronize()


def test_threads_and_streams(cuda):
    makers = [(train, training_state(cuda, 3)), (served, server_state(cuda, 4)),
              (served, server_state(cuda, 5, (1, 1, 1))), (train, training_state(cuda, 6))]
    want = [{k: v.clone() for k, v in f(st).items()} for f, st in makers]
    torch.cuda.synchronize()
    got, errors = [None] * len(makers), []

    def work(i):
        try:
            f, st = makers[i]
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(5):
                    r = f(st)
                got[i] = {k: v.clone() for k, v in r.items()}
            s.synchronize()
        except Exception as e:  # reported by the main thread
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(makers))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for a, b in zip(got, want):
        equal(a, b)

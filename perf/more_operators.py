"""Rotary positions, norms of queries and keys, and the paged cache with the
attention that reads it, as a training or serving program calls them, over the
range of sizes those calls see.  Where ``own`` is false the operators are
computed in their plain form, elementary torch operations in 32 bits (angles
and long sums in 64) rounded once at the end.

Kinds (a case's "kind"):
  rotary           heads rotated by their token's position: half or interleaved
                   layout, the first values of a head or all, forward or
                   inverse (the gradient)
  qk_norm          RMS norm of each query and key head, then the rotation
  qk_norm_bwd      its gradients of queries, keys and both weights
  paged_append     new tokens' keys rotated and stored with their values in the
                   pages of a cache, their queries rotated
  paged_attention  a chunk of new tokens per sequence over the pages, causal
"""
import math
import os
import random
import sys

import torch

own = False

F64 = torch.float64
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6


def _nh():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                       "nova-compiler_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import nova_hip
    return nova_hip


# ---- cases ---------------------------------------------------------------------
# "seqs": new tokens and cache rows (the new ones among them) of each sequence.

_PROMPTS = "4096:4096,2049:2049,1023:1023,517:517,333:333,64:64,37:37,1:1"


def listed():
    lens = random.Random(8)
    cache = ",".join(f"1:{lens.randint(1500, 8192)}" for _ in range(31)) + ",1:8192"
    return [
        # One token of one sequence, the smallest call: latency.
        {"name": "rotary_bf16_1x8x64", "kind": "rotary", "dtype": "bf16", "tokens": 1, "heads": 8,
         "dim": 64, "rot": 64, "interleaved": False, "inverse": False, "fused": False, "far": 4096},
        # Queries and keys of packed prompts, where the projection left them.
        {"name": "rotary_bf16_8120x40x128", "kind": "rotary", "dtype": "bf16", "tokens": 8120, "heads": 40,
         "dim": 128, "rot": 128, "interleaved": False, "inverse": False, "fused": True, "far": 131072},
        # The training step's gradient, 8 x 1024 tokens of width 384, half of each head rotated.
        {"name": "rotary_grad_f32_8192x12x64", "kind": "rotary", "dtype": "f32", "tokens": 8192, "heads": 12,
         "dim": 64, "rot": 32, "interleaved": True, "inverse": True, "fused": False, "far": 1024},
        # 32 sequences' single tokens ...
        {"name": "qk_norm_bf16_32x32", "kind": "qk_norm", "dtype": "bf16", "tokens": 32, "heads": 32,
         "kv_heads": 8, "dim": 128, "rot": 128, "interleaved": False, "weight": "bf16", "fused": True,
         "far": 8192},
        # ... and packed prompts.
        {"name": "qk_norm_bf16_8120x32", "kind": "qk_norm", "dtype": "bf16", "tokens": 8120, "heads": 32,
         "kv_heads": 8, "dim": 128, "rot": 128, "interleaved": False, "weight": "bf16", "fused": True,
         "far": 4096},
        # The backward pass over packed prompts ...
        {"name": "qk_norm_bwd_bf16_8120x32", "kind": "qk_norm_bwd", "dtype": "bf16", "tokens": 8120,
         "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "interleaved": False, "weight": "f32",
         "fused": True, "far": 4096},
        # ... and of one short answer, heads of 80 of which 32 values are rotated.
        {"name": "qk_norm_bwd_f16_333x6", "kind": "qk_norm_bwd", "dtype": "f16", "tokens": 333, "heads": 6,
         "kv_heads": 6, "dim": 80, "rot": 32, "interleaved": True, "weight": "f16", "fused": False,
         "far": 1024},
        # One token of each of 32 sequences ...
        {"name": "append_bf16_32x1", "kind": "paged_append", "dtype": "bf16", "seqs": cache, "heads": 32,
         "kv_heads": 8, "dim": 128, "rot": 128, "interleaved": False, "page": 16, "by_head": False},
        # ... and prompts, into an empty cache.
        {"name": "append_bf16_prompts", "kind": "paged_append", "dtype": "bf16", "seqs": _PROMPTS,
         "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "interleaved": False, "page": 64,
         "by_head": False},
        # One token of one sequence: latency.
        {"name": "attention_f16_1x1000", "kind": "paged_attention", "dtype": "f16", "seqs": "1:1000",
         "heads": 6, "kv_heads": 6, "dim": 64, "page": 16, "room": 1024, "by_head": False},
        # One token of each of 32 sequences over long caches in pages of 16.
        {"name": "attention_bf16_32x8192", "kind": "paged_attention", "dtype": "bf16", "seqs": cache,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 16, "room": 8192, "by_head": False},
        # A server's step: chunks of prompts, a first prompt and single tokens together.
        {"name": "attention_bf16_mixed", "kind": "paged_attention", "dtype": "bf16",
         "seqs": "2048:2048,1024:5000,512:8192,129:4133,37:37,1:8000,1:333", "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "room": 8192, "by_head": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rotary", "qk_norm", "qk_norm_bwd", "paged_append", "paged_attention"])
    dim = rng.choice([32, 64, 80, 96, 128])
    kv = rng.choice([1, 2, 6, 8])
    heads = kv * rng.choice([1, 2, 4, 7]) if kv < 8 else 32
    case = {"kind": kind, "dtype": rng.choice(["bf16", "f16"])}
    if kind in ("rotary", "qk_norm", "qk_norm_bwd"):
        if rng.random() < 0.25:
            case["dtype"] = "f32"
        case.update(tokens=_log(rng, 1, 8192), heads=heads, dim=dim,
                    rot=rng.choice([dim, dim, dim // 16 * 8, 16]), interleaved=rng.random() < 0.4,
                    fused=rng.random() < 0.5, far=_log(rng, 1024, 131072))
        if kind == "rotary":
            case["inverse"] = rng.random() < 0.4
        else:
            case.update(kv_heads=kv, weight=rng.choice(["f32", case["dtype"]]))
        size = 4 if case["dtype"] == "f32" else 2
        while case["tokens"] * (heads + kv) * dim * size > 8120 * 40 * 128 * 2:
            case["tokens"] //= 2
        return case
    if kind == "paged_append":
        seqs, room = [], 8192
        for _ in range(_log(rng, 1, 32)):
            new = min(rng.choice([1, _log(rng, 1, 4096)]), room)
            if new == 0:
                break
            seqs.append((new, new + rng.choice([0, _log(rng, 1, 8192)])))
            room -= new
        case.update(rot=rng.choice([dim, dim, dim // 16 * 8, 16]), interleaved=rng.random() < 0.4)
    else:
        seqs, room, cost = [], 4096, 1.5e11 / (4 * heads * dim)
        single = rng.random() < 0.5
        for _ in range(_log(rng, 1, 32)):
            new = 1 if single else min(rng.choice([1, _log(rng, 1, 2048)]), room)
            if new == 0:
                break
            rows = new + rng.choice([0, _log(rng, 1, 8192 - new)])
            if new * rows > cost:
                continue
            seqs.append((new, rows))
            room -= new
            cost -= new * rows
        seqs = seqs or [(1, _log(rng, 1, 8192))]
        case["room"] = max(n for _, n in seqs) + rng.choice([0, 0, _log(rng, 1, 8192)])
    case.update(seqs=",".join(f"{a}:{b}" for a, b in seqs), heads=heads, kv_heads=kv, dim=dim,
                page=rng.choice([16, 16, 32, 48, 64, 128]), by_head=rng.random() < 0.5)
    return case


def _seqs(case):
    return [tuple(int(x) for x in s.split(":")) for s in case["seqs"].split(",")]


# ---- inputs ----------------------------------------------------------------------

def _freqs(rot, dev):
    return (10000.0 ** (-torch.arange(0, rot, 2, dtype=F64) / rot)).float().to(dev)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DT[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0, to=dt):
        x = torch.empty(shape, dtype=torch.float32, device=dev).normal_(mean, std, generator=g)
        return x.to(to)

    st = {"case": case}
    kind, H, D = case["kind"], case["heads"], case["dim"]
    if kind in ("rotary", "qk_norm", "qk_norm_bwd"):
        T, G = case["tokens"], case.get("kv_heads", 0)
        st["freqs"] = _freqs(case["rot"], dev)
        # Sequences packed one behind the other start at positions of their own.
        start = torch.randint(0, case["far"], (1 + T // 512,), generator=g, device=dev)
        t = torch.arange(T, device=dev)
        st["positions"] = ((start[t // 512] + t % 512) % case["far"]).int()
        if case["fused"]:  # in the output of one projection, values behind them
            x = normal(T, H + 2 * max(G, 1), D)
            st["x"], st["q"], st["k"] = x[:, :H], x[:, :H], x[:, H:H + G]
        else:
            st["x"] = st["q"] = normal(T, H, D)
            st["k"] = normal(T, G, D)
        if kind != "rotary":
            st["wq"], st["wk"] = (normal(D, std=0.2, mean=1.0, to=DT[case["weight"]]) for _ in range(2))
        if kind == "qk_norm_bwd":
            st["gq"], st["gk"] = normal(T, H, D), normal(T, G, D)
        return st
    seqs, G, P = _seqs(case), case["kv_heads"], case["page"]
    T = sum(n for n, _ in seqs)
    need = [-(-rows // P) for _, rows in seqs]
    width = max(-(-case.get("room", 0) // P), max(need))
    pool = sum(need) + 3
    order = torch.randperm(pool, generator=g, device=dev).int()
    table = torch.full((len(seqs), width), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    st["table"] = table
    off = [0]
    for n, _ in seqs:
        off.append(off[-1] + n)
    st["offsets"] = torch.tensor(off, dtype=torch.int32, device=dev)
    st["lengths"] = torch.tensor([rows for _, rows in seqs], dtype=torch.int32, device=dev)
    if case["by_head"]:
        st["kp"], st["vp"] = (normal(pool, G, P, D).transpose(1, 2) for _ in range(2))
    else:
        st["kp"], st["vp"] = normal(pool, P, G, D), normal(pool, P, G, D)
    qkv = normal(T, H + 2 * G, D)
    st["q"], st["k"], st["v"] = qkv[:, :H], qkv[:, H:H + G], qkv[:, H + G:]
    if kind == "paged_append":
        st["freqs"] = _freqs(case["rot"], dev)
    else:
        st["q"], st["scale"] = st["q"].contiguous(), 1.0 / math.sqrt(D)
    return st


# ---- plain forms -------------------------------------------------------------------

def _rotate(x, positions, freqs, interleaved, inverse=False):
    """x [tokens, heads, D] f32 with its first 2 len(freqs) values rotated."""
    angle = positions.double()[:, None] * freqs.double()
    c, s = angle.cos().float()[:, None], angle.sin().float()[:, None]
    if inverse:
        s = -s
    rot, rest = x[..., :2 * len(freqs)], x[..., 2 * len(freqs):]
    if interleaved:
        a, b = rot[..., 0::2], rot[..., 1::2]
        y = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    else:
        a, b = rot[..., :len(freqs)], rot[..., len(freqs):]
        y = torch.cat([a * c - b * s, b * c + a * s], -1)
    return torch.cat([y, rest], -1)


def _norm_plain(st, x, w):
    case, xf = st["case"], x.float()
    y = xf * ((xf * xf).mean(-1, keepdim=True) + EPS).rsqrt() * w.float()
    return _rotate(y, st["positions"], st["freqs"], case["interleaved"]).to(x.dtype)


def _norm_bwd_plain(st, grad, x, w):
    xf, wf = x.float(), w.float()
    r = ((xf * xf).mean(-1, keepdim=True) + EPS).rsqrt()
    g = _rotate(grad.float(), st["positions"], st["freqs"], st["case"]["interleaved"], inverse=True)
    n = xf * r
    dw = (g * n).sum(1).double().sum(0).float()
    t = g * wf
    dx = r * (t - n * (t * n).mean(-1, keepdim=True))
    return dx.to(x.dtype), dw


def _slots(st):
    """Page, row in it and position of every new token."""
    P, page, row, pos = st["case"]["page"], [], [], []
    for b, (new, rows) in enumerate(_seqs(st["case"])):
        at = torch.arange(rows - new, rows, device=st["table"].device)
        page.append(st["table"][b].long()[at // P])
        row.append(at % P)
        pos.append(at)
    return torch.cat(page), torch.cat(row), torch.cat(pos)


def _append_plain(st):
    page, row, pos = _slots(st)
    q, k = (_rotate(st[n].float(), pos, st["freqs"], st["case"]["interleaved"]).to(st[n].dtype)
            for n in ("q", "k"))
    st["kp"][page, row] = k
    st["vp"][page, row] = st["v"]
    return q, st["kp"], st["vp"]


def _rows(st, name, b, rows):
    """The first rows of a sequence's pages, [kv heads, rows, dim]."""
    P = st["case"]["page"]
    pages = st["table"][b, :-(-rows // P)].long()
    return st[name][pages].flatten(0, 1)[:rows].transpose(0, 1)


def _paged_plain(st):
    case, q = st["case"], st["q"]
    rep, D, start = case["heads"] // case["kv_heads"], case["dim"], 0
    out = torch.empty_like(q)
    for b, (new, rows) in enumerate(_seqs(case)):
        k, v = _rows(st, "kp", b, rows).float(), _rows(st, "vp", b, rows).float()
        qs = q[start:start + new].float().unflatten(1, (-1, rep)).permute(1, 2, 0, 3).reshape(len(k), -1, D)
        seen = torch.arange(rows, device=q.device) <= torch.arange(rows - new, rows, device=q.device)[:, None]
        for h in range(len(k)):
            x = (qs[h] @ k[h].t().contiguous() * st["scale"]).unflatten(0, (rep, new))
            x = x.masked_fill(~seen, -math.inf)
            p = (x - x.amax(-1, keepdim=True)).exp_()
            o = (p @ v[h]) / p.sum(-1, keepdim=True)
            out[start:start + new, h * rep:(h + 1) * rep] = o.transpose(0, 1).to(q.dtype)
        start += new
    return out


# ---- one pass ------------------------------------------------------------------------

def run(state):
    st, case = state, state["case"]
    kind = case["kind"]
    if not own:
        if kind == "rotary":
            return _rotate(st["x"].float(), st["positions"], st["freqs"], case["interleaved"],
                           case["inverse"]).to(st["x"].dtype)
        if kind == "qk_norm":
            return _norm_plain(st, st["q"], st["wq"]), _norm_plain(st, st["k"], st["wk"])
        if kind == "qk_norm_bwd":
            dq, dwq = _norm_bwd_plain(st, st["gq"], st["q"], st["wq"])
            dk, dwk = _norm_bwd_plain(st, st["gk"], st["k"], st["wk"])
            return dq, dk, dwq, dwk
        return _append_plain(st) if kind == "paged_append" else _paged_plain(st)
    nh = _nh()
    if kind == "rotary":
        return nh.rotary(st["x"], st["positions"], st["freqs"], interleaved=case["interleaved"],
                         inverse=case["inverse"])
    if kind == "qk_norm":
        return nh.qk_norm_rotary(st["q"], st["k"], st["wq"], st["wk"], st["positions"], st["freqs"],
                                 eps=EPS, interleaved=case["interleaved"])
    if kind == "qk_norm_bwd":
        return nh.qk_norm_rotary_backward(st["gq"], st["gk"], st["q"], st["k"], st["wq"], st["wk"],
                                          st["positions"], st["freqs"], eps=EPS,
                                          interleaved=case["interleaved"])
    if kind == "paged_append":
        q = nh.paged_append(st["k"], st["v"], st["kp"], st["vp"], st["offsets"], st["lengths"],
                            st["table"], freqs=st["freqs"], interleaved=case["interleaved"], q=st["q"])
        return q, st["kp"], st["vp"]
    # A server knows the longest chunk of its step.
    return nh.paged_attention(st["q"], st["kp"], st["vp"], st["offsets"], st["lengths"], st["table"],
                              scale=st["scale"], max_queries=max(n for n, _ in _seqs(case)))


# ---- what a pass cannot do without ------------------------------------------------------

def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    kind, H, D = case["kind"], case["heads"], case["dim"]
    if kind == "rotary":
        n = case["tokens"] * H
        return {"bytes": 2 * n * D * size + 4 * case["tokens"], "flops": 3 * n * case["rot"]}
    if kind in ("qk_norm", "qk_norm_bwd"):
        n = case["tokens"] * (H + case["kv_heads"])
        back = kind == "qk_norm_bwd"
        return {"bytes": (3 if back else 2) * n * D * size + 4 * case["tokens"],
                "flops": n * ((11 if back else 4) * D + 3 * case["rot"])}
    seqs, G = _seqs(case), case["kv_heads"]
    T = sum(n for n, _ in seqs)
    if kind == "paged_append":
        return {"bytes": 2 * T * (H + 2 * G) * D * size, "flops": 3 * T * (H + G) * case["rot"]}
    pairs = sum(n * rows - n * (n - 1) // 2 for n, rows in seqs)
    return {"bytes": (2 * T * H + 2 * G * sum(rows for _, rows in seqs)) * D * size,
            "flops": 4 * D * H * pairs}


# ---- 64 bits -------------------------------------------------------------------------------

def _turned(x, positions, freqs, interleaved, sign=1.0):
    """Pairs as complex numbers times exp(i angle)."""
    n = len(freqs)
    turn = torch.polar(torch.ones(len(x), 1, n, dtype=F64, device=x.device),
                       sign * positions.double()[:, None, None] * freqs.double())
    y = x.double().clone()
    at = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if interleaved else (slice(0, n), slice(n, 2 * n))
    z = torch.complex(y[..., at[0]], y[..., at[1]]) * turn
    y[..., at[0]], y[..., at[1]] = z.real, z.imag
    return y


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "rotary":
        return _turned(st["x"], st["positions"], st["freqs"], case["interleaved"],
                       -1.0 if case["inverse"] else 1.0)
    if kind in ("qk_norm", "qk_norm_bwd"):
        back, first, second = kind == "qk_norm_bwd", [], []
        for x, w, grad in ((st["q"], st["wq"], st.get("gq")), (st["k"], st["wk"], st.get("gk"))):
            x, w = x.double().requires_grad_(back), w.double().requires_grad_(back)
            y = x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS) * w
            if not back:
                first.append(_turned(y, st["positions"], st["freqs"], case["interleaved"]))
                continue
            # A rotation's transpose is its inverse.
            up = _turned(grad, st["positions"], st["freqs"], case["interleaved"], -1.0)
            dx, dw = torch.autograd.grad(y, (x, w), up)
            first.append(dx)
            second.append(dw)
        return tuple(first + second)
    if kind == "paged_append":
        q, k, v, kp, vp = (st[n].double() for n in ("q", "k", "v", "kp", "vp"))
        table, t, pos = st["table"].tolist(), 0, []
        for new, rows in _seqs(case):
            pos += range(rows - new, rows)
        pos = torch.tensor(pos, device=q.device)
        q, k = (_turned(x, pos, st["freqs"], case["interleaved"]) for x in (q, k))
        P = case["page"]
        for b, (new, rows) in enumerate(_seqs(case)):
            at = rows - new
            while at < rows:  # a run inside one page
                n = min(P - at % P, rows - at)
                page = table[b][at // P]
                kp[page, at % P:at % P + n], vp[page, at % P:at % P + n] = k[t:t + n], v[t:t + n]
                at, t = at + n, t + n
        return q, kp, vp
    H, G = case["heads"], case["kv_heads"]
    out, start = torch.zeros(st["q"].shape, dtype=F64, device=st["q"].device), 0
    for b, (new, rows) in enumerate(_seqs(case)):
        last = torch.arange(new, device=out.device) + (rows - new)
        hidden = torch.arange(rows, device=out.device)[None, :] > last[:, None]
        for h in range(H):
            if h % (H // G) == 0:
                k, v = (_rows(st, n, b, rows)[h * G // H].double() for n in ("kp", "vp"))
            x = torch.mm(st["q"][start:start + new, h].double(), k.t().contiguous()) * st["scale"]
            x[hidden] = -math.inf
            out[start:start + new, h] = torch.mm(torch.softmax(x, 1), v)
        start += new
    return out

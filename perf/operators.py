"""Attention over packed sequences and the losses of preference and policy
training, as a training or serving program calls them, over the range of sizes
those calls see.  Where ``own`` is false the operators are computed in their
plain form, elementary torch operations in 32 bits rounded once at the end.

Kinds (a case's "kind"):
  attention        softmax(scale Q K^T) V of sequences packed one behind the
                   other, causal or not, heads shared by groups; outputs the
                   result and the rows' log-sum-exp
  attention_bwd    its gradients of Q, K and V, from the forward's outputs
  attention_decode one query per sequence over a padded cache of given lengths
  token_logp       the log-probability of each row's label
  policy           the clipped policy loss with a KL term over tokens, and the
                   gradient of the logits
  preference       the paired log-ratio loss over packed (chosen, rejected)
                   sequences, and the gradient of the logits
"""
import math
import os
import random
import sys

import torch

own = False

F64 = torch.float64
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BETA, SMOOTHING = 0.1, 0.05           # preference loss
CLIP_LOW, CLIP_HIGH, KL = 0.2, 0.28, 0.04  # policy loss


def _nh():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                       "nova-compiler_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import nova_hip
    return nova_hip


# ---- cases ---------------------------------------------------------------------

_RAGGED = "4096,2049,1023,517,333,64,37,1"


def listed():
    lens = random.Random(8)
    cache = ",".join(str(lens.randint(1500, 8192)) for _ in range(31)) + ",8192"
    return [
        # One layer's attention of 8 images x 12 heads of 64 over 197 tokens.
        {"name": "attention_f16_8x197", "kind": "attention", "dtype": "f16", "lens": ",".join(["197"] * 8),
         "heads": 12, "kv_heads": 12, "dim": 64, "causal": False, "fused": False},
        # One layer of 4096 columns over prompts packed without padding.
        {"name": "attention_bf16_ragged", "kind": "attention", "dtype": "bf16", "lens": _RAGGED,
         "heads": 32, "kv_heads": 8, "dim": 128, "causal": True, "fused": True},
        # The training step's attention, 8 x 1024 tokens of width 384 ...
        {"name": "attention_bwd_bf16_8x1024", "kind": "attention_bwd", "dtype": "bf16",
         "lens": ",".join(["1024"] * 8), "heads": 6, "kv_heads": 6, "dim": 64, "causal": True,
         "fused": True},
        # ... and of packed prompts with heads in groups of four.
        {"name": "attention_bwd_bf16_ragged", "kind": "attention_bwd", "dtype": "bf16", "lens": _RAGGED,
         "heads": 32, "kv_heads": 8, "dim": 128, "causal": True, "fused": False},
        # One token of one sequence: latency.
        {"name": "decode_bf16_1x1000", "kind": "attention_decode", "dtype": "bf16", "lens": "1000",
         "cache": 1024, "heads": 6, "kv_heads": 6, "dim": 64, "bhsd": False},
        # One token of each of 32 sequences over a long cache.
        {"name": "decode_bf16_32x8192", "kind": "attention_decode", "dtype": "bf16", "lens": cache,
         "cache": 8192, "heads": 32, "kv_heads": 8, "dim": 128, "bhsd": True},
        # The reference model's log-probabilities of a batch ...
        {"name": "token_logp_bf16_4096x32000", "kind": "token_logp", "dtype": "bf16", "rows": 4096,
         "classes": 32000, "masked": 0.3},
        # ... and of one short answer.
        {"name": "token_logp_f32_61x50304", "kind": "token_logp", "dtype": "f32", "rows": 61,
         "classes": 50304, "masked": 0.0},
        # A policy step over 8 x 1024 tokens of the training step's vocabulary ...
        {"name": "policy_f32_8192x50304", "kind": "policy", "dtype": "f32", "rows": 8192,
         "classes": 50304, "masked": 0.2, "kl": True},
        # ... and a small micro-batch without the KL term.
        {"name": "policy_bf16_64x32000", "kind": "policy", "dtype": "bf16", "rows": 64,
         "classes": 32000, "masked": 0.2, "kl": False},
        # Preference pairs packed into 8 x 1024 rows ...
        {"name": "preference_bf16_8192x50304", "kind": "preference", "dtype": "bf16",
         "lens": "1024,777,1001,1024,513,400,600,853,300,301,1000,399", "classes": 50304, "masked": 0.3},
        # ... and one pair of short answers.
        {"name": "preference_f32_212x32000", "kind": "preference", "dtype": "f32", "lens": "97,115",
         "classes": 32000, "masked": 0.3},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention", "attention_bwd", "attention_decode", "token_logp", "policy",
                       "preference"])
    if kind in ("attention", "attention_bwd"):
        # Up to 16 sequences of 1 to 4096 tokens, 8192 in all.
        lens, room = [], 8192
        for _ in range(_log(rng, 1, 16)):
            n = min(_log(rng, 1, 4096), room)
            if n == 0:
                break
            lens.append(n)
            room -= n
        kv = rng.choice([1, 2, 6, 8])
        heads, dim, causal = kv * rng.choice([1, 2, 3, 4]), rng.choice([32, 64, 80, 96, 128]), rng.random() < 0.75
        cost = (1 if causal else 2) * heads * dim
        while sum(n * n for n in lens) * cost > 9e10:  # no more than the largest listed case
            lens.remove(max(lens))
        return {"kind": kind, "dtype": rng.choice(["bf16", "f16"]), "lens": ",".join(map(str, lens)),
                "heads": heads, "kv_heads": kv, "dim": dim, "causal": causal,
                "fused": rng.random() < 0.5}
    if kind == "attention_decode":
        cache, batch = _log(rng, 16, 8192), _log(rng, 1, 32)
        kv = rng.choice([1, 2, 6, 8])
        return {"kind": kind, "dtype": rng.choice(["bf16", "f16"]),
                "lens": ",".join(str(_log(rng, 1, cache)) for _ in range(batch)), "cache": cache,
                "heads": kv * rng.choice([1, 2, 4, 7, 8]) if kv < 8 else 32, "kv_heads": kv,
                "dim": rng.choice([32, 64, 80, 96, 128]), "bhsd": rng.random() < 0.5}
    dtype = rng.choice(["f32", "bf16", "f16"])
    classes = rng.choice([50304, 32000, _log(rng, 100, 50304), _log(rng, 10000, 50304)])
    masked = rng.choice([0.0, 0.2, 0.5])
    if kind == "preference":
        lens = [_log(rng, 1, 1024) for _ in range(2 * _log(rng, 1, 6))]
        while sum(lens) > 8192:
            lens = lens[:-2]
        return {"kind": kind, "dtype": dtype, "lens": ",".join(map(str, lens)), "classes": classes,
                "masked": masked}
    case = {"kind": kind, "dtype": dtype, "rows": _log(rng, 1, 8192), "classes": classes,
            "masked": masked}
    if kind == "policy":
        case["kl"] = rng.random() < 0.6
    return case


def _lens(case):
    return [int(n) for n in case["lens"].split(",")]


# ---- inputs ----------------------------------------------------------------------

def _offsets(lens, device):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device=device)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DT[case["dtype"]]

    def normal(*shape, std=1.0, to=dt):
        x = torch.empty(shape, dtype=torch.float32, device=dev).normal_(0.0, std, generator=g)
        return x.to(to)

    st = {"case": case}
    if case["kind"] in ("attention", "attention_bwd"):
        lens = _lens(case)
        T, H, G, D = sum(lens), case["heads"], case["kv_heads"], case["dim"]
        if case["fused"]:  # the three parts of one projection's output
            qkv = normal(T, H + 2 * G, D)
            st["q"], st["k"], st["v"] = qkv[:, :H], qkv[:, H:H + G], qkv[:, H + G:]
        else:
            st["q"], st["k"], st["v"] = normal(T, H, D), normal(T, G, D), normal(T, G, D)
        st["offsets"], st["scale"] = _offsets(lens, dev), 1.0 / math.sqrt(D)
        if case["kind"] == "attention_bwd":
            st["out"], st["lse"] = _attention_plain(st)
            st["grad_out"] = normal(T, H, D)
    elif case["kind"] == "attention_decode":
        lens = _lens(case)
        B, S, H, G, D = len(lens), case["cache"], case["heads"], case["kv_heads"], case["dim"]
        st["q"] = normal(B, H, D)
        if case["bhsd"]:
            st["k"], st["v"] = (normal(B, G, S, D).transpose(1, 2) for _ in range(2))
        else:
            st["k"], st["v"] = normal(B, S, G, D), normal(B, S, G, D)
        st["lengths"] = torch.tensor(lens, dtype=torch.int32, device=dev)
        st["scale"] = 1.0 / math.sqrt(D)
    else:
        pref = case["kind"] == "preference"
        lens = _lens(case) if pref else None
        R, C = sum(lens) if pref else case["rows"], case["classes"]
        x = normal(R, C, std=2.0)
        labels = torch.randint(0, C, (R,), generator=g, device=dev, dtype=torch.int32)
        # A trained model gives its labels far more than their share.
        rows = torch.arange(R, device=dev)
        x[rows, labels.long()] += 8.0
        labels[torch.rand(R, generator=g, device=dev) < case["masked"]] = -1  # prompts and padding
        st["logits"], st["labels"] = x, labels
        if case["kind"] == "policy":
            lp, _ = _token_logp_plain(x, labels)
            step = torch.empty(R, dtype=torch.float32, device=dev).normal_(0.0, 0.15, generator=g)
            # Ratios keep off the points where the clip's gradient jumps.
            for edge in (math.log(1.0 - CLIP_LOW), math.log(1.0 + CLIP_HIGH)):
                near = (step - edge).abs() < 2e-3
                step = torch.where(near, torch.full_like(step, edge + 4e-3), step)
            st["old_logp"] = lp - step
            st["ref_logp"] = lp + torch.empty_like(lp).normal_(0.0, 0.2, generator=g) if case["kl"] else None
            st["advantage"] = torch.empty_like(lp).normal_(0.0, 1.0, generator=g)
            valid = labels >= 0
            st["weight"] = valid.float() / valid.sum().clamp(min=1)
        if pref:
            st["offsets"] = _offsets(lens, dev)
            lp, _ = _token_logp_plain(x, labels)
            ref = torch.stack([p.sum() for p in lp.split(lens)])
            st["ref_logp"] = ref + torch.empty_like(ref).normal_(0.0, 8.0, generator=g)
    return st


# ---- plain forms -------------------------------------------------------------------

def _blocks(case, budget=1 << 28):
    """(first token, one past the last, kv heads' slice) per block of scores."""
    G, rep = case["kv_heads"], case["heads"] // case["kv_heads"]
    s = 0
    for n in _lens(case):
        step = max(1, min(G, budget // max(1, n * n * rep)))
        for h in range(0, G, step):
            yield s, s + n, h, min(G, h + step)
        s += n


def _grouped(t, s, e, h0, h1, rep, dtype):
    """Rows s:e of heads h0*rep:h1*rep as [kv heads, rep, rows, dim]."""
    x = t[s:e, h0 * rep:h1 * rep].to(dtype)
    return x.reshape(e - s, h1 - h0, rep, -1).permute(1, 2, 0, 3).contiguous()


def _scores(st, s, e, h0, h1, rep, dtype):
    q = _grouped(st["q"], s, e, h0, h1, rep, dtype)
    k = _grouped(st["k"], s, e, h0, h1, 1, dtype)
    x = (q @ k.transpose(2, 3).contiguous()) * st["scale"]
    if st["case"]["causal"]:
        n = e - s
        keep = torch.ones(n, n, dtype=torch.bool, device=x.device).tril_()
        x = x.masked_fill(~keep, -math.inf)
    return q, k, x


def _attention_plain(st):
    case, q = st["case"], st["q"]
    H, rep = case["heads"], case["heads"] // case["kv_heads"]
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(H, q.shape[0], dtype=torch.float32, device=q.device)
    for s, e, h0, h1 in _blocks(case):
        _, _, x = _scores(st, s, e, h0, h1, rep, torch.float32)
        v = _grouped(st["v"], s, e, h0, h1, 1, torch.float32)
        m = x.amax(-1, keepdim=True)
        p = (x - m).exp_()
        l = p.sum(-1, keepdim=True)
        o = (p @ v) / l
        out[s:e, h0 * rep:h1 * rep] = o.permute(2, 0, 1, 3).reshape(e - s, -1, o.shape[-1]).to(q.dtype)
        lse[h0 * rep:h1 * rep, s:e] = (m + l.log()).reshape(-1, e - s)
    return out, lse


def _attention_bwd_plain(st):
    case, q, k = st["case"], st["q"], st["k"]
    rep = case["heads"] // case["kv_heads"]
    dq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    dk, dv = (torch.empty(k.shape, dtype=q.dtype, device=q.device) for _ in range(2))
    for s, e, h0, h1 in _blocks(case, 1 << 27):
        qs, ks, x = _scores(st, s, e, h0, h1, rep, torch.float32)
        v = _grouped(st["v"], s, e, h0, h1, 1, torch.float32)
        go = _grouped(st["grad_out"], s, e, h0, h1, rep, torch.float32)
        o = _grouped(st["out"], s, e, h0, h1, rep, torch.float32)
        p = (x - st["lse"][h0 * rep:h1 * rep, s:e].reshape(h1 - h0, rep, e - s, 1)).exp_()
        ds = go @ v.transpose(2, 3).contiguous()
        ds = (ds - (go * o).sum(-1, keepdim=True)) * p * st["scale"]
        gq = ds @ ks
        gk = (ds.transpose(2, 3).contiguous() @ qs).sum(1)
        gv = (p.transpose(2, 3).contiguous() @ go).sum(1)
        dq[s:e, h0 * rep:h1 * rep] = gq.permute(2, 0, 1, 3).reshape(e - s, -1, gq.shape[-1]).to(q.dtype)
        dk[s:e, h0:h1] = gk.transpose(0, 1).to(q.dtype)
        dv[s:e, h0:h1] = gv.transpose(0, 1).to(q.dtype)
    return dq, dk, dv


def _attention_decode_plain(st):
    case, q = st["case"], st["q"]
    G, rep, D = case["kv_heads"], case["heads"] // case["kv_heads"], case["dim"]
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    for b, n in enumerate(_lens(case)):
        qs = q[b].float().reshape(G, rep, D)
        k = st["k"][b, :n].float().permute(1, 2, 0).contiguous()
        v = st["v"][b, :n].float().transpose(0, 1).contiguous()
        x = (qs @ k) * st["scale"]
        p = (x - x.amax(-1, keepdim=True)).exp_()
        out[b] = ((p @ v) / p.sum(-1, keepdim=True)).reshape(-1, D).to(q.dtype)
    return out


def _token_logp_plain(logits, labels):
    x = logits.float()
    m = x.amax(1, keepdim=True)
    lse = m[:, 0] + (x - m).exp_().sum(1).log()
    at = x.gather(1, labels.clamp(min=0).long()[:, None])[:, 0]
    lp = torch.where(labels >= 0, at - lse, torch.zeros_like(at))
    return lp, lse


def _logits_grad(st, lse, coef):
    """coef[row] (onehot(label) - softmax), zero in rows without a label."""
    x, labels = st["logits"], st["labels"]
    coef = torch.where(labels >= 0, coef, torch.zeros_like(coef))
    grad = (x.float() - lse[:, None]).exp_().mul_(-coef[:, None])
    grad.scatter_add_(1, labels.clamp(min=0).long()[:, None], coef[:, None])
    return grad.to(x.dtype)


def _policy_plain(st):
    lp, lse = _token_logp_plain(st["logits"], st["labels"])
    adv, w = st["advantage"], st["weight"]
    ratio = (lp - st["old_logp"]).exp()
    plain = ratio * adv
    clipped = ratio.clamp(1.0 - CLIP_LOW, 1.0 + CLIP_HIGH) * adv
    loss = -torch.minimum(plain, clipped)
    coef = torch.where(plain <= clipped, -plain, torch.zeros_like(plain))
    if st["ref_logp"] is not None:
        d = st["ref_logp"] - lp
        loss = loss + KL * (d.exp() - d - 1.0)
        coef = coef + KL * (1.0 - d.exp())
    loss = torch.where(st["labels"] >= 0, loss * w, torch.zeros_like(loss))
    total = loss.double().sum().float().reshape(1)
    return total, lp, _logits_grad(st, lse, coef * w)


def _preference_plain(st):
    lens = _lens(st["case"])
    lp, lse = _token_logp_plain(st["logits"], st["labels"])
    seq = torch.stack([p.double().sum() for p in lp.split(lens)])
    r = (seq - st["ref_logp"].double()).reshape(-1, 2)
    h = BETA * (r[:, 0] - r[:, 1])
    n = h.shape[0]
    soft = torch.log1p(torch.exp(-h.abs()))
    loss = ((1.0 - SMOOTHING) * (soft + (-h).clamp(min=0)) + SMOOTHING * (soft + h.clamp(min=0))).sum() / n
    sig = 1.0 / (1.0 + torch.exp(h))  # sigmoid(-h)
    c = BETA * (SMOOTHING * (1.0 - sig) - (1.0 - SMOOTHING) * sig) / n
    per_seq = torch.stack([c, -c], 1).reshape(-1)
    coef = torch.cat([per_seq[i].float().expand(k) for i, k in enumerate(lens)])
    return loss.float().reshape(1), seq.float(), _logits_grad(st, lse, coef)


# ---- one pass ------------------------------------------------------------------------

def run(state):
    st, kind = state, state["case"]["kind"]
    if not own:
        if kind == "attention":
            return _attention_plain(st)
        if kind == "attention_bwd":
            return _attention_bwd_plain(st)
        if kind == "attention_decode":
            return _attention_decode_plain(st)
        if kind == "token_logp":
            return _token_logp_plain(st["logits"], st["labels"])[0]
        return _policy_plain(st) if kind == "policy" else _preference_plain(st)
    nh = _nh()
    if kind == "attention":
        return nh.attention(st["q"], st["k"], st["v"], st["offsets"], st["offsets"],
                            causal=st["case"]["causal"], scale=st["scale"])
    if kind == "attention_bwd":
        return nh.attention_backward(st["grad_out"], st["q"], st["k"], st["v"], st["out"], st["lse"],
                                     st["offsets"], st["offsets"], causal=st["case"]["causal"],
                                     scale=st["scale"])
    if kind == "attention_decode":
        return nh.attention_decode(st["q"], st["k"], st["v"], st["lengths"], scale=st["scale"])
    if kind == "token_logp":
        return nh.token_logp(st["logits"], st["labels"])
    if kind == "policy":
        return nh.policy_loss(st["logits"], st["labels"], st["old_logp"], st["advantage"],
                              st["weight"], ref_logp=st["ref_logp"], clip=(CLIP_LOW, CLIP_HIGH),
                              kl_coef=KL if st["ref_logp"] is not None else 0.0)
    return nh.preference_loss(st["logits"], st["labels"], st["offsets"], st["ref_logp"], beta=BETA,
                              smoothing=SMOOTHING)


# ---- what a pass cannot do without ------------------------------------------------------

def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    kind = case["kind"]
    if kind in ("attention", "attention_bwd"):
        lens, H, G, D = _lens(case), case["heads"], case["kv_heads"], case["dim"]
        T = sum(lens)
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lens)
        q, kv, lse = T * H * D * size, 2 * T * G * D * size, 4 * T * H
        if kind == "attention":
            return {"bytes": 2 * q + kv + lse, "flops": 4 * D * H * pairs}
        return {"bytes": 4 * q + 2 * kv + lse, "flops": 10 * D * H * pairs}
    if kind == "attention_decode":
        n, H, G, D = sum(_lens(case)), case["heads"], case["kv_heads"], case["dim"]
        return {"bytes": (2 * n * G * D + 2 * len(_lens(case)) * H * D) * size, "flops": 4 * n * H * D}
    R = sum(_lens(case)) if kind == "preference" else case["rows"]
    C = case["classes"]
    read = int(R * (1.0 - case["masked"])) * C * size
    if kind == "token_logp":
        return {"bytes": read + 8 * R, "flops": 4 * read // size}
    return {"bytes": read + R * C * size + 24 * R, "flops": 8 * read // size}


# ---- 64 bits -------------------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind in ("attention", "attention_bwd"):
        return _attention_exact(st)
    if kind == "attention_decode":
        return _decode_exact(st)
    x, y = st["logits"], st["labels"].long()
    R, C = x.shape
    lp = torch.zeros(R, dtype=F64, device=x.device)
    rows = (y >= 0).nonzero()[:, 0]
    for part in rows.split(1024):
        z = torch.log_softmax(x[part].double(), 1)
        lp[part] = z[torch.arange(len(part), device=x.device), y[part]]
    if kind == "token_logp":
        return lp
    slope = torch.zeros_like(lp)
    if kind == "policy":
        u = lp[rows].requires_grad_()
        adv, w = st["advantage"].double()[rows], st["weight"].double()[rows]
        ratio = torch.exp(u - st["old_logp"].double()[rows])
        obj = torch.min(ratio * adv, torch.clip(ratio, 1.0 - CLIP_LOW, 1.0 + CLIP_HIGH) * adv)
        per = -obj
        if st["ref_logp"] is not None:
            d = st["ref_logp"].double()[rows] - u
            per = per + KL * (torch.expm1(d) - d)
        loss = (w * per).sum()
        slope[rows] = torch.autograd.grad(loss, u)[0]
        first = (loss.detach().reshape(1), lp)
    else:
        u = lp.clone().requires_grad_()
        seq = torch.stack([p.sum() for p in u.split(_lens(case))])
        ratios = seq - st["ref_logp"].double()
        h = BETA * (ratios[0::2] - ratios[1::2])
        logsig = torch.nn.functional.logsigmoid
        loss = -((1.0 - SMOOTHING) * logsig(h) + SMOOTHING * logsig(-h)).mean()
        slope = torch.autograd.grad(loss, u)[0] * (y >= 0)
        first = (loss.detach().reshape(1), seq.detach())
    grad = torch.zeros(R, C, dtype=F64, device=x.device)
    for part in rows.split(1024):
        p = -torch.softmax(x[part].double(), 1)
        p[torch.arange(len(part), device=x.device), y[part]] += 1.0
        grad[part] = p * slope[part][:, None]
    return first + (grad,)


def _attention_exact(st):
    case = st["case"]
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    T = st["q"].shape[0]
    dev = st["q"].device
    back = case["kind"] == "attention_bwd"
    out, lse = torch.zeros(T, H, D, dtype=F64, device=dev), torch.zeros(H, T, dtype=F64, device=dev)
    dq = torch.zeros(T, H, D, dtype=F64, device=dev)
    dk, dv = (torch.zeros(T, G, D, dtype=F64, device=dev) for _ in range(2))
    start = 0
    for n in _lens(case):
        sl = slice(start, start + n)
        for h in range(H):
            kh = h * G // H
            q, k, v = st["q"][sl, h].double(), st["k"][sl, kh].double(), st["v"][sl, kh].double()
            x = torch.mm(q, k.t().contiguous()) * st["scale"]
            if case["causal"]:
                i = torch.arange(n, device=dev)
                x[i[None, :] > i[:, None]] = -math.inf
            if not back:
                lse[h, sl] = torch.logsumexp(x, 1)
                out[sl, h] = torch.mm(torch.softmax(x, 1), v)
                continue
            # By the operator's definition: from the forward's rounded outputs.
            go, o = st["grad_out"][sl, h].double(), st["out"][sl, h].double()
            p = torch.exp(x - st["lse"][h, sl].double()[:, None])
            dv[sl, kh] += torch.mm(p.t().contiguous(), go)
            ds = p * (torch.mm(go, v.t().contiguous()) - (go * o).sum(1)[:, None]) * st["scale"]
            dq[sl, h] = torch.mm(ds, k)
            dk[sl, kh] += torch.mm(ds.t().contiguous(), q)
        start += n
    return (dq, dk, dv) if back else (out, lse)


def _decode_exact(st):
    case = st["case"]
    H, G = case["heads"], case["kv_heads"]
    out = torch.zeros(st["q"].shape, dtype=F64, device=st["q"].device)
    for b, n in enumerate(_lens(case)):
        for g in range(G):
            heads = slice(g * (H // G), (g + 1) * (H // G))
            x = torch.mm(st["q"][b, heads].double(), st["k"][b, :n, g].double().t().contiguous())
            out[b, heads] = torch.mm(torch.softmax(x * st["scale"], 1), st["v"][b, :n, g].double())
    return out

"""Cases of the decoder-step operators: rotary positions, normalised and turned heads, the experts' router and the
linear cross entropy.  Each case runs either in a plain form (elementary torch operations in 32 bits, rounded once at
the end) or, with ``own`` set, through the framework's public functions.

A case is a dict with ``op`` and the operator's sizes:

* ``rope`` / ``qknorm``: tokens ``s`` x ``b``, query groups ``g`` with ``hpg`` query heads each, head size ``d``, ``rot``
  turned channels, ``inter`` (pairs side by side) or halves, ``per_seq`` (one table for each sequence of the batch);
* ``route``: tokens ``t``, experts ``e``, ``k`` choices, ``score`` function, ``bias``, ``groups`` of which ``top_groups`` stay,
  ``renorm``, ``scaling``;
* ``lce``: tokens ``t``, vocabulary ``v``, hidden size ``h``, one in ``ignore`` labels is ignored (0: none).

``train`` adds the gradients of every input that has one.
"""
from __future__ import annotations

import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_EPS = 1e-5
_TINY = 1e-20
_IGNORE = -100


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one token of the 8-group, 32-head layout without gradients: what a call costs at least
        dict(name="rope_one_token", op="rope", s=1, b=1, g=8, hpg=4, d=128, rot=128, inter=True, per_seq=False,
             dtype="bf16", train=False),
        # ragged sizes in fp32: 5 groups of 3 heads of 96 channels, a quarter of them turned, packed sequences whose
        # positions differ along the batch
        dict(name="rope_ragged_partial", op="rope", s=777, b=3, g=5, hpg=3, d=96, rot=24, inter=False, per_seq=True,
             dtype="fp32", train=True),
        # a long sequence of the 8-group layout with interleaved pairs on half of each head
        dict(name="rope_long", op="rope", s=8192, b=2, g=8, hpg=4, d=128, rot=64, inter=True, per_seq=False,
             dtype="bf16", train=True),
        # one short sequence of the smallest configuration (8 heads of 64), a training step's latency
        dict(name="qknorm_short", op="qknorm", s=64, b=1, g=8, hpg=1, d=64, rot=64, inter=False, per_seq=False,
             dtype="bf16", train=True),
        # an ordinary micro-batch: 4096 tokens, 32 heads without sharing, in half precision
        dict(name="qknorm_step", op="qknorm", s=4096, b=1, g=32, hpg=1, d=128, rot=128, inter=False, per_seq=False,
             dtype="fp16", train=True),
        # the largest: four long sequences with shared heads
        dict(name="qknorm_long", op="qknorm", s=8192, b=4, g=8, hpg=4, d=128, rot=128, inter=False, per_seq=False,
             dtype="bf16", train=True),
        # a single token's choice among 8 experts
        dict(name="route_one_token", op="route", t=1, e=8, k=2, score="softmax", bias=False, groups=1, top_groups=1,
             renorm=True, scaling=1.0, dtype="fp32", train=False),
        # an ordinary micro-batch on 64 experts, softmax scores with a balancing bias, bf16 logits, odd token count
        dict(name="route_step", op="route", t=4099, e=64, k=6, score="softmax", bias=True, groups=1, top_groups=1,
             renorm=False, scaling=1.0, dtype="bf16", train=True),
        # many fine experts: sigmoid scores, bias, 4 of 8 groups, renormalised and scaled
        dict(name="route_groups", op="route", t=32768, e=256, k=8, score="sigmoid", bias=True, groups=8, top_groups=4,
             renorm=True, scaling=2.5, dtype="fp32", train=True),
        # a small model's head on a short ragged batch with ignored labels
        dict(name="lce_small", op="lce", t=250, v=32001, h=512, ignore=5, dtype="bf16", train=True),
        # the 32000-word head of a 4096-wide model for one micro-batch
        dict(name="lce_step", op="lce", t=4096, v=32000, h=4096, ignore=0, dtype="bf16", train=True),
        # the largest: the padded 128256-word vocabulary at 8192 tokens
        dict(name="lce_large_vocab", op="lce", t=8192, v=129024, h=4096, ignore=16, dtype="bf16", train=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "qknorm", "route", "lce"])
    train = rng.random() < 0.75
    if op in ("rope", "qknorm"):
        d = rng.choice([64, 80, 96, 128, 128, 256])
        inter = rng.random() < 0.5
        rot = rng.choice([d, d, d // 2, d // 4])
        g, hpg = _log_int(rng, 1, 32), rng.choice([1, 1, 2, 3, 4, 7, 8])
        b = rng.choice([1, 1, 2, 3, 4])
        most = (8192 * 4 * 48 * 128 if op == "qknorm" else 8192 * 2 * 48 * 128) // (b * g * (hpg + 2) * d)
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        if dtype == "fp32":
            most //= 2
        return dict(op=op, s=_log_int(rng, 1, max(1, min(65536, most))), b=b, g=g, hpg=hpg, d=d, rot=rot, inter=inter,
                    per_seq=rng.random() < 0.3, dtype=dtype, train=train)
    if op == "route":
        e = rng.choice([8, 16, 40, 60, 64, 96, 128, 160, 256, 384, 512])
        k = rng.choice([1, 2, 4, 6, 8])
        groups = rng.choice([1, 1, 2, 4, 8]) if e % 8 == 0 else 1
        top_groups = 1 if groups == 1 else rng.choice([x for x in (1, 2, 4) if x <= groups and k % x == 0
                                                       and x * (e // groups) >= k and k // x <= 2] or [groups])
        if groups > 1 and (top_groups * (e // groups) < k or k // top_groups > 2):
            groups = top_groups = 1
        return dict(op=op, t=_log_int(rng, 1, min(32768, 32768 * 256 // e)), e=e, k=k,
                    score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.6, groups=groups,
                    top_groups=top_groups, renorm=rng.random() < 0.6, scaling=rng.choice([1.0, 2.5, 1.3]),
                    dtype=rng.choice(["fp32", "fp32", "bf16", "fp16"]), train=train)
    h = 8 * _log_int(rng, 32, 640)
    v = _log_int(rng, 1000, 129024)
    most = min(8192, 8192 * 129024 * 4096 // (v * h))
    return dict(op=op, t=_log_int(rng, 1, most), v=v, h=h, ignore=rng.choice([0, 0, 3, 16]), dtype="bf16", train=train)


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dt = _TYPES[case["dtype"]]

    def randn(*shape, dtype=torch.float32):
        return torch.randn(*shape, device="cuda", generator=gen, dtype=dtype)

    def rand(*shape):
        return torch.rand(*shape, device="cuda", generator=gen)

    st = {"case": dict(case)}
    if case["op"] in ("rope", "qknorm"):
        s, b, g, hpg, d, r = (case[n] for n in ("s", "b", "g", "hpg", "d", "rot"))
        # head channels differ in size, as those of a trained projection do
        x = randn(s, b, g, hpg + 2, d) * torch.exp(0.5 * randn(d))
        # positions anywhere in a long context; one table for all sequences or one for each
        start = torch.randint(0, 100000, (b if case["per_seq"] else 1,), device="cuda", generator=gen)
        pos = (torch.arange(s, device="cuda")[:, None] + start[None, :]).double()
        inv = 500000.0 ** (-torch.arange(0, r, 2, device="cuda", dtype=torch.float64) / r)
        ang = pos[:, :, None] * inv
        if not case["per_seq"]:
            ang = ang[:, 0]
        st["cos"], st["sin"] = ang.cos().float().contiguous(), ang.sin().float().contiguous()
        st["qkv"] = x.to(dt).requires_grad_(case["train"])
        if case["op"] == "qknorm":
            for n in ("wq", "wk"):
                st[n] = (1.0 + 0.2 * randn(d)).to(dt).requires_grad_(case["train"])
        if case["train"]:
            st["dy"] = (randn(s, b, g, hpg + 2, d) * 1e-2).to(dt)
    elif case["op"] == "route":
        t, e, k = case["t"], case["e"], case["k"]
        # tokens' scores over a common preference for some experts
        st["logits"] = (randn(t, e) * 1.2 + 0.8 * randn(e)).to(dt).requires_grad_(case["train"])
        # the bias of loss-free balancing: steps of 0.001 towards the less used experts
        st["bias"] = 1e-3 * torch.randint(-100, 101, (e,), device="cuda", generator=gen).float() if case["bias"] else None
        if case["train"]:
            st["dweights"], st["dscore"] = randn(t, k) * 1e-2, randn(e) * 1e-3
    else:
        t, v, h = case["t"], case["v"], case["h"]
        w = randn(v, h, dtype=torch.float32).mul_(0.02).to(dt)
        labels = torch.randint(0, v, (t,), device="cuda", generator=gen)
        # normalised states that lean towards their label's row by a different amount each: from untrained tokens to
        # tokens that the model is sure of
        x = randn(t, h) + 50.0 * 0.4 * rand(t, 1).square() * w[labels].float()
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS)
        if case["ignore"]:
            labels[rand(t) < 1.0 / case["ignore"]] = _IGNORE
        st["x"] = x.to(dt).requires_grad_(case["train"])
        st["w"] = w.requires_grad_(case["train"])
        st["labels"] = labels
        if case["train"]:
            st["dloss"] = (0.5 + rand(t)) / t
    return st


# ------------------------------------------------------------------------------------------------ plain forms
def _turn(x, cos, sin, inter):
    """Turns the first 2 * cos.shape[-1] channels of x [s, b, ..., d] by the tables [s, (b,) r/2]."""
    h = cos.shape[-1]
    shape = (x.shape[0], cos.shape[1] if cos.dim() == 3 else 1) + (1,) * (x.dim() - 3) + (h,)
    c, n = cos.reshape(shape), sin.reshape(shape)
    if inter:
        a, b = x[..., 0:2 * h:2], x[..., 1:2 * h:2]
        y = torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2)
    else:
        a, b = x[..., :h], x[..., h:2 * h]
        y = torch.cat([a * c - b * n, b * c + a * n], -1)
    return torch.cat([y, x[..., 2 * h:]], -1)


def _plain_rope(qkv, cos, sin, hpg, inter, wq=None, wk=None):
    x = qkv.float()
    q, k, v = x[..., :hpg, :], x[..., hpg:hpg + 1, :], x[..., hpg + 1:, :]
    if wq is not None:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + _EPS) * wq.float()
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + _EPS) * wk.float()
    return torch.cat([_turn(q, cos, sin, inter), _turn(k, cos, sin, inter), v], -2).to(qkv.dtype)


def _plain_route(logits, bias, c):
    x = logits.float()
    t, e = x.shape
    k, n, m = c["k"], c["groups"], c["top_groups"]
    if c["score"] == "softmax":
        ex = torch.exp(x - x.max(-1, keepdim=True).values)
        # the sum is held in 64 bits, so that which experts are chosen does not hang on the order of the additions
        s = ex / ex.double().sum(-1, keepdim=True).float()
        part = s
    else:
        s = 1.0 / (1.0 + torch.exp(-x))
        part = s / (s.sum(-1, keepdim=True) + _TINY)
    pick = s.detach() if bias is None else s.detach() + bias
    if bias is None and m == n:
        pick = x.detach()  # the scores' own order, also where they round to the same value
    if n > m:
        best = torch.sort(pick.view(t, n, e // n), dim=-1, descending=True).values[..., :max(1, k // m)]
        total = best.sum(-1)
        order = torch.sort(total, dim=-1, descending=True, stable=True).indices[:, :m]
        keep = torch.zeros_like(total, dtype=torch.bool).scatter(1, order, True)
        pick = pick.masked_fill(~keep.repeat_interleave(e // n, 1), -math.inf)
    top = torch.sort(pick, dim=-1, descending=True, stable=True).indices[:, :k]
    w = s.gather(1, top)
    if c["renorm"]:
        w = w / (w.sum(-1, keepdim=True) + _TINY)
    counts = torch.zeros(e, device=x.device, dtype=torch.int64).index_add(
        0, top.reshape(-1), torch.ones(t * k, device=x.device, dtype=torch.int64))
    return w * c["scaling"], top.to(torch.int32), part.sum(0), counts.to(torch.int32)


def _plain_lce(x, w, labels):
    z = x.float() @ w.float().t()
    m = z.detach().max(-1, keepdim=True).values
    lse = m.squeeze(-1) + torch.log(torch.exp(z - m).sum(-1))
    live = labels >= 0
    at = z.gather(1, labels.clamp(min=0)[:, None]).squeeze(1)
    return torch.where(live, lse - at, torch.zeros_like(lse))


def _forward(st):
    c = st["case"]
    if own:
        from elasticmegatron_b200.ops import functional as F_

        if c["op"] == "rope":
            return F_.rope_qkv(st["qkv"], st["cos"], st["sin"], c["hpg"] + 1, interleaved=c["inter"])
        if c["op"] == "qknorm":
            return F_.qk_norm_rope_qkv(st["qkv"], st["wq"], st["wk"], st["cos"], st["sin"], _EPS,
                                       interleaved=c["inter"])
        if c["op"] == "route":
            return F_.moe_route(st["logits"], c["k"], score_function=c["score"], bias=st["bias"],
                                num_groups=c["groups"], group_topk=c["top_groups"], renormalize=c["renorm"],
                                scaling=c["scaling"])
        return F_.linear_cross_entropy(st["x"], st["w"], st["labels"], ignore_index=_IGNORE)
    if c["op"] == "rope":
        return _plain_rope(st["qkv"], st["cos"], st["sin"], c["hpg"], c["inter"])
    if c["op"] == "qknorm":
        return _plain_rope(st["qkv"], st["cos"], st["sin"], c["hpg"], c["inter"], st["wq"], st["wk"])
    if c["op"] == "route":
        return _plain_route(st["logits"], st["bias"], c)
    return _plain_lce(st["x"], st["w"], st["labels"])


def run(st):
    c = st["case"]
    if not c["train"]:
        with torch.no_grad():
            out = _forward(st)
        return dict(zip(("weights", "experts", "score_sum", "counts"), out)) if c["op"] == "route" else {"out": out}
    out = _forward(st)
    if c["op"] == "rope":
        dx, = torch.autograd.grad(out, st["qkv"], st["dy"])
        return {"out": out, "dqkv": dx}
    if c["op"] == "qknorm":
        dx, dwq, dwk = torch.autograd.grad(out, [st["qkv"], st["wq"], st["wk"]], st["dy"])
        return {"out": out, "dqkv": dx, "dwq": dwq, "dwk": dwk}
    if c["op"] == "route":
        weights, experts, score_sum, counts = out
        dl, = torch.autograd.grad([weights, score_sum], st["logits"], [st["dweights"], st["dscore"]])
        return {"weights": weights, "experts": experts, "score_sum": score_sum, "counts": counts, "dlogits": dl}
    dx, dw = torch.autograd.grad(out, [st["x"], st["w"]], st["dloss"])
    return {"out": out, "dx": dx, "dw": dw}


# ------------------------------------------------------------------------------------------------ work
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] in ("rope", "qknorm"):
        tok, heads = case["s"] * case["b"], case["g"] * (case["hpg"] + 2)
        n = tok * heads * case["d"]
        qk = tok * case["g"] * (case["hpg"] + 1) * case["d"]
        table = case["s"] * (case["b"] if case["per_seq"] else 1) * case["rot"] * 4
        ways = 2 if case["train"] else 1
        byts = ways * (2 * n * size + table)
        flops = ways * 3 * qk
        if case["op"] == "qknorm":
            byts += (qk * size if case["train"] else 0) + 2 * ways * case["d"] * size
            flops += qk * (4 + (10 if case["train"] else 0))
        return {"bytes": byts, "flops": flops}
    if case["op"] == "route":
        t, e, k = case["t"], case["e"], case["k"]
        byts = t * e * size + t * k * 8 + e * 8
        flops = t * e * (6 + k)
        if case["train"]:
            byts += 2 * t * e * size + t * k * 12 + e * 4
            flops += t * e * 10
        return {"bytes": byts, "flops": flops}
    t, v, h = case["t"], case["v"], case["h"]
    mats = (t + v) * h * size
    if not case["train"]:
        return {"bytes": mats + t * 12, "flops": 2 * t * v * h}
    return {"bytes": 3 * mats + t * 24, "flops": 6 * t * v * h}


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    """The outputs of ``run`` from the definitions in 64 bits, with the gradients written out."""
    st = prepare(case, seed)
    with torch.no_grad():
        return {"rope": _exact_heads, "qknorm": _exact_heads, "route": _exact_route, "lce": _exact_lce}[case["op"]](st)


def _exact_heads(st):
    c = st["case"]
    hpg, r, d = c["hpg"], c["rot"], c["d"]
    x = st["qkv"].double()
    first = torch.arange(0, r, 2, device=x.device) if c["inter"] else torch.arange(r // 2, device=x.device)
    second = first + (1 if c["inter"] else r // 2)
    # the turn as complex products of the pairs with cos + i sin
    rot = torch.complex(st["cos"].double(), st["sin"].double())
    rot = rot[:, :, None, None, :] if c["per_seq"] else rot[:, None, None, None, :]

    def turned(v, by):
        z = torch.complex(v[..., first], v[..., second]) * by
        y = v.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return y

    norm = c["op"] == "qknorm"
    inv, w = torch.ones_like(x[..., :1]), torch.ones(hpg + 2, d, device=x.device, dtype=torch.float64)
    if norm:
        inv = 1.0 / (x.pow(2).sum(-1, keepdim=True) / d + _EPS).sqrt()
        inv[..., hpg + 1, :] = 1.0
        w[:hpg], w[hpg] = st["wq"].double(), st["wk"].double()
    y = x * inv * w
    y[..., :hpg + 1, :] = turned(y[..., :hpg + 1, :], rot)
    if not c["train"]:
        return {"out": y}
    g = st["dy"].double()
    g[..., :hpg + 1, :] = turned(g[..., :hpg + 1, :], rot.conj())
    if not norm:
        return {"out": y, "dqkv": g}
    xh = x * inv
    dw = (g * xh).sum((0, 1, 2))
    gw = g * w
    dx = inv * (gw - xh * (gw * xh).sum(-1, keepdim=True) / d)
    dx[..., hpg + 1, :] = g[..., hpg + 1, :]
    return {"out": y, "dqkv": dx, "dwq": dw[:hpg].sum(0), "dwk": dw[hpg]}


def _exact_route(st):
    c = st["case"]
    x = st["logits"].double()
    t, e = x.shape
    k, n, m = c["k"], c["groups"], c["top_groups"]
    s = torch.softmax(x, -1) if c["score"] == "softmax" else torch.sigmoid(x)
    pick = s + (st["bias"].double() if st["bias"] is not None else 0.0)
    if n > m:
        of = pick.view(t, n, -1).topk(max(1, k // m), -1).values.sum(-1)
        gone = torch.ones_like(of, dtype=torch.bool).scatter(1, of.argsort(dim=-1, descending=True, stable=True)[:, :m], False)
        pick = pick.masked_fill(gone[:, :, None].expand(t, n, e // n).reshape(t, e), -math.inf)
    # equal scores go to the lowest expert
    top = pick.argsort(dim=-1, descending=True, stable=True)[:, :k]
    chosen = torch.zeros(t, e, device=x.device, dtype=torch.bool).scatter(1, top, True)
    d = (s * chosen).sum(-1, keepdim=True) + _TINY if c["renorm"] else torch.ones(t, 1, device=x.device, dtype=x.dtype)
    u = s / d * chosen
    total = s.sum(-1, keepdim=True) + (_TINY if c["score"] == "sigmoid" else 0.0)
    p = s / total
    out = {"weights": c["scaling"] * u.gather(1, top), "experts": None, "score_sum": p.sum(0), "counts": None}
    if not c["train"]:
        return out
    dw = torch.zeros_like(x).scatter(1, top, st["dweights"].double() * c["scaling"])
    ds = dw / d
    if c["renorm"]:
        ds = ds - chosen * (dw * u).sum(-1, keepdim=True) / d
    dp = st["dscore"].double()[None]
    if c["score"] == "softmax":
        g = ds + dp
        dl = s * (g - (s * g).sum(-1, keepdim=True))
    else:
        dl = s * torch.sigmoid(-x) * (ds + (dp - (dp * p).sum(-1, keepdim=True)) / total)
    out["dlogits"] = dl
    return out


def _exact_lce(st):
    c = st["case"]
    x, w, labels = st["x"].double(), st["w"].double(), st["labels"]
    t, train = c["t"], c["train"]
    out = torch.zeros(t, device=x.device, dtype=torch.float64)
    dx, dw = (torch.zeros_like(x), torch.zeros_like(w)) if train else (None, None)
    for a in range(0, t, 2048):
        sl = slice(a, min(t, a + 2048))
        lab = labels[sl]
        live = torch.nonzero(lab != _IGNORE).squeeze(1)
        z = x[sl] @ w.t()
        lse = torch.logsumexp(z, -1)
        out[sl][live] = lse[live] - z[live, lab[live]]
        if train:
            p = torch.exp(z - lse[:, None])
            p[live, lab[live]] -= 1.0
            p *= (st["dloss"][sl].double() * (lab != _IGNORE))[:, None]
            dx[sl] = p @ w
            dw += p.t() @ x[sl]
    return {"out": out, "dx": dx, "dw": dw} if train else {"out": out}

"""Plain-PyTorch implementations of every hot op.

These are (1) the CPU path used by gloo-rank tests and (2) the fp32 oracles every CUDA kernel is tested
against.  They are never used for CUDA tensors: the dispatch in ``ops/functional.py`` raises if the native
extension is missing on a GPU.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
import torch.nn.functional as F


def rmsnorm_fwd(x: torch.Tensor, w: torch.Tensor, eps: float) -> Tuple[torch.Tensor, torch.Tensor]:
    xf = x.float()
    rstd = torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)
    y = (xf * rstd * w.float()).to(x.dtype)
    return y, rstd.squeeze(-1)


def rmsnorm_bwd(dy, x, w, rstd) -> Tuple[torch.Tensor, torch.Tensor]:
    xf, dyf, wf = x.float(), dy.float(), w.float()
    r = rstd.unsqueeze(-1)
    xhat = xf * r
    dw = (dyf * xhat).reshape(-1, x.shape[-1]).sum(0)
    g = dyf * wf
    dx = r * (g - xhat * (g * xhat).mean(-1, keepdim=True))
    return dx.to(x.dtype), dw


def rope_cos_sin(positions: torch.Tensor, dim: int, base: float):
    inv = 1.0 / (base ** (torch.arange(0, dim, 2, dtype=torch.float64, device=positions.device) / dim))
    ang = positions.to(torch.float64)[:, None] * inv[None, :]
    return ang.cos().float(), ang.sin().float()


def rope_apply(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, inverse: bool = False) -> torch.Tensor:
    """x: [s, b, n, d] rotate-half convention on pairs (i, i + d/2); cos/sin: [s, d/2]."""
    d2 = x.shape[-1] // 2
    xf = x.float()
    x1, x2 = xf[..., :d2], xf[..., d2:]
    c = cos[:, None, None, :]
    s = sin[:, None, None, :]
    if inverse:
        s = -s
    return torch.cat([x1 * c - x2 * s, x2 * c + x1 * s], -1).to(x.dtype)


def swiglu_fwd(h: torch.Tensor) -> torch.Tensor:
    """h: [..., 2f] = [gate | up] -> silu(gate) * up."""
    g, u = h.float().chunk(2, -1)
    return (F.silu(g) * u).to(h.dtype)


def swiglu_bwd(dy: torch.Tensor, h: torch.Tensor) -> torch.Tensor:
    g, u = h.float().chunk(2, -1)
    dyf = dy.float()
    sg = torch.sigmoid(g)
    silu = g * sg
    dg = dyf * u * (sg * (1 + g * (1 - sg)))
    du = dyf * silu
    return torch.cat([dg, du], -1).to(h.dtype)


def attention_fwd(q, k, v, causal: bool = True, scale: Optional[float] = None):
    """q: [b, hq, s, d], k/v: [b, hkv, t, d] (GQA) -> (o [b,hq,s,d], lse [b,hq,s] fp32)."""
    hq, hkv = q.shape[1], k.shape[1]
    if hq != hkv:
        k = k.repeat_interleave(hq // hkv, 1)
        v = v.repeat_interleave(hq // hkv, 1)
    scale = scale or 1.0 / math.sqrt(q.shape[-1])
    s = torch.matmul(q.float(), k.float().transpose(-1, -2)) * scale
    if causal:
        S, T = q.shape[2], k.shape[2]
        mask = torch.ones(S, T, dtype=torch.bool, device=q.device).tril(T - S)
        s = s.masked_fill(~mask, float("-inf"))
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse.unsqueeze(-1))
    o = torch.matmul(p, v.float())
    return o.to(q.dtype), lse


def cross_entropy(logits: torch.Tensor, labels: torch.Tensor) -> torch.Tensor:
    return F.cross_entropy(logits.float(), labels, reduction="none")


def adam_step(master, exp_avg, exp_avg_sq, grad, lr, beta1, beta2, eps, wd, step, clip_coef=1.0):
    """Decoupled AdamW with bias correction on fp32 tensors, in place (torch.optim.AdamW semantics)."""
    g = grad.float() * clip_coef
    exp_avg.mul_(beta1).add_(g, alpha=1 - beta1)
    exp_avg_sq.mul_(beta2).addcmul_(g, g, value=1 - beta2)
    bc1 = 1 - beta1 ** step
    bc2 = 1 - beta2 ** step
    denom = (exp_avg_sq / bc2).sqrt_().add_(eps)
    if wd != 0.0:
        master.mul_(1 - lr * wd)
    master.addcdiv_(exp_avg, denom, value=-lr / bc1)


# ------------------------------------------------------------------------------------------ rotary positions
def rope_rotate(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, interleaved: bool = False,
                inverse: bool = False) -> torch.Tensor:
    """Turns the first ``r = 2 * cos.shape[-1]`` channels of x [s, b, ..., d] (fp32 result); the tables are
    [s, r/2] or [s, b, r/2] and the pairs (i, i + r/2) or, interleaved, (2i, 2i + 1)."""
    h = cos.shape[-1]
    shape = (x.shape[0], cos.shape[1] if cos.dim() == 3 else 1) + (1,) * (x.dim() - 3) + (h,)
    c, s = cos.reshape(shape), sin.reshape(shape)
    if inverse:
        s = -s
    xf = x.float()
    y = xf.clone()
    a, b = (slice(0, 2 * h, 2), slice(1, 2 * h, 2)) if interleaved else (slice(0, h), slice(h, 2 * h))
    y[..., a] = xf[..., a] * c - xf[..., b] * s
    y[..., b] = xf[..., b] * c + xf[..., a] * s
    return y


def heads_fwd(qkv, cos, sin, nq, nk, interleaved, wq=None, wk=None, eps=0.0) -> torch.Tensor:
    """Rotary positions of the first nq + nk slots of each group of qkv [s, b, G, S, d], after an RMSNorm of every
    head where weights are given."""
    y = qkv.float().clone()
    n = nq + nk
    if wq is not None:
        x = y[:, :, :, :n]
        w = torch.cat([wq.float().expand(nq, -1), wk.float().expand(nk, -1)])
        y[:, :, :, :n] = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps) * w
    y[:, :, :, :n] = rope_rotate(y[:, :, :, :n], cos, sin, interleaved)
    return y.to(qkv.dtype)


def heads_bwd(dy, qkv, cos, sin, nq, nk, interleaved, wq=None, wk=None, eps=0.0):
    """(dqkv, dwq, dwk) of :func:`heads_fwd`; the weight gradients are fp32 (None without norm)."""
    n = nq + nk
    dx = dy.float().clone()
    g = rope_rotate(dx[:, :, :, :n], cos, sin, interleaved, inverse=True)
    if wq is None:
        dx[:, :, :, :n] = g
        return dx.to(dy.dtype), None, None
    x = qkv[:, :, :, :n].float()
    rstd = torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps)
    xh = x * rstd
    dw = (g * xh).sum((0, 1, 2))
    gw = g * torch.cat([wq.float().expand(nq, -1), wk.float().expand(nk, -1)])
    dx[:, :, :, :n] = rstd * (gw - xh * (gw * xh).mean(-1, keepdim=True))
    return dx.to(dy.dtype), dw[:nq].sum(0), dw[nq:].sum(0)


# ------------------------------------------------------------------------------------------ router
_TINY = 1e-20


def _route_scores(x, sigmoid):
    """(scores, what the normalised scores of the statistics are divided by)."""
    if sigmoid:
        s = 1.0 / (1.0 + torch.exp(-x))
        return s, s.sum(-1, keepdim=True) + _TINY
    m = x.max(-1, keepdim=True).values
    e = torch.where(x == -math.inf, torch.zeros_like(x), torch.exp(x - m))
    # the sum is held in 64 bits so that the choice does not depend on the order of the additions
    z = e.double().sum(-1, keepdim=True).float()
    return e / torch.where(z == 0, torch.ones_like(z), z), torch.ones_like(z)


def moe_route_fwd(logits, k, sigmoid, bias, groups, topg, renorm, scaling):
    """(weights [T, k], experts [T, k] int32, score_sum [E], counts [E] int32); see ``csrc/moe/route.cu``."""
    x = logits.float()
    T, E = x.shape
    s, norm = _route_scores(x, sigmoid)
    c = s if bias is None else s + bias
    if bias is None and topg == groups:
        c = x  # the scores' own order, also where they round to the same value
    # masked and NaN entries come after every other expert, experts of dropped groups after those
    c = torch.where((x > -math.inf) & ~c.isnan(), c, torch.full_like(c, -math.inf))
    lost = torch.zeros(T, E, dtype=torch.bool, device=x.device)
    if groups > topg:
        best = c.view(T, groups, E // groups).sort(-1, descending=True).values
        best = best[..., :min(max(1, k // topg), E // groups)]
        value = torch.where(best == -math.inf, torch.zeros_like(best), best).sum(-1)
        value = torch.where(best[..., 0] == -math.inf, best[..., 0], value)
        order = value.sort(dim=-1, descending=True, stable=True).indices[:, :topg]
        lost = torch.ones_like(value, dtype=torch.bool).scatter(1, order, False).repeat_interleave(E // groups, 1)
    order = c.sort(dim=-1, descending=True, stable=True).indices
    kept = (~lost).gather(1, order)  # in order, the experts of dropped groups moved to the end
    order = order.gather(1, kept.to(torch.int8).sort(dim=-1, descending=True, stable=True).indices)
    top = order[:, :k]
    w = s.gather(1, top)
    if renorm:
        w = w / (w.sum(-1, keepdim=True) + _TINY)
    counts = torch.bincount(top.reshape(-1), minlength=E).to(torch.int32)
    return w * scaling, top.to(torch.int32), (s / norm).sum(0), counts


def moe_route_bwd(logits, experts, dweights, dscore, sigmoid, renorm, scaling):
    x = logits.float()
    s, norm = _route_scores(x, sigmoid)
    top = experts.long()
    u = s.gather(1, top)
    a = dweights.float() * scaling if dweights is not None else torch.zeros_like(u)
    if renorm:
        den = u.sum(-1, keepdim=True) + _TINY
        a = (a - (a * u / den).sum(-1, keepdim=True)) / den
    ds = torch.zeros_like(s).scatter(1, top, a)
    q = dscore.float()[None] if dscore is not None else torch.zeros(1, x.shape[1], device=x.device)
    if sigmoid:
        e = torch.exp(-x.abs())
        dl = e / (1 + e) ** 2 * (ds + (q - (q * s).sum(-1, keepdim=True) / norm) / norm)
    else:
        g = ds + q
        dl = s * (g - (s * g).sum(-1, keepdim=True))
    return dl.to(logits.dtype)


# ------------------------------------------------------------------------------------------ linear cross entropy
def _ce_rows(labels, col0, vocab, ignore, V):
    """(rows whose label counts, those whose label is one of the columns [col0, col0 + V), its column there)."""
    counts = (labels >= 0) & (labels < vocab) & (labels != ignore)
    own = counts & (labels >= col0) & (labels < col0 + V)
    return counts, own, torch.where(own, labels - col0, torch.zeros_like(labels))


def linear_ce_fwd(x, w, labels, col0, vocab, ignore, raw):
    """(loss, maximum, sum of exponentials) over this rank's columns; with ``raw`` the label's logit (0 where another
    rank holds it), maximum, sum, and the sum for the loss (the kernels exchange the label's own term there)."""
    z = x.float() @ w.float().t()
    m = z.max(-1).values
    s = torch.exp(z - m[:, None]).sum(-1)
    counts, own, col = _ce_rows(labels, col0, vocab, ignore, w.shape[0])
    t = torch.where(own, z.gather(1, col[:, None]).squeeze(1), torch.zeros_like(m))
    if raw:
        return t, m, s, s
    return torch.where(counts, torch.log(s) + (m - t), torch.zeros_like(m)), m, s


def linear_ce_bwd(dloss, x, w, labels, top, total, col0, vocab, ignore, want_dx, want_dw, dw_accum, piece):
    """(dx, dw), the logits computed again for ``piece`` columns of the vocabulary at a time (0: all)."""
    V = w.shape[0]
    counts, own, col = _ce_rows(labels, col0, vocab, ignore, V)
    g = torch.where(counts, dloss.float(), torch.zeros_like(top))
    xf = x.float()
    dx = torch.zeros_like(xf)
    dw = [] if dw_accum is None else None
    for v0 in range(0, V, piece or V):
        wf = w[v0:v0 + (piece or V)].float()
        p = torch.exp(xf @ wf.t() - top[:, None]) * (g / total)[:, None]
        here = torch.nonzero(own & (col >= v0) & (col < v0 + wf.shape[0])).squeeze(1)
        p[here, col[here] - v0] -= g[here]
        p[~counts] = 0.0
        if want_dx:
            dx += p @ wf
        if dw_accum is not None:
            dw_accum[v0:v0 + wf.shape[0]] += p.t() @ xf
        elif want_dw:
            dw.append((p.t() @ xf).to(w.dtype))
    return dx.to(x.dtype) if want_dx else None, torch.cat(dw) if dw else None

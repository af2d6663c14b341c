"""Host forms of the decoder-step operators (general rotary positions, normalised heads, general router) against plain
64-bit formulas, gradients against differences, and their refusals."""
import math

import pytest
import torch

from elasticmegatron_b200.config import RopeScaling
from elasticmegatron_b200.ops import functional as F_


def _turn(x, cos, sin, inter):
    """64-bit rotation of the first 2 * cos.shape[-1] channels, as complex products."""
    h = cos.shape[-1]
    z = torch.complex(cos.double(), sin.double())
    z = z[:, :, None, None, :] if cos.dim() == 3 else z[:, None, None, None, :]
    i = torch.arange(0, 2 * h, 2) if inter else torch.arange(h)
    j = i + (1 if inter else h)
    y = x.clone()
    p = torch.complex(x[..., i], x[..., j]) * z
    y[..., i], y[..., j] = p.real, p.imag
    return y


def _heads(qkv, n, cos, sin, inter, w=None, eps=0.0):
    x = qkv.double()
    h = x[:, :, :, :n]
    if w is not None:
        h = h / (h.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double()
    return torch.cat([_turn(h, cos, sin, inter), x[:, :, :, n:]], 3)


def _tables(s, b, r, per_seq, seed=0):
    g = torch.Generator().manual_seed(seed)
    a = torch.rand((s, b, r // 2) if per_seq else (s, r // 2), generator=g) * 6.28
    return a.cos(), a.sin()


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("s,b,G,hpg,d,r,per_seq", [(1, 1, 1, 1, 16, 16, False), (5, 2, 3, 2, 12, 6, True),
                                                   (3, 1, 2, 1, 10, 2, False)])
def test_heads(s, b, G, hpg, d, r, per_seq, inter):
    g = torch.Generator().manual_seed(1)
    qkv = torch.randn(s, b, G, hpg + 2, d, generator=g).requires_grad_()
    wq, wk = (1 + 0.1 * torch.randn(2, d, generator=g)).unbind(0)
    wq, wk = wq.clone().requires_grad_(), wk.clone().requires_grad_()
    cos, sin = _tables(s, b, r, per_seq)
    dy = torch.randn(qkv.shape, generator=g)
    # one rounding of O(10) fp32 operations on O(1..10) values: below 1e-5
    out = F_.rope_qkv(qkv, cos, sin, hpg + 1, interleaved=inter)
    x64 = qkv.detach().double().requires_grad_()
    want = _heads(x64, hpg + 1, cos, sin, inter)
    torch.testing.assert_close(out.double(), want, atol=1e-5, rtol=1e-5)
    torch.testing.assert_close(torch.autograd.grad(out, qkv, dy)[0].double(),
                               torch.autograd.grad(want, x64, dy.double())[0], atol=1e-5, rtol=1e-5)
    out = F_.qk_norm_rope_qkv(qkv, wq, wk, cos, sin, 1e-5, interleaved=inter)
    w64 = [wq.detach().double().requires_grad_(), wk.detach().double().requires_grad_()]
    want = _heads(x64, hpg + 1, cos, sin, inter, torch.cat([w64[0].expand(hpg, d), w64[1].expand(1, d)]), 1e-5)
    torch.testing.assert_close(out.double(), want, atol=1e-5, rtol=1e-5)
    got = torch.autograd.grad(out, [qkv, wq, wk], dy)
    for a, e in zip(got, torch.autograd.grad(want, [x64] + w64, dy.double())):
        torch.testing.assert_close(a.double(), e, atol=5e-5, rtol=5e-5)


def test_heads_main_grad():
    d = 16
    qkv = torch.randn(4, 2, 2, 3, d)
    cos, sin = _tables(4, 2, d, False)
    grads = []
    for main in (False, True):
        wq, wk = torch.nn.Parameter(torch.ones(d)), torch.nn.Parameter(torch.ones(d))
        ready = []
        if main:
            for w in (wq, wk):
                w.main_grad = torch.ones(d)
                w._grad_ready = lambda: ready.append(1)
        F_.qk_norm_rope_qkv(qkv, wq, wk, cos, sin, 1e-5).square().sum().backward()
        grads.append([(w.main_grad - 1) if main else w.grad for w in (wq, wk)])
        assert len(ready) == (2 if main else 0) and (not main or wq.grad is None)
    for a, e in zip(*grads):
        torch.testing.assert_close(a, e, atol=1e-4, rtol=1e-5)


def test_heads_refusals():
    qkv = torch.randn(4, 2, 2, 3, 16)
    cos, sin = _tables(4, 2, 16, False)
    w = torch.ones(16)
    for bad in (lambda: F_.rope_qkv(qkv[0], cos, sin, 2, interleaved=True),
                lambda: F_.rope_qkv(qkv, cos[:3], sin[:3], 2, interleaved=True),
                lambda: F_.rope_qkv(qkv, cos, sin[:, :4], 2, interleaved=True),
                lambda: F_.rope_qkv(qkv, cos, sin, 4, interleaved=True),
                lambda: F_.rope_qkv(qkv[..., :14], cos, sin, 2, interleaved=True),
                lambda: F_.rope_qkv(qkv[..., :15], cos[:, :6], sin[:, :6], 2, interleaved=True),
                lambda: F_.qk_norm_rope_qkv(qkv, w[:8], w, cos, sin, 1e-5),
                lambda: F_.qk_norm_rope_qkv(qkv, w, w.double(), cos, sin, 1e-5),
                lambda: F_.qk_norm_rope_qkv(qkv[:, :, :, :2], w, w, cos, sin, 1e-5)):
        with pytest.raises(ValueError):
            bad()


def test_rope_tables_scaling():
    pos = torch.arange(0, 40000, 997)
    base = 500000.0
    c0, s0 = F_.rope_tables(pos, 64, base)
    # linear: the angles of positions divided by the factor
    c, s = F_.rope_tables(pos, 64, base, RopeScaling("linear", 4.0))
    c1, s1 = F_.rope_tables(pos.double() / 4, 64, base)
    torch.testing.assert_close(c, c1)
    torch.testing.assert_close(s, s1)
    # llama3: short wavelengths keep their angle, long ones are divided by the factor
    c, s = F_.rope_tables(pos, 64, base, RopeScaling("llama3", 8.0, 8192))
    torch.testing.assert_close(c[:, 0], c0[:, 0])
    inv = base ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64)
    long = 8192 * inv / (2 * math.pi) < 1.0
    assert 0 < int(long.sum()) < 32
    want = (pos.double()[:, None] * inv / 8.0).cos().float()
    torch.testing.assert_close(c[:, long], want[:, long])
    # yarn: the same ends and the attention temperature on both tables
    c, s = F_.rope_tables(pos, 64, base, RopeScaling("yarn", 8.0, 8192))
    amp = 0.1 * math.log(8.0) + 1.0
    torch.testing.assert_close(c.square() + s.square(), torch.full_like(c, amp * amp))
    torch.testing.assert_close(c[:, 0], amp * c0[:, 0])
    torch.testing.assert_close(c[:, -1], amp * want[:, -1])
    for kw in (dict(kind="ntk"), dict(factor=0.5), dict(low_freq_factor=4.0, high_freq_factor=4.0)):
        with pytest.raises(ValueError):
            RopeScaling(**kw)


# ------------------------------------------------------------------------------------------------ router
def brute_route(row, k, sigmoid, bias, groups, topg, renorm, scaling):
    """One token in 64-bit Python numbers, straight from the definition."""
    E = len(row)
    live = [x > -math.inf for x in row]
    if sigmoid:
        s = [1.0 / (1.0 + math.exp(-x)) if x > -700 else 0.0 for x in row]
        norm = sum(s) + 1e-20
    else:
        m = max(row)
        e = [math.exp(x - m) if x > -math.inf else 0.0 for x in row]
        s = [v / (sum(e) or 1.0) for v in e]
        norm = 1.0
    c = [(s[i] + (bias[i] if bias is not None else 0.0)) if live[i] else -math.inf for i in range(E)]
    if bias is None and topg == groups:
        c = list(row)
    per = E // groups
    allowed = set(range(E))
    if groups > 1:
        value = []
        for g in range(groups):
            best = sorted((v for v in c[g * per:(g + 1) * per] if v > -math.inf), reverse=True)[:max(1, k // topg)]
            value.append(sum(best) if best else -math.inf)
        kept = sorted(range(groups), key=lambda g: (-value[g], g))[:topg]
        allowed = {e for g in kept for e in range(g * per, (g + 1) * per)}
    top = sorted(allowed, key=lambda e: (-c[e], e))[:k]
    w = [s[e] for e in top]
    if renorm:
        d = sum(w) + 1e-20
        w = [v / d for v in w]
    return [v * scaling for v in w], top, [v / norm for v in s]


ROUTES = [  # E, k, sigmoid, bias, groups, topg, renorm
    (1, 1, False, False, 1, 1, True),
    (8, 2, False, False, 1, 1, True),
    (8, 8, True, False, 1, 1, False),
    (12, 3, False, True, 3, 2, False),
    (40, 5, True, True, 1, 1, True),
    (64, 6, False, True, 8, 3, True),
    (64, 8, True, True, 8, 4, True),
    (256, 8, True, True, 8, 4, True),
    (512, 32, True, False, 32, 32, True),
    (64, 8, True, True, 4, 2, True),    # groups valued by four experts
    (24, 6, False, True, 3, 2, False),  # by three, eight to a group
    (60, 8, True, True, 4, 1, True),    # by eight, groups that are no whole lanes
    (60, 2, False, True, 4, 1, False),
    (320, 8, True, True, 8, 4, True),
]


def route_inputs(T, E, bias, seed=0, special=True):
    """Logits on a coarse grid (many ties); from row 3 on one row each of all masked, one expert left, the type's
    lowest value and far apart values."""
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(T, E, generator=g) * 8).round() / 4
    if special and T >= 8:
        x[3] = -math.inf
        x[4] = -math.inf
        x[4, E // 2] = 0.5
        x[5, ::2] = torch.finfo(torch.float32).min
        x[6] = torch.linspace(-300, 300, E) if E > 1 else 7.0
        x[7, : E // 2] = -math.inf
    b = (torch.randn(E, generator=g) * 64).round() / 256 if bias else None
    return x, b


@pytest.mark.parametrize("E,k,sigmoid,bias,groups,topg,renorm", ROUTES)
def test_route(E, k, sigmoid, bias, groups, topg, renorm):
    x, b = route_inputs(24, E, bias)
    w, e, ss, cnt = F_.moe_route(x, k, "sigmoid" if sigmoid else "softmax", b, groups, topg, renorm, 1.5)
    want = [brute_route(r, k, sigmoid, b.tolist() if bias else None, groups, topg, renorm, 1.5) for r in x.tolist()]
    assert e.tolist() == [v[1] for v in want]
    torch.testing.assert_close(w.double(), torch.tensor([v[0] for v in want], dtype=torch.float64), atol=1e-6, rtol=1e-5)
    torch.testing.assert_close(ss.double(), torch.tensor([v[2] for v in want], dtype=torch.float64).sum(0), atol=1e-5,
                               rtol=1e-5)
    assert cnt.tolist() == torch.bincount(e.reshape(-1).long(), minlength=E).tolist() and cnt.sum() == 24 * k


@pytest.mark.parametrize("E,k,sigmoid,bias,groups,topg,renorm", ROUTES[1:7])
def test_route_gradient_by_differences(E, k, sigmoid, bias, groups, topg, renorm):
    """dlogits against central differences of the 64-bit definition (at logits without ties, so that the choice does
    not change within a step)."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(3, E, generator=g).requires_grad_()
    b = torch.randn(E, generator=g) * 0.1 if bias else None
    w, e, ss, _ = F_.moe_route(x, k, "sigmoid" if sigmoid else "softmax", b, groups, topg, renorm, 1.5)
    dw, dq = torch.randn(3, k, generator=g), torch.randn(E, generator=g)
    got, = torch.autograd.grad([w, ss], x, [dw, dq])

    def value(rows):
        tot = 0.0
        for t, r in enumerate(rows):
            ww, top, p = brute_route(r, k, sigmoid, b.tolist() if bias else None, groups, topg, renorm, 1.5)
            assert top == e[t].tolist()
            tot += sum(a * c for a, c in zip(ww, dw[t].tolist())) + sum(a * c for a, c in zip(p, dq.tolist()))
        return tot

    rows, h = x.detach().double().tolist(), 1e-6
    for t in range(3):
        for i in range(0, E, max(1, E // 8)):
            at = rows[t][i]
            rows[t][i] = at + h
            up = value(rows)
            rows[t][i] = at - h
            down = value(rows)
            rows[t][i] = at
            # differences: h^2 terms and 1e-16 / h rounding (1e-9); fp32 gradient of O(1) terms (1e-5)
            assert abs(got[t, i].item() - (up - down) / (2 * h)) < 2e-5


def test_route_refusals():
    x = torch.randn(4, 16)
    for bad in (lambda: F_.moe_route(x[0], 2), lambda: F_.moe_route(x, 0), lambda: F_.moe_route(x, 17),
                lambda: F_.moe_route(x, 2, "relu"), lambda: F_.moe_route(x, 2, num_groups=3),
                lambda: F_.moe_route(x, 8, num_groups=4, group_topk=1),
                lambda: F_.moe_route(x, 2, num_groups=4, group_topk=5),
                lambda: F_.moe_route(x, 2, bias=torch.zeros(8)),
                lambda: F_.moe_route(x, 2, bias=torch.zeros(16, dtype=torch.float64)),
                lambda: F_.moe_route(torch.randn(2, 600), 2)):
        with pytest.raises(ValueError):
            bad()


def test_route_empty():
    x = torch.empty(0, 8, requires_grad=True)
    w, e, ss, c = F_.moe_route(x, 2)
    assert w.shape == (0, 2) and e.shape == (0, 2) and ss.tolist() == [0.0] * 8 and c.tolist() == [0] * 8

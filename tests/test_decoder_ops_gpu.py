"""Kernels of the decoder-step operators (csrc/ops/heads.cu, csrc/moe/route.cu) against plain 64-bit formulas."""
import math

import pytest
import torch

from elasticmegatron_b200.ops import functional as F_
from test_decoder_ops_cpu import ROUTES, brute_route, route_inputs

pytestmark = pytest.mark.gpu

# One rounding to the type plus the fp32 arithmetic before it, for values up to about 8 (2^3) in size.
ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -20}


def _turn(x, cos, sin, inter):
    h = cos.shape[-1]
    z = torch.complex(cos.double(), sin.double())
    z = z[:, :, None, None, :] if cos.dim() == 3 else z[:, None, None, None, :]
    i = torch.arange(0, 2 * h, 2, device=x.device) if inter else torch.arange(h, device=x.device)
    j = i + (1 if inter else h)
    y = x.clone()
    p = torch.complex(x[..., i], x[..., j]) * z
    y[..., i], y[..., j] = p.real, p.imag
    return y


def _heads64(x, n, cos, sin, inter, w=None, eps=0.0):
    h = x[:, :, :, :n]
    if w is not None:
        h = h / (h.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w
    return torch.cat([_turn(h, cos, sin, inter), x[:, :, :, n:]], 3)


def _close(a, e, dt, scale=1.0):
    torch.testing.assert_close(a.double(), e, atol=scale * ROUND[dt], rtol=ROUND[dt])


HEADS = [  # s, b, G, hpg, d, r, per_seq
    (1, 1, 1, 1, 64, 64, False),
    (1, 1, 8, 4, 128, 128, False),
    (37, 3, 5, 3, 96, 24, True),    # quarter of a head: pairs that do not fill 8-channel vectors
    (33, 2, 3, 7, 80, 80, False),   # lanes without a pair
    (29, 1, 2, 1, 80, 40, True),
    (65, 2, 1, 8, 256, 128, False),
    (17, 1, 2, 2, 512, 512, True),
    (9, 2, 2, 1, 10, 6, True),      # a head of single channels
    (7, 1, 1, 2, 72, 32, False),    # an odd number of vectors
    (5, 1, 1, 1, 500, 250, False),
    (600, 1, 8, 1, 64, 16, False),
    (1500, 2, 8, 4, 64, 64, False),  # from here on enough heads to be streamed
    (2100, 1, 8, 1, 128, 32, False),
    (901, 3, 6, 2, 80, 80, True),
    (700, 1, 8, 8, 256, 256, False),
    (13, 1, 2, 1, 96, 24, False),
    (1500, 2, 8, 4, 96, 24, False),  # turns of 8 mod 16 channels
    (801, 3, 6, 2, 80, 40, True),
    (40, 1, 3, 1, 72, 8, False),
    (6, 2, 1, 2, 512, 264, False),
    (3, 1, 1, 2, 64, 0, False),     # nothing turns
]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("s,b,G,hpg,d,r,per_seq", HEADS)
def test_heads(s, b, G, hpg, d, r, per_seq, inter, dt):
    g = torch.Generator(device="cuda").manual_seed(s * 1000 + d)
    qkv = torch.randn(s, b, G, hpg + 2, d, generator=g, device="cuda").to(dt).requires_grad_()
    wq, wk = (1 + 0.2 * torch.randn(2, d, generator=g, device="cuda")).to(dt).unbind(0)
    wq, wk = wq.clone().requires_grad_(), wk.clone().requires_grad_()
    ang = torch.rand((s, b, r // 2) if per_seq else (s, r // 2), generator=g, device="cuda") * 6.28
    cos, sin = ang.cos(), ang.sin()
    dy = torch.randn(qkv.shape, generator=g, device="cuda").to(dt)
    x64 = qkv.detach().double().requires_grad_()
    out = F_.rope_qkv(qkv, cos, sin, hpg + 1, interleaved=inter)
    want = _heads64(x64, hpg + 1, cos, sin, inter)
    assert out.dtype == dt and out.is_contiguous()
    _close(out, want, dt)
    assert torch.equal(out[:, :, :, hpg + 1], qkv[:, :, :, hpg + 1])
    _close(torch.autograd.grad(out, qkv, dy)[0], torch.autograd.grad(want, x64, dy.double())[0], dt)

    out = F_.qk_norm_rope_qkv(qkv, wq, wk, cos, sin, 1e-5, interleaved=inter)
    w64 = [wq.detach().double().requires_grad_(), wk.detach().double().requires_grad_()]
    want = _heads64(x64, hpg + 1, cos, sin, inter, torch.cat([w64[0].expand(hpg, d), w64[1].expand(1, d)]), 1e-5)
    _close(out, want, dt)
    dx, dwq, dwk = torch.autograd.grad(out, [qkv, wq, wk], dy)
    ex, eq, ek = torch.autograd.grad(want, [x64] + w64, dy.double())
    # rstd can be a few units for a short head of small values
    _close(dx, ex, dt, 4.0)
    # sums of n products of unit-variance values: n^1/2 in size, rounded once (n 2^-24 of fp32 sums at most)
    for a, e, n in ((dwq, eq, s * b * G * hpg), (dwk, ek, s * b * G)):
        assert a.dtype == dt
        _close(a, e, dt, 4.0 * math.sqrt(n))


def test_heads_views_and_streams():
    """Views with other strides over s and b, rows off the 16-byte grid, and a side stream."""
    g = torch.Generator(device="cuda").manual_seed(5)
    s, b, G, hpg, d = 21, 3, 2, 2, 64
    n = G * (hpg + 2) * d
    cos, sin = (torch.rand(s, d // 2, generator=g, device="cuda") * 6.28).cos(), torch.zeros(s, d // 2, device="cuda")
    wq, wk = torch.ones(2, d, device="cuda").bfloat16().unbind(0)
    wk = wk.clone()
    base = torch.randn(b, s, n + 24, generator=g, device="cuda").bfloat16()
    for x in (base[:, :, :n], base[:, :, 8:n + 8], base[:, :, 3:n + 3]):
        v = x.unflatten(-1, (G, hpg + 2, d)).transpose(0, 1)
        want = F_.qk_norm_rope_qkv(v.contiguous(), wq, wk, cos, sin, 1e-5)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = F_.qk_norm_rope_qkv(v, wq, wk, cos, sin, 1e-5)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got, want)
    # inner dimensions that are not dense, and a gradient that is a broadcast
    v = torch.randn(s, b, G, hpg + 2, 2 * d, generator=g, device="cuda").bfloat16()[..., ::2]
    assert torch.equal(F_.qk_norm_rope_qkv(v, wq, wk, cos, sin, 1e-5),
                       F_.qk_norm_rope_qkv(v.contiguous(), wq, wk, cos, sin, 1e-5))
    x = v.contiguous().requires_grad_()
    out = F_.qk_norm_rope_qkv(x, wq, wk, cos, sin, 1e-5)
    one = torch.ones((), device="cuda").bfloat16()
    assert torch.equal(torch.autograd.grad(out, x, one.expand(out.shape), retain_graph=True)[0],
                       torch.autograd.grad(out, x, torch.ones_like(out))[0])


def test_heads_main_grad_and_determinism():
    g = torch.Generator(device="cuda").manual_seed(6)
    s, b, G, hpg, d = 513, 2, 4, 3, 128
    qkv = torch.randn(s, b, G, hpg + 2, d, generator=g, device="cuda").bfloat16()
    dy = torch.randn(qkv.shape, generator=g, device="cuda").bfloat16()
    ang = torch.rand(s, d // 2, generator=g, device="cuda") * 6.28
    cos, sin = ang.cos(), ang.sin()
    got = []
    for _ in range(3):
        wq = torch.nn.Parameter(torch.ones(d, device="cuda").bfloat16())
        wk = torch.nn.Parameter(torch.ones(d, device="cuda").bfloat16())
        ready = []
        for w in (wq, wk):
            w.main_grad = torch.ones(d, device="cuda")
            w._grad_ready = lambda: ready.append(1)
        F_.qk_norm_rope_qkv(qkv, wq, wk, cos, sin, 1e-5).backward(dy)
        assert len(ready) == 2 and wq.grad is None and wk.grad is None
        got.append(torch.stack([wq.main_grad, wk.main_grad]))
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
    x64 = qkv.double()
    xh = x64 / (x64.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt()
    gr = _turn(dy.double(), cos, -sin, False)
    dw = (gr * xh).sum((0, 1, 2))
    want = torch.stack([dw[:hpg].sum(0), dw[hpg]]) + 1
    # sums of about 12000 products: 110 in size, each fp32 addition off by at most 2^-24 of it
    torch.testing.assert_close(got[0].double(), want, atol=1e-3, rtol=1e-5)


def test_heads_empty():
    for shape in ((0, 2, 2, 3, 64), (4, 0, 2, 3, 64)):
        x = torch.empty(shape, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        cos = torch.ones(shape[0], 32, device="cuda")
        w = torch.ones(64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
        y = F_.qk_norm_rope_qkv(x, w, w, cos, cos, 1e-5)
        dx, dw = torch.autograd.grad(y, [x, w], torch.empty_like(y))
        assert y.shape == shape and dx.shape == shape and dw.abs().sum() == 0
        assert F_.rope_qkv(x, cos, cos, 2, interleaved=True).shape == shape


def test_heads_refusals():
    x = torch.zeros(4, 2, 2, 3, 64, device="cuda", dtype=torch.bfloat16)
    cos = torch.ones(4, 32, device="cuda")
    w = torch.ones(64, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        F_.rope_qkv(x, cos[:3], cos[:3], 2, interleaved=True)
    for bad in (lambda: F_.rope_qkv(x, cos.double(), cos.double(), 2, interleaved=True),
                lambda: F_.rope_qkv(x, cos.cpu(), cos.cpu(), 2, interleaved=True),
                lambda: F_.rope_qkv(x.double(), cos, cos, 2, interleaved=True),
                lambda: F_.rope_qkv(x, cos.t().contiguous().t(), cos, 2, interleaved=True),
                lambda: F_.qk_norm_rope_qkv(x, w.cpu(), w, cos, cos, 1e-5)):
        with pytest.raises(RuntimeError):
            bad()


# ------------------------------------------------------------------------------------------------ router
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("E,k,sigmoid,bias,groups,topg,renorm", ROUTES)
def test_route(E, k, sigmoid, bias, groups, topg, renorm, dt):
    T = 41
    x, b = route_inputs(T, E, bias, seed=E)
    if dt == torch.float16:
        x = x.clamp(min=-60000.0).masked_fill(x == -math.inf, -math.inf)
    x = x.to(dt)
    dev = x.cuda().requires_grad_()
    bd = b.cuda() if bias else None
    w, e, ss, cnt = F_.moe_route(dev, k, "sigmoid" if sigmoid else "softmax", bd, groups, topg, renorm, 1.5)
    want = [brute_route(r, k, sigmoid, b.tolist() if bias else None, groups, topg, renorm, 1.5)
            for r in x.float().tolist()]
    assert e.tolist() == [v[1] for v in want]
    torch.testing.assert_close(w.cpu().double(), torch.tensor([v[0] for v in want], dtype=torch.float64), atol=1e-6,
                               rtol=1e-5)
    torch.testing.assert_close(ss.cpu().double(), torch.tensor([v[2] for v in want], dtype=torch.float64).sum(0),
                               atol=1e-5, rtol=1e-5)
    assert cnt.tolist() == torch.bincount(e.reshape(-1).long(), minlength=E).tolist()
    # gradient against the host form (whose own is tested against differences)
    g = torch.Generator().manual_seed(1)
    dw, dq = torch.randn(T, k, generator=g), torch.randn(E, generator=g)
    xc = x.clone().requires_grad_()
    wc, ec, sc, _ = F_.moe_route(xc, k, "sigmoid" if sigmoid else "softmax", b, groups, topg, renorm, 1.5)
    assert torch.equal(ec, e.cpu())
    for outs, gouts in (((w, ss), (dw, dq)), ((w,), (dw,)), ((ss,), (dq,))):
        got, = torch.autograd.grad(outs, dev, [v.cuda() for v in gouts], retain_graph=True)
        exp, = torch.autograd.grad((wc, sc) if len(outs) == 2 else (wc,) if outs[0] is w else (sc,), xc, gouts,
                                   retain_graph=True)
        assert got.dtype == dt
        tol = {torch.float32: 2e-5, torch.bfloat16: 2.0 ** -7, torch.float16: 2.0 ** -10}[dt]
        torch.testing.assert_close(got.cpu().float(), exp.float(), atol=2e-5, rtol=tol)


@pytest.mark.parametrize("T,E,k,sigmoid,groups,topg", [(1, 8, 2, False, 1, 1), (5000, 60, 4, False, 4, 2),
                                                       (3001, 256, 8, True, 8, 4), (700, 384, 6, False, 1, 1),
                                                       (2111, 512, 8, True, 16, 4)])
def test_route_many_tokens(T, E, k, sigmoid, groups, topg):
    """Continuous logits: the choice is the one of the host form bit for bit, whatever the order of additions, and
    nothing changes from run to run."""
    g = torch.Generator(device="cuda").manual_seed(T)
    x = torch.randn(T, E, generator=g, device="cuda")
    b = torch.randn(E, generator=g, device="cuda") * 0.05
    first = F_.moe_route(x, k, "sigmoid" if sigmoid else "softmax", b, groups, topg, True, 2.5)
    again = F_.moe_route(x, k, "sigmoid" if sigmoid else "softmax", b, groups, topg, True, 2.5)
    for u, v in zip(first, again):
        assert torch.equal(u, v)
    from elasticmegatron_b200.ops import reference as ref

    w, e, ss, cnt = ref.moe_route_fwd(x, k, sigmoid, b, groups, topg, True, 2.5)
    assert torch.equal(first[1], e) and torch.equal(first[3], cnt)
    torch.testing.assert_close(first[0], w, atol=1e-6, rtol=1e-5)
    torch.testing.assert_close(first[2], ss, atol=1e-4, rtol=1e-5)


def test_route_rows_stay_in_range():
    """NaN and infinite logits: every index is an expert, rows without them are unaffected."""
    x = torch.randn(6, 16, device="cuda")
    x[1, 3] = math.nan
    x[2] = math.nan
    x[3, 5] = math.inf
    x[4] = -math.inf
    for fn in ("softmax", "sigmoid"):
        for kw in ({}, dict(bias=torch.zeros(16, device="cuda")), dict(num_groups=4, group_topk=2)):
            w, e, _, cnt = F_.moe_route(x, 4, fn, **kw)
            assert int(e.min()) >= 0 and int(e.max()) < 16 and int(cnt.sum()) == 24
            assert all(len(set(r)) == 4 for r in e.tolist())
            ok = [0, 5]
            w1, e1, _, _ = F_.moe_route(x[ok], 4, fn, **kw)
            assert torch.equal(w[ok], w1) and torch.equal(e[ok], e1)
            assert w[4].abs().sum() == 0 and e[4].tolist() == [0, 1, 2, 3]


def test_route_strided_rows_and_empty():
    x = torch.randn(33, 40, device="cuda")
    for v in (x[:, 4:20], x[:, ::2][:, :16], x.t()[:33, :16]):
        a, b = F_.moe_route(v, 2, renormalize=True), F_.moe_route(v.contiguous(), 2, renormalize=True)
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    w, e, ss, c = F_.moe_route(torch.empty(0, 8, device="cuda"), 2)
    assert w.shape == (0, 2) and ss.tolist() == [0.0] * 8 and c.tolist() == [0] * 8
    with pytest.raises(RuntimeError):
        F_.moe_route(torch.zeros(4, 8, device="cuda", dtype=torch.float64), 2)
    with pytest.raises(RuntimeError):
        F_.moe_route(torch.zeros(4, 8, device="cuda"), 2, bias=torch.zeros(8))


# ------------------------------------------------------------------------------------------------ long tensors
def test_offsets_past_32_bits():
    """More than 2^31 elements: the last tokens come out as in a call of their own."""
    torch.cuda.empty_cache()
    g = torch.Generator(device="cuda").manual_seed(9)
    s, G, hpg, d = 700000, 4, 4, 128
    x = torch.empty(s, 1, G, hpg + 2, d, device="cuda", dtype=torch.bfloat16).normal_(generator=g)
    assert x.numel() > 2 ** 31
    ang = torch.rand(s, d // 2, generator=g, device="cuda") * 6.28
    cos, sin = ang.cos(), ang.sin()
    w = (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).bfloat16()
    y = F_.qk_norm_rope_qkv(x, w, w, cos, sin, 1e-5)
    n = 70000
    assert torch.equal(y[-n:], F_.qk_norm_rope_qkv(x[-n:], w, w, cos[-n:].clone(), sin[-n:].clone(), 1e-5))
    del y
    # strided rows (the direct kernel): every other token of twice as many
    v = x[::2]
    assert torch.equal(F_.rope_qkv(v, cos[::2].contiguous(), sin[::2].contiguous(), hpg + 1, interleaved=True)[-9:],
                       F_.rope_qkv(v[-9:], cos[::2][-9:].contiguous(), sin[::2][-9:].contiguous(), hpg + 1,
                                   interleaved=True))
    del x, v
    logits = torch.empty(4300000, 512, device="cuda").normal_(generator=g)
    assert logits.numel() > 2 ** 31
    a, b = F_.moe_route(logits, 4, "sigmoid", num_groups=8, group_topk=2), F_.moe_route(logits[-999:], 4, "sigmoid",
                                                                                    num_groups=8, group_topk=2)
    assert torch.equal(a[0][-999:], b[0]) and torch.equal(a[1][-999:], b[1]) and int(a[3].sum()) == 4 * 4300000
    del logits, a, b
    torch.cuda.empty_cache()

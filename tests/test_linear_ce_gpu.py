"""Linear cross entropy kernels (csrc/gemm/linear_ce.cu) against 64 bits.

The gradient of the logits P is rounded to bf16 (8 significant bits: at most 2^-8 relative) before the two products and
the result once more, so an element of dx is off by at most 2^-8 (|P| |w| + |dx|), one of dw by 2^-8 (|P|^T |x| + |dw|); fp32 sums and exponentials
add far less (bounded here by a tenth of that)."""
import math

import pytest
import torch

from elasticmegatron_b200.ops import functional as F_

pytestmark = pytest.mark.gpu


def make(T, V, H, seed=0, ignore=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = (torch.randn(V, H, generator=g, device="cuda") * 0.05).bfloat16()
    labels = torch.randint(0, V, (T,), generator=g, device="cuda")
    # from untrained to certain tokens
    x = torch.randn(T, H, generator=g, device="cuda") + 8 * torch.rand(T, 1, generator=g, device="cuda") * w[labels].float() / 0.05 / math.sqrt(H)
    if ignore and T > 3:
        labels[1], labels[2], labels[3] = -100, V, -7
    return x.bfloat16(), w, labels, torch.randn(T, generator=g, device="cuda")


def exact(x, w, labels, dloss):
    """(loss, dx, dw) in 64 bits and the bounds of the gradients' errors."""
    x, w, V = x.double(), w.double(), w.shape[0]
    z = x @ w.t()
    ok = (labels >= 0) & (labels < V)
    at = torch.where(ok, labels, 0)[:, None]
    lse = torch.logsumexp(z, -1)
    loss = torch.where(ok, lse - z.gather(1, at).squeeze(1), 0.0)
    p = torch.exp(z - lse[:, None])
    p.scatter_add_(1, at, -torch.ones_like(at, dtype=torch.float64))
    p *= (dloss.double() * ok)[:, None]
    dx, dw = p @ w, p.t() @ x
    u = 1.1 * 2.0 ** -8
    return loss, dx, dw, u * (p.abs() @ w.abs()), u * (p.t().abs() @ x.abs())


def check(a, e, bound, rounded=True):
    lim = bound + (1.1 * 2.0 ** -8 * e.abs() if rounded else 0) + 1e-7
    over = (a.double() - e).abs() - lim
    assert float(over.max()) <= 0, (float(over.max()), float(lim.max()))


SIZES = [(1, 1000, 64), (1, 5, 8), (3, 257, 72), (128, 513, 256), (129, 4097, 136), (250, 32001, 512), (300, 2049, 1024),
         (1, 32000, 1024), (777, 1025, 264), (1500, 6000, 520), (64, 50001, 128),
         (4000, 300, 64), (3000, 100, 72), (2500, 1000, 264), (100, 3000, 520), (128, 700, 1032)]


@pytest.mark.parametrize("T,V,H", SIZES)
def test_against_64_bits(T, V, H):
    x, w, labels, dloss = make(T, V, H)
    loss, dx, dw, bx, bw = exact(x, w, labels, dloss)
    x.requires_grad_(), w.requires_grad_()
    got = F_.linear_cross_entropy(x, w, labels)
    # logits: fp32 sums of H products of O(1); the loss adds a few units in the last place of values up to 50
    torch.testing.assert_close(got.double(), loss, atol=3e-5, rtol=1e-6)
    gx, gw = torch.autograd.grad(got, [x, w], dloss)
    assert gx.dtype == torch.bfloat16 and gw.dtype == torch.bfloat16
    check(gx, dx, bx)
    check(gw, dw, bw)
    if T > 3:
        assert got[1] == 0 and got[2] == 0 and got[3] == 0 and gx[1:4].abs().sum() == 0


@pytest.mark.parametrize("T,V,H,piece", [(300, 2049, 256, 256), (300, 2049, 256, 1024), (40, 3001, 128, 512),
                                         (2000, 5000, 512, 2048), (1, 2000, 64, 256), (700, 1281, 4096, 256),
                                         (2600, 300, 128, 1024), (3000, 100, 72, 256), (120, 2000, 256, 512)])
def test_pieces_main_grad_and_determinism(T, V, H, piece, monkeypatch):
    x, w, labels, dloss = make(T, V, H, seed=3)
    loss, dx, dw, bx, bw = exact(x, w, labels, dloss)
    monkeypatch.setattr(F_, "LINEAR_CE_PIECE", piece)
    runs = []
    for _ in range(3):
        p = torch.nn.Parameter(w.clone())
        p.main_grad = torch.ones(V, H, device="cuda")
        xi = x.clone().requires_grad_()
        got = F_.linear_cross_entropy(xi, p, labels)
        got.backward(dloss)
        assert p.grad is None
        runs.append((got.detach(), xi.grad, p.main_grad))
    check(runs[0][1], dx, bx)
    # the sum with the ones in the buffer is rounded to fp32
    check(runs[0][2] - 1, dw, bw + 3e-7 * (1 + dw.abs()), rounded=False)
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


def test_only_wanted_gradients_views_and_streams():
    x, w, labels, dloss = make(200, 3000, 256, seed=5)
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    loss = F_.linear_cross_entropy(xg, wg, labels)
    gx, gw = torch.autograd.grad(loss, [xg, wg], dloss)
    l1 = F_.linear_cross_entropy(xg, w, labels)
    assert torch.equal(torch.autograd.grad(l1, xg, dloss)[0], gx)
    l2 = F_.linear_cross_entropy(x, wg, labels)
    assert torch.equal(torch.autograd.grad(l2, wg, dloss)[0], gw)
    # rows with other strides, rows off the 16-byte grid, strided labels, a broadcast gradient, another stream
    wide = torch.zeros(200, 264, device="cuda", dtype=torch.bfloat16)
    wide[:, 8:] = x
    odd = torch.zeros(3000, 257, device="cuda", dtype=torch.bfloat16)
    odd[:, 1:] = w
    lab2 = torch.stack([labels, labels], 1)[:, 0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        l3 = F_.linear_cross_entropy(wide[:, 8:], odd[:, 1:], lab2)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(l3, loss)
    one = torch.ones((), device="cuda")
    a = torch.autograd.grad(F_.linear_cross_entropy(xg, w, labels), xg, one.expand(200))[0]
    b = torch.autograd.grad(F_.linear_cross_entropy(xg, w, labels).sum(), xg)[0]
    assert torch.equal(a, b)


def test_all_ignored_and_empty():
    x, w, labels, dloss = make(130, 1000, 64, ignore=False)
    labels[:] = -100
    x.requires_grad_(), w.requires_grad_()
    loss = F_.linear_cross_entropy(x, w, labels)
    gx, gw = torch.autograd.grad(loss, [x, w], dloss)
    assert loss.abs().sum() == 0 and gx.abs().sum() == 0 and gw.abs().sum() == 0
    loss = F_.linear_cross_entropy(x[:0], w, labels[:0])
    gx, gw = torch.autograd.grad(loss, [x, w], loss)
    assert loss.shape == (0,) and gx.abs().sum() == 0 and gw.abs().sum() == 0


def test_nan_stays_in_its_row():
    x, w, labels, dloss = make(140, 1000, 64, ignore=False)
    x[7] = math.nan
    loss = F_.linear_cross_entropy(x, w, labels)
    assert torch.isnan(loss[7]) and int(torch.isnan(loss).sum()) == 1
    labels[7] = -100  # an ignored row gives no gradient whatever it holds
    x.requires_grad_()
    loss = F_.linear_cross_entropy(x, w, labels)
    gx, = torch.autograd.grad(loss, x, dloss)
    assert loss[7] == 0 and gx[7].abs().sum() == 0 and bool(torch.isfinite(gx).all())


def test_raw_statistics_join_like_ranks():
    """The per-rank statistics of two halves of the vocabulary give the whole loss (what a tensor-parallel group
    reduces), and the gradients of the halves are those of the whole."""
    from elasticmegatron_b200.ops.native import ext

    x, w, labels, dloss = make(300, 2048, 128, seed=8)
    whole, top, total = ext().linear_ce_fwd(x, w, labels, 0, 2048, -100, False)
    dx, dw = ext().linear_ce_bwd(dloss, x, w, labels, top, total, 0, 2048, -100, True, True, None, 0)
    st = [ext().linear_ce_fwd(x, w[h * 1024:(h + 1) * 1024], labels, h * 1024, 2048, -100, True) for h in (0, 1)]
    m = torch.maximum(st[0][1], st[1][1])
    joined = sum(s * torch.exp(t - m) for _, t, _, s in st)
    target = st[0][0] + st[1][0]
    ok = (labels >= 0) & (labels < 2048)
    torch.testing.assert_close(torch.where(ok, torch.log(joined) + m - target, 0.0), whole, atol=1e-5, rtol=1e-6)
    dxs = torch.zeros_like(x, dtype=torch.float32)
    for h in (0, 1):
        px, pw = ext().linear_ce_bwd(dloss, x, w[h * 1024:(h + 1) * 1024], labels, top, total, h * 1024, 2048, -100, True, True,
                                     None, 0)
        dxs += px.float()
        assert torch.equal(pw, dw[h * 1024:(h + 1) * 1024])
    torch.testing.assert_close(dxs, dx.float(), atol=2e-2, rtol=2.0 ** -6)


def test_refusals():
    x, w, labels, _ = make(20, 100, 64)
    with pytest.raises(ValueError):
        F_.linear_cross_entropy(x[:, :60], w[:, :60], labels)
    for bad in (lambda: F_.linear_cross_entropy(x.float(), w.float(), labels),
                lambda: F_.linear_cross_entropy(x, w, labels.cpu()), lambda: F_.linear_cross_entropy(x, w.cpu(), labels)):
        with pytest.raises(RuntimeError):
            bad()


def test_offsets_past_32_bits():
    """A weight and a piece of P of more than 2^31 elements: the loss and gradients of labels at the end of the vocabulary."""
    torch.cuda.empty_cache()
    g = torch.Generator(device="cuda").manual_seed(11)
    T, V, H = 9, 140000, 16384
    w = torch.empty(V, H, device="cuda", dtype=torch.bfloat16).normal_(0, 0.02, generator=g)
    assert w.numel() > 2 ** 31
    x = torch.randn(T, H, generator=g, device="cuda").bfloat16()
    labels = V - 1 - torch.arange(T, device="cuda")
    z = torch.cat([x.double() @ w[v:v + 10000].double().t() for v in range(0, V, 10000)], 1)
    want = torch.logsumexp(z, -1) - z.gather(1, labels[:, None]).squeeze(1)
    w.requires_grad_()
    loss = F_.linear_cross_entropy(x, w, labels)
    p = torch.softmax(z, -1)
    # the tensor cores cut their fp32 sum off at each of the H / 16 steps, by at most 2^-23 of a partial sum that grows to
    # the logit: 2^-24 H / 16 of it in all.  The log of the sum moves by the softmax average of that.
    bound = 3e-5 + 2.0 ** -24 * H / 16 * (p * z.abs()).sum(-1)
    assert bool(((loss.double() - want).abs() <= bound).all())
    gw, = torch.autograd.grad(loss.sum(), w)
    p[torch.arange(T), labels] -= 1.0
    for rows in (slice(0, 64), slice(V - 64, V)):
        e = p[:, rows].t() @ x.double()
        check(gw[rows], e, 1.1 * 2.0 ** -8 * (p[:, rows].t().abs() @ x.double().abs()))
    del w, gw, z, p
    # P of one piece: 20000 tokens by 110000 words
    T, V, H = 20000, 110000, 64
    x = torch.randn(T, H, generator=g, device="cuda").bfloat16().requires_grad_()
    w = (torch.randn(V, H, generator=g, device="cuda") * 0.05).bfloat16()
    labels = torch.randint(0, V, (T,), generator=g, device="cuda")
    whole = {}
    for piece in (V, 4096):
        F_.LINEAR_CE_PIECE, keep = piece, F_.LINEAR_CE_PIECE
        try:
            loss = F_.linear_cross_entropy(x, w, labels)
            whole[piece] = torch.autograd.grad(loss.sum(), x)[0].float()
        finally:
            F_.LINEAR_CE_PIECE = keep
    # the same P and fp32 sums, in another order, rounded once
    torch.testing.assert_close(whole[V], whole[4096], atol=1e-5, rtol=2.0 ** -7)
    torch.cuda.empty_cache()


def test_captured_in_a_graph():
    """A step of all operators in one CUDA graph gives what the calls give one by one."""
    g = torch.Generator(device="cuda").manual_seed(13)
    x, w, labels, dloss = make(300, 3001, 128, seed=13)
    x.requires_grad_(), w.requires_grad_()
    qkv = torch.randn(2000, 2, 4, 6, 64, generator=g, device="cuda").bfloat16().requires_grad_()
    nw = torch.ones(64, device="cuda").bfloat16().requires_grad_()
    ang = torch.rand(2000, 32, generator=g, device="cuda")
    cos, sin = ang.cos(), ang.sin()
    logits = torch.randn(3000, 64, generator=g, device="cuda").requires_grad_()

    def step():
        y = F_.qk_norm_rope_qkv(qkv, nw, nw, cos, sin, 1e-5)
        z = F_.rope_qkv(y, cos, sin, 5, interleaved=True)
        wt, ex, ss, ct = F_.moe_route(logits, 4, "sigmoid", num_groups=8, group_topk=2, renormalize=True)
        loss = F_.linear_cross_entropy(x, w, labels)
        grads = torch.autograd.grad([z, wt, ss, loss], [qkv, nw, logits, x, w],
                                    [torch.ones_like(z), wt.detach(), ss.detach(), dloss])
        return [z, wt, ex, ss, ct, loss, *grads]

    want = [t.detach().clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(2):
        for t in got:
            t.detach().zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))

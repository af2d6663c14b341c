"""Linear cross entropy: host form against 64-bit autograd, pieces of the vocabulary, ignored labels, tensor parallelism
on gloo ranks, refusals."""
import pytest
import torch

from elasticmegatron_b200.ops import functional as F_
from tests.dist_utils import run_distributed


def make(T, V, H, seed=0, ignore=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, H, generator=g)
    w = torch.randn(V, H, generator=g) * 0.3
    labels = torch.randint(0, V, (T,), generator=g)
    if ignore and T > 3:
        labels[1], labels[2], labels[3] = -100, V, -7
    return x, w, labels, torch.randn(T, generator=g)


def exact(x, w, labels, dloss, ignore=-100):
    """64-bit (loss, dx, dw) by autograd over the kept logits."""
    x, w = x.double().requires_grad_(), w.double().requires_grad_()
    z = x @ w.t()
    ok = (labels >= 0) & (labels < w.shape[0]) & (labels != ignore)
    loss = torch.zeros(x.shape[0], dtype=torch.float64, device=x.device)
    loss = torch.where(ok, torch.logsumexp(z, -1) - z.gather(1, torch.where(ok, labels, 0)[:, None]).squeeze(1), loss)
    return (loss.detach(),) + torch.autograd.grad(loss, [x, w], dloss.double())


@pytest.mark.parametrize("piece", [0, 1, 7, 1000])
@pytest.mark.parametrize("T,V,H", [(1, 1, 8), (5, 37, 16), (40, 300, 64)])
def test_against_autograd(T, V, H, piece, monkeypatch):
    monkeypatch.setattr(F_, "LINEAR_CE_PIECE", piece)
    x, w, labels, dloss = make(T, V, H)
    want = exact(x, w, labels, dloss)
    x.requires_grad_(), w.requires_grad_()
    loss = F_.linear_cross_entropy(x, w, labels)
    assert loss.dtype == torch.float32
    got = (loss,) + torch.autograd.grad(loss, [x, w], dloss)
    for a, e in zip(got, want):  # fp32 sums of at most 300 terms of O(1)
        torch.testing.assert_close(a.double(), e, atol=1e-4, rtol=1e-5)
    if T > 3:
        assert loss[1] == 0 and loss[2] == 0 and loss[3] == 0 and got[1][1:4].abs().sum() == 0


def test_matches_the_unfused_pair_and_main_grad():
    x, w, labels, _ = make(24, 96, 32, seed=2, ignore=False)
    out = []
    for fused in (False, True):
        p = torch.nn.Parameter(w.clone())
        p.main_grad = torch.ones(96, 32)
        ready = []
        p._grad_ready = lambda: ready.append(1)
        xi = x.clone().requires_grad_()
        if fused:
            loss = F_.linear_cross_entropy(xi, p, labels)
        else:
            loss = F_.vocab_parallel_cross_entropy(F_.linear(xi, p), labels, 0, None)
        loss.mean().backward()
        assert ready == [1] and p.grad is None
        out.append((loss.detach(), xi.grad, p.main_grad))
    for a, e in zip(*out):
        torch.testing.assert_close(a, e, atol=1e-5, rtol=1e-5)


def test_differences():
    x, w, labels, dloss = make(3, 11, 8, seed=4, ignore=False)
    x.requires_grad_(), w.requires_grad_()
    dx, dw = torch.autograd.grad(F_.linear_cross_entropy(x, w, labels), [x, w], dloss)
    h = 1e-6

    def value(a, b):
        z = a @ b.t()
        return ((torch.logsumexp(z, -1) - z.gather(1, labels[:, None]).squeeze(1)) * dloss.double()).sum().item()

    for which, grad in ((0, dx), (1, dw)):
        for i in range(0, grad.numel(), 5):
            up, down = [x.detach().double(), w.detach().double()], [x.detach().double(), w.detach().double()]
            up[which] = up[which].clone()
            down[which] = down[which].clone()
            up[which].view(-1)[i] += h
            down[which].view(-1)[i] -= h
            assert abs(grad.view(-1)[i].item() - (value(*up) - value(*down)) / (2 * h)) < 1e-5


def _tp(rank, world, mode):
    import torch.distributed as dist

    g = dist.group.WORLD
    T, V, H = 12, 64, 16
    x, w, labels, dloss = make(T, V, H, seed=6)
    n = V // world
    wl = torch.nn.Parameter(w[rank * n:(rank + 1) * n].clone())
    wl.main_grad = torch.zeros(n, H)
    xl = (x[rank * (T // world):(rank + 1) * (T // world)] if mode == "col_sp" else x).clone().requires_grad_()
    loss = F_.linear_cross_entropy(xl, wl, labels, rank * n, mode, g)
    loss.backward(dloss)
    return loss.detach(), xl.grad, wl.main_grad


@pytest.mark.parametrize("mode", ["col", "col_sp"])
def test_tensor_parallel(mode):
    x, w, labels, dloss = make(12, 64, 16, seed=6)
    loss, dx, dw = exact(x, w, labels, dloss)
    res = run_distributed(_tp, 2, mode)
    for r, (l, gx, gw) in enumerate(res):
        torch.testing.assert_close(l.double(), loss, atol=1e-5, rtol=1e-5)
        torch.testing.assert_close(gw.double(), dw[r * 32:(r + 1) * 32], atol=1e-5, rtol=1e-5)
        torch.testing.assert_close(gx.double(), dx[r * 6:(r + 1) * 6] if mode == "col_sp" else dx, atol=1e-5, rtol=1e-5)


def test_refusals():
    x, w, labels, _ = make(6, 20, 16)
    for bad in (lambda: F_.linear_cross_entropy(x[0], w, labels), lambda: F_.linear_cross_entropy(x, w[:, :8], labels),
                lambda: F_.linear_cross_entropy(x, w.double(), labels), lambda: F_.linear_cross_entropy(x, w, labels[:5]),
                lambda: F_.linear_cross_entropy(x, w, labels.int()), lambda: F_.linear_cross_entropy(x, w[:0], labels),
                lambda: F_.linear_cross_entropy(x[:, :12], w[:, :12], labels),
                lambda: F_.linear_cross_entropy(x, w, labels, vocab_start=4)):
        with pytest.raises(ValueError):
            bad()

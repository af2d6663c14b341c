"""Linear cross entropy kernels (csrc/gemm/linear_ce.cu) in rarer uses."""
import math

import pytest
import torch

from elasticmegatron_b200.ops import functional as F_
from elasticmegatron_b200.ops.native import ext
from test_linear_ce_gpu import exact, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [20, 300])
def test_nan_in_a_row_of_w(T):
    """A NaN in a row of w is in every token's sum, whichever label the token has; ignored tokens keep loss 0."""
    x, w, labels, _ = make(T, 1000, 64, seed=1)
    w[777] = math.nan
    labels[labels == 777] = 5
    labels[0] = 777
    counts = (labels >= 0) & (labels < 1000)
    loss = F_.linear_cross_entropy(x, w, labels)
    assert bool(torch.isnan(loss[counts]).all()) and loss[~counts].abs().sum() == 0
    # a rank's share of the vocabulary passes it on in both sums, the other rank's share is unaffected
    for lo, hi, bad in ((0, 512, False), (512, 1000, True)):
        target, top, total, loss_total = ext().linear_ce_fwd(x, w[lo:hi], labels, lo, 1000, -100, True)
        assert bool((torch.isnan(total) == bad).all()) and bool((torch.isnan(loss_total) == bad).all())


@pytest.mark.parametrize("main", [False, True])
@pytest.mark.parametrize("T", [20, 300])
def test_loss_changes_in_place(T, main):
    """The loss is a tensor of its own: scaled, masked and filled in place as any other, without touching what the
    backward pass has kept."""
    x, w, labels, _ = make(T, 1000, 64, seed=2)
    mask = (torch.arange(T, device="cuda") % 3 > 0).float()
    grads = []
    for inplace in (False, True):
        xi, p = x.clone().requires_grad_(), torch.nn.Parameter(w.clone())
        if main:
            p.main_grad = torch.zeros(1000, 64, device="cuda")
        loss = F_.linear_cross_entropy(xi, p, labels)
        if inplace:
            loss *= mask
            loss /= 2.0
            loss.masked_fill_(labels < 0, 0.0)
        else:
            loss = torch.where(labels < 0, 0.0, loss * mask / 2.0)
        loss.sum().backward()
        grads.append((loss.detach(), xi.grad, p.main_grad if main else p.grad))
    for a, b in zip(*grads):
        assert torch.equal(a, b)
    # without gradients, and after the pass that kept the statistics
    xi = x.clone().requires_grad_()
    loss = F_.linear_cross_entropy(xi, w, labels)
    with torch.no_grad():
        loss.zero_()
    loss.sum().backward()
    xj = x.clone().requires_grad_()
    F_.linear_cross_entropy(xj, w, labels).sum().backward()
    assert torch.equal(xi.grad, xj.grad)


@pytest.mark.parametrize("T,H,V,piece", [(1024, 1024, 16384, 256), (100, 1024, 16384, 256), (2048, 512, 32768, 4096),
                                         (100, 512, 32768, 0), (1500, 1024, 2048, 0)])
def test_backward_memory(T, H, V, piece, monkeypatch):
    """Beside the gradients: a bf16 [rows, piece] buffer, one fp32 [T, H] sum and, where a product is split over the
    SMs, one fp32 part of 128 x 256 for each of them.  Smaller pieces take less, not more."""
    monkeypatch.setattr(F_, "LINEAR_CE_PIECE", piece)
    x, w, labels, dloss = make(T, V, H, seed=4)
    x.requires_grad_(), w.requires_grad_()
    loss = F_.linear_cross_entropy(x, w, labels)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    start = torch.cuda.memory_allocated()
    grads = torch.autograd.grad(loss, [x, w], dloss)
    torch.cuda.synchronize()
    used = torch.cuda.max_memory_allocated() - start
    rows = 2 * T if T <= 128 else T
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    bound = 2 * (T + V) * H + 2 * rows * min(piece or V, V) + 4 * T * H + 4 * sms * 128 * 256
    if T <= 128:
        bound += 2 * rows * H  # x twice, for the product with both rows of a token
    # small vectors, and what the allocator rounds each block up to (2 MB for blocks over 1 MB)
    assert used <= bound + 6 * 2 ** 21, (used, bound)
    assert len(grads) == 2


@pytest.mark.parametrize("T", [40, 128, 129, 700])
def test_error_of_the_gradients(T):
    """Relative error (2-norms) of dx and dw against rounding the exact gradients to bf16 alone.  Rounding each term of a
    sum of terms of random signs costs as much again, independently: a factor of 2^1/2, of which up to 128 tokens
    2^-8 of the second summand is left.  5 % for the fp32 sums and the chance in both figures."""
    V, H = 6000, 256
    x, w, labels, _ = make(T, V, H, seed=6, ignore=False)
    dloss = torch.full((T,), 1.0 / T, device="cuda")
    _, dx, dw, _, _ = exact(x, w, labels, dloss)
    x.requires_grad_(), w.requires_grad_()
    got = torch.autograd.grad(F_.linear_cross_entropy(x, w, labels), [x, w], dloss)
    for a, e in zip(got, (dx, dw)):
        rel = float((a.double() - e).norm()) / float((e.bfloat16().double() - e).norm())
        assert rel < 1.05 * (1.0 if T <= 128 else math.sqrt(2.0)), rel

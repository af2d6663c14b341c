"""Whole bf16 heads in halves with one table (the model's default form of rope_qkv): what it accepts, and refusals."""
import pytest
import torch

from elasticmegatron_b200.ops import functional as F_
from test_decoder_ops_gpu import _close, _heads64

pytestmark = pytest.mark.gpu


def _inputs(s, b, G, S, d, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ang = torch.rand(s, d // 2, generator=g, device="cuda") * 6.28
    qkv, dy = torch.randn(2, s, b, G, S, d, generator=g, device="cuda").bfloat16().unbind(0)
    return qkv.clone(), dy.clone(), ang.cos(), ang.sin()


@pytest.mark.parametrize("s,b,G,hpg,d", [(9, 2, 2, 1, 8), (5, 1, 3, 2, 24), (33, 2, 1, 4, 40), (17, 1, 2, 1, 72),
                                         (2100, 2, 4, 2, 88), (12, 2, 2, 2, 64), (7, 1, 1, 1, 10)])
def test_any_even_head_size(s, b, G, hpg, d):
    qkv, dy, cos, sin = _inputs(s, b, G, hpg + 2, d)
    x64 = qkv.double().requires_grad_()
    want = _heads64(x64, hpg + 1, cos, sin, False)
    qkv.requires_grad_()
    out = F_.rope_qkv(qkv, cos, sin, hpg + 1)
    _close(out, want, torch.bfloat16)
    _close(torch.autograd.grad(out, qkv, dy)[0], torch.autograd.grad(want, x64, dy.double())[0], torch.bfloat16)


@pytest.mark.parametrize("off", [1, 3, 4, 8])
def test_dense_views_off_the_vector_grid(off):
    s, b, G, S, d = 21, 2, 2, 4, 64
    qkv, dy, cos, sin = _inputs(s, b, G, S, d, seed=off)
    x = qkv.clone().requires_grad_()
    want = F_.rope_qkv(x, cos, sin, 3)
    wdx, = torch.autograd.grad(want, x, dy)
    pad = torch.zeros(qkv.numel() + off, device="cuda", dtype=torch.bfloat16)

    def moved(t):
        v = pad.clone()[off:]
        v.copy_(t.reshape(-1))
        return v.view(t.shape)

    y = moved(qkv).requires_grad_()
    assert y.is_contiguous()
    out = F_.rope_qkv(y, cos, sin, 3)
    assert torch.equal(out, want) and torch.equal(torch.autograd.grad(out, y, moved(dy))[0], wdx)


def test_refusals():
    qkv, _, cos, sin = _inputs(4, 2, 2, 3, 64)
    both = torch.cat([cos, sin], -1)
    for bad in (lambda: F_.rope_qkv(qkv, cos[:3], sin[:3], 2), lambda: F_.rope_qkv(qkv, cos, sin[:3], 2),
                lambda: F_.rope_qkv(qkv, cos, sin[:, :16].contiguous(), 2), lambda: F_.rope_qkv(qkv, cos, sin[0], 2),
                lambda: F_.rope_qkv(qkv, cos, sin, 4), lambda: F_.rope_qkv(qkv, cos, sin, -1),
                lambda: F_.rope_qkv(qkv[0], cos, sin, 2)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: F_.rope_qkv(qkv, cos, sin.cpu(), 2), lambda: F_.rope_qkv(qkv, cos.cpu(), sin, 2),
                lambda: F_.rope_qkv(qkv, cos, sin.double(), 2), lambda: F_.rope_qkv(qkv, *both.chunk(2, -1), 2),
                lambda: F_.rope_qkv(qkv, torch.cat([cos, cos])[::2], sin, 2),
                lambda: F_.rope_qkv(qkv, cos, sin[:1].expand(4, -1), 2)):
        with pytest.raises(RuntimeError):
            bad()

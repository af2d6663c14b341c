"""One parameter as query and key weight of the normalised heads, on the kernels."""
import pytest
import torch

from elasticmegatron_b200.ops import functional as F_
from test_shared_head_norm_cpu import _main_grads

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("s,d", [(7, 64), (40, 100), (3000, 128)])  # direct kernel, single channels, streamed kernel
def test_one_weight_with_main_grad(s, d):
    g = torch.Generator(device="cuda").manual_seed(s)
    qkv, dy = torch.randn(2, s, 2, 2, 5, d, generator=g, device="cuda").bfloat16().unbind(0)
    ang = torch.rand(s, d // 2, generator=g, device="cuda")
    args = (qkv, dy, ang.cos(), ang.sin(), d)
    (q, k), n = _main_grads(False, *args)
    # the query heads' sum is added to 0, then the key heads' to that; the same in every run
    for _ in range(5):
        (both,), once = _main_grads(True, *args)
        assert torch.equal(both, q + k) and once == 1
    assert n == 2
    # accumulators that overlap without being the same: the words in common get both
    w = [torch.nn.Parameter(torch.ones(d, device="cuda").bfloat16()) for _ in range(2)]
    buf = torch.zeros(d + 4, device="cuda")
    w[0].main_grad, w[1].main_grad = buf[:d], buf[4:]
    F_.qk_norm_rope_qkv(qkv, w[0], w[1], *args[2:4], 1e-5).backward(dy)
    want = torch.zeros_like(buf)
    want[:d] += q
    want[4:] += k
    assert torch.equal(buf, want)

"""One parameter as query and key weight of the normalised heads."""
import torch

from elasticmegatron_b200.ops import functional as F_


def _main_grads(shared, qkv, dy, cos, sin, d):
    """Gradients of the query and key weights, as one parameter or two, and how often a hook was called."""
    ready = []
    ws = []
    for _ in range(1 if shared else 2):
        w = torch.nn.Parameter(torch.ones(d, device=qkv.device, dtype=qkv.dtype))
        w.main_grad = torch.zeros(d, device=qkv.device)
        w._grad_ready = lambda: ready.append(1)
        ws.append(w)
    F_.qk_norm_rope_qkv(qkv, ws[0], ws[-1], cos, sin, 1e-5).backward(dy)
    return [w.main_grad for w in ws], len(ready)


def test_one_weight_with_main_grad():
    g = torch.Generator().manual_seed(3)
    qkv, dy = torch.randn(2, 5, 2, 2, 4, 16, generator=g).unbind(0)
    ang = torch.rand(5, 8, generator=g)
    args = (qkv, dy, ang.cos(), ang.sin(), 16)
    (q, k), n = _main_grads(False, *args)
    (both,), once = _main_grads(True, *args)
    # the query heads' sum is added to 0, then the key heads' to that
    assert torch.equal(both, q + k) and n == 2 and once == 1

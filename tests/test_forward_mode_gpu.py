"""Forward-mode differentiation of the decoder-step operators on CUDA."""
import pytest
import torch

from elasticmegatron_b200.ops import functional as F_

pytestmark = pytest.mark.gpu


def test_forward_mode_is_refused():
    """No operator has a forward-mode rule: an input with a tangent is refused, as on the host, not taken as constant."""
    import torch.autograd.forward_ad as fwAD

    g = torch.Generator(device="cuda").manual_seed(2)
    qkv = torch.randn(4, 2, 2, 3, 64, generator=g, device="cuda").bfloat16()
    w = torch.ones(64, device="cuda").bfloat16()
    cos = torch.ones(4, 32, device="cuda")
    logits = torch.randn(5, 8, generator=g, device="cuda")
    x, wo = torch.randn(45, 64, generator=g, device="cuda").bfloat16().split([5, 40])
    labels = torch.arange(5, device="cuda")
    for refuse, of in (
            (lambda t: F_.rope_qkv(t, cos, cos, 2), qkv), (lambda t: F_.rope_qkv(t, cos, cos, 2, interleaved=True), qkv),
            (lambda t: F_.rope_qkv(qkv, t, cos, 2, interleaved=True), cos),
            (lambda t: F_.qk_norm_rope_qkv(t, w, w, cos, cos, 1e-5), qkv),
            (lambda t: F_.qk_norm_rope_qkv(qkv, w, t, cos, cos, 1e-5), w),
            (lambda t: F_.qk_norm_rope_qkv(qkv, w, w, cos, t, 1e-5), cos),
            (lambda t: F_.moe_route(t, 2), logits), (lambda t: F_.moe_route(logits, 2, bias=t), cos[0, :8].clone()),
            (lambda t: F_.linear_cross_entropy(t, wo, labels), x), (lambda t: F_.linear_cross_entropy(x, t, labels), wo)):
        with fwAD.dual_level():
            with pytest.raises(NotImplementedError):
                refuse(fwAD.make_dual(of, torch.ones_like(of)))
        refuse(of)

"""Head norms without a weight are refused."""
import pytest
import torch

from elasticmegatron_b200.ops import functional as F_


def refuse_missing_weights(device, dtype):
    qkv = torch.randn(4, 2, 2, 3, 64, device=device).to(dtype)
    w, cos = torch.ones(64, device=device).to(dtype), torch.ones(4, 32, device=device)
    for q, k in ((None, w), (w, None), (None, None)):
        with pytest.raises(ValueError):
            F_.qk_norm_rope_qkv(qkv, q, k, cos, cos, 1e-5)


def test_missing_weights():
    refuse_missing_weights("cpu", torch.float32)


@pytest.mark.gpu
def test_missing_weights_on_a_gpu():
    refuse_missing_weights("cuda", torch.bfloat16)

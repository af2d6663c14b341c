"""Whole heads in halves with one table (the model's default) are checked like every other form of rope_qkv."""
import pytest
import torch

from elasticmegatron_b200.ops import functional as F_


def test_refusals():
    qkv = torch.randn(4, 2, 2, 3, 16)
    cos, sin = torch.ones(4, 8), torch.zeros(4, 8)
    for bad in (lambda: F_.rope_qkv(qkv[0], cos, sin, 2), lambda: F_.rope_qkv(qkv, cos[:3], sin[:3], 2),
                lambda: F_.rope_qkv(qkv, cos, sin[:1], 2), lambda: F_.rope_qkv(qkv, cos, sin[:, :1], 2),
                lambda: F_.rope_qkv(qkv, cos, sin[:, :4], 2), lambda: F_.rope_qkv(qkv, cos, sin, 4),
                lambda: F_.rope_qkv(qkv, cos, sin, -1)):
        with pytest.raises(ValueError):
            bad()
    assert F_.rope_qkv(qkv, cos, sin, 3).shape == qkv.shape

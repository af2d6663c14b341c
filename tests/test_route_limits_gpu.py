"""Router kernels (csrc/moe/route.cu) at the limits of what they accept."""
import math

import pytest
import torch

from elasticmegatron_b200.ops import functional as F_

pytestmark = pytest.mark.gpu


WIDE = [  # E, k, sigmoid, groups, topg: more than 256 experts in 31 or 32 groups, valued from shared memory
    (288, 4, False, 32, 4), (310, 8, True, 31, 4), (384, 8, False, 32, 4), (480, 8, True, 32, 31), (496, 9, True, 31, 3),
    (512, 8, True, 32, 2), (512, 32, False, 32, 3)]


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("E,k,sigmoid,groups,topg", WIDE)
def test_many_groups_of_many_experts(E, k, sigmoid, groups, topg, dt):
    """Against 64 bits, for the tokens whose choice does not hang on less than 1e-5 (fp32 scores of at most 1 and sums of at
    most 16 of them are off by less than 2e-6)."""
    T = 67
    g = torch.Generator(device="cuda").manual_seed(E + k)
    x = (3 * torch.randn(T, E, generator=g, device="cuda")).to(dt).requires_grad_()
    bias = 0.05 * torch.randn(E, generator=g, device="cuda")
    w, e, ss, cnt = F_.moe_route(x, k, "sigmoid" if sigmoid else "softmax", bias, groups, topg, True, 1.5)
    s = (torch.sigmoid if sigmoid else lambda v: torch.softmax(v, -1))(x.detach().double())
    c = s + bias.double()
    per, best = E // groups, max(1, k // topg)
    value = c.view(T, groups, per).topk(min(best, per), -1).values.sum(-1).sort(-1, descending=True)
    kept = torch.zeros(T, groups, dtype=torch.bool, device="cuda").scatter(1, value.indices[:, :topg], True)
    c = c.masked_fill(~kept.repeat_interleave(per, 1), -math.inf).sort(-1, descending=True)
    gap = c.values[:, :k] - c.values[:, 1:k + 1]
    sure = (gap.min(-1).values > 1e-5) & (value.values[:, topg - 1] - value.values[:, topg] > 1e-5)
    assert int(sure.sum()) > T // 2
    assert torch.equal(e[sure].long(), c.indices[sure, :k])
    u = s.gather(1, e.long())
    # relative error of a score and of the sum it is divided by: below 1e-6 each
    torch.testing.assert_close(w.double(), 1.5 * u / u.sum(-1, keepdim=True), atol=1e-7, rtol=1e-5)
    p = s / s.sum(-1, keepdim=True)
    torch.testing.assert_close(ss.double(), p.sum(0), atol=1e-5, rtol=1e-5)
    assert torch.equal(cnt.long(), torch.bincount(e.reshape(-1).long(), minlength=E)) and int(cnt.sum()) == T * k
    assert torch.autograd.grad(w.sum() + ss.sum(), x)[0].shape == x.shape

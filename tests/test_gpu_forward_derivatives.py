"""A forward-mode tangent on an upstream gradient is refused, and calls inside a
dual level on tensors without one are as outside."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from spider_web_moe_b200.fp8_blocks import fp8_block_linear
from spider_web_moe_b200.routing import route_experts

pytestmark = pytest.mark.gpu


def test_upstream_tangents(cuda_device):
    z = lambda *s: torch.randn(*s, device=cuda_device)  # noqa: E731
    logits, x, w = z(5, 8).requires_grad_(), z(5, 32).requires_grad_(), z(16, 32)
    want = route_experts(logits, 2)[1], fp8_block_linear(x, w)
    with fwd.dual_level():
        for leaf, call, ref in ((logits, lambda: route_experts(logits, 2)[1], want[0]),
                                (x, lambda: fp8_block_linear(x, w), want[1])):
            y = call()
            assert torch.equal(y, ref)
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad(y, leaf, fwd.make_dual(torch.ones_like(y), torch.ones_like(y)))

"""Tensors with a forward-mode tangent are refused, not read as if they had none.
The refusal comes before any look at the device, so it is tested without one."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from spider_web_moe_b200.fp8_blocks import (Fp8BlockExperts, Fp8BlockTensor, fp8_block_linear, fp8_expert_delta,
                                            quantize_fp8_blocks)
from spider_web_moe_b200.routing import route_experts


def dual(*shape):
    return fwd.make_dual(torch.zeros(*shape), torch.ones(*shape))


def packed(r, c):
    return Fp8BlockTensor(torch.zeros(r, c, dtype=torch.float8_e4m3fn), torch.ones(-(-r // 128), -(-c // 128)), 128)


class Experts(Fp8BlockExperts):
    """The argument checks' view of packed experts."""

    def __init__(self):
        self.hidden, self.num_experts, self.device = 32, 4, torch.device("cpu")


CALLS = [
    lambda z, d: route_experts(d(4, 8), 2),
    lambda z, d: route_experts(z(4, 8), 2, bias=d(8)),
    lambda z, d: fp8_block_linear(d(4, 32), z(8, 32)),
    lambda z, d: fp8_block_linear(z(4, 32), d(8, 32)),
    lambda z, d: fp8_block_linear(d(4, 32), packed(8, 32)),
    lambda z, d: quantize_fp8_blocks(d(4, 32)),
    lambda z, d: fp8_expert_delta(d(4, 32), torch.zeros(4, 2, dtype=torch.int32), z(4, 2), Experts()),
    lambda z, d: fp8_expert_delta(z(4, 32), torch.zeros(4, 2, dtype=torch.int32), d(4, 2), Experts()),
    lambda z, d: Experts().delta(d(4, 32), torch.zeros(4, 2, dtype=torch.int32), z(4, 2)),
]


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("grad", [False, True])
def test_refused(call, grad):
    with fwd.dual_level(), torch.set_grad_enabled(grad):
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(torch.zeros, dual)

"""Sizes that the kernels' 32-bit arguments or grids cannot hold are refused by name,
before any look at the device, instead of wrapping around; so are arguments of
Fp8BlockExperts.delta that do not fit the experts.  Expanded tensors: no memory."""
import ctypes as C

import pytest
import torch

from spider_web_moe_b200 import _lib as L
from spider_web_moe_b200.fp8_blocks import (Fp8BlockExperts, Fp8BlockTensor, fp8_block_linear, fp8_block_matmul,
                                            fp8_expert_delta, quantize_fp8_blocks)
from spider_web_moe_b200.routing import route_experts

BIG = 2 ** 32 + 5  # as a C int: 5


def wide(*shape, dtype=torch.float32):
    return torch.zeros(1, dtype=dtype).expand(*shape)


class Experts(Fp8BlockExperts):
    """The argument checks' view of packed experts."""

    def __init__(self):
        self.hidden, self.num_experts, self.device = 32, 4, torch.device("cpu")


@pytest.mark.parametrize("call", [
    lambda: route_experts(wide(BIG, 1), 1),
    lambda: route_experts(wide(2 ** 31, 1), 1),
    lambda: route_experts(wide(2 ** 16, 2 ** 16, 1), 1),
    lambda: quantize_fp8_blocks(wide(BIG, 1)),
    lambda: quantize_fp8_blocks(wide(2, BIG)),
    lambda: quantize_fp8_blocks(wide(2, 2 ** 24 + 1)),
    lambda: quantize_fp8_blocks(wide(BIG, 1, 1)),
    lambda: quantize_fp8_blocks(wide(65536, 1, 1)),
    lambda: quantize_fp8_blocks(wide(65535 * 128 + 1, 1), 128),
    lambda: quantize_fp8_blocks(torch.zeros(2, 65535 * 128 + 1, dtype=torch.bfloat16).t()),
    lambda: fp8_block_linear(wide(BIG, 1), wide(4, 1)),
    lambda: fp8_block_linear(wide(4, 2 ** 24 + 1), wide(4, 2 ** 24 + 1)),
    lambda: fp8_block_linear(wide(4, 1), wide(65535 * 128 + 1, 1)),
    # the gradients sum over the rows of x, and quantise the transposed weight
    lambda: fp8_block_linear(wide(2 ** 24 + 1, 1), torch.zeros(4, 1, requires_grad=True)),
    lambda: fp8_block_linear(torch.zeros(4, 65535 * 128 + 1, requires_grad=True), wide(4, 65535 * 128 + 1)),
    lambda: fp8_expert_delta(wide(BIG, 32), wide(BIG, 1, dtype=torch.int32), wide(BIG, 1), Experts()),
    lambda: fp8_expert_delta(wide(2 ** 27, 32), wide(2 ** 27, 16, dtype=torch.int32), wide(2 ** 27, 16), Experts()),
])
def test_sizes(call):
    with pytest.raises(ValueError, match="at most"):
        call()


def test_product_sizes():
    q, s = torch.zeros(1, dtype=torch.float8_e4m3fn), torch.zeros(1)
    t = object.__new__(Fp8BlockTensor)
    t.q, t.scale, t.block_rows = q.expand(BIG, 16), s.expand(BIG, 1), 1
    b = Fp8BlockTensor(torch.zeros(4, 16, dtype=torch.float8_e4m3fn), torch.ones(1, 1), 128)
    for args in ((t, b), (Fp8BlockTensor(b.q, torch.ones(4, 1), 1), t)):
        with pytest.raises(ValueError, match="at most"):
            fp8_block_matmul(*args)


@pytest.mark.parametrize("m,i,w,kw,err", [
    ((5, 31), (5, 2), (5, 2), {}, ValueError), ((5, 32), (5, 2), (5, 3), {}, ValueError),
    ((5, 32), (4, 2), (4, 2), {}, ValueError), ((5, 1, 32), (5, 1, 2), (5, 1, 2), {}, ValueError),
    ((5, 32), (5, 0), (5, 0), {}, ValueError), ((5, 32), (5, 65), (5, 65), {}, ValueError),
    ((5, 32), (5, 2), (5, 2), dict(out_dtype=torch.float16), TypeError),
    ((5, 32), (5, 2), (5, 2), dict(rank=2, world=2), ValueError),
])
def test_delta_arguments(m, i, w, kw, err):
    with pytest.raises(err):
        Experts().delta(torch.zeros(m), torch.zeros(i, dtype=torch.int32), torch.zeros(w), **kw)
    with pytest.raises(TypeError):
        Experts().delta(torch.zeros(5, 32), torch.zeros(5, 2), torch.zeros(5, 2))
    with pytest.raises(NotImplementedError):
        Experts().delta(torch.zeros(5, 32), torch.zeros(5, 2, dtype=torch.int32), torch.zeros(5, 2, requires_grad=True))


def test_c_abi_sizes():
    """Sizes near the end of 32 bits, where rounding up to tiles would overflow."""
    lib, p, top = L.load(), 4096, 0x7fffffff
    assert lib.sb_route_experts(p, 0, 8, top, 8, 2, 0, None, 1, 1, 2, 1, 1.0, p, p, None) == L.SB_ERR_ARG
    assert lib.sb_route_experts_backward(p, 0, 8, top, 8, 2, 0, None, 1, 1.0, p, p, p, 8, None) == L.SB_ERR_ARG
    q = dict(x=p, dtype=0, block_rows=1, batch=1, rows=4, cols=8, x_row=8, x_col=1, q=p, ldq=16, scale=p)
    for bad in (dict(rows=top), dict(rows=top, block_rows=128), dict(cols=top, ldq=2 ** 31), dict(batch=65536)):
        assert lib.sb_fp8_quantize_blocks(C.byref(L.Fp8QuantizeArgs(**{**q, **bad})), None) == L.SB_ERR_ARG, bad
    m = dict(epilogue=L.SB_EPI_LINEAR, out_dtype=0, num_groups=1, max_rows=4, n=8, k=32, a=p, lda=32, a_scale=p, b=p,
             ldb=32, b_scale=p, b_block_rows=128, out=p, ldo=8)
    for bad in (dict(max_rows=top), dict(n=top, ldo=2 ** 31), dict(k=top, lda=2 ** 31, ldb=2 ** 31)):
        assert lib.sb_fp8_matmul(C.byref(L.Fp8MatmulArgs(**{**m, **bad})), None) == L.SB_ERR_ARG, bad
    for bad in ((top, 8, 32), (4, top, 32), (4, 8, top)):
        assert lib.sb_fp8_linear_workspace_bytes(*bad, 0) == 0
        assert lib.sb_fp8_linear_backward_workspace_bytes(*bad) == 0
    e = L.Fp8Experts(num_experts=4, hidden=64, ffn=32, activation=L.SB_ACT_GELU, ld_in=64, ld_ffn=32)
    assert lib.sb_fp8_expert_delta_workspace_bytes(C.byref(e), top, 1) == 0
    assert lib.sb_fp8_expert_delta_workspace_bytes(C.byref(e), 2 ** 30, 2) == 0

"""GELU and SiLU in the products' quantising epilogue, value by value.

With zero operands the output is gelu(bias), and a block whose other biases are 0
has the scale |gelu(bias)| / 448: the scale shows the epilogue's fp32 value.
Tolerance: the formula's bound of erfc, 1.5e-7, times |x| / 2; fp32 steps of the
result and of its factors, of which exp(-x^2 / 2) is the worst: 2 + 1.17 x^2 / 2
units of 2^-23, below 2^-18 for |x| <= 6.  Relative to the value the bound is
1.0e-3 at x = -3.8 (e4m3 rounds by up to 6e-2).  SiLU: 2 + 1.17 |x| units of the
exponential, one of the sum, two of the division.  The scale adds two half steps.
"""
import ctypes as C

import pytest
import torch

from spider_web_moe_b200 import _lib as L
from spider_web_moe_b200 import fp8_blocks as F

pytestmark = pytest.mark.gpu


def by_scale(epilogue, values, rows, device, grouped=True):
    """fp32 |gelu(v)|, or |silu(v)| with up values of 1, for every v, from every one of `rows` rows."""
    blocks, n = len(values), 128 * len(values)
    bias = torch.zeros(blocks, 128, device=device)
    bias[torch.arange(blocks), torch.arange(blocks) % 128] = values.to(device)
    a = torch.zeros(rows, 128, dtype=torch.uint8, device=device)
    b = torch.zeros(n, 128, dtype=torch.uint8, device=device)
    one = torch.ones(max(rows, blocks), device=device)
    off = torch.tensor([0, rows], dtype=torch.int32, device=device)
    out = torch.empty(rows, n, dtype=torch.uint8, device=device)
    scale = torch.empty(blocks, rows, device=device)
    gate = epilogue == L.SB_EPI_SWIGLU
    ups = torch.ones(blocks, 128, device=device) if gate else bias
    m = L.Fp8MatmulArgs(epilogue=epilogue, num_groups=1, max_rows=rows, n=n, k=128, a=a.data_ptr(), lda=128,
                        a_scale=one.data_ptr(), a_scale_row=1, a_scale_block=rows, b=b.data_ptr(), ldb=128,
                        b_scale=one.data_ptr(), b_scale_row=1, b_scale_block=1, b_block_rows=128, bias=ups.data_ptr(),
                        b_gate=b.data_ptr(), b_gate_scale=one.data_ptr(), bias_gate=bias.data_ptr(),
                        offsets=off.data_ptr() if grouped else None, out=out.data_ptr(), ldo=n, out_scale=scale.data_ptr(), out_scale_row=1,
                        out_scale_block=rows, status=F._status_ptr(device))
    L.check(L.load().sb_fp8_matmul(C.byref(m), torch.cuda.current_stream().cuda_stream), "sb_fp8_matmul")
    F.check_status(device)
    return scale.double().cpu() * 448


# decode columns of 16, 32, 64; tiles of 128 rows
SCHEDULES = [(3, True), (20, True), (40, False), (200, True)]


@pytest.mark.parametrize("rows,grouped", SCHEDULES)
def test_gelu_values(rows, grouped, cuda_device):
    v = torch.cat([torch.linspace(-6, 6, 479), torch.tensor([-1e-3, 1e-3, 2.0 ** -20, -(2.0 ** -20), 30.0])])
    got = by_scale(L.SB_EPI_GELU, v, rows, cuda_device, grouped)
    x = v.double()
    want = (0.5 * x * torch.special.erfc(-x * 0.5 ** 0.5)).abs()[:, None]
    tol = 1.5e-7 * 0.5 * x.abs()[:, None] + 2.0 ** -18 * want + 2.0 ** -100
    err = (got - want).abs()
    assert (err <= tol).all(), [(float(v[i]), float((err / want)[i].max())) for i in (err > tol).any(1).nonzero().flatten()][:8]


@pytest.mark.parametrize("rows,grouped", SCHEDULES)
def test_silu_values(rows, grouped, cuda_device):
    v = torch.cat([torch.linspace(-60, 60, 479), torch.tensor([-1e-3, 1e-3, 2.0 ** -20, -(2.0 ** -20), -86.0, -1e4, 1e4])])
    got = by_scale(L.SB_EPI_SWIGLU, v, rows, cuda_device, grouped)
    x = v.double()
    want = (x * torch.sigmoid(x)).abs().clamp_min(2.0 ** -100)[:, None]  # the format's floor of a block's amax
    tol = (6 + 1.2 * x.abs()[:, None]) * 2.0 ** -23 * want + 2.0 ** -100
    assert ((got - want).abs() <= tol).all(), float(((got - want).abs() / tol).max())

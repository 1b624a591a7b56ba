"""The products' sums have fp32's 24 bits, in the tensor core too.

First, exactly: beside a product of 2^16 a single product of 2^-7 or more is kept
whole, whichever of a block's four instructions (32 elements each) either is in.
Hence the tolerance of random operands, with S = sum_k |a_k b_k|: an instruction
loses less than 2^-23 of its largest addend from each of its 32 and from the running
sum, 33 * 2^-23 in all, below 2^-17 of its part of S (and of the running sum's);
four instructions: 2^-17 + 4 * 2^-23 of a block's S.  Scaling and the running sum
over KB blocks: (KB + 4) 2^-24 S.
"""
import pytest
import torch

from spider_web_moe_b200.fp8_blocks import Fp8BlockTensor, check_status, fp8_block_matmul, quantize_fp8_blocks

pytestmark = pytest.mark.gpu

# decode columns of 16, 32, 64; tiles of 128 rows; pairs
SHAPES = [(2, 40), (20, 40), (50, 40), (100, 9700), (300, 9000)]


def tensor(v, block_rows):
    q = v.to(torch.float8_e4m3fn)
    assert torch.equal(q.float(), v)
    return Fp8BlockTensor(q, torch.ones(-(-len(v) // block_rows), 1, device=v.device), block_rows)


@pytest.mark.parametrize("m,n", SHAPES)
@pytest.mark.parametrize("at", [0, 45])
@pytest.mark.parametrize("block_rows", [128, 1])
def test_small_beside_large(block_rows, at, m, n, cuda_device):
    pos = [p for p in (1, 8, 31, 32, 40, 63, 64, 96, 127) if p != at]
    a, b = torch.zeros(m, 128, device=cuda_device), torch.zeros(n, 128, device=cuda_device)
    a[:, at], b[:, at] = 256.0, 256.0
    want = torch.full((m, n), 65536.0, device=cuda_device)
    for i, p in enumerate(pos):
        a[:, p] = 2.0 ** -3
        sign = -1.0 if i % 2 else 1.0  # 2^16 - 2^-7 needs one bit more below, which it has
        b[i::len(pos)] = torch.where(torch.arange(128, device=cuda_device) == p, sign * 2.0 ** -4, b[i::len(pos)])
        want[:, i::len(pos)] += sign * 2.0 ** -7
    assert torch.equal(fp8_block_matmul(tensor(a, 1), tensor(b, block_rows), torch.float32), want)
    check_status(cuda_device)


@pytest.mark.parametrize("m,n", SHAPES)
@pytest.mark.parametrize("k", [128, 2048, 5000])
def test_random_operands(k, m, n, cuda_device):
    g = torch.Generator().manual_seed(m + k)
    for block_rows in (128, 1):
        a = quantize_fp8_blocks(torch.randn(m, k, generator=g).to(cuda_device))
        b = quantize_fp8_blocks(torch.randn(n, k, generator=g).to(cuda_device), block_rows)
        av, bv = a.dequantize(torch.float64), b.dequantize(torch.float64)
        # (dequantize rounds q * scale to fp32: 2^-24 of each factor)
        tol = (2.0 ** -17 + 4 * 2.0 ** -23 + (k // 128 + 5 + 2) * 2.0 ** -24) * (av.abs() @ bv.abs().t())
        err = (fp8_block_matmul(a, b, torch.float32).double() - av @ bv.t()).abs()
        assert (err <= tol).all(), float((err / tol).max())

"""Products into a view of a larger tensor leave what is around it as it was, at every
alignment of the view and of its last column."""
import pytest
import torch

from spider_web_moe_b200.fp8_blocks import check_status, fp8_block_matmul, quantize_fp8_blocks

from test_gpu_fp8_blocks import rand

pytestmark = pytest.mark.gpu


# pairs of CTAs (more 128 x 64 items than SMs, or scales per column), one-CTA tiles, decode columns
@pytest.mark.parametrize("m,n0,block_rows", [(709, 4000, 128), (300, 9, 1), (257, 200, 1), (100, 9700, 128), (40, 300, 128)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("k", [10, 300])
def test_surroundings(k, dtype, m, n0, block_rows, cuda_device):
    a = quantize_fp8_blocks(rand(m, k, seed=m).to(cuda_device))
    for n in range(n0, n0 + 9):
        b = quantize_fp8_blocks(rand(n, k, seed=n).to(cuda_device), block_rows)
        want = fp8_block_matmul(a, b, dtype)
        for off in (0, 3, 8, 16):  # in elements: 16-byte boundaries, but for 3
            for pitch in (-(-(n + off) // 8) * 8 + 8, n + off):
                big = torch.full((m + 4, pitch), 7.0, device=cuda_device, dtype=dtype)
                view = big[2:m + 2, off:off + n]
                fp8_block_matmul(a, b, out=view)
                assert torch.equal(view, want), (n, off, pitch)
                view.fill_(7.0)
                assert (big == 7.0).all(), (n, off, pitch)
    check_status(cuda_device)

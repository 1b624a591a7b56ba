"""Block-scaled products whose every step is exact, against 64 bits bit for bit.

Values are small integers, scales, row scales powers of two between 1/2 and 2, biases
integers: with at most 24 blocks of 128 every partial sum is a multiple of 2^-2 (2^-3
with a row scale) below 2^18, so fp32 holds it exactly in any order.  The scales differ from row to row, block
to block and item to item, so that a scale, a bias or a row scale that an epilogue
reads too early, too late or from another item is a wrong output.
"""
import ctypes as C

import pytest
import torch

from spider_web_moe_b200 import _lib as L
from spider_web_moe_b200 import fp8_blocks as F
from spider_web_moe_b200.fp8_blocks import Fp8BlockTensor, check_status, fp8_block_matmul

pytestmark = pytest.mark.gpu


def exact_tensor(r, c, block_rows, g, device, lead=()):
    """Integers of [-2, 2] with scales of 1/2, 1 or 2 (the product of two: 1/4 to 4)."""
    q = torch.zeros(*lead, r, -(-c // 16) * 16)
    q[..., :c] = torch.randint(-2, 3, (*lead, r, c), generator=g).float()
    s = torch.exp2(torch.randint(-1, 2, (*lead, -(-r // block_rows), -(-c // 128)), generator=g).float())
    return Fp8BlockTensor(q.to(torch.float8_e4m3fn).to(device)[..., :c], s.to(device), block_rows)


def values(t):
    return t.dequantize(torch.float64)


# decode columns of 16, 32 and 64 (k split over clusters in the small ones), one-CTA
# tiles, pairs with a full, a part and an empty second CTA, several items per CTA
SHAPES = [(5, 2048, 300), (30, 3071, 260), (60, 1500, 1000), (100, 640, 9700), (700, 1152, 1000), (513, 1040, 3900),
          (900, 3000, 9000), (2600, 300, 4200)]


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("block_rows", [128, 1])
def test_scales_of_every_block(m, k, n, block_rows, cuda_device):
    g = torch.Generator().manual_seed(m + k)
    a, b = exact_tensor(m, k, 1, g, cuda_device), exact_tensor(n, k, block_rows, g, cuda_device)
    want = values(a) @ values(b).t()
    for _ in range(8):
        assert torch.equal(fp8_block_matmul(a, b, torch.float32).double(), want)
    check_status(cuda_device)


@pytest.mark.parametrize("counts", [[1, 0, 3, 9], [30, 0, 60, 40], [70, 128, 90, 129], [600, 0, 300, 257], [1500, 129, 1024, 31]])
def test_bias_and_row_scale_of_every_item(counts, cuda_device):
    """Grouped, with short k, so that an item's bias and row scales follow the last one's closely."""
    e, u, h = len(counts), 1100, 200
    g = torch.Generator().manual_seed(sum(counts))
    off = torch.tensor([0] + counts).cumsum(0).int().to(cuda_device)
    rows = int(off[-1])
    x, w = exact_tensor(rows, h, 1, g, cuda_device), exact_tensor(u, h, 128, g, cuda_device, (e,))
    bias = torch.randint(-8, 9, (e, u), generator=g).float().to(cuda_device)
    rs = torch.exp2(torch.randint(-1, 2, (rows,), generator=g).float()).to(cuda_device)
    out = torch.empty(rows, u, device=cuda_device)
    a = L.Fp8MatmulArgs(epilogue=L.SB_EPI_LINEAR, out_dtype=L.SB_F32, num_groups=e, max_rows=rows, n=u, k=h,
                        a=x.q.data_ptr(), lda=x.pitch, a_scale=x.scale.data_ptr(), a_scale_row=x.scale.stride(0),
                        a_scale_block=x.scale.stride(1), b=w.q.data_ptr(), ldb=w.pitch, b_group_rows=u,
                        b_scale=w.scale.data_ptr(), b_scale_row=w.scale.stride(1), b_scale_block=w.scale.stride(2),
                        b_scale_group=w.scale.stride(0), b_block_rows=128, bias=bias.data_ptr(), bias_group=u,
                        row_scale=rs.data_ptr(), offsets=off.data_ptr(), out=out.data_ptr(), ldo=u,
                        status=F._status_ptr(cuda_device))
    xv, wv = values(x), values(w)
    want = torch.cat([(xv[off[i]:off[i + 1]] @ wv[i].t() + bias[i].double()) for i in range(e)]) * rs[:, None].double()
    for _ in range(8):
        out.fill_(-1e9)
        L.check(L.load().sb_fp8_matmul(C.byref(a), torch.cuda.current_stream().cuda_stream), "sb_fp8_matmul")
        assert torch.equal(out.double(), want)
    check_status(cuda_device)

"""sb_fp8_quantize_blocks with row_count: rows behind the count are not written,
whatever the strides of x."""
import ctypes as C

import pytest
import torch

from spider_web_moe_b200 import _lib as L

from test_gpu_fp8_blocks import plain_quantize, rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,cols,count", [(304, 200, 130), (301, 256, 7), (64, 64, 0), (40, 130, 99)])
@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("indexed", [False, True])
def test_rows_behind_the_count(indexed, transposed, rows, cols, count, dtype, cuda_device):
    x = rand(rows, cols, seed=rows, dtype=dtype)
    order = torch.randperm(rows, generator=torch.Generator().manual_seed(1))
    pitch, cb = -(-cols // 16) * 16, -(-cols // 128)
    d = (x.t().contiguous().t() if transposed else x).to(cuda_device)
    d = d if d.stride() == ((1, rows) if transposed else (cols, 1)) else d.t().contiguous().t()
    assert d.stride() == ((1, rows) if transposed else (cols, 1))
    q = torch.full((rows, pitch), 0x55, dtype=torch.uint8, device=cuda_device)
    scale = torch.full((cb, rows), -1.0, device=cuda_device)
    n, index = torch.tensor([count], dtype=torch.int32, device=cuda_device), order.int().to(cuda_device)
    a = L.Fp8QuantizeArgs(x=d.data_ptr(), dtype=L.SB_F32 if dtype == torch.float32 else L.SB_BF16, block_rows=1,
                          batch=1, rows=rows, cols=cols, x_row=d.stride(0), x_col=d.stride(1),
                          row_index=index.data_ptr() if indexed else None, row_count=n.data_ptr(), q=q.data_ptr(),
                          ldq=pitch, scale=scale.data_ptr(), scale_row=1, scale_col=rows)
    L.check(L.load().sb_fp8_quantize_blocks(C.byref(a), torch.cuda.current_stream().cuda_stream), "quantize")
    live = min(rows, count)
    wq, ws = plain_quantize(x[order] if indexed else x, 1)
    assert torch.equal(q[:live, :cols].cpu(), wq[:live]) and torch.equal(scale.t()[:live].cpu(), ws[:live])
    assert (q[live:] == 0x55).all() and (scale[:, live:] == -1).all()

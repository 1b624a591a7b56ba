"""Block-scaled experts packed by a pass on one stream and used by a pass on another
that does not wait for it."""
import pytest
import torch

from test_gpu_fp8_block_layer import make

pytestmark = pytest.mark.gpu


@torch.no_grad()
def test_packed_on_another_stream(cuda_device):
    layer, h, x0 = make("swiglu", cuda_device, torch.bfloat16)
    layer.quantize_experts_fp8(block_size=128)
    want = layer(h, x0, 0)
    layer.invalidate()
    layer.engine(h.device, h.dtype, 22)
    busy, other = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(busy):
        torch.cuda._sleep(200_000_000)  # 0.1 s: what the stream has yet to do
        layer.fp8_block_experts(cuda_device)
    with torch.cuda.stream(other):
        got = layer(h, x0, 0)
    torch.cuda.synchronize()
    assert torch.equal(got, want)

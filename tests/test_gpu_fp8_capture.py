"""The layer's first pass with block-scaled experts inside a capture: refused, and
the layer works afterwards."""
import pytest
import torch

from test_gpu_fp8_block_layer import make

pytestmark = pytest.mark.gpu


@torch.no_grad()
def test_first_pass_under_capture(cuda_device):
    layer, h, x0 = make("swiglu", cuda_device, torch.bfloat16)
    layer(h, x0, 0)
    layer.quantize_experts_fp8(block_size=128)
    layer.engine(h.device, h.dtype, 22)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="captur"):
        with torch.cuda.graph(graph):
            layer(h, x0, 0)
    want = layer(h, x0, 0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(h, x0, 0)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)

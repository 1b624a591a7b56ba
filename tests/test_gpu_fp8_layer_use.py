"""Block-scaled experts of the layer in use: packed by a pass on one stream and used by
a pass on another that does not wait for it, and under expert parallelism."""
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


@pytest.mark.parametrize("rank", [0, 1])
@torch.no_grad()
def test_expert_parallel_pass(rank, cuda_device, monkeypatch):
    """The layer and fp8_expert_delta as rank 0 and 1 of 2, the other rank's part of
    the delta put in where the all-reduce is: the one-process result, bit for bit (a
    token has two experts, and the sum of two numbers does not depend on the order)."""
    import spider_web_moe_b200.fp8_blocks as F
    import spider_web_moe_b200.layer as layer_module

    layer, h, x0 = make("swiglu", cuda_device, torch.bfloat16)
    layer.quantize_experts_fp8(block_size=128)
    want = layer(h, x0, 1)
    ex = layer.fp8_block_experts(cuda_device)
    msgs, idx, w = layer.engine(h.device, h.dtype, 22).route(h, 1)
    msgs, idx, w = msgs.clone(), idx.clone(), w.clone()
    other = ex.delta(msgs, idx, w, 1 - rank, 2, torch.float32)
    alone = F.fp8_expert_delta(msgs, idx, w, ex)
    helpers = layer_module.ep_helpers
    for owner in (helpers, F):
        monkeypatch.setattr(owner, "ep_enabled", lambda: True)
        monkeypatch.setattr(owner, "get_rank_world", lambda: (rank, 2))
        monkeypatch.setattr(owner, "all_reduce_sum_", lambda t: t.add_(other))
    assert layer.expert_parallel
    assert torch.equal(layer(h, x0, 1), want)
    assert torch.equal(F.fp8_expert_delta(msgs, idx, w, ex), alone)
    assert not torch.equal(ex.delta(msgs, idx, w, rank, 2, torch.float32), other)


def test_status_of_another_stream(cuda_device):
    """check_status waits for every stream of the device: an error that a kernel is
    yet to record on another stream is seen."""
    import spider_web_moe_b200.fp8_blocks as F
    from spider_web_moe_b200 import _lib as L

    F._status_ptr(cuda_device)
    word = F._STATUS[cuda_device][0]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)
        word.fill_(4)
    try:
        with pytest.raises(L.SpiderB200Error, match="0x4"):
            F.check_status(cuda_device)
    finally:
        side.synchronize()
        word.zero_()
        torch.cuda.synchronize()
    F.check_status(cuda_device)

"""SpiderMoELayer with block-scaled fp8 experts: each loop equals the block's own
routing and messages, the fp64 statement of the experts on them (activations
quantised as defined), and the LayerNorm.

Tolerance: the experts' delta is within 2^-5 of its row norm (as in the experts'
own test: activations next to a rounding border), which the LayerNorm passes on
times residual_scale * |delta| / |u - mean(u)|, plus the activation dtype's
rounding of messages and output (2^-8 each in bf16).
"""
import pytest
import torch

from spider_web_moe_b200 import ModelConfig, SpiderMoELayer
from spider_web_moe_b200.fp8_blocks import check_status

from test_gpu_fp8_blocks import delta_oracle

pytestmark = pytest.mark.gpu


def make(activation, device, dtype):
    torch.manual_seed(3)
    cfg = ModelConfig(hidden_size=128, num_heads=4, num_experts=8, top_k=2, edges_per_expert=2, num_loops=3,
                      expert_ffn_size=192, expert_activation=activation)
    layer = SpiderMoELayer(cfg).to(device, dtype).eval()
    g = torch.Generator().manual_seed(4)
    h = torch.randn(2, 11, 128, generator=g).to(device, dtype)
    return layer, h, torch.randn(2, 11, 128, generator=g).to(device, dtype)


@pytest.mark.parametrize("activation", ["gelu", "swiglu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@torch.no_grad()
def test_layer_loop(activation, dtype, cuda_device):
    layer, h, x0 = make(activation, cuda_device, dtype)
    plain = layer(h, x0, 1)
    layer.quantize_experts_fp8(block_size=128)
    out, stats = layer(h, x0, 1, return_stats=True)
    check_status(cuda_device)
    assert torch.equal(out, layer(h, x0, 1)) and out.dtype == dtype and "aux_loss" in stats
    ex = layer.fp8_block_experts(cuda_device)
    msgs, idx, w = layer.engine(h.device, dtype, 22).route(h, 1)
    b = {"up": ex.b_up.cpu(), "down": ex.b_down.cpu(), "gate": None if ex.b_gate is None else ex.b_gate.cpu()}
    delta, _ = delta_oracle(ex, b, msgs.cpu(), idx.cpu(), w.cpu())
    u = h.reshape(22, -1).double().cpu() + layer.residual_scale * delta + layer.reinject_weight * x0.reshape(22, -1).double().cpu()
    c = u - u.mean(1, keepdim=True)
    want = c / (c.var(1, unbiased=False, keepdim=True) + 1e-5).sqrt() * layer.norm.weight.double().cpu() + \
        layer.norm.bias.double().cpu()
    got = out.reshape(22, -1).double().cpu()
    tol = 2 * layer.residual_scale * 2.0 ** -5 * delta.norm(dim=1) / c.norm(dim=1) + 2.0 ** -7
    assert ((got - want).norm(dim=1) / want.norm(dim=1) <= tol).all()
    # all loops in a row, the early-exit driver, and back to the module's own weights
    seq = h
    for l in range(3):
        seq = layer(seq, x0, l)
    assert torch.equal(layer.run_loops(h, x0), seq)
    assert torch.isfinite(layer.run_recurrent_decode(h[:, :1], x0[:, :1])).all()
    layer.dequantize_experts()
    assert torch.equal(layer(h, x0, 1), plain)


@torch.no_grad()
def test_new_weights_are_packed_again(cuda_device):
    layer, h, x0 = make("swiglu", cuda_device, torch.bfloat16)
    layer.quantize_experts_fp8(block_size=128)
    first = layer(h, x0, 0)
    state = {k: (v * 1.5 if "experts" in k else v) for k, v in layer.state_dict().items()}
    layer.load_state_dict(state)
    assert not torch.equal(layer(h, x0, 0), first)
    layer.quantize_experts_fp8()  # per output channel: the block kernels' own format
    assert layer._fp8 is not None and torch.isfinite(layer(h, x0, 0)).all()


@torch.no_grad()
def test_layer_captured(cuda_device):
    layer, h, x0 = make("swiglu", cuda_device, torch.bfloat16)
    layer.quantize_experts_fp8(block_size=128)
    want = layer(h, x0, 0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        layer(h, x0, 0)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(h, x0, 0)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


@torch.no_grad()
def test_layer_decode_and_statistics(cuda_device):
    """The layer's other drivers run these experts too: early exit that never
    exits is the loop over all blocks, and statistics do not change the output."""
    layer, h, x0 = make("swiglu", cuda_device, torch.float32)
    layer.quantize_experts_fp8(block_size=128)
    want = layer.run_loops(h, x0)
    assert torch.equal(layer.run_recurrent_decode(h, x0, early_exit=False), want)
    h1, x1 = h[:, :1].contiguous(), x0[:, :1].contiguous()
    got = layer.run_recurrent_decode(h1, x1, early_exit=True, threshold=2.0)
    assert torch.equal(got, layer.run_loops(h1, x1))
    out, stats = layer(h, x0, 0, return_stats=True)
    assert torch.equal(out, layer(h, x0, 0)) and stats
    check_status(cuda_device)

"""Packing expert weights inside a stream capture is refused: the quantised weights
would be recorded, not written, and would lie in the graph's memory."""
import pytest
import torch

from spider_web_moe_b200 import ModelConfig, SpiderMoELayer
from spider_web_moe_b200.fp8_blocks import Fp8BlockExperts


def layer():
    cfg = ModelConfig(hidden_size=64, num_heads=4, num_experts=4, top_k=2, edges_per_expert=2, num_loops=2,
                      expert_ffn_size=128)
    m = SpiderMoELayer(cfg)
    m.quantize_experts_fp8(block_size=128)
    return m


def test_layer_under_capture(monkeypatch):
    m = layer()
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="captur"):
        m.fp8_block_experts("cuda:0")
    assert m._fp8_experts is None
    packed = m._fp8_experts = object.__new__(Fp8BlockExperts)  # packed before the capture: used as it is
    packed.device = torch.device("cuda:0")
    assert m.fp8_block_experts("cuda:0") is packed

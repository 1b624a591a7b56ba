"""B200-native recurrent Spider-MoE block (forward pass).

A drop-in for the reference block ``SpiderMoELayer`` (spider_moe/model.py:163)
and its ``sparse_expert_delta`` / ``expert_parallel`` helpers.  The compute
runs in hand-written sm_100a CUDA kernels behind a C ABI
(``include/spider_b200.h``); Python holds device memory, streams and
``torch.distributed``.  Submodules are imported lazily so that the config and
the synthetic-data helpers load without the CUDA library.
"""
from .config import ModelConfig, load_config  # noqa: F401

__all__ = ["ModelConfig", "load_config", "SpiderMoELayer", "sparse_expert_delta", "LumenWorkspace",
           "ExpertChunkStore", "CudaGraphDecodeRunner", "load_spiderw", "write_spiderw", "route_experts",
           "quantize_fp8_blocks", "fp8_block_matmul", "fp8_block_linear", "fp8_expert_delta", "Fp8BlockTensor",
           "Fp8BlockExperts"]

_LAZY = {
    "SpiderMoELayer": ("layer", "SpiderMoELayer"),
    "sparse_expert_delta": ("sparse_experts", "sparse_expert_delta"),
    "LumenWorkspace": ("lumen", "LumenWorkspace"),
    "ExpertChunkStore": ("dobu", "ExpertChunkStore"),
    "CudaGraphDecodeRunner": ("cuda_graph", "CudaGraphDecodeRunner"),
    "load_spiderw": ("spiderw", "load_spiderw"),
    "write_spiderw": ("spiderw", "write_spiderw"),
    "route_experts": ("routing", "route_experts"),
    "quantize_fp8_blocks": ("fp8_blocks", "quantize_fp8_blocks"),
    "fp8_block_matmul": ("fp8_blocks", "fp8_block_matmul"),
    "fp8_block_linear": ("fp8_blocks", "fp8_block_linear"),
    "fp8_expert_delta": ("fp8_blocks", "fp8_expert_delta"),
    "Fp8BlockTensor": ("fp8_blocks", "Fp8BlockTensor"),
    "Fp8BlockExperts": ("fp8_blocks", "Fp8BlockExperts"),
}


def __getattr__(name):
    if name in _LAZY:
        import importlib

        mod, attr = _LAZY[name]
        return getattr(importlib.import_module(f".{mod}", __name__), attr)
    raise AttributeError(name)

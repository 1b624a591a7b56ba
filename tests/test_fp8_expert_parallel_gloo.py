"""Expert parallelism of the block-scaled fp8 experts on CPU ranks (gloo, world 2
and 3): every rank runs its own experts on all tokens in fp32, the parts are summed
and rounded once.  The experts' arithmetic is a stand-in: integers, so that the sum is
the one-process result bit for bit."""
import os
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from spider_web_moe_b200 import ModelConfig, SpiderMoELayer
from spider_web_moe_b200.fp8_blocks import Fp8BlockExperts, fp8_expert_delta

N, H, E, K = 7, 16, 5, 3


class Experts(Fp8BlockExperts):
    """delta[t] = sum of w * (e + 1) * messages[t] over the rank's experts."""

    def __init__(self):
        self.hidden, self.num_experts, self.device = H, E, torch.device("cpu")

    def delta(self, messages, top_indices, top_weights, rank=0, world=1, out_dtype=None):
        assert messages.dim() == 2 and top_indices.shape == top_weights.shape == (len(messages), K)
        mine = (top_indices >= 0) & (top_indices < E) & (top_indices % world == rank)
        f = (top_weights * (top_indices + 1) * mine).sum(1, keepdim=True)
        return (f * messages.float()).to(out_dtype or messages.dtype)


class Engine:
    """Routing and epilogue stand-ins of the block."""

    def __init__(self, idx, w):
        self.idx, self.w = idx, w

    def route(self, h, loop_idx):
        return h.reshape(-1, H) + loop_idx, self.idx, self.w

    def epilogue(self, rows, inv, h, x0):
        assert rows.dtype == torch.float32 and rows.is_contiguous() and inv.flatten().tolist() == list(range(N))
        return h + rows.view_as(h) + x0


def inputs():
    g = torch.Generator().manual_seed(3)
    x = torch.randint(-4, 5, (N, H), generator=g).float()
    idx = torch.randint(-1, E + 1, (N, K), generator=g)
    w = torch.randint(1, 4, (N, K), generator=g).float()
    return x, idx, w


def passes():
    x, idx, w = inputs()
    ex = Experts()
    layer = SpiderMoELayer(ModelConfig(hidden_size=H, num_heads=1, num_experts=E, top_k=K, edges_per_expert=1, num_loops=1,
                                       expert_ffn_size=8))
    layer._fp8_experts = ex
    from spider_web_moe_b200.expert_parallel import ep_enabled

    out = layer._forward_fp8_blocks(Engine(idx, w), x, 2 * x, 3, ep_enabled())
    assert set(out[1]) == {"top_idx", "top_w"}
    return [fp8_expert_delta(x, idx, w, ex), fp8_expert_delta(x.view(1, N, H).bfloat16(), idx[None], w[None], ex),
            fp8_expert_delta(x, idx, w, ex, expert_parallel=False), out[0]]


def worker(rank, world, port, q):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    try:
        q.put((rank, [(t.dtype, tuple(t.shape), t.float().tolist()) for t in passes()]))
    finally:
        dist.destroy_process_group()


@pytest.mark.parametrize("world", [2, 3])
def test_ranks_agree_with_one_process(world):
    want = [(t.dtype, tuple(t.shape), t.float().tolist()) for t in passes()]
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=worker, args=(r, world, port, q)) for r in range(world)]
    for p in procs:
        p.start()
    got = dict(q.get(timeout=240) for _ in range(world))
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    assert all(got[r] == want for r in range(world))

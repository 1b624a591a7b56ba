"""NaN routing weights reach the token's output; weights <= 0 do not."""
import pytest
import torch

from spider_web_moe_b200.fp8_blocks import check_status, fp8_expert_delta
from spider_web_moe_b200.routing import route_experts

from test_gpu_fp8_blocks import make_experts, rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [3, 40, 700, 3000])  # decode columns, tiles of 128 rows, pairs; both groupings
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_nan_logit(n, score, cuda_device):
    """A NaN logit's token is NaN, and the other tokens are as without it."""
    ex, _ = make_experts(4, 128, 96, True, 31, cuda_device)
    x = rand(n, 128, seed=n).to(cuda_device)
    logits = rand(n, 4, seed=n + 1)
    clean = fp8_expert_delta(x, *route_experts(logits.to(cuda_device), 2, score=score), ex)
    bad = n // 2
    logits[bad, 3] = float("nan")
    idx, w = route_experts(logits.to(cuda_device), 2, score=score)
    got = fp8_expert_delta(x, idx, w, ex)
    keep = torch.arange(n, device=cuda_device) != bad
    assert torch.isnan(got[bad]).all() and torch.equal(got[keep], clean[keep])
    check_status(cuda_device)


@pytest.mark.parametrize("repeat", [1, 200])
def test_nan_weights(repeat, cuda_device):
    """Given weights: NaN stays NaN, also added to another of the same expert;
    outside [0, E) it is skipped like any other; 0 and below are dropped."""
    ex, _ = make_experts(4, 64, 48, False, 77, cuda_device)
    nan = float("nan")
    idx = torch.tensor([[0, 1], [2, 2], [-1, 3], [4, 0], [0, 1], [3, 3]]).repeat(repeat, 1).to(cuda_device)
    w = torch.tensor([[nan, 1.0], [nan, -5.0], [nan, 1.0], [nan, 0.0], [-1.0, 0.0], [1.0, -1.0]]).repeat(repeat, 1)
    x = rand(6, 64, seed=78).repeat(repeat, 1).to(cuda_device)
    got = fp8_expert_delta(x, idx, w.to(cuda_device), ex).view(repeat, 6, 64)
    assert torch.isnan(got[:, :2]).all()
    assert torch.isfinite(got[:, 2]).all() and (got[:, 2] != 0).any()
    assert (got[:, 3:] == 0).all()

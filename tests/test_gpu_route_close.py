"""route_experts where choices or group scores lie a few fp32 steps apart: the
indices are those of exact arithmetic (fp64 here: its errors, below 2^-44, are far
under the gaps that the inputs can have, so no index hangs on them)."""
import math

import pytest
import torch

from spider_web_moe_b200.routing import route_experts

pytestmark = pytest.mark.gpu


def definition(logits, k, score, bias, num_groups=1, topk_groups=1):
    """(idx, kept groups) in fp64, all rows at once; ties to the lower id."""
    x = logits.double()
    s = torch.softmax(x, -1) if score == "softmax" else torch.sigmoid(x)
    c = s + bias.double()
    if topk_groups < num_groups:
        per = c.view(len(c), num_groups, -1)
        gs = per.topk(2, dim=-1).values.sum(-1)
        keep = gs.sort(dim=-1, descending=True, stable=True).indices[:, :topk_groups]
        gone = torch.ones_like(gs, dtype=torch.bool).scatter_(1, keep, False)
        c = per.masked_fill(gone.unsqueeze(-1), float("-inf")).view_as(c)
    return c.sort(dim=-1, descending=True, stable=True).indices[:, :k].int()


def check(logits, k, score, bias, **kw):
    got = route_experts(logits, k, score=score, bias=bias, **kw)[0]
    for at in range(0, len(logits), 16384):
        want = definition(logits[at:at + 16384], k, score, bias, **kw)
        bad = (got[at:at + 16384] != want).any(1)
        assert not bad.any(), f"{int(bad.sum())} of {len(want)} tokens"


def test_softmax_sum_of_1024_experts(cuda_device):
    """36 additions of a row's sum all round the same way, by half a step of a sum
    of 1: expert 0's score comes out 2^-18.8 too small, and a choice 2.5e-8 below
    its own would be taken if 2^-19 were believed to cover that."""
    logits = torch.full((1, 1024), -100.0)
    logits[0, 0] = 0.0
    small = math.log(2.0 ** -24 * (1 + 2e-5))
    logits[0, 1:32] = small
    logits[0, [32, 64, 128, 256, 512]] = small
    bias = torch.full((1024,), -10.0)
    bias[0], bias[1000] = -1.0, -2.1708e-6
    idx, w = route_experts(logits.to(cuda_device), 1, bias=bias.to(cuda_device), renormalize=False)
    assert definition(logits, 1, "softmax", bias).item() == 0
    assert idx.item() == 0 and abs(w.item() - 1.0) < 1e-5


@pytest.mark.parametrize("e", [40, 200, 500, 513, 777, 1024])
def test_softmax_choices_around_one_value(e, cuda_device):
    """Biases that bring every choice of row 0 within an fp32 step or two of 0, and
    rows that differ from it by little: gaps on both sides of any tolerance."""
    g = torch.Generator().manual_seed(e)
    logits = torch.randn(3000, e, generator=g) * 2
    logits[1:] = logits[0] + torch.randn(2999, e, generator=g) * torch.logspace(-8, -2, 2999)[:, None]
    s = torch.softmax(logits[0].double(), -1)
    bias = (-s * (1 + torch.randn(e, generator=g).double() * 2.0 ** -22)).float()
    check(logits.to(cuda_device), min(8, e), "softmax", bias.to(cuda_device))

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


def test_group_score_of_opposite_signs(cuda_device):
    """Group 0: 15 + 7u and -15, group 1: 15 and -15 + 3u (u = 2^-20, their last
    place): 7u against 3u.  Order keys with the last three bits replaced read -7u
    and +u, a gap of 7.6e-6 that a tolerance relative to the sum does not cover."""
    u = 2.0 ** -20
    logits = torch.zeros(1, 256)             # sigmoid: 0.5, exactly
    bias = torch.full((256,), -1000.0)
    bias[0], bias[1] = 14.5 + 7 * u, -15.5
    bias[128], bias[129] = 14.5, -15.5 + 3 * u
    kw = dict(num_groups=2, topk_groups=1)
    idx = route_experts(logits.to(cuda_device), 1, score="sigmoid", bias=bias.to(cuda_device), **kw)[0]
    assert definition(logits, 1, "sigmoid", bias, **kw).item() == 0 and idx.item() == 0


@pytest.mark.parametrize("e,groups,topk_groups,size", [(1024, 32, 8, 8.0), (256, 8, 4, 16.0), (256, 8, 4, 4096.0),
                                                       (96, 8, 2, 64.0), (480, 4, 3, 300.0), (800, 32, 9, None)])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_groups_with_large_biases(e, groups, topk_groups, size, score, cuda_device):
    """Biases of both signs, so that a group's best two choices cancel; in the last
    case of another magnitude in each group (1 to 4096), so that the groups' scores
    are known to different precision."""
    g = torch.Generator().manual_seed(e + groups)
    n, per = 60000, e // groups
    logits = (torch.randn(n, e, generator=g) * 1.5).to(cuda_device)
    mag = torch.full((groups, 1), size) if size else torch.exp2(torch.randint(0, 13, (groups, 1), generator=g).float())
    bias = -mag * (1 + torch.rand(groups, per, generator=g))
    bias[:, 0] = mag[:, 0]                   # one large positive choice and its opposite, the next best
    bias[:, 1] = -mag[:, 0]
    order = torch.stack([torch.randperm(per, generator=g) for _ in range(groups)])
    bias = bias.gather(1, order).reshape(-1).contiguous().to(cuda_device)
    check(logits, min(8, per), score, bias, num_groups=groups, topk_groups=topk_groups)

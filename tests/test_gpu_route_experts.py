"""route_experts on the GPU against a plain fp64 statement of it: indices exact,
weights and gradients within fp32 rounding.

Tolerances (u = 2^-24, the fp32 half step).  A score is exp of a difference of
magnitude up to 30 here (relative error 30 u), a 2-ulp expf (4 u), a sum of at
most 32 terms per lane and 5 shuffles (37 u), a reciprocal and a product (2 u);
the renormalising sum and division add at most 80 + 7 u: below 2^-16 in all.
A gradient element is a sum of two terms, each at most M = max_j |ds_j| times its
score and each within 2^-15 of its value.
"""
import pytest
import torch

from spider_web_moe_b200.routing import route_experts

pytestmark = pytest.mark.gpu

RTOL = 2.0 ** -16


def oracle(logits, k, score="softmax", bias=None, num_groups=1, topk_groups=None, group_score="top2",
           renormalize=True, scale=1.0):
    """(idx, weights) in fp64; differentiable in logits (fp64 leaf) for the chosen idx."""
    x = logits.double()
    n, e = x.shape
    b = torch.zeros(e, dtype=torch.float64) if bias is None else bias.double()
    masked = (x == float("-inf")) | (b == float("-inf"))
    dead = x == float("-inf")
    if score == "softmax":
        m = torch.where(dead, torch.zeros_like(x), x).detach().masked_fill(dead, float("-inf")).amax(-1, keepdim=True)
        m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
        z = torch.where(dead, torch.zeros_like(x), torch.exp(torch.where(dead, torch.zeros_like(x), x - m)))
        t = z.sum(-1, keepdim=True)
        s = torch.where(t > 0, z / t.clamp_min(1e-300), z)
    else:
        s = torch.where(dead, torch.zeros_like(x), torch.sigmoid(torch.where(dead, torch.zeros_like(x), x)))
    c = torch.where(masked, torch.full_like(s, float("-inf")), s + b).detach()
    if num_groups > 1 and topk_groups not in (None, num_groups):
        per = c.view(n, num_groups, -1)
        srt = per.sort(-1, descending=True).values
        gs = srt[..., :2].sum(-1) if group_score == "top2" else srt[..., 0]
        keep = gs.sort(dim=-1, descending=True, stable=True).indices[:, :topk_groups]
        gone = torch.ones(n, num_groups, dtype=torch.bool).scatter_(1, keep, False)
        # below every candidate, masked ones (-inf) included
        rank = torch.where(gone.unsqueeze(-1).expand_as(per).reshape(n, e), torch.zeros(n, e, dtype=torch.bool), True)
    else:
        rank = torch.ones(n, e, dtype=torch.bool)
    idx = torch.empty(n, k, dtype=torch.long)
    for r in range(n):  # candidates by (choice descending, id ascending)
        order = sorted((i for i in range(e) if rank[r, i]), key=lambda i: (-float(c[r, i]), i))
        idx[r] = torch.tensor(order[:k])
    w = s.gather(1, idx)
    w = torch.where(masked.gather(1, idx), torch.zeros_like(w), w)
    if renormalize:
        w = w / w.sum(-1, keepdim=True).clamp_min(1e-9)
    return idx.int(), w * scale


CASES = [
    (1, 1, 1, {}), (1, 8, 8, {}), (7, 33, 5, dict(renormalize=False)), (64, 128, 8, {}),
    (50, 60, 3, dict(score="sigmoid")), (129, 256, 8, dict(score="sigmoid", bias=True, num_groups=8, topk_groups=4,
                                                           scale=2.5)),
    (65, 160, 6, dict(num_groups=8, topk_groups=3, group_score="max")),
    (65, 160, 6, dict(num_groups=8, topk_groups=3, bias=True)), (40, 24, 4, dict(num_groups=4, topk_groups=2)),
    (33, 32, 32, dict(bias=True)), (17, 1024, 32, dict(score="sigmoid", num_groups=32, topk_groups=2)),
    (40, 512, 7, dict(bias=True)), (20, 96, 2, dict(num_groups=32, topk_groups=1, score="sigmoid", bias=True)),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,e,k,kw", CASES)
def test_matches_fp64(n, e, k, kw, dtype, cuda_device):
    g = torch.Generator().manual_seed(n * 1000 + e)
    logits = (2 * torch.randn(n, e, generator=g)).to(dtype)
    kw = dict(kw)
    bias = torch.randn(e, generator=g) * 0.1 if kw.pop("bias", False) else None
    idx, w = route_experts(logits.to(cuda_device), k, bias=None if bias is None else bias.to(cuda_device), **kw)
    want_i, want_w = oracle(logits, k, bias=bias, **kw)
    assert idx.dtype == torch.int32 and w.dtype == torch.float32
    assert torch.equal(idx.cpu(), want_i)
    torch.testing.assert_close(w.cpu().double(), want_w, rtol=RTOL, atol=1e-30)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_masks_and_ties(score, biased, cuda_device):
    """Equal logits, rows with few or no experts left, the type's lowest value,
    biases of -inf: ids by (choice, id), masked experts last with weight 0."""
    e, k = 16, 4
    inf = float("inf")
    lowest = torch.finfo(torch.float32).min
    rows = torch.zeros(7, e)
    rows[1] = -inf                       # nothing left
    rows[2, :] = -inf
    rows[2, [9, 3]] = torch.tensor([0.5, 0.25])  # fewer than k left
    rows[3] = lowest
    rows[3, 5] = 1.0
    rows[4] = lowest                     # all equal, at the lowest value
    rows[5, ::2] = -inf
    rows[6] = torch.arange(e) * 1e-7     # closer than fp32 scores resolve
    bias = None
    if biased:
        bias = torch.zeros(e)
        bias[0] = -inf
        bias[7] = 2e-8
    kw = dict(score=score, bias=bias)
    idx, w = route_experts(rows.to(cuda_device), k, score=score, bias=None if bias is None else bias.to(cuda_device))
    want_i, want_w = oracle(rows, k, **kw)
    assert torch.equal(idx.cpu(), want_i)
    torch.testing.assert_close(w.cpu().double(), want_w, rtol=RTOL, atol=1e-30)
    assert torch.isfinite(w).all()


def test_close_choices_are_decided_exactly(cuda_device):
    """Choices spread over a few fp32 steps: the order is that of exact arithmetic."""
    g = torch.Generator().manual_seed(5)
    logits = torch.randn(200, 64, generator=g)
    s = torch.sigmoid(logits.double())
    bias = (0.75 - s[0]).float()  # row 0: every choice within 2^-24 or so of 0.75
    logits[1:100] = logits[0] + torch.randn(99, 64, generator=g) * 1e-6
    kw = dict(score="sigmoid", num_groups=8, topk_groups=4)
    idx, _ = route_experts(logits.to(cuda_device), 8, bias=bias.to(cuda_device), **kw)
    want, _ = oracle(logits, 8, bias=bias, **kw)
    assert torch.equal(idx.cpu(), want)


def test_nan_is_seen(cuda_device):
    rows = torch.zeros(3, 40)
    rows[1, 17] = float("nan")
    idx, w = route_experts(rows.to(cuda_device), 3, score="sigmoid")
    assert idx[1, 0].item() == 17 and torch.isnan(w[1]).all() and torch.isfinite(w[0]).all() and torch.isfinite(w[2]).all()
    idx, w = route_experts(rows.to(cuda_device), 3)
    assert torch.isnan(w[1]).all() and idx[1].tolist() == [0, 1, 2] and torch.isfinite(w[2]).all()


def test_shapes_strides_and_streams(cuda_device):
    g = torch.Generator().manual_seed(6)
    base = torch.randn(6, 5, 50, generator=g).to(cuda_device)
    view = base[:, 1:4, 3:40]                       # no contiguous rows of rows
    idx, w = route_experts(view, 4)
    want_i, want_w = oracle(view.reshape(-1, 37).cpu(), 4)
    assert idx.shape == (6, 3, 4) and torch.equal(idx.reshape(-1, 4).cpu(), want_i)
    pitched = base.view(30, 50)[:, :37]             # a row pitch of its own
    assert torch.equal(route_experts(pitched, 4)[0].cpu(), oracle(pitched.cpu(), 4)[0])
    cols = base[0].t()                              # column-contiguous
    assert torch.equal(route_experts(cols, 2)[0].cpu(), oracle(cols.cpu(), 2)[0])
    assert route_experts(base[:0], 4)[0].shape == (0, 5, 4)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a = route_experts(view, 4)
    s.synchronize()
    assert torch.equal(a[0], idx) and torch.equal(a[1], w)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,e,k,kw", [(1, 1, 1, {}), (37, 60, 3, {}), (64, 128, 8, dict(renormalize=False)),
                                      (33, 256, 8, dict(score="sigmoid", scale=2.5, bias=True)),
                                      (20, 40, 4, dict(score="sigmoid", renormalize=False)),
                                      (9, 700, 6, dict(bias=True))])
def test_gradient(n, e, k, kw, dtype, cuda_device):
    g = torch.Generator().manual_seed(n + e)
    logits = (2 * torch.randn(n, e, generator=g)).to(dtype)
    gw = torch.randn(n, k, generator=g)
    kw = dict(kw)
    bias = torch.randn(e, generator=g) * 0.1 if kw.pop("bias", False) else None
    leaf = logits.to(cuda_device).requires_grad_()
    idx, w = route_experts(leaf, k, bias=None if bias is None else bias.to(cuda_device), **kw)
    w.backward(gw.to(cuda_device))
    x = logits.double().requires_grad_()
    want_i, want_w = oracle(x, k, bias=bias, **kw)
    assert torch.equal(idx.cpu(), want_i)
    (want,) = torch.autograd.grad(want_w, x, gw.double())
    got = leaf.grad.cpu().double()
    assert leaf.grad.dtype == dtype
    # M: the largest derivative with respect to a score of the row
    s = want_w.detach() / kw.get("scale", 1.0)
    d = 1.0 if not kw.get("renormalize", True) else oracle(logits, k, bias=bias, **{**kw, "renormalize": False,
                                                                                    "scale": 1.0})[1].sum(-1, keepdim=True)
    m = kw.get("scale", 1.0) * (gw.double().abs() + (gw.double() * s).abs().sum(-1, keepdim=True)) / d
    m = m.amax(-1, keepdim=True)
    tol = 2.0 ** -14 * m + (0 if dtype == torch.float32 else 2.0 ** -8 * want.abs())
    assert ((got - want).abs() <= tol).all(), float(((got - want).abs() - tol).max())


def test_gradient_against_differences(cuda_device):
    """Central differences of the fp64 oracle, step 1e-5: their error is about
    1e-10, far below the fp32 tolerance."""
    g = torch.Generator().manual_seed(11)
    logits = torch.randn(3, 12, generator=g, dtype=torch.float64).float()
    gw = torch.randn(3, 4, generator=g)
    for kw in (dict(), dict(renormalize=False), dict(score="sigmoid"), dict(score="sigmoid", renormalize=False)):
        leaf = logits.to(cuda_device).requires_grad_()
        route_experts(leaf, 4, **kw)[1].backward(gw.to(cuda_device))
        num = torch.zeros(3, 12, dtype=torch.float64)
        for i in range(12):
            hi, lo = logits.double().clone(), logits.double().clone()
            hi[:, i] += 1e-5
            lo[:, i] -= 1e-5
            num[:, i] = ((oracle(hi, 4, **kw)[1] - oracle(lo, 4, **kw)[1]) * gw.double()).sum(-1) / 2e-5
        assert (leaf.grad.cpu().double() - num).abs().max() < 1e-5


def test_equal_upstream_gradients_cancel_exactly(cuda_device):
    """Renormalised weights sum to a constant: with the same upstream gradient for
    all of a token's weights (a single expert's among them) the gradient is 0."""
    x = torch.randn(50, 40, device=cuda_device)
    for score in ("softmax", "sigmoid"):
        for k in (1, 5):
            leaf = x.clone().requires_grad_()
            _, w = route_experts(leaf, k, score=score)
            w.backward(torch.randn(50, 1, device=cuda_device).expand(50, k))
            assert (leaf.grad == 0).all()


def test_masked_rows_have_zero_gradient(cuda_device):
    rows = torch.randn(3, 8)
    rows[0] = float("-inf")
    rows[1, 1:] = float("-inf")
    bias = torch.zeros(8)
    bias[5:] = float("-inf")
    for score in ("softmax", "sigmoid"):
        leaf = rows.to(cuda_device).requires_grad_()
        _, w = route_experts(leaf, 6, score=score, bias=bias.to(cuda_device))
        w.backward(torch.ones_like(w) * 3)
        assert torch.isfinite(leaf.grad).all()
        assert (leaf.grad[0] == 0).all() and (leaf.grad[1, 1:] == 0).all()


def test_not_twice_differentiable(cuda_device):
    leaf = torch.randn(3, 8, device=cuda_device, requires_grad=True)
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(route_experts(leaf, 2)[1].sum(), leaf, create_graph=True)
    idx, w = route_experts(leaf, 2)
    assert not idx.requires_grad and w.requires_grad
    with torch.no_grad():
        assert not route_experts(leaf, 2)[1].requires_grad


def test_captured(cuda_device):
    g = torch.Generator().manual_seed(12)
    x = torch.randn(70, 64, generator=g).to(cuda_device)
    buf = x.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        route_experts(buf, 4)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        idx, w = route_experts(buf, 4)
    for i in range(3):
        buf.copy_(x.roll(i, 0))
        graph.replay()
        want = route_experts(x.roll(i, 0), 4)
        assert torch.equal(idx, want[0]) and torch.equal(w, want[1])


def test_offsets_past_32_bits(cuda_device):
    """More than 2^31 logits: the last tokens' routing and gradient are those of a small call."""
    n, e = 2_200_000, 1000
    logits = torch.zeros(n, e, dtype=torch.bfloat16, device=cuda_device)
    tail = torch.randn(257, e, generator=torch.Generator().manual_seed(1)).to(cuda_device, torch.bfloat16)
    logits[-257:] = tail
    grad = torch.ones(n, 4, device=cuda_device)
    grad[:, 1] = 3.0
    out = []
    for x in (logits, tail):
        x.requires_grad_()
        idx, w = route_experts(x, 4)
        w.backward(grad[:x.shape[0]])
        out.append((idx[-257:], w[-257:], x.grad[-257:]))
        assert (idx[0] == torch.arange(4, device=cuda_device)).all() or x is tail
    assert all(torch.equal(a, b) for a, b in zip(*out))

"""Expert routing from router logits (``sb_route_experts``), with its gradient.

``SpiderMoELayer`` routes with the reference's softmax router inside its block
kernels (spider_moe/model.py:254-258).  ``route_experts`` is the routing on its
own, for given logits and with the choices larger expert counts are served and
trained with: softmax or sigmoid scores, a balance bias that moves the choice
but not the weight, groups of experts of which only the best take part, and
optional renormalisation and scaling of the weights.  Its results are the
``top_indices`` / ``top_weights`` that ``sparse_expert_delta``,
``fp8_expert_delta`` and the ``forge_ep`` dispatch take.
"""
from __future__ import annotations

import torch

from . import _lib as L

SCORES = {"softmax": L.SB_SCORE_SOFTMAX, "sigmoid": L.SB_SCORE_SIGMOID}
GROUP_SCORES = {"max": 1, "top2": 2}
MAX_EXPERTS, MAX_TOP_K, MAX_GROUPS = 1024, 32, 32


def _dtype_code(dtype: torch.dtype) -> int:
    if dtype == torch.float32:
        return L.SB_F32
    if dtype == torch.bfloat16:
        return L.SB_BF16
    raise TypeError(f"router logits must be float32 or bfloat16, got {dtype}")


def _rows(logits: torch.Tensor) -> torch.Tensor:
    """[..., E] as [n, E] with unit column stride (a copy only if there is no such view)."""
    x = logits if logits.dim() == 2 else logits.reshape(-1, logits.shape[-1])
    return x if x.stride(1) == 1 and x.stride(0) >= x.shape[1] else x.contiguous()


def _launch(logits, top_k, score, bias, num_groups, topk_groups, group_top, renormalize, scale):
    x = _rows(logits)
    n, e = x.shape
    idx = x.new_empty((n, top_k), dtype=torch.int32)
    w = x.new_empty((n, top_k), dtype=torch.float32)
    rc = L.on_device(x.device, L.load().sb_route_experts, x.data_ptr(), _dtype_code(x.dtype), max(x.stride(0), e), n,
                     e, top_k, score, L.ptr(bias), num_groups, topk_groups, group_top, renormalize, scale,
                     idx.data_ptr(), w.data_ptr())
    L.check(rc, "sb_route_experts")
    if logits.dim() == 2:
        return idx, w
    lead = logits.shape[:-1]
    return idx.view(*lead, top_k), w.view(*lead, top_k)


class _RouteExperts(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, bias, top_k, score, num_groups, topk_groups, group_top, renormalize, scale):
        idx, w = _launch(logits, top_k, score, bias, num_groups, topk_groups, group_top, renormalize, scale)
        ctx.save_for_backward(logits, idx, bias)
        ctx.args = (score, renormalize, scale)
        ctx.mark_non_differentiable(idx)
        ctx.set_materialize_grads(False)
        return idx, w

    @staticmethod
    def backward(ctx, _, grad_w):
        if grad_w is None:
            return (None,) * 9
        if torch.is_grad_enabled():
            raise RuntimeError("route_experts is not twice differentiable")
        L.refuse_forward_ad("route_experts", grad_w)
        logits, idx, bias = ctx.saved_tensors
        score, renormalize, scale = ctx.args
        x = _rows(logits)
        n, e = x.shape
        k = idx.shape[-1]
        g = grad_w.reshape(n, k).to(torch.float32).contiguous()
        dl = x.new_empty((n, e))
        rc = L.on_device(x.device, L.load().sb_route_experts_backward, x.data_ptr(), _dtype_code(x.dtype),
                         max(x.stride(0), e), n, e, k, score, L.ptr(bias), renormalize, scale, idx.data_ptr(),
                         g.data_ptr(), dl.data_ptr(), e)
        L.check(rc, "sb_route_experts_backward")
        return dl.view(logits.shape), None, None, None, None, None, None, None, None


def route_experts(logits: torch.Tensor, top_k: int, *, score: str = "softmax", bias: torch.Tensor | None = None,
                  num_groups: int = 1, topk_groups: int | None = None, group_score: str = "top2",
                  renormalize: bool = True, scale: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """logits [..., E] (float32 or bfloat16, CUDA) -> (top_idx int32, top_w float32), both [..., top_k].

    scores ``s`` = softmax or sigmoid of the logits, choices ``s + bias``; with
    ``num_groups`` > 1 only the best ``topk_groups`` groups of E / num_groups
    neighbouring experts take part, a group's score being the sum of its best
    two choices ("top2") or its best one ("max"); the ``top_k`` best choices,
    descending, equal ones by lower id.  Weights are the chosen scores (without
    the bias), divided by max(their sum, 1e-9) with ``renormalize``, times
    ``scale``.  An expert whose logit or bias is -inf ranks last, with weight 0.

    Differentiable in ``logits`` through the weights, the choice held fixed; the
    bias has no gradient; no second and no forward-mode derivatives.  To capture a backward pass into a CUDA graph, drop
    eager graphs of the same logits first: autograd ties their gradient to the
    stream those were built on.
    """
    _dtype_code(logits.dtype)
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise ValueError("route_experts needs logits [..., E] with E >= 1")
    e = logits.shape[-1]
    if score not in SCORES:
        raise ValueError(f"score must be one of {sorted(SCORES)}, got {score!r}")
    if group_score not in GROUP_SCORES:
        raise ValueError(f"group_score must be one of {sorted(GROUP_SCORES)}, got {group_score!r}")
    if e > MAX_EXPERTS:
        raise ValueError(f"at most {MAX_EXPERTS} experts, got {e}")
    if not 1 <= top_k <= min(e, MAX_TOP_K):
        raise ValueError(f"top_k must be in [1, min(E, {MAX_TOP_K})], got {top_k}")
    if not 1 <= num_groups <= MAX_GROUPS or e % num_groups:
        raise ValueError(f"num_groups must divide the {e} experts and be at most {MAX_GROUPS}, got {num_groups}")
    topk_groups = num_groups if topk_groups is None else topk_groups
    if not 1 <= topk_groups <= num_groups or top_k > topk_groups * (e // num_groups):
        raise ValueError(f"topk_groups {topk_groups} of {num_groups} groups must hold top_k {top_k} experts")
    if logits.numel() > L.MAX_EXTENT:  # else there are fewer tokens than that, too
        L.check_extent("tokens", logits.numel() // e)
    L.refuse_forward_ad("route_experts", logits, bias)
    if bias is not None:
        if bias.shape != (e,) or bias.device != logits.device:
            raise ValueError("bias must be [E] on the logits' device")
        if bias.dtype != torch.float32 or bias.requires_grad or not bias.is_contiguous():
            bias = bias.detach().to(torch.float32).contiguous()
    if not logits.is_cuda:
        raise RuntimeError("spider_b200 route_experts runs on CUDA tensors only")
    args = (int(top_k), SCORES[score], int(num_groups), int(topk_groups), GROUP_SCORES[group_score],
            int(bool(renormalize)), float(scale))
    if torch.is_grad_enabled() and logits.requires_grad:
        return _RouteExperts.apply(logits, bias, *args)
    return _launch(logits.detach(), args[0], args[1], bias, *args[2:])

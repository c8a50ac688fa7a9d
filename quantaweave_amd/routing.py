"""Routing of tokens to experts by scores: softmax or sigmoid, a balance bias,
groups of experts, top-k and renormalised weights, with its gradient.

The reference routes by softmax probabilities with a plain top-k
(src/quantweave_moe_model.py:124-137); this is the form of layers with many
experts, whose choice is limited to a few groups and balanced by a bias.
"""

from __future__ import annotations

import math
from functools import lru_cache
from typing import Optional

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _hip, _lib

SCORES = {"softmax": 0, "sigmoid": 1}
GROUP_SCORES = {"max": 1, "top2": 2}
MAX_TOP_K = 64


@lru_cache(maxsize=256)
def check_rule(experts: int, top_k: int, score: str, groups: int, top_groups: int, group_score: str,
               scale: float) -> None:
    """Raises ValueError for a routing rule that no kernel takes (one that some kernel takes is looked at once)."""
    if score not in SCORES:
        raise ValueError(f"score must be softmax or sigmoid, got {score!r}")
    if group_score not in GROUP_SCORES:
        raise ValueError(f"group_score must be top2 or max, got {group_score!r}")
    if not 1 <= experts <= 1024:
        raise ValueError(f"experts must be in [1, 1024], got {experts}")
    if groups < 1 or experts % groups:
        raise ValueError(f"groups must divide the experts, got {groups} and {experts}")
    if not 1 <= top_groups <= groups:
        raise ValueError(f"top_groups must be in [1, {groups}], got {top_groups}")
    if not 1 <= top_k <= min(MAX_TOP_K, top_groups * (experts // groups)):
        raise ValueError(f"top_k must be in [1, {min(MAX_TOP_K, top_groups * (experts // groups))}], got {top_k}")
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")


class _RouteExperts(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits: Tensor, rule: tuple):
        ctx.set_materialize_grads(False)
        index, weight, scores = _route(logits.detach(), *rule)
        ctx.save_for_backward(scores, index)
        ctx.rule = rule
        ctx.mark_non_differentiable(index)
        return index, weight, scores

    @staticmethod
    @once_differentiable
    def backward(ctx, _index, d_weight, d_scores):
        scores, index = ctx.saved_tensors
        top_k, score, _bias, _groups, _top_groups, _group_score, renormalize, scale = ctx.rule
        if not ctx.needs_input_grad[0]:
            return None, None
        _hip.note_stream(ctx.next_functions[0][0], "route_experts", scores.device)
        e = scores.size(-1)
        t = scores.numel() // e
        out = torch.empty_like(scores)
        if t:
            dw = None if d_weight is None else d_weight.float().contiguous()
            ds = None if d_scores is None else d_scores.float().contiguous()
            _hip.call_on(scores.device, "qw_moe_route_scored_backward", _hip.ptr(scores), _hip.ptr(index), _hip.ptr(dw),
                         _hip.ptr(ds), t, e, top_k, SCORES[score], int(renormalize), scale, _hip.ptr(out), _hip.raw_stream(scores.device))
        return out, None


def _route(logits: Tensor, top_k: int, score: str, bias: Optional[Tensor], groups: int, top_groups: int,
           group_score: str, renormalize: bool, scale: float) -> tuple[Tensor, Tensor, Tensor]:
    dev, lead, e = logits.device, logits.shape[:-1], logits.size(-1)
    logits = logits.contiguous()
    t = logits.numel() // e
    scores = torch.empty_like(logits)
    index = torch.empty((*lead, top_k), dtype=torch.int32, device=dev)
    weight = torch.empty((*lead, top_k), dtype=torch.float32, device=dev)
    if t:
        _hip.call_on(dev, "qw_moe_route_scored_from_logits", _hip.ptr(logits), t, e, top_k, SCORES[score],
                     _hip.ptr(bias), groups, top_groups, GROUP_SCORES[group_score], int(renormalize), scale,
                     _hip.ptr(scores), _hip.ptr(index), _hip.ptr(weight), _hip.raw_stream(dev))
    return index, weight, scores


def route_experts(logits: Tensor, top_k: int, *, score: str = "softmax", bias: Optional[Tensor] = None,
                  groups: int = 1, top_groups: Optional[int] = None, group_score: str = "top2",
                  renormalize: bool = True, scale: float = 1.0) -> tuple[Tensor, Tensor, Tensor]:
    """Chooses experts from the router's logits [..., experts] (float32).

    Returns (index int32 [..., top_k], weight [..., top_k], scores [..., experts]):

    * scores: softmax(logits), or sigmoid(logits) per expert;
    * the choice goes by scores + bias (bias [experts], taken in float32, no
      gradient): of the
      `groups` equal runs of experts the `top_groups` with the highest value
      stay (`group_score`: the sum of the run's two highest, or its highest),
      and of their experts the top_k highest are taken, in descending order.
      It is the choice of 64-bit arithmetic; equal values go to the lowest
      index and a NaN counts as -infinity;
    * weight: scores[index], divided by their sum plus 1e-20 where `renormalize`,
      times `scale`.

    Differentiable in logits through weight and scores; second and
    forward-mode derivatives are refused."""
    if not logits.is_cuda:
        _hip.require_device(logits, "route_experts")
    if logits.dtype != torch.float32 or logits.dim() < 1:
        raise ValueError(f"route_experts: logits are float32 [..., experts], got {logits.dtype} {tuple(logits.shape)}")
    _hip.refuse_tangent(logits, "route_experts")
    experts = logits.size(-1)
    top_groups = groups if top_groups is None else top_groups
    check_rule(experts, top_k, score, groups, top_groups, group_score, scale)
    if bias is not None:
        if tuple(bias.shape) != (experts,) or bias.device != logits.device:
            raise ValueError(f"route_experts: bias is [{experts}] on {logits.device}")
        bias = bias.detach().float().contiguous()
    rule = (top_k, score, bias, groups, top_groups, group_score, bool(renormalize), float(scale))
    if logits.requires_grad and torch.is_grad_enabled():
        node = _hip.gradient_node(logits)  # held until the result's graph holds it
        return _RouteExperts.apply(logits, rule)
    return _route(logits.detach(), *rule)

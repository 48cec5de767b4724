"""Routing from a router's logits, and the expert order of the routed pairs.

`MoELayer` routes behind its own gate GEMM (Gate.forward, model.py:569-589) without expert groups. These
take the logits of any router: K3's KimiMoEGate, the M2.5 engine's F.linear (m25_stage.py:412-416), with
group-limited selection where the model has it.

    w, ids = topk(logits, 8, bias=b, score="sigmoid", n_group=8, topk_group=4, group_score="top2")
    order = expert_order(ids, n_experts)

CUDA tensors only; on the tensors' device, the current stream or `stream`, without synchronising.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import _lib, fp4
from ._lib import check
from .fp4 import _away, _elsewhere

_SCORE = _lib.SCORE
_GROUP_SCORE = {"max": 0, "top2": 1}


class ExpertOrder(NamedTuple):
    """The (token, slot) pairs sorted by expert, in token order within one: expert e's are
    offsets[e] .. offsets[e + 1] - 1."""
    offsets: torch.Tensor     # int32 [E + 1]
    tokens: torch.Tensor      # int32 [T k]: the token at each place (-1 behind offsets[E])
    places: torch.Tensor      # int32 [T, k]: each pair's place (-1: its id is no expert)


def topk(logits: torch.Tensor, k: int, bias: Optional[torch.Tensor] = None, score: str = "sigmoid", n_group: int = 1,
         topk_group: int = 1, group_score: str = "max", renormalize: bool = True, scale: float = 1.0, stream=None):
    """logits [T, E] (bf16, fp16 or fp32, any row stride) -> (weights fp32 [T, k], indices int64 [T, k]), best first.

    score        "softmax", "sigmoid" or "sqrtsoftplus" of the logits
    bias         fp32 [E], added for the selection only
    n_group      groups of E / n_group consecutive experts; only the topk_group best compete, a group
                 scored by its best expert ("max") or the sum of its two best ("top2")
    renormalize  divide the chosen experts' unbiased scores by their sum; then times `scale`

    Values are compared as real numbers (sums with a bias, or of two: in 64 bits), ties go to the lower id. An expert whose logit is NaN, -inf or the
    type's lowest value is masked: after all others of the kept groups, with weight 0. A bias of -inf keeps an
    expert behind the others too."""
    sc, gs = _SCORE.get(score), _GROUP_SCORE.get(group_score)
    if sc is None or gs is None:
        raise ValueError(f"topk: score {score!r}, group_score {group_score!r}")
    if _away("topk", logits, stream):
        with _elsewhere(logits.device, stream):
            return topk(logits, k, bias, score, n_group, topk_group, group_score, renormalize, scale)
    r = (fp4._HOST or fp4.host()).topk(logits, k, bias, sc, n_group, topk_group, gs, renormalize, scale)
    if type(r) is int:
        check(r, "sb_route_topk")
    return r


def expert_order(indices: torch.Tensor, n_experts: int, stream=None) -> ExpertOrder:
    """indices int64 [T, k] -> ExpertOrder. Pairs whose id is outside [0, n_experts) (dropped tokens, padding) are
    left out."""
    if _away("expert_order", indices, stream):
        with _elsewhere(indices.device, stream):
            return expert_order(indices, n_experts)
    r = (fp4._HOST or fp4.host()).expert_order(indices, n_experts)
    if type(r) is int:
        check(r, "sb_expert_order")
    return ExpertOrder(*r)

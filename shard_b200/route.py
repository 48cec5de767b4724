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

from . import _lib
from ._lib import check, lib
from .fp4 import DTYPES, _current_device, _current_stream, _elsewhere, _empty, _same_device

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

    Values are compared as real numbers, ties go to the lower id. An expert whose logit is NaN, -inf or the
    type's lowest value is masked: after all others of the kept groups, with weight 0."""
    sc, gs, dt = _SCORE.get(score), _GROUP_SCORE.get(group_score), DTYPES.get(logits.dtype)
    if sc is None or gs is None:
        raise ValueError(f"topk: score {score!r}, group_score {group_score!r}")
    if dt is None or not logits.is_cuda or logits.dim() != 2:
        raise ValueError("topk: logits must be a CUDA tensor [T, E] of bf16, fp16 or fp32")
    dev = logits.get_device()
    if stream is not None or dev != _current_device():
        with _elsewhere(logits.device, stream):
            return topk(logits, k, bias, score, n_group, topk_group, group_score, renormalize, scale)
    t, e = logits.shape
    stride, inner = logits.stride()
    if inner != 1 and e > 1:
        logits = logits.contiguous()
        stride = e
    pb = None
    if bias is not None:
        if bias.dtype != torch.float32 or tuple(bias.shape) != (e,) or not bias.is_contiguous():
            raise ValueError(f"topk: bias must be contiguous fp32 [{e}]")
        _same_device("topk", logits, bias)
        pb = bias.data_ptr()
    w = _empty((t, k), dtype=torch.float32, device=logits.device)
    ids = _empty((t, k), dtype=torch.int64, device=logits.device)
    rc = lib().sb_route_topk(logits.data_ptr(), dt, t, e, stride if t > 1 else e, pb, k, sc, n_group, topk_group, gs,
                             renormalize, scale, w.data_ptr(), ids.data_ptr(), _current_stream(dev))
    if rc:
        check(rc, "sb_route_topk")
    return w, ids


def expert_order(indices: torch.Tensor, n_experts: int, stream=None) -> ExpertOrder:
    """indices int64 [T, k] -> ExpertOrder. Pairs whose id is outside [0, n_experts) (dropped tokens, padding) are
    left out."""
    if not indices.is_cuda or indices.dtype != torch.int64 or indices.dim() != 2 or not indices.is_contiguous():
        raise ValueError("expert_order: indices must be a contiguous CUDA int64 tensor [T, k]")
    dev = indices.get_device()
    if stream is not None or dev != _current_device():
        with _elsewhere(indices.device, stream):
            return expert_order(indices, n_experts)
    t, k = indices.shape
    if k < 1:
        raise ValueError("expert_order: no slots")
    pairs = t * k
    L = lib()
    need = L.sb_expert_order_workspace_bytes(pairs, n_experts) if pairs > 1024 else 0
    # one allocation: places, tokens, offsets, the kernels' counts
    n0, n1, n2, n3 = pairs, pairs, n_experts + 1, need >> 2
    buf = _empty(n0 + n1 + n2 + n3, dtype=torch.int32, device=indices.device)
    base = buf.data_ptr()
    rc = L.sb_expert_order(indices.data_ptr(), t, k, n_experts, base + 4 * (n0 + n1), base + 4 * n0, base,
                           base + 4 * (n0 + n1 + n2) if need else None, need, _current_stream(dev))
    if rc:
        check(rc, "sb_expert_order")
    places, tokens, offsets, _ = buf.split_with_sizes((n0, n1, n2, n3))
    return ExpertOrder(offsets, tokens, places.view(t, k))

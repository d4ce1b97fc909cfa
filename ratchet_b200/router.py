"""The router of a mixture-of-experts layer: top-k experts and combine weights
from logits, and the gradient of the logits.  Its ids and weights are what
ExpertParallelMoE.forward takes; zipf_routing in moe.py draws synthetic ones.
"""
from __future__ import annotations

import torch

from . import _lib, ops

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_SCORES = {"softmax": 0, "sigmoid": 1}
MAX_EXPERTS = 1024
MAX_TOPK = 32


def _logits(logits: torch.Tensor, topk: int, score: str):
    if (logits.dim() != 2 or logits.dtype not in _DTYPES or not logits.is_cuda
            or not logits.is_contiguous()):
        raise ValueError("logits must be a contiguous [T, E] fp32, bf16 or fp16 CUDA tensor")
    tokens, experts = int(logits.shape[0]), int(logits.shape[1])
    if not 1 <= experts <= MAX_EXPERTS:
        raise ValueError(f"{experts} experts outside [1, {MAX_EXPERTS}]")
    if not 1 <= topk <= min(experts, MAX_TOPK):
        raise ValueError(f"topk={topk} outside [1, {min(experts, MAX_TOPK)}]")
    if score not in _SCORES:
        raise ValueError(f"score={score!r}: 'softmax' or 'sigmoid'")
    if tokens > 2**31 - 1:
        raise ValueError(f"{tokens} tokens are too many")
    return tokens, experts


def moe_router(logits: torch.Tensor, topk: int, *, score: str = "softmax",
               bias: torch.Tensor | None = None, renormalize: bool = True, scale: float = 1.0):
    """(ids int32 [T, topk], weights fp32 [T, topk]) of router logits [T, E].

    Scores s are the softmax or the sigmoid of a token's logits.  The topk experts
    with the largest s + bias are chosen (bias: fp32 [E], for the choice only, e.g.
    a load balancing term), largest first, ties to the lowest index; their weights
    are s -- over the sum of the chosen ones' with renormalize -- times scale.
    A logit (or a bias) of -inf masks an expert; routes that are left over carry
    id -1 and weight 0, which the layer treats as absent.  A row that holds a NaN
    logit (softmax: or +inf) has NaN weights.  E <= 1024, topk <= 32."""
    tokens, experts = _logits(logits, topk, score)
    dev = logits.device
    if bias is not None and (bias.dtype is not torch.float32 or tuple(bias.shape) != (experts,)
                             or bias.device != dev or not bias.is_contiguous()):
        raise ValueError(f"bias must be a contiguous fp32 [{experts}] tensor on {dev}")
    with ops._on(dev):
        ids = torch.empty((tokens, topk), dtype=torch.int32, device=dev)
        weights = torch.empty((tokens, topk), dtype=torch.float32, device=dev)
        _lib.check(_lib.lib().fgg_moe_router(
            logits.data_ptr(), _DTYPES[logits.dtype], tokens, experts, topk, _SCORES[score],
            None if bias is None else bias.data_ptr(), 1 if renormalize else 0, float(scale),
            ids.data_ptr(), weights.data_ptr(), ops._stream_ptr(dev)), "moe_router")
    return ids, weights


def moe_router_backward(dweights: torch.Tensor, logits: torch.Tensor, ids: torch.Tensor, *,
                        score: str = "softmax", renormalize: bool = True,
                        scale: float = 1.0) -> torch.Tensor:
    """The gradient of moe_router's logits, [T, E] in their type.

    dweights fp32 [T, topk]; logits, score, renormalize and scale as in the
    forward call; ids int32 [T, topk] as it returned them (an id outside [0, E) is
    an absent route; an expert named twice gets both shares).  The choice itself
    has no gradient, so neither has the bias."""
    if dweights.dim() != 2:
        raise ValueError(f"dweights must be [T, topk], got {list(dweights.shape)}")
    topk = int(dweights.shape[1])
    tokens, experts = _logits(logits, topk, score)
    dev = logits.device
    for name, t, dt in (("dweights", dweights, torch.float32), ("ids", ids, torch.int32)):
        if (t.dtype is not dt or tuple(t.shape) != (tokens, topk) or t.device != dev
                or not t.is_contiguous()):
            raise ValueError(f"{name} must be a contiguous {dt} [{tokens}, {topk}] tensor on {dev}")
    with ops._on(dev):
        dlogits = torch.empty_like(logits)
        _lib.check(_lib.lib().fgg_moe_router_backward(
            dweights.data_ptr(), logits.data_ptr(), _DTYPES[logits.dtype], ids.data_ptr(), tokens,
            experts, topk, _SCORES[score], 1 if renormalize else 0, float(scale),
            dlogits.data_ptr(), ops._stream_ptr(dev)), "moe_router_backward")
    return dlogits

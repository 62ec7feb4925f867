"""Expert choice from router logits on B200.

``route_topk`` turns the logits of any MoE router into the ``(top_k_weights,
top_k_index)`` pair that the expert modules take
(``Gemma4TextExpertsNVFP4`` / ``Gemma4TextExpertsFP8`` /
``Gemma4TextExpertsFP8Block``): softmax or sigmoid scores, a bias that only
the choice sees (load balancing), groups of experts, top-k and renormalised
weights in one launch (``csrc/route.cu``). The Gemma-4 router keeps its own
kernel, which fuses the projection (``bridges.gemma4.router``). The
reference has no such function: its router is HF transformers' code.

Forward only, like the expert modules: the outputs carry no gradient.
"""
from __future__ import annotations

import torch

from .. import _capi as A

_SCORES = {"softmax": A.SCORE_SOFTMAX, "sigmoid": A.SCORE_SIGMOID}
_GROUP_SCORES = {"max": A.GROUP_MAX, "top2": A.GROUP_TOP2}
_LOGITS = (torch.bfloat16, torch.float16, torch.float32)


def route_topk(logits: torch.Tensor, k: int, *, score: str = "softmax", bias: torch.Tensor | None = None,
               n_group: int = 1, topk_group: int = 1, group_score: str = "max", renormalize: bool = True,
               scale: float = 1.0) -> tuple[torch.Tensor, torch.Tensor]:
    """The k experts of each token and their weights.

    Args:
        logits: (T, E) bfloat16, float16 or float32 router logits; an expert
            masked with ``-inf`` is never chosen.
        k: experts per token, at most ``min(E, 32)``; E is at most 1024.
        score: ``"softmax"`` over the E logits, or ``"sigmoid"`` of each.
        bias: (E,) added to the scores for the choice alone; the weights are
            the unbiased scores.
        n_group, topk_group: the experts form ``n_group`` equal runs (at most
            32); only those of the best ``topk_group`` runs can be chosen.
        group_score: a run's worth: its ``"max"`` choice value or the sum of
            its ``"top2"``.
        renormalize: divide the k weights by their sum.
        scale: factor on the weights.

    Returns ``(weights (T, k) float32, ids (T, k) int64)``, experts in
    descending order of score + bias in 64-bit arithmetic; equal ones by the
    larger logit, then by the lower index (equal groups by the logit of their
    best expert), so that a bias that is the same for all changes nothing. A
    slot for which no expert is left has id E and weight 0 (the expert
    forwards skip it); a row that holds a NaN (for softmax, or +inf) has NaN
    weights.
    """
    if logits.ndim != 2:
        raise ValueError(f"logits must be 2D (tokens, experts); got shape {tuple(logits.shape)}")
    if logits.dtype not in _LOGITS:
        raise ValueError(f"logits must be bfloat16, float16 or float32, got {logits.dtype}")
    if score not in _SCORES:
        raise ValueError(f"score must be 'softmax' or 'sigmoid', got {score!r}")
    if group_score not in _GROUP_SCORES:
        raise ValueError(f"group_score must be 'max' or 'top2', got {group_score!r}")
    T, E = logits.shape
    if bias is not None:
        if tuple(bias.shape) != (E,):
            raise ValueError(f"bias must have shape ({E},), got {tuple(bias.shape)}")
        if bias.dtype not in _LOGITS:
            raise ValueError(f"bias must be bfloat16, float16 or float32, got {bias.dtype}")
    dev = A.cuda_index(logits, bias)
    if not 1 <= k <= E:
        raise ValueError(f"route_topk: k ({k}) must be in [1, min(num_experts, 32)]")
    if logits.stride(1) != 1 or logits.stride(0) < E:
        logits = logits.contiguous()
    with A.on_device(dev):
        if bias is not None:
            bias = bias.detach().to(torch.float32).contiguous()
        weights = torch.empty((T, k), dtype=torch.float32, device=logits.device)
        ids = torch.empty((T, k), dtype=torch.int64, device=logits.device)
        A.check(A.load().aeoq_route_topk(
            logits.data_ptr(), A.dtype_code(logits.dtype), logits.stride(0) if T > 1 else E, T, E, k, _SCORES[score],
            A.ptr(bias), n_group, topk_group, _GROUP_SCORES[group_score], int(bool(renormalize)), float(scale),
            weights.data_ptr(), ids.data_ptr(), A.raw_stream(dev)))
    return weights, ids

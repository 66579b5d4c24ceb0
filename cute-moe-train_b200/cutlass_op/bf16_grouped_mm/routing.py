"""Router of the MoE block: top-k experts per token with their weights, with autograd.

Between a model's router projection and the grouped products: ``moe_route`` turns logits [tokens, E] into
the expert ids that :func:`permute.moe_permute` (and the expert-parallel ``EPMoEFFN``) take and the fp32
weights that :func:`permute.moe_unpermute` applies.  One kernel forward (``grouped_mm::moe_route``) and
one backward (``grouped_mm::moe_route_bwd``).
"""

from __future__ import annotations

import torch

from . import _ext  # noqa: F401  (registers the operators)
from .optimer import timed

# include/moe_gemm.h: enum mgf_route_score, with MGF_ROUTE_BIAS_ON_SCORE for the biased ones
_SCORES = {"softmax": 0, "sigmoid": 1, "biased_softmax": 0x100, "biased_sigmoid": 0x101}


@torch.library.register_fake("grouped_mm::moe_route")
def _moe_route_fake(logits, topk, score, renormalize, scale, bias, token_mask):
    shape = (logits.size(0), topk)
    return (torch.empty(shape, dtype=torch.float32, device=logits.device),
            torch.empty(shape, dtype=torch.int64, device=logits.device))


@torch.library.register_fake("grouped_mm::moe_route_bwd")
def _moe_route_bwd_fake(logits, expert_idx, grad_weights, score, renormalize, scale):
    return torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)


def moe_route(logits: torch.Tensor, topk: int, score: str = "softmax", renormalize: bool = True,
              scale: float = 1.0, bias: torch.Tensor | None = None,
              token_mask: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Top-k routing of every token.

    Args:
        logits: [tokens, E] bf16, fp16 or fp32 (any row stride), E <= 1024.
        topk: experts per token, at most min(E, 32).
        score: ``"softmax"`` or ``"sigmoid"`` of the logits; ``"biased_softmax"`` or ``"biased_sigmoid"``: the same
            weights, with ``bias`` added to the score itself (of the softmax: over all experts) for the selection.
        renormalize: divide by the chosen experts' sum; for softmax that is the softmax over the chosen
            logits (GPT-OSS), without it the softmax over all E.
        scale: factor on the weights.
        bias: fp32 [E], for the selection only (load balancing), no gradient.  It is added to the **logits**, unless
            ``score`` is one of the biased ones.  The two choose different experts, since neither score is linear:
            logits (4, 1) with bias (0, 0.4) choose expert 0, their sigmoids (0.982, 0.731) with it expert 1.  A bias
            that was trained on the scores, as loss-free balancing does, needs ``"biased_sigmoid"``.
        token_mask: bool [tokens]; tokens with False (padding) are not routed.

    Returns:
        (weights fp32 [tokens, topk], expert_idx int64 [tokens, topk]), the largest logit (or score) + bias first
        and ties to the lowest expert.  Experts whose logit (or sum with the bias) is -inf are never chosen; slots
        left over that way and the slots of masked tokens have id -1 and weight 0, and such copies are
        dropped by ``moe_permute``.  NaN sorts first, as in ``torch.topk``, and its weights are NaN.
        The logits' gradient is zero at experts that the weights do not depend on.
    """
    if score not in _SCORES:
        raise ValueError(f"moe_route: score must be one of {sorted(_SCORES)}, got {score!r}")
    with timed("moe_route"):
        return torch.ops.grouped_mm.moe_route.default(logits, topk, _SCORES[score], renormalize, scale, bias, token_mask)

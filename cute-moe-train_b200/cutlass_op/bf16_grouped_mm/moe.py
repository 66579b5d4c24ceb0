"""The MoE block on one GPU: router logits and tokens in, combined expert outputs out, with autograd.

route -> permute -> expert FFN -> unpermute over the operators of :mod:`routing`, :mod:`permute`, the bf16
FFN (``grouped_mm_ffn``) and :mod:`fp8_block`; the single-GPU counterpart of
``expert_parallel.EPMoEFFN``.  Nothing is read on the host, so the whole block can be captured in a graph.
"""

from __future__ import annotations

import torch

from . import grouped_mm_ffn
from .fp8_block import (grouped_mm_ffn_fp8_block, grouped_mm_fp8_block, grouped_mm_swiglu_fp8_block,
                        quantize_rows_block, quantize_weights_block)
from .permute import moe_permute, moe_permute_fp8, moe_unpermute
from .routing import moe_route

PRECISIONS = ("bf16", "fp8_block")


def moe_ffn(x: torch.Tensor, logits: torch.Tensor, topk: int, w_up: torch.Tensor, w_down: torch.Tensor,
            b_up: torch.Tensor, b_down: torch.Tensor | None = None, *, precision: str = "bf16",
            score: str = "softmax", renormalize: bool = True, route_scale: float = 1.0,
            route_bias: torch.Tensor | None = None, token_mask: torch.Tensor | None = None,
            swiglu_alpha: float = 1.702, swiglu_limit: float = 7.0,
            up_codes: tuple[torch.Tensor, torch.Tensor] | None = None,
            down_codes: tuple[torch.Tensor, torch.Tensor] | None = None) -> torch.Tensor:
    """out[t] = sum_j weights[t, j] * FFN_expert(t, j)(x[t]).

    x [tokens, H] bf16, logits [tokens, E], w_up [E, H, 2I] (gate and up interleaved), w_down [E, I, H],
    biases bf16.  ``score`` ... ``token_mask`` as in :func:`routing.moe_route` (masked tokens get zeros).
    ``precision="fp8_block"`` runs the products and input gradients in block-scaled e4m3 (see
    :func:`fp8_block.grouped_mm_ffn_fp8_block`, also for ``up_codes`` / ``down_codes``); without gradients the
    tokens go straight to codes in expert order and no bf16 rows are written.
    """
    if precision not in PRECISIONS:
        raise ValueError(f"moe_ffn: precision must be one of {PRECISIONS}, got {precision!r}")
    if logits.shape[1] != w_up.shape[0]:
        raise ValueError(f"moe_ffn: logits are for {logits.shape[1]} experts, the weights for {w_up.shape[0]}")
    weights, expert_idx = moe_route(logits, topk, score, renormalize, route_scale, route_bias, token_mask)
    num_experts = w_up.shape[0]
    if precision == "bf16":
        if up_codes is not None or down_codes is not None:
            raise ValueError("moe_ffn: up_codes and down_codes need precision='fp8_block'")
        rows, plan = moe_permute(x, expert_idx, num_experts)
        y = grouped_mm_ffn(rows, w_up, w_down, plan.offs, b_up, b_down, swiglu_alpha, swiglu_limit)
    elif torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, w_up, w_down, b_up, b_down)):
        rows, plan = moe_permute(x, expert_idx, num_experts)
        y = grouped_mm_ffn_fp8_block(rows, w_up, w_down, plan.offs, b_up, b_down, swiglu_alpha, swiglu_limit,
                                     up_codes, down_codes)
    else:
        q_up, s_up = up_codes if up_codes is not None else quantize_weights_block(w_up)
        q_down, s_down = down_codes if down_codes is not None else quantize_weights_block(w_down)
        qx, sx, plan = moe_permute_fp8(x, expert_idx, num_experts)
        s, _ = grouped_mm_swiglu_fp8_block(qx, q_up, plan.offs, sx, s_up, b_up, swiglu_alpha, swiglu_limit)
        qs, ss = quantize_rows_block(s)
        y = grouped_mm_fp8_block(qs, q_down, plan.offs, ss, s_down, b_down)
    return moe_unpermute(y, plan, weights)

"""Tokens sorted by expert and back on one GPU, with the router's weights applied, with autograd.

``moe_permute`` gives the rows and the ``offs`` that the grouped products take; ``moe_unpermute`` brings
their outputs back to the tokens::

    weights, expert_idx = moe_route(logits, topk)
    rows, plan = moe_permute(x, expert_idx, num_experts)
    y = grouped_mm_ffn(rows, w_up, w_down, plan.offs, b_up, b_down)
    out = moe_unpermute(y, plan, weights)

Dropped copies (id -1: masked tokens, slots without an expert, a capacity limit of the caller) have no
row and contribute nothing; the rows behind ``offs[-1]`` are zeros.  The plan is built by one kernel
(``grouped_mm::moe_sort``) and never read on the host.  Sums are fp32 in slot order, without atomics.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import _ext  # noqa: F401  (registers the operators)
from .custom_op import _padded, refuse_tangents
from .optimer import timed


class MoEPlan(NamedTuple):
    """Where every routed copy goes (copy = token * topk + slot).

    offs: int32 [E], cumulative row ends per expert; row_of_copy: int32 [tokens, topk], the copy's row or
    -1 if it was dropped; copy_of_row: int32 [tokens * topk], the row's copy or -1 behind offs[-1].
    """

    offs: torch.Tensor
    row_of_copy: torch.Tensor
    copy_of_row: torch.Tensor


def _plan_fake(expert_idx, num_experts):
    def i32(*shape):
        return torch.empty(shape, dtype=torch.int32, device=expert_idx.device)

    return i32(num_experts), i32(*expert_idx.shape), i32(expert_idx.numel())


def _rows_fake(rows, cols, dtype, device):
    return torch.empty_strided((rows, cols), (_padded(cols, dtype), 1), dtype=dtype, device=device)


@torch.library.register_fake("grouped_mm::moe_sort")
def _moe_sort_fake(expert_idx, num_experts):
    return _plan_fake(expert_idx, num_experts)


@torch.library.register_fake("grouped_mm::moe_permute")
def _moe_permute_fake(x, expert_idx, num_experts):
    return (_rows_fake(expert_idx.numel(), x.size(1), x.dtype, x.device), *_plan_fake(expert_idx, num_experts))


@torch.library.register_fake("grouped_mm::moe_permute_rows")
def _moe_permute_rows_fake(x, offs, row_of_copy):
    return _rows_fake(row_of_copy.numel(), x.size(1), x.dtype, x.device)


@torch.library.register_fake("grouped_mm::moe_unpermute")
def _moe_unpermute_fake(rows, offs, row_of_copy, weights):
    return _rows_fake(row_of_copy.size(0), rows.size(1), rows.dtype, rows.device)


@torch.library.register_fake("grouped_mm::moe_unpermute_bwd")
def _moe_unpermute_bwd_fake(grad_out, rows, offs, row_of_copy, weights, need_rows, need_weights):
    g_rows = _rows_fake(rows.size(0), rows.size(1), rows.dtype, rows.device) if need_rows else rows.new_empty(0)
    shape = row_of_copy.shape if need_weights else (0,)
    return g_rows, torch.empty(shape, dtype=torch.float32, device=rows.device)


def _codes_fake(rows, cols, device):
    return (_rows_fake(rows, cols, torch.float8_e4m3fn, device),
            _rows_fake(rows, (cols + 127) // 128, torch.float32, device))


@torch.library.register_fake("grouped_mm::moe_permute_fp8")
def _moe_permute_fp8_fake(x, expert_idx, num_experts):
    return (*_codes_fake(expert_idx.numel(), x.size(1), x.device), *_plan_fake(expert_idx, num_experts))


@torch.library.register_fake("grouped_mm::moe_permute_rows_fp8")
def _moe_permute_rows_fp8_fake(x, offs, row_of_copy):
    return _codes_fake(row_of_copy.numel(), x.size(1), x.device)


def moe_sort(expert_idx: torch.Tensor, num_experts: int) -> MoEPlan:
    """The plan of a stable sort of the routed copies by expert.

    expert_idx: int64 [tokens, topk], ids in [-1, num_experts), -1 = dropped; the same expert may occur
    twice in a token.  Other ids drop their copy and are reported by ``check_device_status()``.
    num_experts <= 1024.
    """
    with timed("moe_sort"):
        return MoEPlan(*torch.ops.grouped_mm.moe_sort.default(expert_idx, num_experts))


def moe_permute(x: torch.Tensor, expert_idx: torch.Tensor | None = None, num_experts: int | None = None,
                plan: MoEPlan | None = None) -> tuple[torch.Tensor, MoEPlan]:
    """x [tokens, hidden] (bf16, fp16 or fp32) -> (rows [tokens * topk, hidden] in expert order, plan).

    Pass ``expert_idx`` and ``num_experts`` to sort, or the ``plan`` of an earlier call.  The gradient of x
    is the sum of its copies' row gradients.
    """
    with timed("moe_permute"):
        if plan is not None:
            return torch.ops.grouped_mm.moe_permute_rows.default(x, plan.offs, plan.row_of_copy), plan
        if expert_idx is None or num_experts is None:
            raise ValueError("moe_permute needs expert_idx and num_experts, or a plan")
        rows, *p = torch.ops.grouped_mm.moe_permute.default(x, expert_idx, num_experts)
        return rows, MoEPlan(*p)


def moe_permute_fp8(x: torch.Tensor, expert_idx: torch.Tensor | None = None, num_experts: int | None = None,
                    plan: MoEPlan | None = None) -> tuple[torch.Tensor, torch.Tensor, MoEPlan]:
    """``quantize_rows_block`` of the rows of ``moe_permute`` (bf16 x) in one pass over x: (e4m3 codes
    [tokens * topk, hidden], fp32 scales [tokens * topk, ceil(hidden / 128)], plan).  Rows behind offs[-1]
    have zero codes and scales.  No autograd: the codes feed inference, or a backward that uses x."""
    refuse_tangents("moe_permute_fp8", x)
    with timed("moe_permute_fp8"):
        if plan is not None:
            return (*torch.ops.grouped_mm.moe_permute_rows_fp8.default(x.detach(), plan.offs, plan.row_of_copy), plan)
        if expert_idx is None or num_experts is None:
            raise ValueError("moe_permute_fp8 needs expert_idx and num_experts, or a plan")
        q, scale, *p = torch.ops.grouped_mm.moe_permute_fp8.default(x.detach(), expert_idx, num_experts)
        return q, scale, MoEPlan(*p)


def moe_unpermute(rows: torch.Tensor, plan: MoEPlan, weights: torch.Tensor | None = None) -> torch.Tensor:
    """out[t] = sum_j weights[t, j] * rows[plan.row_of_copy[t, j]] (weights fp32 [tokens, topk], or 1),
    summed in fp32 and rounded once.  Gradients: rows and weights, from one pass over the rows."""
    with timed("moe_unpermute"):
        return torch.ops.grouped_mm.moe_unpermute.default(rows, plan.offs, plan.row_of_copy, weights)

"""e4m3 with a scale for each block of 128: quantisers, grouped products and the FFN with autograd.

The recipe of :mod:`fp8` gives a whole row or column one scale, so one outlier costs all of it its small
values.  Here every 1 x 128 block of an activation row and every 128 x 128 block of a weight has its own.
The scales are powers of two (the smallest s with amax / s <= 448), so quantising rounds only once, in the
code; the grouped product takes any fp32 scales.  The weights' codes keep the weights' layout: one set is
the forward's operand and, transposed, the input gradient's.

``grouped_mm_fp8_block``, ``grouped_mm_swiglu_fp8_block`` and ``grouped_mm_swiglu_bwd_fp8_block`` are the
ragged-M products with the bias, SwiGLU and SwiGLU-backward epilogues; every block's product is scaled and
added in fp32.  ``grouped_mm_ffn_fp8_block`` chains them into the MoE FFN with autograd: both forward products
and both input gradients in e4m3, the weight and bias gradients in bf16 (``grouped_mm::mm_wgrad_bias``) from the
unquantised activations -- they contract over tokens, where the 1 x 128 blocks of either operand do not lie.
"""

from __future__ import annotations

import torch

from . import _ext  # noqa: F401  (registers the operators)
from .custom_op import _padded, refuse_tangents
from .optimer import timed
from .permute import _codes_fake

BLOCK = 128
E4M3_MAX = 448.0


def _blocks(n: int) -> int:
    return (n + BLOCK - 1) // BLOCK


@torch.library.register_fake("grouped_mm::fp8_quantize_rows_block")
def _quantize_rows_block_fake(x):
    return _codes_fake(x.size(0), x.size(1), x.device)


@torch.library.register_fake("grouped_mm::fp8_quantize_weights_block")
def _quantize_weights_block_fake(w):
    e, k, n = w.shape
    if w.stride(2) != 1 and n > 1:
        q, s = _quantize_weights_block_fake(w.transpose(1, 2))
        return q.transpose(1, 2), s.transpose(1, 2)
    p = (n + 15) // 16 * 16
    return (torch.empty_strided((e, k, n), (k * p, p, 1), dtype=torch.float8_e4m3fn, device=w.device),
            torch.empty((e, _blocks(k), _blocks(n)), dtype=torch.float32, device=w.device))


def quantize_rows_block(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """bf16 [M, K] -> (e4m3 [M, K], fp32 [M, ceil(K / 128)]), both with a 16-byte row pitch:
    x[m, k] ~= q[m, k] * scale[m, k // 128].  Non-finite elements become NaN codes and do not enter their
    block's scale."""
    refuse_tangents("quantize_rows_block", x)
    with timed("fp8_quantize"):
        return torch.ops.grouped_mm.fp8_quantize_rows_block.default(x.detach())


def quantize_weights_block(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """bf16 [E, K, N] (unit stride along N or along K) -> (e4m3 [E, K, N] in the same layout, fp32
    [E, ceil(K / 128), ceil(N / 128)]): w[e, k, n] ~= q[e, k, n] * scale[e, k // 128, n // 128].
    ``q.transpose(1, 2), scale.transpose(1, 2)`` are the codes of ``w.transpose(1, 2)``."""
    refuse_tangents("quantize_weights_block", w)
    with timed("fp8_quantize"):
        return torch.ops.grouped_mm.fp8_quantize_weights_block.default(w.detach())


def dequantize_rows_block(q: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    return q.float() * scale.repeat_interleave(BLOCK, 1)[:, :q.shape[1]]


def dequantize_weights_block(q: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    s = scale.repeat_interleave(BLOCK, 1)[:, :q.shape[1]].repeat_interleave(BLOCK, 2)[:, :, :q.shape[2]]
    return q.float() * s


def _out_fake(mat_a, cols):
    return torch.empty_strided((mat_a.size(0), cols), (_padded(cols, torch.bfloat16), 1), dtype=torch.bfloat16,
                               device=mat_a.device)


@torch.library.register_fake("grouped_mm::mm_fp8_block")
def _mm_fp8_block_fake(mat_a, mat_b, offs, scale_a, scale_b, bias):
    return _out_fake(mat_a, mat_b.size(2))


@torch.library.register_fake("grouped_mm::mm_swiglu_fp8_block")
def _mm_swiglu_fp8_block_fake(mat_a, mat_b, offs, scale_a, scale_b, bias, swiglu_alpha, swiglu_limit):
    return _out_fake(mat_a, mat_b.size(2) // 2), _out_fake(mat_a, mat_b.size(2))


@torch.library.register_fake("grouped_mm::mm_swiglu_bwd_fp8_block")
def _mm_swiglu_bwd_fp8_block_fake(grad_output, down_w_t, offs, aux_biased_acc, scale_a, scale_b, swiglu_alpha,
                                  swiglu_limit):
    return _out_fake(grad_output, 2 * down_w_t.size(2))


def grouped_mm_fp8_block(mat_a: torch.Tensor, mat_b: torch.Tensor, offs: torch.Tensor, scale_a: torch.Tensor,
                         scale_b: torch.Tensor, bias: torch.Tensor | None = None) -> torch.Tensor:
    """Ragged-M grouped product of block-scaled e4m3 operands (+ per-expert bf16 bias) -> bf16 [total_M, N].

    mat_a e4m3 [total_M, K] row-major and mat_b e4m3 [E, K, N] with unit stride along N or K (rows 16 bytes
    apart), scale_a fp32 [total_M, ceil(K / 128)], scale_b fp32 [E, ceil(K / 128), ceil(N / 128)] (any strides),
    offs int32 [E] cumulative row ends, N a multiple of 8.  Rows behind offs[-1] are not written.
    """
    refuse_tangents("grouped_mm_fp8_block", scale_a, scale_b, bias)
    with timed("fp8_block_mm"):
        return torch.ops.grouped_mm.mm_fp8_block.default(mat_a, mat_b, offs, scale_a, scale_b, bias)


def grouped_mm_swiglu_fp8_block(mat_a: torch.Tensor, mat_b: torch.Tensor, offs: torch.Tensor, scale_a: torch.Tensor,
                                scale_b: torch.Tensor, bias: torch.Tensor, swiglu_alpha: float = 1.702,
                                swiglu_limit: float = 7.0) -> tuple[torch.Tensor, torch.Tensor]:
    """The product + bias + clamped SwiGLU -> (swiglu_out [total_M, I], aux_biased_acc [total_M, 2I]), the
    activation computed from the stored (bf16) aux; mat_b's columns interleave gate and up."""
    refuse_tangents("grouped_mm_swiglu_fp8_block", scale_a, scale_b, bias)
    with timed("fp8_block_up_swiglu_fwd"):
        return torch.ops.grouped_mm.mm_swiglu_fp8_block.default(mat_a, mat_b, offs, scale_a, scale_b, bias, swiglu_alpha,
                                                        swiglu_limit)


def grouped_mm_swiglu_bwd_fp8_block(grad_output: torch.Tensor, down_w_t: torch.Tensor, offs: torch.Tensor,
                                    aux_biased_acc: torch.Tensor, scale_a: torch.Tensor, scale_b: torch.Tensor,
                                    swiglu_alpha: float = 1.702, swiglu_limit: float = 7.0) -> torch.Tensor:
    """SwiGLU backward of the product grad_output @ down_w_t against aux -> grad_aux bf16 [total_M, 2I]
    (interleaved like aux)."""
    refuse_tangents("grouped_mm_swiglu_bwd_fp8_block", aux_biased_acc, scale_a, scale_b)
    with timed("fp8_block_down_dgrad_swiglu_bwd"):
        return torch.ops.grouped_mm.mm_swiglu_bwd_fp8_block.default(grad_output, down_w_t, offs, aux_biased_acc, scale_a,
                                                            scale_b, swiglu_alpha, swiglu_limit)


class _FFNFp8Block(torch.autograd.Function):
    """The MoE FFN with block-scaled e4m3 products and input gradients, bf16 weight gradients."""

    @staticmethod
    def forward(ctx, x, w_up, b_up, w_down, b_down, offs, alpha, limit, up_codes, down_codes):
        q_up, s_up = up_codes if up_codes is not None else quantize_weights_block(w_up)
        q_down, s_down = down_codes if down_codes is not None else quantize_weights_block(w_down)
        qx, sx = quantize_rows_block(x)
        s, aux = grouped_mm_swiglu_fp8_block(qx, q_up, offs, sx, s_up, b_up, alpha, limit)
        qs, ss = quantize_rows_block(s)
        out = grouped_mm_fp8_block(qs, q_down, offs, ss, s_down, b_down)
        ctx.save_for_backward(x, s, aux, offs, q_up, s_up, q_down, s_down)
        ctx.alpha, ctx.limit, ctx.has_b_down = alpha, limit, b_down is not None
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        x, s, aux, offs, q_up, s_up, q_down, s_down = ctx.saved_tensors
        g = g.contiguous()
        g_x = g_wu = g_bu = g_wd = g_bd = None
        if ctx.needs_input_grad[3] or ctx.needs_input_grad[4]:
            with timed("down_wgrad_bias"):
                g_wd, g_bd = torch.ops.grouped_mm.mm_wgrad_bias(s.transpose(-2, -1), g, offs)
        if any(ctx.needs_input_grad[:3]):
            qg, sg = quantize_rows_block(g)
            grad_aux = grouped_mm_swiglu_bwd_fp8_block(qg, q_down.transpose(1, 2), offs, aux, sg,
                                                       s_down.transpose(1, 2), ctx.alpha, ctx.limit)
            if ctx.needs_input_grad[0]:
                qa, sa = quantize_rows_block(grad_aux)
                g_x = grouped_mm_fp8_block(qa, q_up.transpose(1, 2), offs, sa, s_up.transpose(1, 2))
            if ctx.needs_input_grad[1] or ctx.needs_input_grad[2]:
                with timed("up_wgrad_bias"):
                    g_wu, g_bu = torch.ops.grouped_mm.mm_wgrad_bias(x.transpose(-2, -1), grad_aux, offs)
        return g_x, g_wu, g_bu, g_wd, g_bd if ctx.has_b_down else None, None, None, None, None, None


def grouped_mm_ffn_fp8_block(x: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, offs: torch.Tensor,
                             b_up: torch.Tensor, b_down: torch.Tensor | None = None, swiglu_alpha: float = 1.702,
                             swiglu_limit: float = 7.0, up_codes: tuple[torch.Tensor, torch.Tensor] | None = None,
                             down_codes: tuple[torch.Tensor, torch.Tensor] | None = None) -> torch.Tensor:
    """The MoE expert FFN of ``grouped_mm_ffn`` with block-scaled e4m3 forward products and input gradients;
    bf16 inputs, parameters, output and gradients.  ``up_codes`` / ``down_codes``: the weights'
    ``quantize_weights_block`` kept by the caller between optimizer steps (or for inference); quantised in
    the call where absent.  The rows behind offs[-1] of the output (and of x's gradient) are not written."""
    return _FFNFp8Block.apply(x, w_up, b_up, w_down, b_down, offs, swiglu_alpha, swiglu_limit, up_codes, down_codes)

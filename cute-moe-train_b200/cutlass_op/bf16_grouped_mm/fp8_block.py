"""e4m3 with a scale for each block of 128: quantisers.

The recipe of :mod:`fp8` gives a whole row or column one scale, so one outlier costs all of it its small
values.  Here every 1 x 128 block of an activation row and every 128 x 128 block of a weight has its own.
The scales are powers of two (the smallest s with amax / s <= 448), so quantising rounds only once, in the
code; the grouped product takes any fp32 scales.  The weights' codes keep the weights' layout: one set is
the forward's operand and, transposed, the input gradient's.
"""

from __future__ import annotations

import torch

from . import _ext  # noqa: F401  (registers the operators)
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
    with timed("fp8_quantize"):
        return torch.ops.grouped_mm.fp8_quantize_rows_block(x.detach())


def quantize_weights_block(w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """bf16 [E, K, N] (unit stride along N or along K) -> (e4m3 [E, K, N] in the same layout, fp32
    [E, ceil(K / 128), ceil(N / 128)]): w[e, k, n] ~= q[e, k, n] * scale[e, k // 128, n // 128].
    ``q.transpose(1, 2), scale.transpose(1, 2)`` are the codes of ``w.transpose(1, 2)``."""
    with timed("fp8_quantize"):
        return torch.ops.grouped_mm.fp8_quantize_weights_block(w.detach())


def dequantize_rows_block(q: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    return q.float() * scale.repeat_interleave(BLOCK, 1)[:, :q.shape[1]]


def dequantize_weights_block(q: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    s = scale.repeat_interleave(BLOCK, 1)[:, :q.shape[1]].repeat_interleave(BLOCK, 2)[:, :, :q.shape[2]]
    return q.float() * s

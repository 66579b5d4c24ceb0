"""Forward-mode derivatives are refused: a tangent must never be lost without an error (shape inference only, no GPU)."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad


def _meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


def _refused(f, x):
    """`f` refuses a dual tensor (with and without requires_grad) and torch.func.jvp, and takes the plain one."""
    for grad in (False, True):
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(x.clone().requires_grad_(grad), torch.empty_like(x))
            with pytest.raises((RuntimeError, NotImplementedError)):
                f(dual)
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(f, (x,), (torch.empty_like(x),))
    f(x)
    with forward_ad.dual_level():
        f(x)  # a level without a tangent on this input


def _plan():
    from cutlass_op.bf16_grouped_mm.permute import moe_sort

    return moe_sort(_meta(10, 4, dtype=torch.int64), 8)


def _ffn():
    return [_meta(8, 128, 256), _meta(8, 128, 128), _meta(8, 256), _meta(8, 128)]


def test_router_and_permutation():
    from cutlass_op.bf16_grouped_mm.permute import moe_permute, moe_permute_fp8, moe_unpermute
    from cutlass_op.bf16_grouped_mm.routing import moe_route

    plan = _plan()
    _refused(lambda t: moe_route(t, 4)[0], _meta(10, 8, dtype=torch.float32))
    _refused(lambda t: moe_permute(t, _meta(10, 4, dtype=torch.int64), 8)[0], _meta(10, 64))
    _refused(lambda t: moe_permute(t, plan=plan)[0], _meta(10, 64))
    _refused(lambda t: moe_permute_fp8(t, plan=plan)[1], _meta(10, 64))
    _refused(lambda t: moe_unpermute(t, plan), _meta(40, 64))
    _refused(lambda t: moe_unpermute(_meta(40, 64), plan, t), _meta(10, 4, dtype=torch.float32))


def test_block_scaled_products():
    from cutlass_op.bf16_grouped_mm import fp8_block as f

    _refused(lambda t: f.quantize_rows_block(t)[1], _meta(10, 128))
    _refused(lambda t: f.quantize_weights_block(t)[1], _meta(2, 128, 128))
    e4m3 = torch.float8_e4m3fn
    a = (_meta(10, 128, dtype=e4m3), _meta(2, 128, 256, dtype=e4m3), _meta(2, dtype=torch.int32))
    s = (_meta(10, 1, dtype=torch.float32), _meta(2, 1, 2, dtype=torch.float32))
    _refused(lambda t: f.grouped_mm_fp8_block(*a, *s, t), _meta(2, 256))
    _refused(lambda t: f.grouped_mm_fp8_block(*a, t, s[1]), s[0])
    _refused(lambda t: f.grouped_mm_swiglu_fp8_block(*a, *s, t)[0], _meta(2, 256))
    _refused(lambda t: f.grouped_mm_swiglu_bwd_fp8_block(*a, t, *s), _meta(10, 512))


@pytest.mark.parametrize("precision", ["bf16", "fp8_block"])
def test_moe_block(precision):
    from cutlass_op.bf16_grouped_mm.moe import moe_ffn

    w = _ffn()
    logits = _meta(10, 8, dtype=torch.float32)
    _refused(lambda t: moe_ffn(t, logits, 2, *w, precision=precision), _meta(10, 128))
    _refused(lambda t: moe_ffn(_meta(10, 128), t, 2, *w, precision=precision), logits)
    for i, t in enumerate(w):
        _refused(lambda t, i=i: moe_ffn(_meta(10, 128), logits, 2, *w[:i], t, *w[i + 1:], precision=precision), t)


def test_bf16_and_row_scaled_products():
    import cutlass_op.bf16_grouped_mm as m
    from cutlass_op.bf16_grouped_mm import fp8

    offs = _meta(2, dtype=torch.int32)
    x, w, b, aux = _meta(10, 128), _meta(2, 128, 256), _meta(2, 256), _meta(10, 512)
    _refused(lambda t: m.grouped_mm(t, w, offs, b), x)
    _refused(lambda t: m.grouped_mm(x, t, offs, b), w)
    _refused(lambda t: m.grouped_mm(x, w, offs, t), b)
    _refused(lambda t: m.grouped_mm_swiglu(t, w, offs, b)[0], x)
    _refused(lambda t: m.grouped_mm_swiglu(x, t, offs, b)[0], w)
    _refused(lambda t: m.grouped_mm_swiglu(x, w, offs, t)[0], b)
    _refused(lambda t: m.grouped_mm_downproj(t, w, offs, b, aux), x)
    _refused(lambda t: m.grouped_mm_downproj(x, t, offs, b, aux), w)
    _refused(lambda t: m.grouped_mm_downproj(x, w, offs, t, aux), b)
    _refused(lambda t: m.grouped_mm_downproj(x, w, offs, b, t), aux)
    e4m3, f32 = torch.float8_e4m3fn, torch.float32
    a = (_meta(10, 128, dtype=e4m3), _meta(2, 256, 128, dtype=e4m3).transpose(1, 2), offs)
    s = (_meta(10, dtype=f32), _meta(2, 256, dtype=f32))
    _refused(lambda t: fp8.grouped_mm_fp8(*a, *s, t), b)
    _refused(lambda t: fp8.grouped_mm_fp8(*a, t, s[1]), s[0])
    _refused(lambda t: fp8.grouped_mm_swiglu_fp8(*a, *s, t)[0], b)
    _refused(lambda t: fp8.grouped_mm_swiglu_bwd_fp8(*a, t, *s), aux)

"""NaN through the products' SwiGLU epilogues: what is not a number on the way in is none on the way out, and
nothing else changes.

The clamps of the formula keep NaN (as ``torch.clamp`` does): the activation of a NaN gate or up is NaN.  The
gradients are those of the formula too: the clamped range's derivative is 0, and a NaN input lies outside the
unclamped range, so its own gradient is 0 while it makes the other one's NaN; a NaN accumulator makes NaN wherever
the input is not clamped.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

ALPHA, LIMIT = 1.702, 7.0


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _same_but_for_nan(got, clean, nan):
    """`got` is NaN exactly where `nan` says and bit for bit `clean` everywhere else."""
    assert torch.equal(got.isnan(), nan), f"{int(got.isnan().sum())} NaN, expected {int(nan.sum())}"
    assert torch.equal(got[~nan], clean[~nan])


def _pairs(gate, up):
    return torch.stack([gate, up], 2).flatten(1)


def _spoilt(aux):
    """`aux` with a NaN gate, a NaN up and a pair of both; (aux, NaN gates, NaN ups)."""
    out = aux.clone()
    out[3, 0], out[5, 3], out[8, 10], out[8, 11] = math.nan, math.nan, math.nan, math.nan
    return out, out[:, 0::2].isnan(), out[:, 1::2].isnan()


FORMS = [("0", "1", "256"), ("0", "2", "256"), ("0", "1", "128"), ("1", "1", "256"), ("1", "2", "256")]


@pytest.mark.parametrize("mx,cg,bn", FORMS)
def test_block_scaled_swiglu_keeps_nan(mx, cg, bn, monkeypatch):
    from cutlass_op.bf16_grouped_mm import fp8_block

    for name, value in (("MGF_BLOCK_MX", mx), ("MGF_CTA_GROUP", cg), ("MGF_BN", bn)):
        monkeypatch.setenv(name, value)
    g = _gen(1)
    E, K, N, rows = 2, 320, 272, 150
    x = _randn(g, rows, K).to(torch.bfloat16)
    w = (_randn(g, E, K, N) / math.sqrt(K)).to(torch.bfloat16)
    bias = (0.1 * _randn(g, E, N)).to(torch.bfloat16)
    offs = torch.tensor([70, rows], dtype=torch.int32, device="cuda")
    qb, sb = fp8_block.quantize_weights_block(w)
    f = fp8_block.grouped_mm_swiglu_fp8_block
    qa, sa = fp8_block.quantize_rows_block(x)
    s0, aux0 = f(qa, qb, offs, sa, sb, bias, ALPHA, LIMIT)
    assert not s0.isnan().any() and not aux0.isnan().any()
    x[7, 300] = math.nan
    x[100, 5] = math.inf  # a NaN code too
    na, nsa = fp8_block.quantize_rows_block(x)
    bad = torch.zeros(rows, dtype=torch.bool, device="cuda")
    bad[[7, 100]] = True
    s, aux = f(na, qb, offs, nsa, sb, bias, ALPHA, LIMIT)
    _same_but_for_nan(aux, aux0, bad[:, None].expand(rows, N))
    _same_but_for_nan(s, s0, bad[:, None].expand(rows, N // 2))
    # a NaN gate, a NaN up (of one group's bias): the activation of that pair alone
    b = bias.clone()
    b[0, 6], b[1, 9] = math.nan, math.nan
    nan = torch.zeros(rows, N // 2, dtype=torch.bool, device="cuda")
    nan[:70, 3], nan[70:, 4] = True, True
    _same_but_for_nan(f(qa, qb, offs, sa, sb, b, ALPHA, LIMIT)[0], s0, nan)


@pytest.mark.parametrize("mx,cg,bn", FORMS)
def test_block_scaled_swiglu_backward_keeps_nan(mx, cg, bn, monkeypatch):
    from cutlass_op.bf16_grouped_mm import fp8_block

    for name, value in (("MGF_BLOCK_MX", mx), ("MGF_CTA_GROUP", cg), ("MGF_BN", bn)):
        monkeypatch.setenv(name, value)
    g = _gen(2)
    E, K, I, rows = 2, 320, 272, 150
    grad = _randn(g, rows, K).to(torch.bfloat16)
    w = (_randn(g, E, K, I) / math.sqrt(K)).to(torch.bfloat16)
    aux = (4 * _randn(g, rows, 2 * I)).to(torch.bfloat16)
    offs = torch.tensor([70, rows], dtype=torch.int32, device="cuda")
    qb, sb = fp8_block.quantize_weights_block(w)
    f = fp8_block.grouped_mm_swiglu_bwd_fp8_block
    qa, sa = fp8_block.quantize_rows_block(grad)
    clean = f(qa, qb, offs, aux, sa, sb, ALPHA, LIMIT)
    assert not clean.isnan().any()
    gate, up = aux[:, 0::2].float(), aux[:, 1::2].float()
    grad[9, 17] = math.nan
    na, nsa = fp8_block.quantize_rows_block(grad)
    nan = torch.zeros_like(aux, dtype=torch.bool)
    nan[9] = _pairs(gate <= LIMIT, up.abs() <= LIMIT)[9]
    assert nan[9].any() and not nan[9].all()
    _same_but_for_nan(f(na, qb, offs, aux, nsa, sb, ALPHA, LIMIT), clean, nan)
    bad, ng, nu = _spoilt(aux)
    want = clean.clone()
    want[:, 0::2][ng], want[:, 1::2][nu] = 0.0, 0.0
    nan = _pairs(nu & (gate <= LIMIT) & ~ng, ng & (up.abs() <= LIMIT) & ~nu)
    assert nan.any()
    _same_but_for_nan(f(qa, qb, offs, bad, sa, sb, ALPHA, LIMIT), want, nan)


def test_block_scaled_moe_ffn_keeps_the_nan_of_a_token():
    _moe_ffn_keeps_nan("fp8_block")


def _moe_ffn_keeps_nan(precision):
    from cutlass_op.bf16_grouped_mm.moe import moe_ffn

    g = _gen(3)
    T, E, H, I = 40, 4, 128, 64
    x = _randn(g, T, H).to(torch.bfloat16)
    logits = _randn(g, T, E)
    w = [t.to(torch.bfloat16) for t in (_randn(g, E, H, 2 * I) / math.sqrt(H), _randn(g, E, I, H) / math.sqrt(I),
                                        0.1 * _randn(g, E, 2 * I), 0.1 * _randn(g, E, H))]
    clean = moe_ffn(x, logits, 2, *w, precision=precision)
    bad = x.clone()
    bad[11, 3] = math.nan
    nan = torch.zeros_like(clean, dtype=torch.bool)
    nan[11] = True
    _same_but_for_nan(moe_ffn(bad, logits, 2, *w, precision=precision), clean, nan)
    leaf = bad.clone().requires_grad_(True)
    _same_but_for_nan(moe_ffn(leaf, logits, 2, *w, precision=precision).detach(), clean, nan)


# ------------------------------------------------------------------------------------------------ bf16, e4m3 with row scales
def test_bf16_moe_ffn_keeps_the_nan_of_a_token():
    _moe_ffn_keeps_nan("bf16")


@pytest.mark.parametrize("rows,cg", [(150, "1"), (150, "2")])
@pytest.mark.parametrize("store_aux", [True, False])
def test_bf16_swiglu_keeps_nan(rows, cg, store_aux, monkeypatch):
    from cutlass_op.bf16_grouped_mm import grouped_mm_swiglu

    monkeypatch.setenv("MGF_CTA_GROUP", cg)
    g = _gen(4)
    E, K, N = 2, 320, 272
    x = _randn(g, rows, K).to(torch.bfloat16)
    w = (_randn(g, E, K, N) / math.sqrt(K)).to(torch.bfloat16)
    bias = (0.1 * _randn(g, E, N)).to(torch.bfloat16)
    offs = torch.tensor([70, rows], dtype=torch.int32, device="cuda")

    def f(x, bias):
        if store_aux:
            return grouped_mm_swiglu(x, w, offs, bias)[0]
        return torch.ops.grouped_mm.mm_swiglu_noaux(x, w, offs, bias, ALPHA, LIMIT)

    s0 = f(x, bias)
    assert not s0.isnan().any()
    bad = x.clone()
    bad[7, 300] = math.nan
    nan = torch.zeros(rows, N // 2, dtype=torch.bool, device="cuda")
    nan[7] = True
    _same_but_for_nan(f(bad, bias), s0, nan)
    b = bias.clone()
    b[0, 6], b[1, 9] = math.nan, math.nan
    nan = torch.zeros(rows, N // 2, dtype=torch.bool, device="cuda")
    nan[:70, 3], nan[70:, 4] = True, True
    _same_but_for_nan(f(x, b), s0, nan)


@pytest.mark.parametrize("e4m3", [False, True])
@pytest.mark.parametrize("cg", ["1", "2"])
def test_swiglu_backward_keeps_nan(cg, e4m3, monkeypatch):
    from cutlass_op.bf16_grouped_mm import fp8

    monkeypatch.setenv("MGF_CTA_GROUP", cg)
    g = _gen(5)
    E, K, I, rows = 2, 320, 272, 150
    grad = _randn(g, rows, K).to(torch.bfloat16)
    w = (_randn(g, E, K, I) / math.sqrt(K)).to(torch.bfloat16)
    aux = (4 * _randn(g, rows, 2 * I)).to(torch.bfloat16)
    offs = torch.tensor([70, rows], dtype=torch.int32, device="cuda")
    if e4m3:
        (qg, sg), (qw, sw) = fp8.quantize_rows(grad), fp8.quantize_weights(w)

        def f(aux):
            return fp8.grouped_mm_swiglu_bwd_fp8(qg, qw, offs, aux, sg, sw, ALPHA, LIMIT)
    else:
        def f(aux):
            return torch.ops.grouped_mm.mm_swiglu_bwd(grad, w, offs, aux, ALPHA, LIMIT)
    clean = f(aux)
    assert not clean.isnan().any()
    gate, up = aux[:, 0::2].float(), aux[:, 1::2].float()
    bad, ng, nu = _spoilt(aux)
    want = clean.clone()
    want[:, 0::2][ng], want[:, 1::2][nu] = 0.0, 0.0
    nan = _pairs(nu & (gate <= LIMIT) & ~ng, ng & (up.abs() <= LIMIT) & ~nu)
    _same_but_for_nan(f(bad), want, nan)


def test_e4m3_row_scaled_swiglu_keeps_nan():
    from cutlass_op.bf16_grouped_mm import fp8

    g = _gen(6)
    E, K, N, rows = 2, 320, 272, 150
    x = _randn(g, rows, K).to(torch.bfloat16)
    w = (_randn(g, E, K, N) / math.sqrt(K)).to(torch.bfloat16)
    bias = (0.1 * _randn(g, E, N)).to(torch.bfloat16)
    offs = torch.tensor([70, rows], dtype=torch.int32, device="cuda")
    (qx, sx), (qw, sw) = fp8.quantize_rows(x), fp8.quantize_weights(w)
    s0, _ = fp8.grouped_mm_swiglu_fp8(qx, qw, offs, sx, sw, bias, ALPHA, LIMIT)
    bias[1, 8] = math.nan
    nan = torch.zeros(rows, N // 2, dtype=torch.bool, device="cuda")
    nan[70:, 4] = True
    _same_but_for_nan(fp8.grouped_mm_swiglu_fp8(qx, qw, offs, sx, sw, bias, ALPHA, LIMIT)[0], s0, nan)

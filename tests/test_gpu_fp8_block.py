"""e4m3 with a scale per block of 128: quantisers against their definition (bit for bit)."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _scale_ref(amax):
    """Smallest power of two (not below 2^-126) with amax / s <= 448, 1 where amax is 0, in 64 bits."""
    a = amax.double()
    s = torch.full_like(a, 2.0 ** -126)
    for _ in range(256):
        s = torch.where(a > 448 * s, 2 * s, s)
    return torch.where(a > 0, s, torch.ones_like(s))


def _code_ref(v, s):
    """e4m3 values of v / s: four significant bits, steps of 2^-9 below 2^-6, ties to even, NaN kept."""
    t = v.double() / s
    t = torch.where(torch.isfinite(t), t, torch.full_like(t, math.nan))
    step = torch.exp2(torch.floor(torch.log2(t.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(t / step) * step


def _rows_ref(x):
    m, k = x.shape
    nb = -(-k // 128)
    full = torch.zeros(m, nb * 128, dtype=torch.float64, device=x.device)
    full[:, :k] = x.double()
    b = full.view(m, nb, 128)
    s = _scale_ref(torch.where(torch.isfinite(b), b, 0.0).abs().amax(2))
    return _code_ref(b, s[:, :, None]).reshape(m, -1)[:, :k], s


def _weights_ref(w):
    e, k, n = w.shape
    kb, nb = -(-k // 128), -(-n // 128)
    full = torch.zeros(e, kb * 128, nb * 128, dtype=torch.float64, device=w.device)
    full[:, :k, :n] = w.double()
    b = full.view(e, kb, 128, nb, 128)
    s = _scale_ref(torch.where(torch.isfinite(b), b, 0.0).abs().amax((2, 4)))
    return _code_ref(b, s[:, :, None, :, None]).reshape(e, kb * 128, nb * 128)[:, :k, :n], s


def _same(q, ref):
    q = q.double()
    assert torch.equal(q.isnan(), ref.isnan())
    assert torch.equal(q[~q.isnan()], ref[~ref.isnan()])


def _special(x):
    """Rows with the values that a scale can go wrong at."""
    v = [0.0, -0.0, 448.0, 449.0, 1.75, 1.7578125, 2.0 ** -126, 2.0 ** -133, 3.3e38, -3.3e38]
    for i, c in enumerate(v[:x.shape[0]]):
        x[i] = 0
        x[i, x.shape[1] // 2] = c
        x[i, 0] = c / 3
    return x


@pytest.mark.parametrize("M,K", [(0, 128), (1, 1), (1, 128), (12, 129), (33, 2880), (7, 7168), (300, 520), (64, 15)])
def test_row_blocks(M, K):
    from cutlass_op.bf16_grouped_mm import fp8_block

    x = torch.randn(M, K, generator=_gen(M + K), device="cuda") * torch.logspace(-6, 6, K, device="cuda")
    x = _special(x.to(torch.bfloat16))
    q, s = fp8_block.quantize_rows_block(x)
    assert q.stride(0) % 16 == 0 and s.stride(0) % 4 == 0 and s.shape == (M, -(-K // 128))
    ref_q, ref_s = _rows_ref(x)
    assert torch.equal(s.double(), ref_s)
    _same(q, ref_q)
    # columns of a wider matrix that start off a 16-byte boundary
    wide = torch.randn(M, K + 9, generator=_gen(1), device="cuda").to(torch.bfloat16)
    q, s = fp8_block.quantize_rows_block(wide[:, 3:K + 3])
    ref_q, ref_s = _rows_ref(wide[:, 3:K + 3])
    assert torch.equal(s.double(), ref_s)
    _same(q, ref_q)


def test_non_finite_elements_become_nan_codes_alone():
    from cutlass_op.bf16_grouped_mm import fp8_block

    x = torch.randn(4, 256, generator=_gen(2), device="cuda").to(torch.bfloat16)
    clean_q, clean_s = fp8_block.quantize_rows_block(x)
    x[1, 5], x[2, 130], x[3, 200] = math.nan, math.inf, -math.inf
    ref_q, ref_s = _rows_ref(x)
    q, s = fp8_block.quantize_rows_block(x)
    assert torch.equal(s.double(), ref_s)
    _same(q, ref_q)
    assert torch.isnan(q.float()).sum() == 3 and torch.equal(q[0].float(), clean_q[0].float())
    w = x.view(1, 4, 256)
    q, s = fp8_block.quantize_weights_block(w)
    ref_q, ref_s = _weights_ref(w)
    assert torch.equal(s.double(), ref_s)
    _same(q, ref_q)


@pytest.mark.parametrize("E,K,N", [(1, 1, 1), (2, 128, 128), (3, 130, 257), (2, 2880, 320), (4, 64, 1000), (0, 8, 8)])
@pytest.mark.parametrize("layout", ["n", "k", "slice"])
def test_weight_blocks(E, K, N, layout):
    from cutlass_op.bf16_grouped_mm import fp8_block

    g = _gen(E + K + N)
    w = torch.randn(E, K, N + 5, generator=g, device="cuda") * torch.logspace(-4, 4, N + 5, device="cuda")
    w = w.to(torch.bfloat16)
    w = w[:, :, 2:N + 2] if layout == "slice" else w[:, :, :N].contiguous()
    if layout == "k":
        w = w.transpose(1, 2)
    q, s = fp8_block.quantize_weights_block(w)
    ref_q, ref_s = _weights_ref(w)
    assert q.shape == w.shape and torch.equal(s.double(), ref_s)
    _same(q, ref_q)
    if w.numel() > 1 and min(K, N) > 1:
        inner = 1 if layout == "k" else 2
        assert q.stride(inner) == 1 and q.stride(3 - inner) % 16 == 0
    back = fp8_block.dequantize_weights_block(q, s)
    assert ((back - w.float()).abs() <= 2.0 ** -4 * w.float().abs() + 2.0 ** -10 * s.amax((1, 2), keepdim=True)).all() \
        if w.numel() else True


@pytest.mark.parametrize("T,k,E,H,drop", [(1, 1, 1, 128, 0), (50, 4, 8, 2880, 0), (31, 8, 16, 136, 0.3), (9, 2, 4, 77, 0),
                                          (5, 3, 4, 256, 1.1)])
def test_permute_fp8_equals_quantised_rows(T, k, E, H, drop):
    import cutlass_op.bf16_grouped_mm as m
    from cutlass_op.bf16_grouped_mm import fp8_block
    from cutlass_op.bf16_grouped_mm.permute import moe_permute, moe_permute_fp8

    g = _gen(T + H)
    x = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
    idx = torch.randint(0, E, (T, k), generator=g, device="cuda")
    idx = torch.where(torch.rand(T, k, generator=g, device="cuda") < drop, torch.full_like(idx, -1), idx)
    rows, plan = moe_permute(x, idx, E)
    q, s, p = moe_permute_fp8(x, idx, E)
    assert all(torch.equal(a, b) for a, b in zip(plan, p))
    kept = int(plan.offs[-1])
    ref_q, ref_s = fp8_block.quantize_rows_block(rows)
    assert torch.equal(q[:kept].view(torch.uint8), ref_q[:kept].view(torch.uint8)) and torch.equal(s[:kept], ref_s[:kept])
    assert (q[kept:].float() == 0).all() and (s[kept:] == 0).all()
    again = moe_permute_fp8(x, plan=plan)
    assert torch.equal(again[0].view(torch.uint8), q.view(torch.uint8)) and torch.equal(again[1], s)
    m.check_device_status()


def test_quantiser_refusals():
    from cutlass_op.bf16_grouped_mm import fp8_block

    with pytest.raises(RuntimeError, match="BFloat16"):
        fp8_block.quantize_rows_block(torch.zeros(2, 128, device="cuda"))
    with pytest.raises(RuntimeError, match="unit stride"):
        fp8_block.quantize_rows_block(torch.zeros(128, 2, device="cuda", dtype=torch.bfloat16).t())
    with pytest.raises(RuntimeError, match="unit stride"):
        fp8_block.quantize_weights_block(torch.zeros(2, 8, 8, 2, device="cuda", dtype=torch.bfloat16)[..., 0])
    with pytest.raises(RuntimeError, match="bf16"):
        fp8_block.quantize_weights_block(torch.zeros(8, 8, device="cuda", dtype=torch.bfloat16))

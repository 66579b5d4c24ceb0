"""Tensors of more than 2^31 elements: the last rows of a long batch are where 32-bit offsets would go wrong."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

T, H = 300_032, 7168  # 2.15e9 elements


@pytest.fixture(autouse=True)
def _memory_back():
    yield
    torch.cuda.empty_cache()


def _rows(seed, cols=H):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.empty(T, cols, dtype=torch.bfloat16, device="cuda")
    block = torch.randn(4096, cols, generator=g, device="cuda").to(torch.bfloat16)
    for i in range(0, T, 4096):  # each stretch of rows differs from the others by a factor
        n = min(4096, T - i)
        x[i:i + n] = block[:n] * (1 + i // 4096 % 7)
    return x


def test_permute_unpermute_and_quantise():
    from cutlass_op.bf16_grouped_mm.fp8_block import quantize_rows_block
    from cutlass_op.bf16_grouped_mm.permute import moe_permute, moe_permute_fp8, moe_unpermute

    x = _rows(1)
    idx = torch.randint(0, 16, (T, 1), generator=torch.Generator(device="cuda").manual_seed(2), device="cuda")
    rows, plan = moe_permute(x, idx, 16)
    probe = torch.cat([torch.arange(64), torch.arange(T - 4096, T, 37)]).cuda()
    at = plan.row_of_copy.flatten().long()[probe]
    assert torch.equal(rows[at], x[probe])
    assert int(plan.row_of_copy.max()) == T - 1 and torch.equal(rows[-1], x[plan.copy_of_row[-1].long()])
    q, s, _ = moe_permute_fp8(x, plan=plan)
    ref_q, ref_s = quantize_rows_block(x[probe])
    assert torch.equal(q.view(torch.uint8)[at], ref_q.view(torch.uint8)) and torch.equal(s[at], ref_s)
    del q, s
    out = moe_unpermute(rows, plan, torch.full((T, 1), 2.0, device="cuda"))
    assert torch.equal(out[probe], 2 * x[probe])
    del out
    q, s = quantize_rows_block(x)
    assert torch.equal(q.view(torch.uint8)[probe], ref_q.view(torch.uint8)) and torch.equal(s[probe], ref_s)


@pytest.mark.parametrize("mx", ["0", "1"])
def test_products(mx, monkeypatch):
    from cutlass_op.bf16_grouped_mm import fp8_block

    monkeypatch.setenv("MGF_BLOCK_MX", mx)
    x = _rows(3, 128)
    g = torch.Generator(device="cuda").manual_seed(4)
    w = torch.randn(2, 128, H, generator=g, device="cuda").to(torch.bfloat16)
    bias = torch.randn(2, H, generator=g, device="cuda").to(torch.bfloat16)
    qx, sx = fp8_block.quantize_rows_block(x)
    qw, sw = fp8_block.quantize_weights_block(w)
    last = 517
    offs = torch.tensor([T - last, T], dtype=torch.int32, device="cuda")
    few = torch.tensor([0, last], dtype=torch.int32, device="cuda")
    tail = (qx[-last:], qw, few, sx[-last:])
    s, aux = fp8_block.grouped_mm_swiglu_fp8_block(qx, qw, offs, sx, sw, bias)
    s1, aux1 = fp8_block.grouped_mm_swiglu_fp8_block(*tail, sw, bias)
    assert torch.equal(aux[-last:], aux1) and torch.equal(s[-last:], s1)
    del s
    half = qw[:, :, :H // 2], sw[:, :, :H // 256]
    d = fp8_block.grouped_mm_swiglu_bwd_fp8_block(qx, half[0], offs, aux, sx, half[1])
    d1 = fp8_block.grouped_mm_swiglu_bwd_fp8_block(qx[-last:], half[0], few, aux1, sx[-last:], half[1])
    assert torch.equal(d[-last:], d1)


def test_router():
    from cutlass_op.bf16_grouped_mm.routing import moe_route

    E, n = 1024, 2_100_000
    g = torch.Generator(device="cuda").manual_seed(5)
    tail = torch.randn(300, E, generator=g, device="cuda").to(torch.bfloat16)
    logits = torch.zeros(n, E, dtype=torch.bfloat16, device="cuda")
    logits[-300:] = tail
    logits.requires_grad_(True)
    w, idx = moe_route(logits, 4)
    w1, idx1 = moe_route(tail.requires_grad_(True), 4)
    assert torch.equal(w[-300:], w1) and torch.equal(idx[-300:], idx1) and idx[0].tolist() == [0, 1, 2, 3]
    gw = torch.randn(n, 4, generator=g, device="cuda")
    (dl,) = torch.autograd.grad(w, logits, gw)
    (dl1,) = torch.autograd.grad(w1, tail, gw[-300:])
    assert torch.equal(dl[-300:], dl1)

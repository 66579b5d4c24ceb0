"""Kernels that stop early with copies in flight: they let them land, report and leave the device usable.

The launcher's test hook MGF_TEST_STALL_PRODUCER=2 loads but multiplies nothing: every stage is filled, every wait behind
that gives up after 1.5 s, and the copies' barriers are then waited for.  MGF_DEV_DRAIN_TIMEOUT would say that a wait
for them had run out.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _case(rows=700, E=2, K=1400, N=528):
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn(rows, K, generator=g, device="cuda").to(torch.bfloat16)
    w = (torch.randn(E, K, N, generator=g, device="cuda") / math.sqrt(K)).to(torch.bfloat16)
    return x, w, torch.tensor([300, rows], dtype=torch.int32, device="cuda")


def _stalls_and_recovers(f, monkeypatch):
    from cutlass_op.bf16_grouped_mm._ext import DEV_WAIT_TIMEOUT, device_status

    device_status()
    want = f()
    assert device_status() == 0
    monkeypatch.setenv("MGF_TEST_STALL_PRODUCER", "2")
    f()
    assert device_status() == DEV_WAIT_TIMEOUT
    monkeypatch.delenv("MGF_TEST_STALL_PRODUCER")
    for a, b in zip(f(), want):
        assert torch.equal(a, b)
    assert device_status() == 0


@pytest.mark.parametrize("mx,cg,bn", [("0", "1", "256"), ("0", "2", "256"), ("0", "1", "128"), ("1", "1", "256"),
                                      ("1", "2", "256")])
@pytest.mark.parametrize("layout", ["kn", "nk"])
def test_block_scaled_products(mx, cg, bn, layout, monkeypatch):
    from cutlass_op.bf16_grouped_mm import fp8_block

    for name, value in (("MGF_BLOCK_MX", mx), ("MGF_CTA_GROUP", cg), ("MGF_BN", bn)):
        monkeypatch.setenv(name, value)
    x, w, offs = _case()
    if layout == "nk":
        w = w.transpose(1, 2).contiguous().transpose(1, 2)
    qa, sa = fp8_block.quantize_rows_block(x)
    qb, sb = fp8_block.quantize_weights_block(w)
    _stalls_and_recovers(lambda: [fp8_block.grouped_mm_fp8_block(qa, qb, offs, sa, sb)], monkeypatch)


@pytest.mark.parametrize("cg", ["1", "2"])
@pytest.mark.parametrize("what", ["mm", "mm_nk", "swiglu", "fp8", "wgrad", "wgrad_short", "wgrad_fp8"])
def test_bf16_and_row_scaled_products(what, cg, monkeypatch):
    import cutlass_op.bf16_grouped_mm as m
    from cutlass_op.bf16_grouped_mm import fp8

    monkeypatch.setenv("MGF_CTA_GROUP", cg)
    x, w, offs = _case()
    g = torch.randn(700, 528, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(torch.bfloat16)
    if what == "mm":
        f = lambda: [m.grouped_mm(x, w, offs)]  # noqa: E731
    elif what == "mm_nk":
        wt = w.transpose(1, 2).contiguous().transpose(1, 2)
        f = lambda: [m.grouped_mm(x, wt, offs)]  # noqa: E731
    elif what == "swiglu":
        f = lambda: m.grouped_mm_swiglu(x, w, offs, g[:2])  # noqa: E731
    elif what == "fp8":
        (qx, sx), (qw, sw) = fp8.quantize_rows(x), fp8.quantize_weights(w)
        f = lambda: [fp8.grouped_mm_fp8(qx, qw, offs, sx, sw)]  # noqa: E731
    elif what == "wgrad_fp8":
        (qx, sx), (qg, sg) = fp8.quantize_cols(x), fp8.quantize_cols(g)
        f = lambda: [t for t in fp8.grouped_mm_wgrad_fp8(qx, qg, offs, sx, sg) if t is not None]  # noqa: E731
    else:
        ends = offs if what == "wgrad" else torch.arange(10, 701, 10, dtype=torch.int32, device="cuda")
        f = lambda: torch.ops.grouped_mm.mm_wgrad_bias(x.transpose(0, 1), g, ends)  # noqa: E731
    _stalls_and_recovers(f, monkeypatch)

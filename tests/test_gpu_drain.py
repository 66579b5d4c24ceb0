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

"""Calls of the MoE block's operators next to their limits."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,k", [(1, 1), (5, 2), (300, 3)])
def test_gradients_of_rows_of_one_element_broadcast_over_the_tokens(T, k, dtype):
    """``out.sum()`` of [T, 1]: its gradient is one element seen T times (stride 0)."""
    from cutlass_op.bf16_grouped_mm.permute import moe_permute, moe_unpermute

    g = _gen(T)
    idx = torch.randint(0, 4, (T, k), generator=g, device="cuda")
    x = torch.randn(T, 1, generator=g, device="cuda").to(dtype).requires_grad_(True)
    rows, plan = moe_permute(x, idx, 4)
    rows.sum().backward()
    assert torch.equal(x.grad, torch.full_like(x.grad, k))
    y = rows.detach().clone().requires_grad_(True)
    w = torch.rand(T, k, generator=g, device="cuda").requires_grad_(True)
    moe_unpermute(y, plan, w).sum().backward()
    c = plan.copy_of_row.long()
    assert torch.equal(y.grad.flatten(), w.detach().flatten()[c].to(dtype))
    assert torch.equal(w.grad.flatten()[c], y.detach().flatten().float())


@pytest.mark.parametrize("sms_left", [1, 2, 3])
@pytest.mark.parametrize("rows", [1100, 3000])
def test_products_on_the_few_sms_that_a_carve_out_leaves(rows, sms_left, monkeypatch):
    from cutlass_op.bf16_grouped_mm import fp8_block

    monkeypatch.setenv("MGF_BLOCK_MX", "1")
    for name in ("MGF_CTA_GROUP", "MGF_BN"):
        monkeypatch.delenv(name, raising=False)
    g = _gen(rows)
    x = torch.randn(rows, 256, generator=g, device="cuda").to(torch.bfloat16)
    w = torch.randn(1, 256, 512, generator=g, device="cuda").to(torch.bfloat16)
    offs = torch.tensor([rows], dtype=torch.int32, device="cuda")
    qa, sa = fp8_block.quantize_rows_block(x)
    qb, sb = fp8_block.quantize_weights_block(w)
    want = fp8_block.grouped_mm_fp8_block(qa, qb, offs, sa, sb)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    torch._C._set_sm_carveout_experimental(sms - sms_left)
    try:
        got = fp8_block.grouped_mm_fp8_block(qa, qb, offs, sa, sb)
    finally:
        torch._C._set_sm_carveout_experimental(None)
    assert torch.equal(got, want)

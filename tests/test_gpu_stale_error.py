"""An error of an earlier runtime call is not reported as an operator's own."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _leave_an_error():
    """A call of the library's that the CUDA runtime refuses on the host: the address is no mapping of its."""
    from cutlass_op.bf16_grouped_mm import _ext

    assert _ext.lib.mgf_ipc_close(1 << 40) != 0


def _calls():
    import cutlass_op.bf16_grouped_mm as m
    from cutlass_op.bf16_grouped_mm import fp8, fp8_block, permute, routing

    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(64, 128, generator=g, device="cuda").to(torch.bfloat16)
    w = (torch.randn(4, 128, 256, generator=g, device="cuda") / math.sqrt(128)).to(torch.bfloat16)
    logits = torch.randn(64, 4, generator=g, device="cuda")
    offs = torch.tensor([10, 20, 50, 64], dtype=torch.int32, device="cuda")
    weights, idx = routing.moe_route(logits, 2)
    many = torch.randint(0, 4, (9000, 1), generator=g, device="cuda")
    rows, plan = permute.moe_permute(x, idx, 4)
    qa, sa = fp8_block.quantize_rows_block(x)
    qb, sb = fp8_block.quantize_weights_block(w)

    def grad(f, *leaves):
        leaves = [t.detach().clone().requires_grad_(True) for t in leaves]
        return torch.autograd.grad(f(*leaves).float().sum(), leaves)

    return {
        "moe_route": lambda: routing.moe_route(logits, 2),
        "moe_route_bwd": lambda: grad(lambda t: routing.moe_route(t, 2)[0], logits),
        "moe_sort": lambda: permute.moe_sort(idx, 4),
        "moe_sort many": lambda: permute.moe_sort(many, 4),
        "moe_permute": lambda: permute.moe_permute(x, idx, 4)[0],
        "moe_permute plan": lambda: permute.moe_permute(x, plan=plan)[0],
        "moe_unpermute": lambda: permute.moe_unpermute(rows, plan, weights),
        "moe_unpermute_bwd": lambda: grad(lambda r, t: permute.moe_unpermute(r, plan, t), rows, weights),
        "moe_permute_fp8": lambda: permute.moe_permute_fp8(x, plan=plan)[1],
        "quantize_rows_block": lambda: fp8_block.quantize_rows_block(x)[1],
        "quantize_weights_block": lambda: fp8_block.quantize_weights_block(w)[1],
        "grouped_mm_fp8_block": lambda: fp8_block.grouped_mm_fp8_block(qa, qb, offs, sa, sb),
        "grouped_mm": lambda: m.grouped_mm(x, w, offs),
        "quantize_rows": lambda: fp8.quantize_rows(x)[1],
        "quantize_rows_cols": lambda: fp8.quantize_rows_cols(x)[1],
        "quantize_cols": lambda: fp8.quantize_cols(x)[1],
        "quantize_weights": lambda: fp8.quantize_weights(w)[1],
        "quantize_weights_both": lambda: fp8.quantize_weights_both(w)[1],
        "gather_rows": lambda: torch.ops.grouped_mm.gather_rows(x, idx.flatten(), None),
        "combine_rows": lambda: torch.ops.grouped_mm.combine_rows(x, idx.flatten(), weights.flatten(), 2),
        "ep_sort": lambda: torch.ops.grouped_mm.ep_sort(idx.flatten(), 4, 2),
    }


def _flat(out):
    return [out] if isinstance(out, torch.Tensor) else list(out)


@pytest.mark.parametrize("mx", ["0", "1"])
def test_operators_after_a_refused_call(mx, monkeypatch):
    monkeypatch.setenv("MGF_BLOCK_MX", mx)
    for name, f in _calls().items():
        want = _flat(f())
        _leave_an_error()
        try:
            got = _flat(f())
        except RuntimeError as e:
            pytest.fail(f"{name}: {e}")
        for a, b in zip(got, want):
            assert torch.equal(a, b), name

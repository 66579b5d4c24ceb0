"""Shape inference and refusals of the MoE block operators (no GPU needed)."""

from __future__ import annotations

import inspect

import pytest
import torch


def _meta(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


def test_signatures():
    from cutlass_op.bf16_grouped_mm import permute, routing

    s = inspect.signature(routing.moe_route)
    assert list(s.parameters) == ["logits", "topk", "score", "renormalize", "scale", "bias", "token_mask"]
    assert list(inspect.signature(permute.moe_permute).parameters) == ["x", "expert_idx", "num_experts", "plan"]
    assert list(inspect.signature(permute.moe_unpermute).parameters) == ["rows", "plan", "weights"]


def test_fake_shapes_of_router_and_permutation():
    from cutlass_op.bf16_grouped_mm.permute import moe_permute, moe_permute_fp8, moe_sort, moe_unpermute
    from cutlass_op.bf16_grouped_mm.routing import moe_route

    logits = _meta(10, 32, dtype=torch.float32).requires_grad_(True)
    w, idx = moe_route(logits, 4)
    assert w.shape == (10, 4) and w.dtype == torch.float32 and w.requires_grad
    assert idx.shape == (10, 4) and idx.dtype == torch.int64 and not idx.requires_grad
    x = _meta(10, 36).requires_grad_(True)
    rows, plan = moe_permute(x, idx, 32)
    assert rows.shape == (40, 36) and rows.stride() == (40, 1) and rows.requires_grad  # 16-byte row pitch
    assert plan.offs.shape == (32,) and plan.row_of_copy.shape == (10, 4) and plan.copy_of_row.shape == (40,)
    assert all(t.dtype == torch.int32 for t in plan)
    out = moe_unpermute(rows, plan, w)
    assert out.shape == (10, 36) and out.dtype == torch.bfloat16 and out.requires_grad
    dl, dx = torch.autograd.grad(out, (logits, x), _meta(10, 36))
    assert dl.shape == logits.shape and dl.dtype == logits.dtype and dx.shape == x.shape
    q, scale, _ = moe_permute_fp8(_meta(10, 200), plan=moe_sort(idx, 32))
    assert q.shape == (40, 200) and q.dtype == torch.float8_e4m3fn and q.stride() == (208, 1)
    assert scale.shape == (40, 2) and scale.stride() == (4, 1)


def test_cpu_tensors_and_wrong_words_are_refused():
    from cutlass_op.bf16_grouped_mm.permute import moe_permute, moe_sort
    from cutlass_op.bf16_grouped_mm.routing import moe_route

    with pytest.raises((RuntimeError, NotImplementedError)):
        moe_route(torch.zeros(2, 4), 2)
    with pytest.raises((RuntimeError, NotImplementedError)):
        moe_sort(torch.zeros(2, 2, dtype=torch.int64), 4)
    with pytest.raises(ValueError, match="score"):
        moe_route(torch.zeros(2, 4), 2, score="tanh")
    with pytest.raises(ValueError, match="plan"):
        moe_permute(torch.zeros(2, 4))


def test_host_refusals_at_the_c_abi():
    """Argument errors answer before any device call."""
    import ctypes

    from cutlass_op.bf16_grouped_mm._ext import lib

    i64, i32, f32, ptr = ctypes.c_int64, ctypes.c_int32, ctypes.c_float, ctypes.c_void_p
    route = lib.mgf_moe_route
    route.argtypes = [ptr, i32, i64, i64, i32, i32, i32, i32, f32, ptr, ptr, ptr, ptr, ptr]

    def r(dtype=0, tokens=4, experts=8, topk=2, score=0, logits=16):
        return route(logits, dtype, 8, tokens, experts, topk, score, 1, 1.0, None, None, None, None, None)

    assert r(dtype=3) == -1 and r(tokens=-1) == -1 and r(experts=0) == -1 and r(experts=1025) == -1
    assert r(topk=0) == -1 and r(topk=9) == -1 and r(experts=64, topk=33) == -1 and r(score=2) == -1
    assert r(logits=None) == -1 and r() == -1  # outputs missing
    assert r(tokens=0) == 0
    sort = lib.mgf_moe_sort
    sort.argtypes = [ptr, i64, i32, ptr, ptr, ptr, ptr, ptr]
    assert sort(None, 4, 8, 16, 16, 16, None, None) == -1 and sort(16, -1, 8, 16, 16, 16, None, None) == -1
    assert sort(16, 1 << 31, 8, 16, 16, 16, 16, None) == -1 and sort(16, 4, 1025, 16, 16, 16, None, None) == -1
    assert sort(16, 9000, 8, 16, 16, 16, None, None) == -1  # needs its workspace
    lib.mgf_moe_sort_workspace_words.restype = i64
    lib.mgf_moe_sort_workspace_words.argtypes = [i64, i32]
    assert lib.mgf_moe_sort_workspace_words(8192, 8) == 0 and lib.mgf_moe_sort_workspace_words(8193, 8) == 40
    quant = lib.mgf_fp8_block_quantize_rows
    quant.argtypes = [ptr, i64, i64, i64, i32, ptr, ptr, ptr, i64, ptr, i64, i64, ptr]
    assert quant(16, 8, 4, 8, 2, None, None, 16, 16, 16, 4, 4, None) == -1   # two rows per token without a plan
    assert quant(16, 8, 4, 8, 1, None, None, 8, 16, 16, 4, 4, None) == -3    # codes not 16-byte aligned
    assert quant(16, 8, 4, 8, 1, None, None, 16, 24, 16, 4, 4, None) == -3   # row pitch of the codes
    perm = lib.mgf_moe_permute
    perm.argtypes = [ptr, i32, i64, i64, i32, i64, ptr, ptr, ptr, i64, i64, ptr]
    assert perm(16, 0, 8, 4, 0, 8, 16, 16, 16, 8, 4, None) == -1  # topk 0
    assert perm(16, 0, 8, 1 << 30, 4, 8, 16, 16, 16, 8, 4, None) == -1  # more copies than 32 bits hold

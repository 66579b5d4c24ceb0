"""Calls of the MoE block's operators next to their limits."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


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


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("score,renorm", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
@pytest.mark.parametrize("T,E,k", [(37, 32, 4), (64, 128, 8), (9, 257, 8), (5, 1000, 32), (33, 1024, 2)])
def test_router_gradient_element_by_element(T, E, k, score, renorm, dtype):
    """Every element within a bound of its own.  u = 2^-24; p is an expert's probability, s its sigmoid, r = sum p g.
    Every factor (p, 1 - s, r's terms) is off by less than 128 u of itself (exp of |z| <= 32: 32 u of the argument's rounding,
    a few u each for exp, log1p and divisions, 37 u for a sum over 1024 terms); r and g - r by 128 u (|g| + sum p |g|)
    together with their sums' roundings.
      chosen, or any expert of a softmax over all: 384 u * scale * p * (|G| + sum p |g|) (G: its g, or 0)
      sigmoid over the chosen, not divided by their sum: 384 u * scale * s (1 - s) |g|
    plus the output's rounding; exactly 0 where the formula is 0.  fp16 outputs below 2^-14 are multiples of 2^-24:
    2^-25 more."""
    from cutlass_op.bf16_grouped_mm.routing import moe_route

    g = _gen(T + E + k)
    scale = 2.5
    leaf = (1.5 * torch.randn(T, E, generator=g, device="cuda")).to(dtype).requires_grad_(True)
    w, idx = moe_route(leaf, k, score, renorm, scale)
    gw = torch.randn(T, k, generator=g, device="cuda")
    (dl,) = torch.autograd.grad(w, leaf, gw)
    z = leaf.detach().double()
    hot = torch.zeros(T, E, dtype=torch.bool, device="cuda").scatter_(1, idx, True)
    G = torch.zeros(T, E, dtype=torch.float64, device="cuda").scatter_(1, idx, gw.double())
    s = torch.sigmoid(z)
    if score == "softmax":
        p = torch.softmax(z.masked_fill(~hot, -math.inf), 1) if renorm else torch.softmax(z, 1)
        slope = torch.ones_like(p)
    else:
        p = torch.where(hot, s, 0.0)
        p = p / p.sum(1, keepdim=True) if renorm else p
        slope = 1 - s
    if score == "sigmoid" and not renorm:
        ref, size = scale * p * slope * G, scale * p * slope * G.abs()
    else:
        chosen = torch.where(hot, p, 0.0)
        r = (chosen * G).sum(1, keepdim=True)
        ref = scale * p * slope * (G - r)
        size = scale * p * slope * (G.abs() + (chosen * G.abs()).sum(1, keepdim=True))
    half = torch.finfo(dtype).eps / 2
    tol = 384 * U * size + half * (ref.abs() + 384 * U * size) + (2.0 ** -25 if dtype == torch.float16 else 0.0) * (size > 0)
    over = (dl.double() - ref).abs() - tol
    assert not over.isnan().any() and float(over.max()) <= 0.0, f"{int((over > 0).sum())} off, worst by {float(over.max()):.3e}"
    assert (dl[size == 0] == 0).all()


class _Desc(ctypes.Structure):  # include/moe_gemm.h: mgf_block_gemm_desc
    i32, i64, ptr, f32 = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p, ctypes.c_float
    _fields_ = [("epilogue", i32), ("num_groups", i32), ("total_rows", i64), ("n", i64), ("k", i64), ("a", ptr), ("lda", i64),
                ("b", ptr), ("ldb", i64), ("ldb_batch", i64), ("b_mn_major", i32), ("sm_carveout", i32), ("offs", ptr),
                ("scale_a", ptr), ("scale_a_stride", i64), ("scale_b", ptr), ("scale_b_stride_e", i64),
                ("scale_b_stride_k", i64), ("scale_b_stride_n", i64), ("bias", ptr), ("bias_stride", i64), ("d", ptr),
                ("ldd", i64), ("d2", ptr), ("ldd2", i64), ("aux", ptr), ("ld_aux", i64), ("swiglu_alpha", f32),
                ("swiglu_limit", f32), ("workspace", ptr)]


@pytest.mark.parametrize("epilogue", [0, 1, 2])
@pytest.mark.parametrize("cg", ["1", "2"])
def test_tensor_core_scales_leave_rows_behind_the_last_group(cg, epilogue, monkeypatch):
    """The form with the scales in the tensor cores (it needs the workspace and powers of two) writes rows of groups only,
    and only the columns of its matrix."""
    from cutlass_op.bf16_grouped_mm import _ext, fp8_block

    monkeypatch.setenv("MGF_BLOCK_MX", "1")
    monkeypatch.setenv("MGF_CTA_GROUP", cg)
    g = _gen(4)
    E, K, N, kept, rows = 3, 256, 272, 135, 335
    x = torch.randn(rows, K, generator=g, device="cuda").to(torch.bfloat16)
    w = torch.randn(E, K, N, generator=g, device="cuda").to(torch.bfloat16)
    bias = torch.randn(E, N, generator=g, device="cuda").to(torch.bfloat16)
    offs = torch.tensor([5, 5, kept], dtype=torch.int32, device="cuda")
    qa, sa = fp8_block.quantize_rows_block(x)
    qb, sb = fp8_block.quantize_weights_block(w)
    aux = torch.randn(rows, 2 * N, generator=g, device="cuda").to(torch.bfloat16)
    if epilogue == 0:
        want = [fp8_block.grouped_mm_fp8_block(qa, qb, offs, sa, sb, bias)]
    elif epilogue == 1:
        want = list(fp8_block.grouped_mm_swiglu_fp8_block(qa, qb, offs, sa, sb, bias))[::-1]
    else:
        want = [fp8_block.grouped_mm_swiglu_bwd_fp8_block(qa, qb, offs, aux, sa, sb)]
    outs = [torch.full((rows, t.shape[1] + 16), 7.0, dtype=torch.bfloat16, device="cuda") for t in want]
    d = _Desc(epilogue, E, rows, N, K, qa.data_ptr(), qa.stride(0), qb.data_ptr(), qb.stride(1), qb.stride(0), 1, 0,
              offs.data_ptr(), sa.data_ptr(), sa.stride(0), sb.data_ptr(), *sb.stride(),
              bias.data_ptr() if epilogue < 2 else None, N, outs[0].data_ptr(), outs[0].stride(0),
              outs[1].data_ptr() if epilogue == 1 else None, outs[1].stride(0) if epilogue == 1 else 0,
              aux.data_ptr() if epilogue == 2 else None, 2 * N, 1.702, 7.0, None)
    lib = _ext.lib
    lib.mgf_block_gemm_desc_size.restype = ctypes.c_size_t
    assert ctypes.sizeof(_Desc) == lib.mgf_block_gemm_desc_size()
    lib.mgf_block_gemm_workspace_bytes.restype = ctypes.c_int64
    lib.mgf_block_gemm_workspace_bytes.argtypes = [ctypes.c_void_p]
    nbytes = lib.mgf_block_gemm_workspace_bytes(ctypes.byref(d))
    assert nbytes > 0
    ws = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    d.workspace = ws.data_ptr()
    lib.mgf_block_gemm_launch.argtypes = [ctypes.c_void_p, ctypes.c_void_p]
    assert lib.mgf_block_gemm_launch(ctypes.byref(d), torch.cuda.current_stream().cuda_stream) == 0
    for out, ref in zip(outs, want):
        n = ref.shape[1]
        assert torch.equal(out[:kept, :n], ref[:kept])
        assert (out[kept:] == 7.0).all() and (out[:, n:] == 7.0).all()


@pytest.mark.parametrize("rows,E", [(32, 32), (700, 5)])
@pytest.mark.parametrize("mx", ["0", "1"])
def test_products_repeat_bit_for_bit(rows, E, mx, monkeypatch):
    from cutlass_op.bf16_grouped_mm import fp8_block

    monkeypatch.setenv("MGF_BLOCK_MX", mx)
    for name in ("MGF_CTA_GROUP", "MGF_BN"):
        monkeypatch.delenv(name, raising=False)
    g = _gen(rows)
    K, N = 2880, 1296
    x = torch.randn(rows, K, generator=g, device="cuda").to(torch.bfloat16)
    w = (torch.randn(E, K, N, generator=g, device="cuda") / math.sqrt(K)).to(torch.bfloat16)
    bias = torch.randn(E, N, generator=g, device="cuda").to(torch.bfloat16)
    offs = torch.randint(0, rows + 1, (E,), generator=g, device="cuda").sort().values.int()
    offs[-1] = rows
    qa, sa = fp8_block.quantize_rows_block(x)
    qb, sb = fp8_block.quantize_weights_block(w)
    first = fp8_block.grouped_mm_swiglu_fp8_block(qa, qb, offs, sa, sb, bias)
    for _ in range(20):
        again = fp8_block.grouped_mm_swiglu_fp8_block(qa, qb, offs, sa, sb, bias)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])

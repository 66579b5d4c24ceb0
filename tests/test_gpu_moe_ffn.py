"""The MoE block as a whole (route -> permute -> FFN -> unpermute) and the block-scaled FFN, with gradients.

The parts are held to their own tolerances in test_gpu_moe_block.py and test_gpu_fp8_block.py; here the
chains must be exactly those parts, and the results must be the formula's as far as the types allow, measured as
the norm of the difference over the norm of the result.
  bf16       each bf16 rounding on the way is at most 2^-9 of a step's value in the mean square sense (2^-8 at
             most, uniform: / sqrt(3)); rounded are aux, the activation, the output, the rows' gradient,
             grad_aux and the sums: below 8 roundings in a row, sqrt(8) * 2^-8 / sqrt(3) < 2^-7.
  fp8_block  an e4m3 rounding is at most 2^-4 of the value, uniform: 2^-4 / sqrt(3) in the mean square sense;
             a product has two, the FFN's output two products and the deepest gradient (x's) four, so at
             most sqrt(8) * 2^-4 / sqrt(3) = 0.102; the SwiGLU slopes of up to 1 + |alpha g| / 4 * ... amplify
             gate errors by less than 1.5: below 0.153.
  logits     dl_j = p_j (d_j - sum_i p_i d_i) with d_j = <y_j, g> over H elements.  Errors e of y_j, independent
             with |e| = b |y_j|, change d_j by <e, g>, b |y_j| |g| / sqrt(H) in the mean square sense -- whatever
             is left of d_j itself after its terms cancel.  Both terms of dl_j have that error, so the
             norm of the difference is held to 2 b times the norm of p_j |y_j| |g| / sqrt(H), not to b times
             the norm of dl.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

ALPHA, LIMIT = 1.702, 7.0
BF16, FP8 = 2.0 ** -7, 0.153


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _params(E, H, I, seed):
    g = _gen(seed)

    def r(*s):
        return torch.randn(*s, generator=g, device="cuda")

    return [t.to(torch.bfloat16) for t in (r(E, H, 2 * I) / math.sqrt(H), r(E, I, H) / math.sqrt(I),
                                           0.02 * r(E, 2 * I), 0.02 * r(E, H))]


def _expert(x, w_up, w_down, b_up, b_down):
    aux = x @ w_up + b_up
    gate, up = aux[:, 0::2].clamp(max=LIMIT), aux[:, 1::2].clamp(-LIMIT, LIMIT)
    return (gate * torch.sigmoid(ALPHA * gate) * (up + 1)) @ w_down + b_down


def _plain(x, logits, k, w_up, w_down, b_up, b_down, mask=None):
    """The block in 64 bits: every expert on all tokens, weighted by softmax over the k largest logits."""
    kth = logits.topk(k, dim=1).values[:, -1:]
    p = torch.softmax(logits.masked_fill(logits < kth, -math.inf), 1)
    out = sum(p[:, e:e + 1] * _expert(x, w_up[e], w_down[e], b_up[e], b_down[e]) for e in range(w_up.shape[0]))
    return out if mask is None else torch.where(mask[:, None], out, 0.0)


def _off(got, ref):
    return float((got.double() - ref).norm() / ref.norm())


@pytest.mark.parametrize("precision,bound", [("bf16", BF16), ("fp8_block", FP8)])
@pytest.mark.parametrize("T,E,k,H,I,masked", [(1, 4, 2, 128, 64, False), (37, 8, 4, 256, 192, False),
                                              (300, 16, 4, 320, 128, True), (64, 32, 1, 136, 72, False)])
def test_block_against_the_formula(precision, bound, T, E, k, H, I, masked):
    import cutlass_op.bf16_grouped_mm as m
    from cutlass_op.bf16_grouped_mm.moe import moe_ffn

    g = _gen(T)
    w = _params(E, H, I, T + 1)
    x = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
    logits = torch.randn(T, E, generator=g, device="cuda")  # fp32: no ties
    mask = torch.rand(T, generator=g, device="cuda") < 0.8 if masked else None
    leaves = [t.clone().requires_grad_(True) for t in (x, logits, *w)]
    out = moe_ffn(leaves[0], leaves[1], k, *leaves[2:], precision=precision, token_mask=mask)
    ref_leaves = [t.double().requires_grad_(True) for t in (x, logits, *w)]
    ref = _plain(ref_leaves[0], ref_leaves[1], k, *ref_leaves[2:], mask=mask)
    assert out.dtype == torch.bfloat16 and _off(out.detach(), ref) <= bound
    if masked:
        assert (out[~mask] == 0).all()
    go = torch.randn(T, H, generator=g, device="cuda").to(torch.bfloat16)
    got = torch.autograd.grad(out, leaves, go)
    want = torch.autograd.grad(ref, ref_leaves, go.double())
    for name, a, b, t in zip(("x", "logits", "w_up", "w_down", "b_up", "b_down"), got, want, leaves):
        assert a.dtype == t.dtype and a.shape == t.shape
        if name == "logits":
            y = torch.stack([_expert(x.double(), *(t[e].double() for t in w)) for e in range(E)], 1)
            kth = logits.topk(k, dim=1).values[:, -1:]
            p = torch.softmax(logits.double().masked_fill(logits < kth, -math.inf), 1)
            size = p * y.norm(dim=2) * go.double().norm(dim=1, keepdim=True) / math.sqrt(H)
            assert (a.double() - b).norm() <= 2 * bound * size.norm(), name
        else:
            assert _off(a, b) <= bound, (name, _off(a, b))
    with torch.no_grad():
        again = moe_ffn(x, logits, k, *w, precision=precision, token_mask=mask)
    assert torch.equal(again, out)  # inference takes codes in expert order: the same codes
    m.check_device_status()


@pytest.mark.parametrize("counts", [[0, 130, 7, 0, 513], [1], [0, 0, 3]])
def test_block_scaled_ffn_is_the_chain_of_its_parts(counts):
    from cutlass_op.bf16_grouped_mm import fp8_block as f

    E, H, I = len(counts), 264, 144
    w_up, w_down, b_up, b_down = _params(E, H, I, 3)
    g = _gen(4)
    M = sum(counts)
    rows = M + 5  # five rows behind the last group
    x = torch.randn(rows, H, generator=g, device="cuda").to(torch.bfloat16)
    go = torch.randn(rows, H, generator=g, device="cuda").to(torch.bfloat16)
    offs = torch.tensor(counts, device="cuda").cumsum(0).int()
    leaves = [t.clone().requires_grad_(True) for t in (x, w_up, w_down, b_up, b_down)]
    out = f.grouped_mm_ffn_fp8_block(leaves[0], leaves[1], leaves[2], offs, leaves[3], leaves[4])
    grads = torch.autograd.grad(out, leaves, go)

    q_up, s_up = f.quantize_weights_block(w_up)
    q_down, s_down = f.quantize_weights_block(w_down)
    qx, sx = f.quantize_rows_block(x)
    s, aux = f.grouped_mm_swiglu_fp8_block(qx, q_up, offs, sx, s_up, b_up)
    qs, ss = f.quantize_rows_block(s)
    assert torch.equal(out[:M], f.grouped_mm_fp8_block(qs, q_down, offs, ss, s_down, b_down)[:M])
    qg, sg = f.quantize_rows_block(go)
    grad_aux = f.grouped_mm_swiglu_bwd_fp8_block(qg, q_down.transpose(1, 2), offs, aux, sg, s_down.transpose(1, 2))
    qa, sa = f.quantize_rows_block(grad_aux)
    gx = f.grouped_mm_fp8_block(qa, q_up.transpose(1, 2), offs, sa, s_up.transpose(1, 2))
    assert torch.equal(grads[0][:M], gx[:M])
    wu, bu = torch.ops.grouped_mm.mm_wgrad_bias(x.t(), grad_aux, offs)
    wd, bd = torch.ops.grouped_mm.mm_wgrad_bias(s.t(), go, offs)
    for a, b in zip(grads[1:], (wu, wd, bu, bd)):
        assert torch.equal(a, b)
    # kept codes, the other layout of the weights, and only some gradients wanted
    kept = f.grouped_mm_ffn_fp8_block(x, w_up, w_down, offs, b_up, b_down, up_codes=(q_up, s_up),
                                      down_codes=(q_down, s_down))
    assert torch.equal(kept[:M], out[:M])
    other = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (w_up, w_down)]
    assert torch.equal(f.grouped_mm_ffn_fp8_block(x, *other, offs, b_up, b_down)[:M], out[:M])
    for i in range(5):
        part = [t.detach().clone().requires_grad_(j == i) for j, t in enumerate(leaves)]
        y = f.grouped_mm_ffn_fp8_block(part[0], part[1], part[2], offs, part[3], part[4])
        (gi,) = torch.autograd.grad(y, part[i], go)
        assert torch.equal(gi[:M] if i == 0 else gi, grads[i][:M] if i == 0 else grads[i])


def test_block_captured_forward_and_backward():
    from cutlass_op.bf16_grouped_mm.moe import moe_ffn

    for precision in ("bf16", "fp8_block"):
        w = [t.requires_grad_(True) for t in _params(8, 128, 64, 1)]
        x = torch.randn(40, 128, generator=_gen(2), device="cuda").to(torch.bfloat16).requires_grad_(True)
        logits = torch.randn(40, 8, generator=_gen(3), device="cuda").requires_grad_(True)
        go = torch.randn(40, 128, generator=_gen(4), device="cuda").to(torch.bfloat16)
        leaves = (x, logits, *w)

        def step():
            out = moe_ffn(x, logits, 4, *w, precision=precision)
            return (out.detach(), *torch.autograd.grad(out, leaves, go))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                got = step()
        torch.cuda.current_stream().wait_stream(side)
        for seed in (5, 6):
            with torch.no_grad():
                x.copy_(torch.randn(40, 128, generator=_gen(seed), device="cuda"))
                logits.copy_(torch.randn(40, 8, generator=_gen(seed + 9), device="cuda"))
            graph.replay()
            want = step()
            for a, b in zip(got, want):
                assert torch.equal(a, b), precision


def test_block_refusals_and_empty_batch():
    from cutlass_op.bf16_grouped_mm.moe import moe_ffn

    w = _params(4, 128, 64, 1)
    x = torch.zeros(3, 128, device="cuda", dtype=torch.bfloat16)
    logits = torch.zeros(3, 4, device="cuda")
    with pytest.raises(ValueError, match="precision"):
        moe_ffn(x, logits, 2, *w, precision="fp4")
    with pytest.raises(ValueError, match="experts"):
        moe_ffn(x, torch.zeros(3, 5, device="cuda"), 2, *w)
    with pytest.raises(ValueError, match="codes"):
        moe_ffn(x, logits, 2, *w, up_codes=(x, x))
    with pytest.raises(RuntimeError):
        moe_ffn(x, torch.zeros(2, 4, device="cuda"), 2, *w)
    for precision in ("bf16", "fp8_block"):
        leaves = [t.clone().requires_grad_(True) for t in w]
        out = moe_ffn(x[:0], logits[:0], 2, *leaves, precision=precision)
        assert out.shape == (0, 128)
        for gr, t in zip(torch.autograd.grad(out.sum(), leaves), leaves):
            assert gr.shape == t.shape and (gr == 0).all()


def test_block_through_a_tracing_compiler():
    """Fake tensors and autograd of every operator agree with what runs (traced forward and backward)."""
    from cutlass_op.bf16_grouped_mm.permute import MoEPlan
    from cutlass_op.bf16_grouped_mm.routing import moe_route

    ops = torch.ops.grouped_mm
    w = _params(4, 64, 32, 1)
    x = torch.randn(6, 64, generator=_gen(1), device="cuda").to(torch.bfloat16)
    logits = torch.randn(6, 4, generator=_gen(2), device="cuda")
    wt, idx = moe_route(logits, 2)
    rows, *plan = ops.moe_permute(x, idx, 4)
    plan = MoEPlan(*plan)
    lg, xg, rg, wg = (t.detach().clone().requires_grad_(True) for t in (logits, x, rows, wt))
    checks = ["test_schema", "test_autograd_registration", "test_faketensor"]
    for op, args in ((ops.moe_route, (lg, 2, 0, True, 1.0, None, None)), (ops.moe_route, (logits, 2, 1, False, 2.0, None, None)),
                     (ops.moe_sort, (idx, 4)), (ops.moe_permute, (xg, idx, 4)),
                     (ops.moe_permute_rows, (xg, plan.offs, plan.row_of_copy)),
                     (ops.moe_unpermute, (rg, plan.offs, plan.row_of_copy, wg)),
                     (ops.moe_unpermute, (rows, plan.offs, plan.row_of_copy, None)),
                     (ops.fp8_quantize_rows_block, (x,)), (ops.fp8_quantize_weights_block, (w[0],)),
                     (ops.fp8_quantize_weights_block, (w[0].transpose(1, 2),)),
                     (ops.moe_permute_fp8, (x, idx, 4))):
        torch.library.opcheck(op.default, args, test_utils=checks)

    def step(lg, xg):
        wt, idx = ops.moe_route(lg, 2, 0, True, 1.0, None, None)
        rows, offs, row_of_copy, _ = ops.moe_permute(xg, idx, 4)
        return ops.moe_unpermute(rows * 2, offs, row_of_copy, wt)

    go = torch.randn(6, 64, generator=_gen(3), device="cuda").to(torch.bfloat16)
    want = step(lg, xg)
    ref = torch.autograd.grad(want, (lg, xg), go)
    out = torch.compile(step, backend="aot_eager", fullgraph=True)(lg, xg)
    assert torch.equal(out, want)
    for a, b in zip(torch.autograd.grad(out, (lg, xg), go), ref):
        assert torch.equal(a, b)

"""Router, permutation and their gradients against plain implementations in 64 bits.

Tolerances count roundings.  u = 2^-24 is half a step of fp32; an output type of machine epsilon eps adds
eps / 2 relative to the value.
  weights    exp of a difference |z| <= 32 rounded to fp32 (32 u), the same for log s (32 u), exp, log1p
             and the division (a few u each), a sum of at most 1024 terms in a tree over 32 lanes of 32
             (37 u): below 128 u relative.
  logits     dl = scale p (g - r): 128 u of every factor, r a sum of k terms: below 384 u * scale * p *
             (|g| + sum p |g|), plus the output rounding.
  unpermute  k fused multiply-adds: k u * sum |w r|, plus the output rounding.
             fp16 outputs below 2^-14 are multiples of 2^-24, whatever their value: half a step there is
             2^-25, not eps / 2 of the value, so 2^-25 is added for fp16 (bf16 and fp32 have the range of
             fp32 and no such values here).
  dweights   a lane adds 8 * ceil(width / 256) products, then 5 shuffles, then 8 warps.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _half(dt):
    return torch.finfo(dt).eps / 2


def _floor(dt):
    """Half a step of the type's smallest values (see above)."""
    return 2.0 ** -25 if dt == torch.float16 else 0.0


def _within(got, ref, tol):
    """Every element within its tolerance (a message of one line, not of whole tensors)."""
    over = (got.double() - ref).abs() - tol
    worst = float(over.max()) if over.numel() else 0.0
    assert not over.isnan().any() and worst <= 0.0, f"{int((over > 0).sum())} of {over.numel()} off, worst by {worst:.3e}"


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _status_ok():
    import cutlass_op.bf16_grouped_mm as m

    m.check_device_status()


# ------------------------------------------------------------------------------------------------ router
def _route_ref(logits, k, score, renorm, scale, bias, mask):
    """(weights fp64, ids, p fp64 of all experts as the weights use them) by sorting; slots without an
    expert: id -1, weight 0."""
    z = logits.double()
    key = logits.float() if bias is None else logits.float() + bias
    # -inf (of the logit or of the key) last and unusable, NaN first, equal keys by expert
    avail = ~((logits.float() == -math.inf) | (key == -math.inf))
    order_key = torch.where(torch.isnan(key), torch.full_like(key, math.inf), key)
    rank = torch.where(torch.isnan(key), torch.zeros_like(key), torch.ones_like(key))
    ids = torch.argsort(rank, dim=1, stable=True)
    by_key = torch.argsort(-torch.gather(order_key, 1, ids), dim=1, stable=True)
    # NaN rows first: a stable sort by -key among [NaN, others] keeps NaN before +inf
    ids = torch.gather(ids, 1, by_key)
    ids = torch.gather(ids, 1, torch.argsort((~torch.gather(avail, 1, ids)).int(), dim=1, stable=True))
    ids = ids[:, :k]
    live = torch.gather(avail, 1, ids)
    if mask is not None:
        live = live & mask[:, None]
    c = torch.gather(z, 1, ids)
    if score == "softmax":
        if renorm:
            e = torch.where(live, torch.exp(c - c.masked_fill(~live, -math.inf).amax(1, keepdim=True)), 0.0)
            p = e / e.sum(1, keepdim=True)
        else:
            p = torch.gather(torch.softmax(z, 1), 1, ids)
    else:
        s = torch.sigmoid(c)
        p = torch.where(live, s, 0.0)
        if renorm:
            p = p / p.sum(1, keepdim=True)
    return torch.where(live, scale * p, 0.0), torch.where(live, ids, -1)


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("score,renorm", [("softmax", True), ("softmax", False), ("sigmoid", True),
                                          ("sigmoid", False)])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (3, 4, 4), (37, 32, 4), (130, 33, 5), (64, 128, 8), (9, 257, 8),
                                   (5, 1000, 32), (2, 1024, 1)])
def test_route_forward_and_gradient(dtype, score, renorm, T, E, k):
    from cutlass_op.bf16_grouped_mm.routing import moe_route

    g = _gen(T * 1000 + E)
    scale = 2.5
    # a wider matrix's columns: a row stride other than E
    wide = (1.5 * torch.randn(T, E + 3, generator=g, device="cuda")).to(DT[dtype])
    logits = wide[:, 1:E + 1]
    bias = 0.3 * torch.randn(E, generator=g, device="cuda") if E % 2 else None
    mask = (torch.rand(T, generator=g, device="cuda") < 0.7) if T % 2 else None
    leaf = logits.detach().requires_grad_(True)
    w, idx = moe_route(leaf, k, score, renorm, scale, bias, mask)
    ref_w, ref_idx = _route_ref(logits, k, score, renorm, scale, bias, mask)
    assert torch.equal(idx, ref_idx)
    _within(w, ref_w, 128 * U * ref_w)
    assert not idx.requires_grad
    gw = torch.randn(T, k, generator=g, device="cuda")
    (dl,) = torch.autograd.grad(w, leaf, gw)
    assert dl.dtype == leaf.dtype and dl.shape == leaf.shape
    z = logits.double().requires_grad_(True)
    sel = ref_idx.clamp(min=0)
    live = ref_idx >= 0
    if score == "softmax":
        full = torch.softmax(z, 1)
        rw = torch.gather(full, 1, sel)
    else:
        full = torch.sigmoid(z)
        rw = torch.gather(full, 1, sel)
    rw = torch.where(live, rw, 0.0)
    if renorm:
        rw = rw / rw.sum(1, keepdim=True).clamp(min=1e-300)
    rw = torch.where(live, rw * scale, 0.0)
    (ref,) = torch.autograd.grad(rw, z, gw.double())
    gmax = gw.abs().amax(1, keepdim=True).double()
    _within(dl, ref, 384 * U * scale * 2 * gmax + _half(DT[dtype]) * ref.abs() + _floor(DT[dtype]))
    _status_ok()


def test_route_gradient_against_differences():
    from cutlass_op.bf16_grouped_mm.routing import moe_route

    g = _gen(5)
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            logits = torch.randn(6, 16, generator=g, device="cuda")
            gw = torch.randn(6, 3, generator=g, device="cuda")
            leaf = logits.clone().requires_grad_(True)
            (dl,) = torch.autograd.grad(moe_route(leaf, 3, score, renorm)[0], leaf, gw)
            d = torch.randn(6, 16, generator=g, device="cuda")
            h = 2.0 ** -9
            _, idx = moe_route(logits, 3, score, renorm)
            hi, ih = moe_route(logits + h * d, 3, score, renorm)
            lo, il = moe_route(logits - h * d, 3, score, renorm)
            same = (ih == idx).all(1) & (il == idx).all(1)
            num = ((hi.double() - lo.double()) * gw).sum(1) / (2 * h)
            ana = (dl.double() * d).sum(1)
            # central differences: h^2 / 6 times a third derivative below 6 |d|^3 |g|, and 4 * 128 u |g| / (2 h)
            size = gw.abs().sum(1).double()
            tol = size * (h * h * d.abs().amax(1).double() ** 3 + 4 * 128 * U / (2 * h))
            assert same.any() and ((num - ana).abs() <= tol)[same].all(), (score, renorm)


def test_route_masked_experts_infinities_and_nan():
    from cutlass_op.bf16_grouped_mm.routing import moe_route

    inf, nan = math.inf, math.nan
    low = torch.finfo(torch.float32).min
    logits = torch.tensor([
        [-inf, 1.0, -inf, 0.0],     # two experts left for three slots
        [-inf, -inf, -inf, -inf],   # none
        [low, low, low, low],       # the type's lowest value is a value: ties go to the lowest expert
        [nan, 0.0, 1.0, 2.0],       # NaN first
        [0.0, -0.0, 0.0, -0.0],     # equal
        [nan, inf, nan, -inf],      # masked token: whatever stands in it
    ], device="cuda")
    mask = torch.tensor([True, True, True, True, True, False], device="cuda")
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            leaf = logits.clone().requires_grad_(True)
            w, idx = moe_route(leaf, 3, score, renorm, token_mask=mask)
            assert idx.tolist() == [[1, 3, -1], [-1, -1, -1], [0, 1, 2], [0, 3, 2], [0, 1, 2], [-1, -1, -1]]
            assert (w[idx < 0] == 0).all()
            if renorm:
                assert torch.allclose(w[2], torch.full((3,), 1 / 3, device="cuda"), rtol=128 * U, atol=0)
            assert torch.isnan(w[3, 0])
            (dl,) = torch.autograd.grad(w, leaf, torch.ones_like(w))
            assert (dl[1] == 0).all() and (dl[5] == 0).all() and (dl[0, [0, 2]] == 0).all()
            assert torch.isfinite(dl[[0, 1, 2, 4, 5]]).all()


def test_route_bias_selects_but_does_not_weigh():
    from cutlass_op.bf16_grouped_mm.routing import moe_route

    logits = torch.tensor([[3.0, 2.0, 1.0, 0.0]], device="cuda")
    bias = torch.tensor([-10.0, 0.0, 0.0, 5.0], device="cuda")
    w, idx = moe_route(logits, 2, "sigmoid", False, bias=bias)
    assert idx.tolist() == [[3, 1]]
    ref = torch.sigmoid(torch.tensor([[0.0, 2.0]], dtype=torch.float64, device="cuda"))
    assert ((w.double() - ref).abs() <= 128 * U * ref).all()


# ------------------------------------------------------------------------------------------------ permutation
def _ids(g, T, k, E, drop):
    idx = torch.randint(0, E, (T, k), generator=g, device="cuda")  # repeats within a token included
    if drop:
        idx = torch.where(torch.rand(T, k, generator=g, device="cuda") < drop, torch.full_like(idx, -1), idx)
    return idx


def _plan_ref(idx, E):
    flat = idx.flatten().tolist()
    offs, copy_of_row = [], []
    for e in range(E):
        copy_of_row += [c for c, v in enumerate(flat) if v == e]
        offs.append(len(copy_of_row))
    row_of_copy = [-1] * len(flat)
    for r, c in enumerate(copy_of_row):
        row_of_copy[c] = r
    return offs, row_of_copy, copy_of_row + [-1] * (len(flat) - len(copy_of_row))


@pytest.mark.parametrize("T,k,E,drop", [(0, 4, 8, 0), (1, 1, 1, 0), (8, 4, 32, 0), (33, 3, 5, 0.3), (700, 8, 256, 0.1),
                                        (5, 2, 1024, 0), (1024, 4, 7, 0), (1025, 4, 7, 0.9), (64, 1, 3, 1.1)])
def test_sort_equals_a_stable_counting_sort(T, k, E, drop):
    from cutlass_op.bf16_grouped_mm.permute import moe_sort

    idx = _ids(_gen(T + E), T, k, E, drop)
    plan = moe_sort(idx, E)
    offs, row_of_copy, copy_of_row = _plan_ref(idx, E)
    assert plan.offs.tolist() == offs
    assert plan.row_of_copy.flatten().tolist() == row_of_copy
    assert plan.copy_of_row.tolist() == copy_of_row
    _status_ok()


@pytest.mark.parametrize("n,E", [(8192, 64), (8193, 16), (4096 * 4 + 1, 1024), (300_001, 128), (700_000, 3)])
def test_sort_of_many_copies(n, E):
    from cutlass_op.bf16_grouped_mm.permute import moe_sort

    idx = _ids(_gen(n), n, 1, E, 0.05)
    plan = moe_sort(idx, E)
    flat = torch.where(idx.flatten() < 0, E, idx.flatten())
    order = torch.sort(flat, stable=True).indices
    kept = int((flat < E).sum())
    assert torch.equal(plan.offs.long(), torch.bincount(flat, minlength=E + 1)[:E].cumsum(0))
    assert torch.equal(plan.copy_of_row[:kept].long(), order[:kept]) and (plan.copy_of_row[kept:] == -1).all()
    inv = torch.full((n,), -1, device="cuda")
    inv[order[:kept]] = torch.arange(kept, device="cuda")
    assert torch.equal(plan.row_of_copy.flatten().long(), inv)


@pytest.mark.parametrize("T,k,E,drop", [(1, 1, 1, 0), (8, 4, 32, 0), (64, 4, 1024, 0.3), (257, 1, 5, 0.2), (250, 4, 3, 0.1),
                                          (128, 8, 1000, 0), (3, 5, 2, 1.1), (1025, 1, 9, 0.1)])
def test_permute_sorts_as_the_sort_does(T, k, E, drop):
    """Few copies are sorted within the permuting launch; the plan is the same."""
    from cutlass_op.bf16_grouped_mm.permute import moe_permute, moe_sort

    idx = _ids(_gen(T * 7 + E), T, k, E, drop)
    x = torch.randn(T, 24, generator=_gen(1), device="cuda")
    rows, plan = moe_permute(x, idx, E)
    for a, b in zip(plan, moe_sort(idx, E)):
        assert torch.equal(a, b)
    assert torch.equal(rows, moe_permute(x, plan=plan)[0])


def test_sort_reports_ids_out_of_range_and_drops_them():
    import cutlass_op.bf16_grouped_mm as m
    from cutlass_op.bf16_grouped_mm._ext import DEV_ROW_OUT_OF_RANGE, device_status
    from cutlass_op.bf16_grouped_mm.permute import moe_sort

    m.device_status()
    plan = moe_sort(torch.tensor([[0, 5], [-2, 1]], device="cuda"), 2)
    assert device_status() == DEV_ROW_OUT_OF_RANGE
    assert plan.offs.tolist() == [1, 2] and plan.row_of_copy.tolist() == [[0, -1], [-1, 1]]
    assert plan.copy_of_row.tolist() == [0, 3, -1, -1]
    from cutlass_op.bf16_grouped_mm.permute import moe_permute

    x = torch.tensor([[1.0], [2.0]], device="cuda")
    rows, same = moe_permute(x, torch.tensor([[0, 5], [-2, 1]], device="cuda"), 2)
    assert device_status() == DEV_ROW_OUT_OF_RANGE
    assert all(torch.equal(a, b) for a, b in zip(same, plan)) and rows.flatten().tolist() == [1.0, 2.0, 0.0, 0.0]


@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,k,E,H,drop,weighted", [
    (1, 1, 1, 1, 0, True), (7, 4, 8, 2880, 0, True), (50, 8, 16, 129, 0.2, True), (300, 3, 5, 8, 0.5, False),
    (19, 5, 4, 4097, 0, False), (260, 11, 9, 264, 0.1, True), (19000, 2, 32, 40, 0.1, True), (6, 2, 4, 64, 1.1, True)])
def test_permute_unpermute_and_gradients(dtype, T, k, E, H, drop, weighted):
    from cutlass_op.bf16_grouped_mm.permute import moe_permute, moe_unpermute

    g = _gen(T + H)
    dt = DT[dtype]
    half = _half(dt) + U
    wide = torch.randn(T, H + 5, generator=g, device="cuda").to(dt)
    x = (wide[:, :H] if H % 2 else wide[:, :H].contiguous()).detach().requires_grad_(True)
    idx = _ids(g, T, k, E, drop)
    rows, plan = moe_permute(x, idx, E)
    kept = int(plan.offs[-1])
    n = T * k
    c = plan.copy_of_row[:kept].long()
    assert rows.shape == (n, H) and (rows.stride(0) * dt.itemsize) % 16 == 0
    assert torch.equal(rows[:kept], x.detach()[c // k]) and (rows[kept:] == 0).all()
    # gradient of x: rows' gradients summed; what stands behind the last row does not enter
    gr = torch.randn(n, H, generator=g, device="cuda").to(dt)
    gr[kept:] = math.nan
    (dx,) = torch.autograd.grad(rows, x, gr)
    ref = torch.zeros(T, H, dtype=torch.float64, device="cuda").index_add_(0, c // k, gr[:kept].double())
    size = torch.zeros(T, H, dtype=torch.float64, device="cuda").index_add_(0, c // k, gr[:kept].double().abs())
    _within(dx, ref, k * U * size + half * ref.abs() + _floor(dt))

    y = torch.randn(n, H, generator=g, device="cuda").to(dt)
    y[kept:] = math.nan
    y.requires_grad_(True)
    w = torch.randn(T, k, generator=g, device="cuda").requires_grad_(True) if weighted else None
    out = moe_unpermute(y, plan, w)
    wc = w.detach().flatten()[c].double() if weighted else torch.ones(kept, dtype=torch.float64, device="cuda")
    terms = wc[:, None] * y.detach()[:kept].double()
    ref = torch.zeros(T, H, dtype=torch.float64, device="cuda").index_add_(0, c // k, terms)
    size = torch.zeros(T, H, dtype=torch.float64, device="cuda").index_add_(0, c // k, terms.abs())
    assert out.dtype == dt
    _within(out.detach(), ref, k * U * size + half * ref.abs() + _floor(dt))
    go = torch.randn(T, H, generator=g, device="cuda").to(dt)
    got = torch.autograd.grad(out, (y, w) if weighted else (y,), go)
    ref = wc[:, None] * go.double()[c // k]
    _within(got[0][:kept], ref, half * ref.abs() + _floor(dt))
    assert (got[0][kept:] == 0).all()
    if weighted:
        prod = y.detach()[:kept].double() * go.double()[c // k]
        dw = torch.zeros(n, dtype=torch.float64, device="cuda")
        dw[c] = prod.sum(1)
        size = torch.zeros(n, dtype=torch.float64, device="cuda")
        size[c] = prod.abs().sum(1)
        steps = 8 * math.ceil(H / 32) + 16
        _within(got[1].flatten(), dw, steps * U * size)
    _status_ok()


def test_permute_with_a_plan_and_only_one_gradient_wanted():
    from cutlass_op.bf16_grouped_mm.permute import moe_permute, moe_sort, moe_unpermute

    g = _gen(3)
    x = torch.randn(40, 96, generator=g, device="cuda").to(torch.bfloat16)
    idx = _ids(g, 40, 4, 6, 0.2)
    plan = moe_sort(idx, 6)
    rows, same = moe_permute(x, plan=plan)
    assert same is plan and torch.equal(rows, moe_permute(x, idx, 6)[0])
    w = torch.rand(40, 4, generator=g, device="cuda")
    go = torch.randn(40, 96, generator=g, device="cuda").to(torch.bfloat16)
    y, wl = rows.detach().clone().requires_grad_(True), w.clone().requires_grad_(True)
    both = torch.autograd.grad(moe_unpermute(y, plan, wl), (y, wl), go)
    (only_rows,) = torch.autograd.grad(moe_unpermute(y, plan, w), y, go)
    (only_w,) = torch.autograd.grad(moe_unpermute(rows, plan, wl), wl, go)
    assert torch.equal(both[0], only_rows) and torch.equal(both[1], only_w)
    # a transposed (column-major) and a broadcast output gradient
    col = go.t().contiguous().t()
    (g1,) = torch.autograd.grad(moe_unpermute(y, plan, w), y, col)
    assert torch.equal(g1, only_rows)
    moe_unpermute(y, plan, w).sum().backward()
    ref = torch.where(plan.copy_of_row >= 0, w.flatten()[plan.copy_of_row.clamp(min=0).long()], 0.0)
    assert torch.equal(y.grad, ref.to(torch.bfloat16)[:, None].expand_as(y.grad))


def test_permute_plan_with_a_row_out_of_range_touches_nothing_else():
    from cutlass_op.bf16_grouped_mm._ext import DEV_ROW_OUT_OF_RANGE, device_status
    from cutlass_op.bf16_grouped_mm.permute import MoEPlan, moe_permute, moe_unpermute

    device_status()
    i32 = dict(dtype=torch.int32, device="cuda")
    plan = MoEPlan(torch.tensor([4], **i32), torch.tensor([[0, 4], [2, 3]], **i32), torch.tensor([0, -1, 2, 3], **i32))
    x = torch.arange(16.0, device="cuda").view(2, 8)
    rows, _ = moe_permute(x, plan=plan)
    assert device_status() == DEV_ROW_OUT_OF_RANGE
    assert torch.equal(rows[[0, 2, 3]], x[[0, 1, 1]])
    out = moe_unpermute(rows[[0, 0, 2, 3]], plan)
    assert device_status() == DEV_ROW_OUT_OF_RANGE and torch.equal(out, torch.stack([x[0], 2 * x[1]]))


def test_refusals_on_the_device():
    from cutlass_op.bf16_grouped_mm.permute import moe_permute, moe_sort, moe_unpermute
    from cutlass_op.bf16_grouped_mm.routing import moe_route

    logits = torch.zeros(4, 8, device="cuda")
    for bad in (dict(topk=0), dict(topk=9), dict(topk=2, bias=torch.zeros(7, device="cuda")),
                dict(topk=2, bias=torch.zeros(8)), dict(topk=2, token_mask=torch.ones(4, device="cuda"))):
        with pytest.raises(RuntimeError):
            moe_route(logits, **bad)
    with pytest.raises(RuntimeError, match="float"):
        moe_route(logits.double(), 2)
    with pytest.raises(RuntimeError, match="unit stride"):
        moe_route(torch.zeros(8, 4, device="cuda").t(), 2)
    idx = torch.zeros(4, 2, dtype=torch.int64, device="cuda")
    with pytest.raises(RuntimeError, match="int64"):
        moe_sort(idx.int(), 8)
    with pytest.raises(RuntimeError, match="1024"):
        moe_sort(idx, 1025)
    with pytest.raises(RuntimeError, match="tokens"):
        moe_permute(torch.zeros(3, 8, device="cuda"), idx, 8)
    with pytest.raises(RuntimeError, match="unit stride"):
        moe_permute(torch.zeros(8, 4, device="cuda").t(), idx, 8)
    rows, plan = moe_permute(torch.zeros(4, 8, device="cuda"), idx, 8)
    with pytest.raises(RuntimeError, match="weights"):
        moe_unpermute(rows, plan, torch.zeros(4, 2, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="weights"):
        moe_unpermute(rows, plan, torch.zeros(4, 3, device="cuda"))
    leaf = torch.zeros(4, 8, device="cuda", requires_grad=True)
    w, _ = moe_route(leaf, 2)
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(w.sum(), leaf, create_graph=True)


# ------------------------------------------------------------------------------------------------ streams and graphs
def test_route_and_permute_captured_and_replayed_with_new_inputs():
    from cutlass_op.bf16_grouped_mm.permute import moe_permute, moe_unpermute
    from cutlass_op.bf16_grouped_mm.routing import moe_route

    g = _gen(11)
    logits = torch.randn(48, 16, generator=g, device="cuda")
    x = torch.randn(48, 72, generator=g, device="cuda").to(torch.bfloat16)

    def step():
        w, idx = moe_route(logits, 4)
        rows, plan = moe_permute(x, idx, 16)
        return moe_unpermute(rows, plan, w), plan.offs

    step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graphs, outs = [], []
        for _ in range(2):
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr):
                outs.append(step())
            graphs.append(gr)
    torch.cuda.current_stream().wait_stream(side)
    for seed in (1, 2):
        logits.copy_(torch.randn(48, 16, generator=_gen(seed), device="cuda"))
        x.copy_(torch.randn(48, 72, generator=_gen(seed + 7), device="cuda"))
        for gr in graphs:
            gr.replay()
        want = step()
        for got in outs:
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])

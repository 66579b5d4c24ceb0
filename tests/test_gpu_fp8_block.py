"""e4m3 with a scale per block of 128: quantisers against their definition (bit for bit), the grouped
products against the same sums in 64 bits.

Tolerances of the products count roundings (u = 2^-24).  A block of 128 products of e4m3 numbers is summed
by the tensor core: the products are exact (8 significant bits), the sum of 128 is allowed 128 roundings that
may truncate instead of round (2 u each); the scale factor sa * sb rounds once, the promotion (one fused
multiply-add per block) once per block.  So |acc - exact| <= (256 + 1 + blocks) u * S with S the sum of the
magnitudes of all products.  Where the tensor core applies the scales (powers of two: exact) it also sums all
k products: 2 k u S.  bf16 output: 2^-8 of the value.  SwiGLU and its backward are computed from
bf16 (exactly known) or fp32 inputs in fp32: a few u times their condition, below 64 u of the terms'
magnitudes, times the output rounding.  The sigmoid is 1 / (1 + e^-z) by an approximate reciprocal that gives 0
where the denominator is over 2^126: an absolute error of up to 2^-126, times the other factors.
"""

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
    return _code_ref(b, s[:, :, None]).reshape(m, nb * 128)[:, :k], s


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


# ------------------------------------------------------------------------------------------------ grouped products
U = 2.0 ** -24
ALPHA, LIMIT = 1.702, 7.0


def _case(E, K, N, counts, layout, seed, extra_rows=0):
    """Operands with arbitrary fp32 scales (not powers of two); groups of `counts` rows and rows behind them."""
    g = _gen(seed)
    M = sum(counts) + extra_rows

    def codes(*shape):
        return torch.randn(*shape, generator=g, device="cuda").mul_(20).to(torch.float8_e4m3fn)

    def pitched(t):
        p = torch.zeros(*t.shape[:-1], (t.shape[-1] + 15) // 16 * 16 + 16, dtype=t.dtype, device="cuda")
        p = p[..., :t.shape[-1]]
        p.copy_(t)
        return p

    kb, nb = -(-K // 128), -(-N // 128)
    a = pitched(codes(M, K))
    b = pitched(codes(E, K, N)) if layout == "kn" else pitched(codes(E, N, K)).transpose(1, 2)
    sa = torch.empty(M, (kb + 3) // 4 * 4, device="cuda")[:, :kb]
    sa.copy_(0.01 + torch.rand(M, kb, generator=g, device="cuda"))
    sb = 0.01 + torch.rand(E, kb, nb, generator=g, device="cuda")
    if layout == "nk":
        sb = sb.transpose(1, 2).contiguous().transpose(1, 2)
    offs = torch.tensor(counts, device="cuda").cumsum(0).int()
    bias = (100 * torch.randn(E, N, generator=g, device="cuda")).to(torch.bfloat16)
    return a, b, offs, sa, sb, bias


def _exact(a, b, offs, sa, sb):
    """(sum, sum of magnitudes) of every output, in 64 bits; rows behind the last group stay zero."""
    K, N = b.shape[1:]
    out = torch.zeros(a.shape[0], N, dtype=torch.float64, device="cuda")
    mag = torch.zeros_like(out)
    ad = a.double() * sa.double().repeat_interleave(128, 1)[:, :K]
    lo = 0
    for e, hi in enumerate(offs.tolist()):
        s = sb[e].double().repeat_interleave(128, 0)[:K].repeat_interleave(128, 1)[:, :N]
        bd = b[e].double() * s
        out[lo:hi] = ad[lo:hi] @ bd
        mag[lo:hi] = ad[lo:hi].abs() @ bd.abs()
        lo = hi
    return out, mag


def _within(name, got, ref, tol):
    over = (got.double() - ref).abs() - tol
    worst = float(over.max()) if over.numel() else 0.0
    assert not over.isnan().any() and worst <= 0.0, f"{name}: {int((over > 0).sum())} of {over.numel()} off by up to {worst:.3e}"


def _row_of(offs, M):
    """Group of every row (the last one's for rows behind it)."""
    return torch.bucketize(torch.arange(M, device="cuda"), offs.long(), right=True).clamp(max=offs.numel() - 1)


SHAPES = [
    (1, 1, 16, [1]),
    (1, 128, 128, [128]),
    (4, 256, 192, [70, 0, 131, 5]),
    (3, 320, 272, [600, 513, 700]),
    (2, 2880, 528, [1029, 640]),
    (5, 100, 48, [0, 1, 127, 129, 0]),
    (2, 1000, 1040, [3, 260]),
    (40, 136, 144, [1] * 40),
]


@pytest.mark.parametrize("form", ["auto", "single", "pair", "narrow", "choice", "powers", "powers pair"])
@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("E,K,N,counts", SHAPES)
def test_products_against_64_bits(E, K, N, counts, layout, form, monkeypatch):
    """auto .. narrow: the launch shapes; choice: arbitrary scales offered to the form that wants powers of two,
    which has to leave them to the other; powers (pair): powers of two, applied by the tensor cores."""
    import cutlass_op.bf16_grouped_mm as m
    from cutlass_op.bf16_grouped_mm import fp8_block

    monkeypatch.setenv("MGF_BLOCK_MX", "1" if form.startswith(("choice", "powers")) else "0")
    if form in ("single", "pair", "powers", "powers pair"):
        monkeypatch.setenv("MGF_CTA_GROUP", "2" if form.endswith("pair") else "1")
    if form == "narrow":
        monkeypatch.setenv("MGF_BN", "128")
    a, b, offs, sa, sb, bias = _case(E, K, N, counts, layout, E * 7 + K, extra_rows=3)
    rows = int(offs[-1])
    steps = 257 + sa.shape[1]
    if form.startswith("powers"):
        steps = 2 * K
        for t in (sa, sb):
            t.copy_(torch.exp2(torch.randint(-6, 7, t.shape, generator=_gen(8), device="cuda").float()))
        sa[rows:] = 0.3  # behind the last group: no scale of the product
    acc, mag = _exact(a, b, offs, sa, sb)
    tol = steps * U * mag
    out = fp8_block.grouped_mm_fp8_block(a, b, offs, sa, sb)
    _within("no bias", out[:rows], acc[:rows], (tol + 2.0 ** -8 * acc.abs())[:rows])
    biased = acc + bias.double()[_row_of(offs, acc.shape[0])]
    tol = tol + U * biased.abs()
    out = fp8_block.grouped_mm_fp8_block(a, b, offs, sa, sb, bias)
    _within("bias", out[:rows], biased[:rows], (tol + 2.0 ** -8 * biased.abs())[:rows])
    # SwiGLU in a range where it is not all clamped
    sa2 = sa * 2.0 ** -10
    sa2 = torch.empty_strided(sa.shape, sa.stride(), device="cuda").copy_(sa2)
    bias2 = (bias.float() / 64).to(torch.bfloat16)
    acc2, mag2 = acc * 2.0 ** -10, mag * 2.0 ** -10
    biased = acc2 + bias2.double()[_row_of(offs, acc.shape[0])]
    s, aux = fp8_block.grouped_mm_swiglu_fp8_block(a, b, offs, sa2, sb, bias2, ALPHA, LIMIT)
    _within("aux", aux[:rows], biased[:rows],
            (steps * U * mag2 + U * biased.abs() + 2.0 ** -8 * biased.abs())[:rows])
    gate, up = aux.double()[:, 0::2].clamp(max=LIMIT), aux.double()[:, 1::2].clamp(-LIMIT, LIMIT)
    ref = gate * torch.sigmoid(ALPHA * gate) * (up + 1)
    # exp of an argument of up to |alpha gate| with a rounding of its own: |z| u; u + 1 loses |up| u absolutely
    cond = (gate * torch.sigmoid(ALPHA * gate)).abs() * ((up + 1).abs() * (8 + 4 * (ALPHA * gate).abs()) + 2 * up.abs())
    _within("swiglu", s[:rows], ref[:rows], (8 * U * cond + 2.0 ** -8 * ref.abs() + 2.0 ** -126 * (gate * (up + 1)).abs())[:rows])
    # SwiGLU backward against an aux with clamped and unclamped values
    aux_in = (4 * torch.randn(a.shape[0], 2 * N, generator=_gen(9), device="cuda")).to(torch.bfloat16)
    got = fp8_block.grouped_mm_swiglu_bwd_fp8_block(a, b, offs, aux_in, sa2, sb, ALPHA, LIMIT)
    g0, u0 = aux_in.double()[:, 0::2], aux_in.double()[:, 1::2]
    gc, uc = g0.clamp(max=LIMIT), u0.clamp(-LIMIT, LIMIT)
    sig = torch.sigmoid(ALPHA * gc)
    err = steps * U * mag2
    fg = (uc + 1) * sig * (1 + ALPHA * gc * (1 - sig)) * (g0 <= LIMIT)
    fu = gc * sig * (u0.abs() <= LIMIT)
    z = (ALPHA * gc).abs()
    cg = sig * ((uc + 1).abs() * (1 + z) * (16 + 8 * z) + 2 * uc.abs() * (1 + z))
    cu = gc.abs() * sig * (8 + 4 * z)
    tiny = 2.0 ** -126 * acc2.abs() * ((uc + 1).abs() + gc.abs()) * (1 + z)
    for name, f, c, part in (("d_gate", fg, cg, got[:, 0::2]), ("d_up", fu, cu, got[:, 1::2])):
        ref = acc2 * f
        _within(name, part[:rows], ref[:rows],
                (err * (f.abs() + 8 * U * c) + 8 * U * c * acc2.abs() + 2.0 ** -8 * ref.abs() + tiny + 1e-37)[:rows])
    m.check_device_status()


def test_rows_behind_the_last_group_stay_as_they_were():
    """The launcher writes rows of groups only: an output that the caller filled keeps the others."""
    import ctypes

    from cutlass_op.bf16_grouped_mm import _ext, fp8_block

    a, b, offs, sa, sb, bias = _case(3, 256, 256, [5, 0, 130], "kn", 1, extra_rows=200)
    want = fp8_block.grouped_mm_fp8_block(a, b, offs, sa, sb, bias)
    out = torch.full((a.shape[0], 256), 7.0, dtype=torch.bfloat16, device="cuda")

    class Desc(ctypes.Structure):  # include/moe_gemm.h: mgf_block_gemm_desc
        i32, i64, ptr, f32 = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p, ctypes.c_float
        _fields_ = [("epilogue", i32), ("num_groups", i32), ("total_rows", i64), ("n", i64), ("k", i64), ("a", ptr),
                    ("lda", i64), ("b", ptr), ("ldb", i64), ("ldb_batch", i64), ("b_mn_major", i32),
                    ("sm_carveout", i32), ("offs", ptr), ("scale_a", ptr), ("scale_a_stride", i64), ("scale_b", ptr),
                    ("scale_b_stride_e", i64), ("scale_b_stride_k", i64), ("scale_b_stride_n", i64), ("bias", ptr),
                    ("bias_stride", i64), ("d", ptr), ("ldd", i64), ("d2", ptr), ("ldd2", i64), ("aux", ptr),
                    ("ld_aux", i64), ("swiglu_alpha", f32), ("swiglu_limit", f32), ("workspace", ptr)]

    _ext.lib.mgf_block_gemm_desc_size.restype = ctypes.c_size_t
    assert ctypes.sizeof(Desc) == _ext.lib.mgf_block_gemm_desc_size()
    d = Desc(0, 3, a.shape[0], 256, 256, a.data_ptr(), a.stride(0), b.data_ptr(), b.stride(1), b.stride(0), 1, 0,
             offs.data_ptr(), sa.data_ptr(), sa.stride(0), sb.data_ptr(), *sb.stride(), bias.data_ptr(), 256,
             out.data_ptr(), 256, None, 0, None, 0, ALPHA, LIMIT, None)
    _ext.lib.mgf_block_gemm_launch.argtypes = [ctypes.c_void_p, ctypes.c_void_p]
    assert _ext.lib.mgf_block_gemm_launch(ctypes.byref(d), torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(out[:135], want[:135]) and (out[135:] == 7.0).all()


def test_malformed_offs_are_clamped_and_reported(monkeypatch):
    from cutlass_op.bf16_grouped_mm import fp8_block
    from cutlass_op.bf16_grouped_mm._ext import DEV_BAD_OFFS, device_status

    device_status()
    a, b, offs, sa, sb, _ = _case(3, 128, 128, [10, 10, 10], "kn", 2)
    for mx in ("0", "1"):
        monkeypatch.setenv("MGF_BLOCK_MX", mx)
        if mx == "1":
            sa.fill_(0.25), sb.fill_(4.0)
        good = fp8_block.grouped_mm_fp8_block(a, b, offs, sa, sb)
        bad = torch.tensor([10, 20, 5000], dtype=torch.int32, device="cuda")
        assert torch.equal(fp8_block.grouped_mm_fp8_block(a, b, bad, sa, sb), good)
        assert device_status() == DEV_BAD_OFFS
        # decreasing: group 0 has rows 0 .. 19, the others none
        bad = torch.tensor([20, 10, 5], dtype=torch.int32, device="cuda")
        fixed = torch.tensor([20, 20, 20], dtype=torch.int32, device="cuda")
        want = fp8_block.grouped_mm_fp8_block(a, b, fixed, sa, sb)[:20]
        assert device_status() == 0
        assert torch.equal(fp8_block.grouped_mm_fp8_block(a, b, bad, sa, sb)[:20], want)
        assert device_status() == DEV_BAD_OFFS


def test_product_refusals():
    from cutlass_op.bf16_grouped_mm import fp8_block

    a, b, offs, sa, sb, bias = _case(2, 256, 256, [10, 10], "kn", 3)
    f = fp8_block.grouped_mm_fp8_block
    for args, words in [
        ((a.float(), b, offs, sa, sb), "float8"),
        ((a, b[:, :128], offs, sa, sb), "contraction"),
        ((a, b[..., :250], offs, sa, sb), "multiple of 8"),
        ((a, b, offs.long(), sa, sb), "int32"),
        ((a, b, offs[:1], sa, sb), "int32"),
        ((a, b, offs, sa[:, :1], sb), "scale_a"),
        ((a, b, offs, sa.double(), sb), "scale_a"),
        ((a, b, offs, sa.t().contiguous().t(), sb), "scale_a"),
        ((a, b, offs, sa, sb[:, :, :1]), "scale_b"),
        ((a, b, offs, sa, sb, bias.float()), "bias"),
        ((a, b, offs, sa, sb, bias[:, :128]), "bias"),
        ((a, b.cpu(), offs, sa, sb), "CUDA"),
        ((a[:, 1:129], b[:, :128], offs, sa[:, :1], sb[:, :1]), "aligned"),
    ]:
        with pytest.raises(RuntimeError, match=words):
            f(*args)
    with pytest.raises(RuntimeError, match="multiple of 16"):
        fp8_block.grouped_mm_swiglu_fp8_block(a, b[..., :248], offs, sa, sb, bias[:, :248].contiguous())
    with pytest.raises(RuntimeError, match="aux"):
        fp8_block.grouped_mm_swiglu_bwd_fp8_block(a, b, offs, torch.zeros(20, 256, device="cuda", dtype=torch.bfloat16),
                                                  sa, sb)


@pytest.mark.parametrize("mx", ["0", "1"])
@pytest.mark.parametrize("cg", ["1", "2"])
def test_waits_that_run_out_are_reported_and_leave_the_device_usable(mx, cg, monkeypatch):
    """The launcher's test hook hands out no tiles, so every consumer's bounded wait gives up with nothing in
    flight; the next launch is right."""
    from cutlass_op.bf16_grouped_mm import fp8_block
    from cutlass_op.bf16_grouped_mm._ext import DEV_WAIT_TIMEOUT, device_status

    monkeypatch.setenv("MGF_BLOCK_MX", mx)
    monkeypatch.setenv("MGF_CTA_GROUP", cg)
    a, b, offs, sa, sb, bias = _case(2, 256, 256, [130, 10], "kn", 4)
    sa.fill_(0.5)
    sb.fill_(2.0)
    device_status()
    want = fp8_block.grouped_mm_fp8_block(a, b, offs, sa, sb, bias)
    assert device_status() == 0
    monkeypatch.setenv("MGF_TEST_STALL_PRODUCER", "1")
    fp8_block.grouped_mm_fp8_block(a, b, offs, sa, sb, bias)
    assert device_status() == DEV_WAIT_TIMEOUT
    monkeypatch.delenv("MGF_TEST_STALL_PRODUCER")
    assert torch.equal(fp8_block.grouped_mm_fp8_block(a, b, offs, sa, sb, bias), want) and device_status() == 0


def test_two_streams_and_a_captured_launch_with_new_scales(monkeypatch):
    """Two launches at once have scratch of their own; a captured launch chooses its form anew on every replay."""
    from cutlass_op.bf16_grouped_mm import fp8_block

    monkeypatch.setenv("MGF_BLOCK_MX", "1")
    a, b, offs, sa, sb, bias = _case(4, 512, 384, [300, 7, 0, 900], "kn", 6)
    powers = torch.exp2(torch.randint(-3, 4, sa.shape, generator=_gen(1), device="cuda").float())
    sa1 = torch.empty_strided(sa.shape, sa.stride(), device="cuda").copy_(powers)
    sb1 = torch.ones_like(sb)
    f = fp8_block.grouped_mm_fp8_block
    want = [f(a, b, offs, sa, sb, bias), f(a, b, offs, sa1, sb1, bias)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(4):
        for s, scales in zip(streams, ((sa, sb), (sa1, sb1))):
            with torch.cuda.stream(s):
                got.append(f(a, b, offs, *scales, bias))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert torch.equal(g, want[i % 2])
    xa, xb = sa.clone(memory_format=torch.preserve_format), sb.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = f(a, b, offs, xa, xb, bias)
    for i, scales in ((1, (sa1, sb1)), (0, (sa, sb)), (1, (sa1, sb1))):
        xa.copy_(scales[0])
        xb.copy_(scales[1])
        graph.replay()
        assert torch.equal(out, want[i])


@pytest.mark.parametrize("powers", [False, True])
def test_few_rows_over_much_weight(powers, monkeypatch):
    """Few rows, but so many blocks of weights that the launcher itself offers them to the form with the scales in the
    tensor cores; which form runs is the scales' matter."""
    import cutlass_op.bf16_grouped_mm as m
    from cutlass_op.bf16_grouped_mm import fp8_block

    for name in ("MGF_BLOCK_MX", "MGF_CTA_GROUP", "MGF_BN"):
        monkeypatch.delenv(name, raising=False)
    K, N = 2200, 4200
    counts = [1, 0, 5, 40, 2, 33] + [1] * 64
    a, b, offs, sa, sb, bias = _case(len(counts), K, N, counts, "kn", 11, extra_rows=2)
    if powers:
        for t in (sa, sb):
            t.copy_(torch.exp2(torch.randint(-6, 7, t.shape, generator=_gen(8), device="cuda").float()))
    acc, mag = _exact(a, b, offs, sa, sb)
    biased = acc + bias.double()[_row_of(offs, acc.shape[0])]
    rows = int(offs[-1])
    tol = (2 * K if powers else 257 + sa.shape[1]) * U * mag + U * biased.abs() + 2.0 ** -8 * biased.abs()
    out = fp8_block.grouped_mm_fp8_block(a, b, offs, sa, sb, bias)
    _within("out", out[:rows], biased[:rows], tol[:rows])
    m.check_device_status()

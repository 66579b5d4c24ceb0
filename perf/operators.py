"""Cases of the operators of a mixture-of-experts block around the grouped products, for measurement.

The operators (package ``cutlass_op.bf16_grouped_mm``):

* ``routing.moe_route``: router logits -> the top-k experts of every token and their weights, and the
  gradient of the logits;
* ``permute.moe_permute`` / ``moe_unpermute``: tokens sorted by expert and back, with the weights
  applied, and the gradients of tokens, rows and weights;
* ``fp8_block.quantize_*_block`` / ``permute.moe_permute_fp8``: e4m3 codes with one power-of-two scale
  for each 1 x 128 block of an activation row and each 128 x 128 block of a weight;
* ``fp8_block.grouped_mm_*_fp8_block``: the grouped product of such operands (bias, SwiGLU and SwiGLU
  backward epilogues).

``own = False`` computes the plain form of each from elementary torch operations in 32 bits; ``own =
True`` makes the calls a user makes.
"""

import math

import torch

own = False

BLOCK = 128
ALPHA, LIMIT = 1.702, 7.0


def _modules():
    import sys

    if "cute-moe-train_b200" not in sys.path:
        sys.path.insert(0, "cute-moe-train_b200")
    from cutlass_op.bf16_grouped_mm import fp8_block, permute, routing

    return routing, permute, fp8_block


# ------------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # one decoding step of eight sequences: latency only
        {"name": "route_decode", "op": "route", "T": 8, "E": 32, "k": 4, "dtype": "bf16", "score": "softmax",
         "renorm": True, "bias": False, "masked": False, "train": False},
        # the router of one training step, weights and the gradient of the logits
        {"name": "route_train", "op": "route", "T": 24576, "E": 128, "k": 4, "dtype": "bf16", "score": "softmax",
         "renorm": True, "bias": False, "masked": False, "train": True},
        # many fine-grained experts, fp32 logits, sigmoid scores with a balancing bias, a padded batch
        {"name": "route_fine", "op": "route", "T": 16384, "E": 256, "k": 8, "dtype": "fp32", "score": "sigmoid",
         "renorm": True, "bias": True, "masked": True, "train": True},
        # decoding: the copies of eight tokens in expert order
        {"name": "permute_decode", "op": "permute", "T": 8, "H": 2880, "E": 32, "k": 4, "dtype": "bf16",
         "drop": 0.0, "train": False},
        # a training step of the GPT-OSS widths, with the tokens' gradient
        {"name": "permute_train", "op": "permute", "T": 24576, "H": 2880, "E": 128, "k": 4, "dtype": "bf16",
         "drop": 0.0, "train": True},
        # decoding: the weighted sums of eight tokens' expert outputs
        {"name": "unpermute_decode", "op": "unpermute", "T": 8, "H": 2880, "E": 32, "k": 4, "dtype": "bf16",
         "drop": 0.0, "train": False},
        # a training step: weighted sums, the rows' and the weights' gradients; a tenth of the copies dropped
        {"name": "unpermute_train", "op": "unpermute", "T": 16384, "H": 7168, "E": 256, "k": 8, "dtype": "bf16",
         "drop": 0.1, "train": True},
        # tokens to e4m3 rows in expert order, what an inference batch feeds the up-projection with
        {"name": "permute_fp8", "op": "permute_fp8", "T": 8192, "H": 7168, "E": 256, "k": 8, "drop": 0.0},
        # the up-projection weights of one layer to codes, once per optimizer step
        {"name": "quantize_weights", "op": "quantize_weights", "E": 32, "K": 2880, "N": 5760},
        # decoding: 32 rows over 32 experts, the experts' weights are what is read
        {"name": "mm_decode", "op": "mm", "epi": "swiglu", "layout": "kn", "rows": 32, "E": 32, "K": 2880, "N": 5760},
        # the up-projection of a training step
        {"name": "mm_train", "op": "mm", "epi": "swiglu", "layout": "kn", "rows": 98304, "E": 32, "K": 2880,
         "N": 5760},
        # fine-grained experts: the down-projection's input gradient through SwiGLU
        {"name": "mm_dgrad_fine", "op": "mm", "epi": "swiglu_bwd", "layout": "nk", "rows": 32768, "E": 256,
         "K": 7168, "N": 2048},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["route", "permute", "unpermute", "permute_fp8", "quantize_weights", "mm", "mm"])
    T, E = _log_int(rng, 1, 24576), _log_int(rng, 4, 256)
    k = rng.randint(1, min(8, E))
    if op == "route":
        return {"op": op, "T": T, "E": E, "k": k, "dtype": rng.choice(["bf16", "fp16", "fp32"]),
                "score": rng.choice(["softmax", "sigmoid"]), "renorm": rng.random() < 0.7, "bias": rng.random() < 0.4,
                "masked": rng.random() < 0.4, "train": rng.random() < 0.7}
    H = _log_int(rng, 16, 7168)
    T = min(T, 16384 * 7168 * 8 // (H * k))
    if op in ("permute", "unpermute"):
        return {"op": op, "T": T, "H": H, "E": E, "k": k, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                "drop": rng.choice([0.0, 0.0, 0.1]), "train": rng.random() < 0.7}
    if op == "permute_fp8":
        return {"op": op, "T": T, "H": 8 * max(2, H // 8), "E": E, "k": k, "drop": rng.choice([0.0, 0.1])}
    K, N = _log_int(rng, 64, 7168), 16 * _log_int(rng, 4, 360)
    while E * K * N > 256 * 7168 * 2048:
        E //= 2
    if op == "quantize_weights":
        E = max(1, min(E, 32 * 2880 * 5760 // (K * N)))
        return {"op": op, "E": E, "K": K, "N": N}
    rows = min(_log_int(rng, 1, 98304), 98304 * 2880 * 5760 // (K * N))
    epi = rng.choice(["bias", "swiglu", "swiglu_bwd"])
    return {"op": op, "epi": epi, "layout": rng.choice(["kn", "nk"]), "rows": rows, "E": E, "K": K, "N": N}


# ------------------------------------------------------------------------------------------------ inputs

_DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 2654435761 % (1 << 31) + 1)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _popularity(g, E):
    """Log weights of the experts: Zipf(1.1) over a random order."""
    order = torch.rand(E, generator=g, device="cuda").argsort()
    return -1.1 * torch.log1p(order.float())


def _expert_ids(g, T, E, k, drop):
    """[T, k] distinct experts per token; a share `drop` of the copies is dropped (-1)."""
    keys = _popularity(g, E) - torch.log(-torch.log(torch.rand(T, E, generator=g, device="cuda").clamp(1e-9, 1 - 1e-6)))
    idx = keys.topk(k, dim=1).indices
    if drop:
        idx = torch.where(torch.rand(T, k, generator=g, device="cuda") < drop, torch.full_like(idx, -1), idx)
    return idx


def _plan(idx, E):
    """(offs, row_of_copy, copy_of_row) of a stable sort of the copies by expert; -1 = no row / no copy."""
    flat = idx.reshape(-1)
    order = torch.sort(torch.where(flat < 0, torch.full_like(flat, E), flat), stable=True).indices
    counts = torch.zeros(E + 1, dtype=torch.int64, device=flat.device)
    counts.index_add_(0, torch.where(flat < 0, torch.full_like(flat, E), flat), torch.ones_like(flat))
    offs = counts[:E].cumsum(0)
    place = torch.arange(flat.numel(), device=flat.device)
    copy_of_row = torch.where(place < offs[-1], order, torch.full_like(order, -1))
    row_of_copy = torch.empty_like(order)
    row_of_copy[order] = torch.where(place < offs[-1], place, torch.full_like(place, -1))
    return offs.int(), row_of_copy.int().view(idx.shape), copy_of_row.int()


def _pitched(t, pitch):
    """`t` with its rows `pitch` elements apart at multiples of it."""
    wide = -(-t.shape[-1] // pitch) * pitch
    out = torch.zeros(*t.shape[:-1], wide, dtype=t.dtype, device=t.device)[..., :t.shape[-1]]
    out.copy_(t)
    return out


def _power_of_two(amax):
    """The smallest power of two s with amax / s <= 448 (1 where amax is 0)."""
    mant, expo = torch.frexp(amax / 1.75)  # amax / 1.75 = mant * 2^expo, mant in [0.5, 1)
    e = torch.where(mant == 0.5, expo - 1, expo) - 8
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), e.clamp(min=-126)), torch.ones_like(amax))


def _blocks(v, dim):
    """`v` with dimension `dim` padded with zeros and split into blocks of 128."""
    n = v.shape[dim]
    pad = -n % BLOCK
    if pad:
        shape = list(v.shape)
        shape[dim] = pad
        v = torch.cat([v, v.new_zeros(shape)], dim)
    return v.unflatten(dim, ((n + pad) // BLOCK, BLOCK))


def _row_codes(x):
    """(e4m3 codes, scales [rows, blocks]) of 1 x 128 blocks."""
    v = _blocks(x.float(), 1)
    s = _power_of_two(v.abs().amax(2))
    return (v / s[..., None]).flatten(1)[:, :x.shape[1]].to(torch.float8_e4m3fn), s


def _weight_codes(w):
    """(e4m3 codes, scales [experts, K blocks, N blocks]) of 128 x 128 blocks."""
    v = _blocks(_blocks(w.float(), 2), 1)
    s = _power_of_two(v.abs().amax((2, 4)))
    q = (v / s[:, :, None, :, None]).flatten(3, 4).flatten(1, 2)[:, :w.shape[1], :w.shape[2]]
    return q.to(torch.float8_e4m3fn), s


def _group_sizes(g, rows, E):
    """Rows of each expert: one draw of a Zipf(1.1) choice per row, as routing gives them."""
    p = torch.softmax(_popularity(g, E), 0)
    pick = torch.multinomial(p, rows, replacement=True, generator=g)
    return torch.zeros(E, dtype=torch.int64, device="cuda").index_add_(0, pick, torch.ones_like(pick))


def prepare(case, seed):
    g = _generator(seed)
    op = case["op"]
    if op == "route":
        T, E, k = case["T"], case["E"], case["k"]
        s = {"case": case, "logits": (1.5 * _randn(g, T, E)).to(_DTYPE[case["dtype"]]), "bias": None, "mask": None}
        if case["bias"]:
            s["bias"] = 0.1 * _randn(g, E)
        if case["masked"]:
            s["mask"] = torch.rand(T, generator=g, device="cuda") < 0.9
        s["grad"] = _randn(g, T, k)
        s["logits"].requires_grad_(case["train"])
        return s
    if op in ("permute", "unpermute", "permute_fp8"):
        T, H, E, k = case["T"], case["H"], case["E"], case["k"]
        dt = _DTYPE[case.get("dtype", "bf16")]
        idx = _expert_ids(g, T, E, k, case["drop"])
        if op != "unpermute":
            x = _randn(g, T, H).to(dt).requires_grad_(case.get("train", False))
            grad = _pitched(_randn(g, T * k, H).to(dt), 16 // dt.itemsize) if case.get("train") else None
            return {"case": case, "x": x, "idx": idx, "grad": grad}
        rows = _pitched(_randn(g, T * k, H).to(dt), 16 // dt.itemsize).detach().requires_grad_(case["train"])
        w = torch.softmax(_randn(g, T, k), 1).detach().requires_grad_(case["train"])
        return {"case": case, "rows": rows, "weights": w, "plan": _plan(idx, E),
                "grad": _randn(g, T, H).to(dt) if case["train"] else None}
    E, K, N = case["E"], case["K"], case["N"]
    if op == "quantize_weights":
        w = torch.empty(E, K, N, dtype=torch.bfloat16, device="cuda")
        for e in range(E):
            w[e] = _randn(g, K, N) / math.sqrt(K)
        return {"case": case, "w": w}
    counts = _group_sizes(g, case["rows"], E)
    sizes = counts.tolist()
    qa, sa = _row_codes(_randn(g, case["rows"], K).to(torch.bfloat16))
    # the weights' codes as a layer keeps them: [E, K, N] with unit stride along N, or (the input
    # gradient's view of the other projection) the transpose of [E, N, K] with unit stride along K
    shape = (E, K, N) if case["layout"] == "kn" else (E, N, K)
    qb = torch.zeros(*shape[:2], -(-shape[2] // 16) * 16, dtype=torch.float8_e4m3fn, device="cuda")[..., :shape[2]]
    sb = torch.empty(E, -(-shape[1] // BLOCK), -(-shape[2] // BLOCK), device="cuda")
    for e in range(E):
        q, sc = _weight_codes((_randn(g, 1, *shape[1:]) / math.sqrt(K)).to(torch.bfloat16))
        qb[e], sb[e] = q[0], sc[0]
    if case["layout"] == "nk":
        qb, sb = qb.transpose(1, 2), sb.transpose(1, 2)
    s = {"case": case, "qa": _pitched(qa, 16), "sa": _pitched(sa, 4), "qb": qb, "sb": sb, "sizes": sizes,
         "offs": counts.cumsum(0).int(), "bias": None, "aux": None}
    if case["epi"] != "swiglu_bwd":
        s["bias"] = (0.02 * _randn(g, E, N)).to(torch.bfloat16)
    else:
        s["aux"] = (1.5 * _randn(g, case["rows"], 2 * N)).to(torch.bfloat16)
    return s


# ------------------------------------------------------------------------------------------------ plain forms

def _route_plain(s):
    case, k = s["case"], s["case"]["k"]
    logits = s["logits"].detach().float()
    key = logits if s["bias"] is None else logits + s["bias"]
    idx = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :k]
    if case["score"] == "softmax":
        if case["renorm"]:
            p = torch.gather(logits, 1, idx)
            p = torch.exp(p - p.amax(1, keepdim=True))
            w = p / p.sum(1, keepdim=True)
        else:
            full = torch.exp(logits - logits.amax(1, keepdim=True))
            full = full / full.sum(1, keepdim=True)
            w = torch.gather(full, 1, idx)
    else:
        chosen = torch.gather(logits, 1, idx)
        sig = 1 / (1 + torch.exp(-chosen))
        w = sig / sig.sum(1, keepdim=True) if case["renorm"] else sig
    out = w
    if s["mask"] is not None:
        out = torch.where(s["mask"][:, None], w, torch.zeros_like(w))
        idx_out = torch.where(s["mask"][:, None], idx, torch.full_like(idx, -1))
    else:
        idx_out = idx
    if not case["train"]:
        return [out, idx_out]
    g = s["grad"] if s["mask"] is None else torch.where(s["mask"][:, None], s["grad"], torch.zeros_like(s["grad"]))
    if case["score"] == "softmax" and not case["renorm"]:
        d = torch.zeros_like(logits).scatter_(1, idx, g)
        d = full * (d - (w * g).sum(1, keepdim=True))
    else:
        d = w * (g - (w * g).sum(1, keepdim=True)) if case["renorm"] else w * g
        if case["score"] == "sigmoid":
            d = d * (1 - sig)
        d = torch.zeros_like(logits).scatter_(1, idx, d)
    return [out, idx_out, d.to(s["logits"].dtype)]


def _take_rows(v, index):
    """v[index], and zeros where the index is -1."""
    picked = v[index.clamp(min=0).long()]
    return torch.where((index >= 0)[..., None], picked, torch.zeros_like(picked))


def _permute_plain(s):
    case = s["case"]
    x = s["x"].detach()
    plan = _plan(s["idx"], case["E"])
    offs, row_of_copy, copy_of_row = plan
    token = torch.where(copy_of_row < 0, copy_of_row, torch.div(copy_of_row, case["k"], rounding_mode="floor"))
    out = {"rows": _take_rows(x, token), "offs": offs, "row_of_copy": row_of_copy, "copy_of_row": copy_of_row}
    if case["train"]:
        out["dx"] = _take_rows(s["grad"].float(), row_of_copy).sum(1).to(x.dtype)
    return out


def _unpermute_plain(s):
    case = s["case"]
    rows, w = s["rows"].detach(), s["weights"].detach()
    _, row_of_copy, copy_of_row = s["plan"]
    copies = _take_rows(rows.float(), row_of_copy)
    out = {"out": (copies * w[..., None]).sum(1).to(rows.dtype)}
    if case["train"]:
        g = s["grad"].float()
        token = torch.where(copy_of_row < 0, copy_of_row, torch.div(copy_of_row, case["k"], rounding_mode="floor"))
        w_row = torch.where(copy_of_row < 0, torch.zeros_like(copy_of_row, dtype=torch.float32),
                            w.reshape(-1)[copy_of_row.clamp(min=0).long()])
        out["drows"] = (_take_rows(g, token) * w_row[:, None]).to(rows.dtype)
        out["dweights"] = (copies * g[:, None, :]).sum(2)
    return out


def _permute_fp8_plain(s):
    case = s["case"]
    offs, row_of_copy, copy_of_row = _plan(s["idx"], case["E"])
    token = torch.where(copy_of_row < 0, copy_of_row, torch.div(copy_of_row, case["k"], rounding_mode="floor"))
    q, scale = _row_codes(s["x"].detach())
    q = q.view(torch.uint8)[token.clamp(min=0).long()]
    q = torch.where((token >= 0)[:, None], q, torch.zeros_like(q)).view(torch.float8_e4m3fn)
    return {"codes": q, "scales": _take_rows(scale, token), "offs": offs, "row_of_copy": row_of_copy,
            "copy_of_row": copy_of_row}


def _spread(s, rows, cols):
    """Block scales [rows / 128, cols / 128] at every element."""
    return s.repeat_interleave(BLOCK, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :cols]


def _swiglu(aux):
    g, u = aux[:, 0::2].float().clamp(max=LIMIT), aux[:, 1::2].float().clamp(-LIMIT, LIMIT)
    return g / (1 + torch.exp(-ALPHA * g)) * (u + 1)


def _swiglu_bwd(gs, aux):
    g, u = aux[:, 0::2].to(gs.dtype), aux[:, 1::2].to(gs.dtype)
    gc, uc = g.clamp(max=LIMIT), u.clamp(-LIMIT, LIMIT)
    sig = 1 / (1 + torch.exp(-ALPHA * gc))
    dg = torch.where(g <= LIMIT, gs * (uc + 1) * sig * (1 + ALPHA * gc * (1 - sig)), torch.zeros_like(gs))
    du = torch.where((u >= -LIMIT) & (u <= LIMIT), gs * gc * sig, torch.zeros_like(gs))
    return torch.stack([dg, du], 2).flatten(1)


def _mm_plain(s):
    case = s["case"]
    K, N = case["K"], case["N"]
    a = (_blocks(s["qa"].float(), 1) * s["sa"][..., None]).flatten(1)[:, :K]
    acc = torch.empty(case["rows"], N, device="cuda")
    at = 0
    for e, m in enumerate(s["sizes"]):  # the experts' products are of different heights
        if m:
            b = s["qb"][e].float() * _spread(s["sb"][e], K, N)
            torch.matmul(a[at:at + m], b, out=acc[at:at + m])
            if s["bias"] is not None:
                acc[at:at + m] += s["bias"][e].float()
            at += m
    if case["epi"] == "bias":
        return [acc.to(torch.bfloat16)]
    if case["epi"] == "swiglu":
        aux = acc.to(torch.bfloat16)
        return [_swiglu(aux).to(torch.bfloat16), aux]
    return [_swiglu_bwd(acc, s["aux"]).to(torch.bfloat16)]


_PLAIN = {"route": _route_plain, "permute": _permute_plain, "unpermute": _unpermute_plain,
          "permute_fp8": _permute_fp8_plain, "quantize_weights": lambda s: list(_weight_codes(s["w"])),
          "mm": _mm_plain}


# ------------------------------------------------------------------------------------------------ the framework's calls

def _run_own(s):
    routing, permute, fp8_block = _modules()
    case = s["case"]
    op = case["op"]
    if op == "route":
        w, idx = routing.moe_route(s["logits"], case["k"], score=case["score"], renormalize=case["renorm"],
                                   bias=s["bias"], token_mask=s["mask"])
        if not case["train"]:
            return [w, idx]
        return [w, idx, torch.autograd.grad(w, s["logits"], s["grad"])[0]]
    if op == "permute":
        rows, plan = permute.moe_permute(s["x"], s["idx"], case["E"])
        out = {"rows": rows, "offs": plan.offs, "row_of_copy": plan.row_of_copy, "copy_of_row": plan.copy_of_row}
        if case["train"]:
            out["dx"] = torch.autograd.grad(rows, s["x"], s["grad"])[0]
        return out
    if op == "unpermute":
        y = permute.moe_unpermute(s["rows"], permute.MoEPlan(*s["plan"]), s["weights"])
        out = {"out": y}
        if case["train"]:
            out["drows"], out["dweights"] = torch.autograd.grad(y, (s["rows"], s["weights"]), s["grad"])
        return out
    if op == "permute_fp8":
        q, scale, plan = permute.moe_permute_fp8(s["x"], s["idx"], case["E"])
        return {"codes": q, "scales": scale, "offs": plan.offs, "row_of_copy": plan.row_of_copy,
                "copy_of_row": plan.copy_of_row}
    if op == "quantize_weights":
        return list(fp8_block.quantize_weights_block(s["w"]))
    a = (s["qa"], s["qb"], s["offs"], s["sa"], s["sb"])
    if case["epi"] == "bias":
        return [fp8_block.grouped_mm_fp8_block(*a, s["bias"])]
    if case["epi"] == "swiglu":
        return list(fp8_block.grouped_mm_swiglu_fp8_block(*a, s["bias"], ALPHA, LIMIT))
    return [fp8_block.grouped_mm_swiglu_bwd_fp8_block(*a[:3], s["aux"], *a[3:], ALPHA, LIMIT)]


def run(state):
    if own:
        return _run_own(state)
    return _PLAIN[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------ what a pass cannot do without

def work(case):
    op = case["op"]
    size = {"bf16": 2, "fp16": 2, "fp32": 4}.get(case.get("dtype", "bf16"))
    if op == "route":
        T, E, k = case["T"], case["E"], case["k"]
        # logits in; weights (fp32) and ids (64 bits) out; the weights' gradient in and the logits' out
        b = T * E * size + T * k * 12 + (4 * E if case["bias"] else 0) + (T if case["masked"] else 0)
        if case["train"]:
            b += T * k * 4 + T * E * size
        return {"bytes": b, "flops": 4 * T * E}
    if op in ("permute", "unpermute", "permute_fp8"):
        T, H, E, k = case["T"], case["H"], case["E"], case["k"]
        n = T * k
        kept = n * (1 - case["drop"])
        if op == "permute":
            b = T * H * size + n * H * size + n * 16 + 4 * E
            if case["train"]:
                b += kept * H * size + T * H * size
            return {"bytes": b, "flops": n * H if case["train"] else 0}
        if op == "permute_fp8":
            return {"bytes": T * H * 2 + n * H + n * -(-H // BLOCK) * 4 + n * 16 + 4 * E, "flops": 2 * T * H}
        b = kept * H * size + T * H * size + n * 8
        if case["train"]:  # output gradient in; rows' and weights' gradients out (the rows are read once)
            b += T * H * size + n * H * size + n * 8
        return {"bytes": b, "flops": (6 if case["train"] else 2) * n * H}
    E, K, N = case["E"], case["K"], case["N"]
    if op == "quantize_weights":
        return {"bytes": 3 * E * K * N + 4 * E * -(-K // BLOCK) * -(-N // BLOCK), "flops": 2 * E * K * N}
    M = case["rows"]
    # the expected number of experts with a row, by the distribution the rows are drawn from
    p = [(i + 1) ** -1.1 for i in range(E)]
    active = sum(1 - (1 - v / sum(p)) ** M for v in p)
    out = {"bias": 2 * N, "swiglu": 3 * N, "swiglu_bwd": 8 * N}[case["epi"]]
    b = M * K + 4 * M * -(-K // BLOCK) + active * (K * N + 4 * -(-K // BLOCK) * -(-N // BLOCK) + 2 * N) + M * out
    return {"bytes": b, "flops": 2 * M * K * N}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "route":
        return _route_exact(s)
    if op == "permute":
        return _permute_exact(s)
    if op == "unpermute":
        return _unpermute_exact(s)
    if op == "permute_fp8":
        x = s["x"].double()
        scale, code = _codes_exact(x, 1)
        owner = _owner_exact(s["idx"], case["E"])
        return {"codes": _by_owner(code, owner), "scales": _by_owner(scale, owner), "offs": None, "row_of_copy": None,
                "copy_of_row": None}
    if op == "quantize_weights":
        codes, scales = [], []
        for e in range(case["E"]):
            scale, code = _codes_exact(s["w"][e].double(), BLOCK)
            codes.append(code.float())
            scales.append(scale)
        return [torch.stack(codes), torch.stack(scales)]
    return _mm_exact(s)


def _route_exact(s):
    case = s["case"]
    z = s["logits"].detach().double()
    T, E, k = case["T"], case["E"], case["k"]
    key = s["logits"].detach().float() if s["bias"] is None else s["logits"].detach().float() + s["bias"]
    # the k largest, the earlier expert first among equals: rank = experts that come before
    chosen = torch.argsort(-key, dim=1, stable=True)[:, :k]
    hot = torch.zeros(T, E, dtype=torch.bool, device="cuda").scatter_(1, chosen, True)
    live = torch.ones(T, 1, dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"][:, None]
    z = z.requires_grad_(True)
    if case["score"] == "softmax":
        w = torch.softmax(z.masked_fill(~hot, -math.inf), 1) if case["renorm"] else torch.softmax(z, 1)
    else:
        w = torch.sigmoid(z)
        w = w / (w * hot).sum(1, keepdim=True) if case["renorm"] else w
    w = torch.gather(w, 1, chosen)
    w = torch.where(live, w, torch.zeros_like(w))
    out = [w.detach(), None]
    if case["train"]:
        out.append(torch.autograd.grad(w, z, s["grad"].double())[0])
    return out


def _owner_exact(idx, E):
    """Token of every row in expert order, -1 behind the last row."""
    T, k = idx.shape
    copies = torch.arange(T * k, device=idx.device)
    rank = torch.where(idx.reshape(-1) < 0, torch.full_like(copies, E), idx.reshape(-1)) * (T * k) + copies
    order = rank.argsort()
    return torch.where(idx.reshape(-1)[order] < 0, torch.full_like(order, -1), order // k)


def _by_owner(v, owner):
    out = torch.zeros(owner.numel(), v.shape[1], dtype=v.dtype, device=v.device)
    out[owner >= 0] = v[owner[owner >= 0]]
    return out


def _permute_exact(s):
    case = s["case"]
    owner = _owner_exact(s["idx"], case["E"])
    out = {"rows": _by_owner(s["x"].detach(), owner), "offs": None, "row_of_copy": None, "copy_of_row": None}
    if case["train"]:
        dx = torch.zeros(case["T"], case["H"], dtype=torch.float64, device="cuda")
        out["dx"] = dx.index_add_(0, owner[owner >= 0], s["grad"][owner >= 0].double())
    return out


def _unpermute_exact(s):
    case = s["case"]
    row_of_copy = s["plan"][1].long()
    y = torch.zeros(case["T"], case["H"], dtype=torch.float64, device="cuda")
    if case["train"]:
        drows = torch.zeros(case["T"] * case["k"], case["H"], dtype=torch.float64, device="cuda")
        dw = torch.zeros(case["T"], case["k"], dtype=torch.float64, device="cuda")
        g = s["grad"].double()
    for j in range(case["k"]):
        there = row_of_copy[:, j] >= 0
        at = row_of_copy[there, j]
        r = s["rows"].detach()[at].double()
        w = s["weights"].detach()[there, j].double()
        y[there] += w[:, None] * r
        if case["train"]:
            drows[at] = w[:, None] * g[there]
            dw[there, j] = (r * g[there]).sum(1)
    return {"out": y, "drows": drows, "dweights": dw} if case["train"] else {"out": y}


def _codes_exact(v, high):
    """(scales, codes as numbers) of `high` x 128 blocks of a matrix in 64 bits."""
    rows, cols = v.shape
    full = torch.zeros(-(-rows // high) * high, -(-cols // BLOCK) * BLOCK, dtype=torch.float64, device="cuda")
    full[:rows, :cols] = v
    tile = full.view(full.shape[0] // high, high, full.shape[1] // BLOCK, BLOCK)
    amax = tile.abs().amax((1, 3))
    e = torch.ceil(torch.log2(torch.where(amax > 0, amax, torch.full_like(amax, 448.0)) / 448.0))
    e = torch.where(torch.exp2(e) * 448.0 < amax, e + 1, e)  # log2 is not exact next to a power of two
    e = torch.where(torch.exp2(e - 1) * 448.0 >= amax, e - 1, e)
    scale = torch.exp2(torch.where(amax > 0, e, torch.zeros_like(e)))
    q = tile / scale[:, None, :, None]
    # e4m3: four significant bits, steps of 2^-9 below 2^-6, ties to even
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 3)
    q = torch.round(q / step) * step
    return scale, q.reshape(full.shape)[:rows, :cols]


def _mm_exact(s):
    case = s["case"]
    K, N, rows = case["K"], case["N"], case["rows"]
    if 2.0 * rows * K * N > 1e13:
        return None
    v = torch.zeros(rows, N, dtype=torch.float64, device="cuda")
    ends = s["offs"].tolist()
    for e, (lo, hi) in enumerate(zip([0] + ends[:-1], ends)):
        if hi > lo:
            for c in range(0, K, 16 * BLOCK):  # strips of the contraction, scaled block by block
                d = min(K, c + 16 * BLOCK)
                sa = s["sa"][lo:hi, c // BLOCK:-(-d // BLOCK)].double().repeat_interleave(BLOCK, 1)[:, :d - c]
                sb = s["sb"][e, c // BLOCK:-(-d // BLOCK)].double().repeat_interleave(BLOCK, 0)[:d - c]
                sb = sb.repeat_interleave(BLOCK, 1)[:, :N]
                v[lo:hi] += (s["qa"][lo:hi, c:d].double() * sa) @ (s["qb"][e, c:d].double() * sb)
            if s["bias"] is not None:
                v[lo:hi] += s["bias"][e].double()
    if case["epi"] == "bias":
        return [v]
    if case["epi"] == "swiglu":
        aux = v.to(torch.bfloat16).double()  # the activation is defined on the stored values
        gate, up = aux[:, 0::2].clamp(max=LIMIT), aux[:, 1::2].clamp(-LIMIT, LIMIT)
        return [gate * torch.sigmoid(ALPHA * gate) * (up + 1), v]
    gate, up = s["aux"][:, 0::2].double(), s["aux"][:, 1::2].double()
    gc, uc = gate.clamp(max=LIMIT), up.clamp(-LIMIT, LIMIT)
    sig = torch.sigmoid(ALPHA * gc)
    out = torch.zeros(rows, 2 * N, dtype=torch.float64, device="cuda")
    out[:, 0::2] = v * (uc + 1) * sig * (1 + ALPHA * gc * (1 - sig)) * (gate <= LIMIT)
    out[:, 1::2] = v * gc * sig * (up.abs() <= LIMIT)
    return [out]

"""The router's selection bias added to the scores ("biased_sigmoid", "biased_softmax"): which experts it chooses,
their weights and the logits' gradient, against the definition in 64 bits.

The kernel's keys are score + bias in fp32.  A sigmoid is off by at most 6 u of itself (u = 2^-24: exp 2 ulp = 4 u, sum
and quotient u each), a softmax over E <= 1024 experts by less than 128 u, and the sum with a bias below 2 rounds by 2 u:
below 130 u in all.  Choices are compared where the k + 1 largest sums of the definition lie further apart than twice that.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _scores(z, score):
    return torch.sigmoid(z) if score == "biased_sigmoid" else torch.softmax(z, 1)


def test_a_bias_on_the_score_chooses_other_experts_than_one_on_the_logit():
    from cutlass_op.bf16_grouped_mm.routing import moe_route

    logits = torch.tensor([[4.0, 1.0]], device="cuda")
    bias = torch.tensor([0.0, 0.4], device="cuda")
    assert moe_route(logits, 1, "sigmoid", bias=bias)[1].tolist() == [[0]]         # 4 against 1.4
    assert moe_route(logits, 1, "biased_sigmoid", bias=bias)[1].tolist() == [[1]]  # 0.982 against 1.131
    logits = torch.tensor([[2.0, 0.0, 1.0]], device="cuda")
    bias = torch.tensor([0.0, 0.7, 0.1], device="cuda")
    assert moe_route(logits, 2, "softmax", bias=bias)[1].tolist() == [[0, 2]]
    assert moe_route(logits, 2, "biased_softmax", bias=bias)[1].tolist() == [[1, 0]]  # 0.790, 0.665, 0.345


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("score", ["biased_sigmoid", "biased_softmax"])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (5, 4, 4), (130, 33, 5), (64, 128, 8), (40, 257, 8), (9, 1000, 32)])
def test_biased_scores_against_64_bits(T, E, k, renorm, score, dtype):
    from cutlass_op.bf16_grouped_mm.routing import moe_route

    g = _gen(T * 100 + E)
    leaf = (1.5 * torch.randn(T, E, generator=g, device="cuda")).to(dtype).requires_grad_(True)
    bias = (0.5 if score == "biased_sigmoid" else 2.0 / E) * torch.randn(E, generator=g, device="cuda")
    mask = torch.rand(T, generator=g, device="cuda") < 0.8 if T > 1 else None
    w, idx = moe_route(leaf, k, score, renorm, 2.5, bias, mask)
    z = leaf.detach().double()
    key = _scores(z, score) + bias.double()
    top = key.topk(min(k + 1, E), dim=1)
    clear = (top.values[:, :-1] - top.values[:, 1:] > 260 * U).all(1)
    live = torch.ones(T, dtype=torch.bool, device="cuda") if mask is None else mask
    assert clear.float().mean() > 0.4 or E > 500
    assert torch.equal(idx[clear & live], top.indices[clear & live][:, :k]) and (idx[~live] == -1).all()
    # whatever was chosen: the sums along the slots do not grow, and none left out is larger
    chosen = torch.gather(key, 1, idx.clamp(min=0))[live]
    assert (chosen[:, 1:] <= chosen[:, :-1] + 260 * U).all()
    rest = key[live].scatter(1, idx[live], -math.inf)
    assert (rest.amax(1) <= chosen[:, -1] + 260 * U).all()
    # weights and gradient are those of the chosen experts' scores, the bias has no part in them
    p = torch.gather(_scores(z, score), 1, idx.clamp(min=0))
    if renorm:
        if score == "biased_softmax":
            p = torch.softmax(torch.gather(z, 1, idx.clamp(min=0)), 1)
        else:
            p = p / p.sum(1, keepdim=True)
    ref = torch.where(live[:, None], 2.5 * p, 0.0)
    assert ((w.double() - ref).abs() <= 128 * U * ref).all()
    gw = torch.randn(T, k, generator=g, device="cuda")
    (dl,) = torch.autograd.grad(w, leaf, gw)
    # the same experts by a bias on the logits that leaves no others: the gradient does not know where the bias was added.
    # Both are off by 384 u * scale * 2 max|g| at most, and by half a step of the output
    picked = torch.full((T, E), -math.inf, device="cuda").scatter_(1, idx.clamp(min=0), 0.0)
    for t in range(min(T, 8)):
        if not live[t]:
            assert (dl[t] == 0).all()
            continue
        one = leaf.detach()[t:t + 1].clone().requires_grad_(True)
        w1, i1 = moe_route(one, k, score[7:], renorm, 2.5, picked[t])
        g1 = torch.zeros(1, E, device="cuda").scatter_(1, idx[t:t + 1], gw[t:t + 1])
        (d1,) = torch.autograd.grad(w1, one, torch.gather(g1, 1, i1))
        tol = 768 * U * 2.5 * 2 * gw[t].abs().max() + torch.finfo(dtype).eps * torch.maximum(dl[t].abs(), d1[0].abs()).float()
        assert ((dl[t].float() - d1[0].float()).abs() <= tol + (2.0 ** -24 if dtype == torch.float16 else 0)).all()


def test_biased_scores_with_masked_experts_infinities_and_nan():
    from cutlass_op.bf16_grouped_mm.routing import moe_route

    inf, nan = math.inf, math.nan
    logits = torch.tensor([[-inf, 1.0, -inf, 0.0], [-inf, -inf, -inf, -inf], [nan, 0.0, 1.0, 2.0], [inf, 0.0, 0.0, -inf],
                           [0.0, 0.0, 0.0, 0.0]], device="cuda")
    zero = torch.zeros(4, device="cuda")
    w, idx = moe_route(logits, 3, "biased_sigmoid", False, bias=zero)
    assert idx.tolist() == [[1, 3, -1], [-1, -1, -1], [0, 3, 2], [0, 1, 2], [0, 1, 2]]
    assert (w[idx < 0] == 0).all() and w[2, 0].isnan() and w[3, 0] == 1
    _, idx = moe_route(logits[:1], 3, "biased_sigmoid", bias=torch.tensor([9.0, -inf, 9.0, 0.0], device="cuda"))
    assert idx.tolist() == [[3, -1, -1]]
    # without a bias: the same as by the logits
    x = torch.randn(40, 64, generator=_gen(1), device="cuda")
    for score in ("softmax", "sigmoid"):
        for a, b in zip(moe_route(x, 6, score), moe_route(x, 6, "biased_" + score)):
            assert torch.equal(a, b)


def test_moe_ffn_takes_a_bias_on_the_score():
    from cutlass_op.bf16_grouped_mm.moe import moe_ffn

    g = _gen(2)
    E, H, I = 4, 64, 32
    w = [torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16) for s in ((E, H, 2 * I), (E, I, H), (E, 2 * I), (E, H))]
    x = torch.randn(1, H, generator=g, device="cuda").to(torch.bfloat16)
    logits = torch.tensor([[4.0, 1.0, 0.0, 0.0]], device="cuda")
    bias = torch.tensor([0.0, 0.4, 0.0, 0.0], device="cuda")
    only = lambda e: moe_ffn(x, torch.where(torch.arange(E, device="cuda") == e, 0.0, -math.inf)[None], 1, *w)  # noqa: E731
    assert torch.equal(moe_ffn(x, logits, 1, *w, score="sigmoid", route_bias=bias), only(0))
    assert torch.equal(moe_ffn(x, logits, 1, *w, score="biased_sigmoid", route_bias=bias), only(1))

"""Gradients of the router's logits where a score is next to 1: what is left of them is a
difference, which has to be taken before it is rounded."""

import pytest
import torch

import opengemm_b200 as og

pytestmark = pytest.mark.gpu

UNIT = 2.0**-24  # a rounding to float32


@pytest.mark.parametrize("experts,top_k", [(1, 1), (8, 2), (61, 8), (256, 8), (1000, 32)])
def test_logistic_scores_near_zero_and_one(experts, top_k):
    g = torch.Generator().manual_seed(experts)
    logits = ((torch.rand(200, experts, generator=g) * 2 - 1) * 30).cuda()
    weights, indices = og.route(logits, top_k, scores="sigmoid", renormalise=False, scale=1.5)
    grad = torch.randn(200, top_k, generator=g).cuda()
    got = og.route_backward(grad, logits, indices, scores="sigmoid", renormalise=False, scale=1.5).double()
    x = logits.double()
    slope = torch.sigmoid(x) * torch.sigmoid(-x)
    want = torch.zeros_like(slope).scatter_(1, indices.long(), grad.double() * 1.5) * slope
    # the factor 1.5, an exponential (2 units of the last place are 4 of these), 1 + e, its square, a
    # quotient (2), the product: each once, and the sum's error twice in its square
    assert ((got - want).abs() <= 16 * UNIT * want.abs() + 1e-38).all()
    assert (got.gather(1, indices.long()) != 0).all()


@pytest.mark.parametrize("renormalise", [False, True])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts,top_k", [(2, 2), (8, 2), (61, 8), (256, 8), (1000, 32)])
def test_one_expert_with_nearly_all_the_weight(experts, top_k, scores, renormalise):
    """ds_i - sum over j of s_j ds_j is sum over j of s_j (ds_i - ds_j): next to a score of 1 the first
    form loses what the second keeps."""
    if scores == "sigmoid" and not renormalise:
        pytest.skip("no difference to take")
    g = torch.Generator().manual_seed(experts + top_k)
    logits = torch.randn(200, experts, generator=g)
    lead = torch.arange(200) / 10.0  # 0 .. 20 above, so that the rest is worth 1 .. 2e-9 of it
    if scores == "sigmoid":
        logits -= lead[:, None]
    logits[torch.arange(200), torch.randint(0, experts, (200,), generator=g)] += lead
    logits = logits.cuda()
    weights, indices = og.route(logits, top_k, scores=scores, renormalise=renormalise)
    grad = torch.randn(200, top_k, generator=g).cuda()
    got = og.route_backward(grad, logits, indices, scores=scores, renormalise=renormalise).double()
    x, at = logits.double(), indices.long()
    s = torch.softmax(x, -1) if scores == "softmax" else torch.sigmoid(x)
    ds = torch.zeros_like(s).scatter_(1, at, grad.double())
    chosen = torch.zeros_like(s).scatter_(1, at, 1.0)
    p = s * chosen / (s * chosen).sum(-1, keepdim=True) if renormalise else s
    difference = ds[:, :, None] - ds[:, None, :]
    size = ds.abs()[:, :, None] + ds.abs()[:, None, :]
    size = torch.where(torch.eye(experts, dtype=torch.bool, device="cuda"), 0.0, size)
    want, terms = p * (difference * p[:, None, :]).sum(-1), p * (size * p[:, None, :]).sum(-1)
    if renormalise and scores == "sigmoid":
        want, terms = want * torch.sigmoid(-x), terms * torch.sigmoid(-x)
    # every term is a product of two scores (40 units each: an exponential, the row's sum and its
    # reciprocal, or the sum of the chosen) and a rounded difference, added in float32: 96 units;
    # twice that because a difference may be taken to an expert with half of the weight instead of each
    assert ((got - want).abs() <= 2 * 96 * UNIT * terms + 1e-38).all()

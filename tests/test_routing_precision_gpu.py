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

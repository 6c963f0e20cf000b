"""`route`, `expert_plan`, `expert_combine` and their gradients against the definitions in 64 bits."""

import pytest
import torch

import opengemm_b200 as og
from opengemm_b200 import capi
from tests.feed_forward_util import assert_within

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["native", "interpreter"], autouse=True)
def host_path(request):
    """Every test runs through the native host path and through the Python one."""
    before = capi.use_front(request.param == "native")
    assert (capi.front() is not None) == (request.param == "native")
    yield
    capi.use_front(before)

INF = float("inf")


def scores_of(logits, scores):
    x = logits.double()
    s = torch.softmax(x, -1) if scores == "softmax" else torch.sigmoid(x)
    return torch.where(x == -INF, 0.0, s)  # a row without a finite logit scores 0


def reference(logits, top_k, scores="softmax", bias=None, groups=1, top_groups=1, group_top=2, renormalise=True, scale=1.0):
    """(weights, indices) by the definition, one token after another."""
    s = scores_of(logits, scores).cpu()
    closed = (logits == -INF).cpu()
    choice = s if bias is None else s + bias.double().cpu()
    choice = choice.masked_fill(closed, -INF)
    tokens, experts = s.shape
    each = experts // groups
    weights = torch.zeros(tokens, top_k, dtype=torch.float64)
    indices = torch.full((tokens, top_k), -1, dtype=torch.int32)
    for t in range(tokens):
        c = choice[t].tolist()
        if groups > 1:
            best = [sum(sorted((v for v in c[g * each:(g + 1) * each] if v != -INF), reverse=True)[:group_top]) if max(c[g * each:(g + 1) * each]) != -INF
                    else -INF for g in range(groups)]
            open_ = sorted((g for g in range(groups) if best[g] != -INF), key=lambda g: (-best[g], g))[:top_groups]
            c = [v if i // each in open_ else -INF for i, v in enumerate(c)]
        order = sorted((i for i in range(experts) if c[i] != -INF), key=lambda i: (-c[i], i))[:top_k]
        for j, i in enumerate(order):
            indices[t, j], weights[t, j] = i, s[t, i]
    if renormalise:
        total = weights.sum(-1, keepdim=True)
        weights = torch.where(total > 0, weights / total.clamp(min=1e-300), 0.0)
    return weights * scale, indices


def logits_of(tokens, experts, dtype, seed=0):
    """Logits that differ by at least 1/64 inside a row, so that no rounding of a score decides an order."""
    g = torch.Generator().manual_seed(seed)
    order = torch.rand(tokens, experts, generator=g).argsort(-1)
    return ((order - experts / 2) / 64).to(dtype).cuda()


# A score is an exponential (2 units), a sum of at most 1024 of them down a tree (12), a division
# and a product: 20 units of float32 cover it, twice that after dividing by the sum of the chosen.
SCORE_ERROR = 40 * 2.0**-24


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("tokens,experts,top_k", [(1, 1, 1), (1, 8, 2), (5, 33, 8), (130, 64, 6), (17, 200, 8), (9, 256, 32), (3, 1000, 10), (4, 1024, 8)])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_choice_and_weights(scores, tokens, experts, top_k, dtype):
    logits = logits_of(tokens, experts, dtype, seed=experts) if dtype is torch.float32 else logits_of(tokens, min(experts, 1024), dtype, seed=experts)
    for renormalise, scale in ((True, 1.0), (False, 2.5)):
        weights, indices = og.route(logits, top_k, scores=scores, renormalise=renormalise, scale=scale)
        want, at = reference(logits, top_k, scores, renormalise=renormalise, scale=scale)
        assert weights.dtype is torch.float32 and indices.dtype is torch.int32
        assert torch.equal(indices.cpu(), at)
        assert_within(weights.cpu(), want, SCORE_ERROR * want.abs())


@pytest.mark.parametrize("groups,each,top_groups,group_top", [(8, 32, 4, 2), (4, 16, 1, 1), (2, 5, 2, 2), (3, 1, 2, 2), (32, 3, 7, 2), (8, 20, 3, 2), (3, 64, 2, 2), (5, 32, 2, 1), (32, 32, 5, 2), (2, 256, 1, 2)])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
def test_groups_and_bias(groups, each, top_groups, group_top, scores, biased):
    experts, tokens = groups * each, 40
    logits = logits_of(tokens, experts, torch.float32, seed=3)
    # steps of 1/4: larger than any score's rounding, smaller than what decides between all experts
    bias = torch.randint(0, 3, (experts,), generator=torch.Generator().manual_seed(1)).float().cuda() / 4 if biased else None
    top_k = min(6, top_groups * each)
    weights, indices = og.route(logits, top_k, scores=scores, bias=bias, groups=groups, top_groups=top_groups, group_top=group_top)
    want, at = reference(logits, top_k, scores, bias, groups, top_groups, group_top)
    assert torch.equal(indices.cpu(), at)
    assert_within(weights.cpu(), want, SCORE_ERROR * want.abs())


def test_equal_scores_take_the_lowest_index():
    logits = torch.zeros(3, 70, device="cuda", dtype=torch.bfloat16)
    logits[1, 40:] = 1.0
    logits[2, ::2] = -0.0
    weights, indices = og.route(logits, 4)
    assert indices.tolist() == [[0, 1, 2, 3], [40, 41, 42, 43], [0, 1, 2, 3]]
    assert torch.allclose(weights, torch.full_like(weights, 0.25))
    _, indices = og.route(logits[:1].contiguous(), 3, groups=7, top_groups=2, group_top=1)
    assert indices.tolist() == [[0, 1, 2]]


def test_masked_infinite_and_nan_logits():
    x = logits_of(7, 64, torch.float32, seed=9)
    x[0] = -INF                      # nothing to choose from
    x[1, 3:] = -INF                  # fewer than top_k
    x[2, ::2] = -INF
    x[3, 5] = float("nan")
    x[4] = torch.finfo(torch.float32).min
    x[5, 60:] = -INF
    for scores in ("softmax", "sigmoid"):
        for groups in (1, 4):
            weights, indices = og.route(x, 8, scores=scores, groups=groups, top_groups=2 if groups > 1 else 1)
            assert indices[0].tolist() == [-1] * 8 and weights[0].tolist() == [0.0] * 8
            assert sorted(indices[1].tolist()) == [-1] * 5 + [0, 1, 2]
            assert weights[1, 3:].tolist() == [0.0] * 5 and abs(weights[1].sum().item() - 1) < 1e-6
            assert all(i % 2 for i in indices[2].tolist())
            if groups == 1:
                assert indices[3, 0].item() == 5
            assert weights[3].isnan().any()
            assert indices[4].tolist() == list(range(8))
            assert weights[5].isfinite().all() and max(indices[5].tolist()) < 60
            if scores == "softmax":
                assert torch.allclose(weights[4], torch.full_like(weights[4], 0.125))
            else:
                assert weights[4].tolist() == [0.0] * 8  # every score underflows: nothing to divide by
    x[6, 7] = INF
    _, indices = og.route(x, 2)
    assert indices[6, 0].item() == 7
    bias = torch.zeros(64, device="cuda")
    bias[10:] = -INF                 # experts switched off
    _, indices = og.route(x[2:3].contiguous(), 8, bias=bias)
    assert sorted(indices[0].tolist()) == [-1, -1, -1, 1, 3, 5, 7, 9]


def test_no_tokens():
    weights, indices = og.route(torch.empty(0, 16, device="cuda"), 4)
    assert weights.shape == indices.shape == (0, 4)
    plan = og.expert_plan(indices, 16)
    assert plan.offsets.tolist() == [0] * 17 and plan.rows == 0
    out = og.expert_combine(torch.empty(0, 64, device="cuda", dtype=torch.bfloat16), weights, plan)
    assert out.shape == (0, 64)
    assert og.route_backward(weights, torch.empty(0, 16, device="cuda"), indices).shape == (0, 16)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalise", [True, False])
@pytest.mark.parametrize("tokens,experts,top_k", [(1, 5, 1), (70, 64, 6), (33, 200, 8), (5, 1024, 32)])
def test_gradient_of_the_logits(tokens, experts, top_k, renormalise, scores, dtype):
    logits = logits_of(tokens, experts, dtype, seed=4)
    logits[0, 1:3] = -INF
    if tokens > 4:
        logits[3] = -INF
    weights, indices = og.route(logits, top_k, scores=scores, renormalise=renormalise, scale=1.5)
    grad = torch.randn(tokens, top_k, device="cuda")
    got = og.route_backward(grad, logits, indices, scores=scores, renormalise=renormalise, scale=1.5)
    assert got.dtype is dtype
    x = logits.double().masked_fill(logits == -INF, -1e300).requires_grad_()
    s = torch.softmax(x, -1) if scores == "softmax" else torch.sigmoid(x)
    s = s * (logits != -INF)
    w = s.gather(1, indices.clamp(min=0).long()) * (indices >= 0)
    if renormalise:
        total = w.sum(-1, keepdim=True)
        w = w / torch.where(total > 0, total, 1.0)
    want, = torch.autograd.grad((w * 1.5 * grad.double()).sum(), x)
    want = torch.where(logits == -INF, 0.0, want)
    # differences of products with |grad| at most `size`: a few units of each term
    size = 1.5 * grad.double().abs().max(-1, keepdim=True).values
    assert_within(got, want, SCORE_ERROR * 4 * size * (1 if renormalise else 1.0))


def test_gradient_against_differences():
    logits = logits_of(6, 24, torch.float32, seed=8)
    grad = torch.randn(6, 4, device="cuda")
    for scores in ("softmax", "sigmoid"):
        _, indices = og.route(logits, 4, scores=scores)
        got = og.route_backward(grad, logits, indices, scores=scores)
        for i in (0, 7, int(indices[2, 0]), int(indices[2, 3])):
            step = torch.zeros_like(logits)
            step[:, i] = 2.0**-9  # less than the logits' spacing, so the choice stays
            up, _ = reference(logits + step, 4, scores)
            down, _ = reference(logits - step, 4, scores)
            want = ((up - down).cuda() * grad.double()).sum(-1) / 2.0**-8
            torch.testing.assert_close(got[:, i].double(), want, rtol=1e-3, atol=1e-5)


def check_plan(indices, experts):
    plan = og.expert_plan(indices, experts)
    flat = indices.flatten().long().cpu()
    valid = (flat >= 0) & (flat < experts)
    counts = torch.bincount(flat[valid], minlength=experts)
    offsets = torch.cat([torch.zeros(1, dtype=torch.long), counts.cumsum(0)])
    order = torch.where(valid, flat, experts).sort(stable=True).indices[: int(offsets[-1])]
    assert torch.equal(plan.offsets.cpu().long(), offsets)
    assert torch.equal(plan.tokens.cpu().long()[: order.numel()], order // indices.size(1))
    positions = torch.full((flat.numel(),), -1)
    positions[order] = torch.arange(order.numel())
    assert torch.equal(plan.positions.cpu().long().flatten(), positions)
    return plan


@pytest.mark.parametrize("tokens,top_k,experts", [(1, 1, 1), (1, 8, 256), (16, 8, 64), (511, 1, 3), (512, 8, 8), (513, 8, 60), (4097, 3, 1024), (20001, 8, 128)])
def test_plan_is_a_stable_sort(tokens, top_k, experts):
    g = torch.Generator().manual_seed(tokens)
    indices = torch.randint(-1, experts + (tokens % 2), (tokens, top_k), generator=g, dtype=torch.int32).cuda()
    check_plan(indices, experts)  # repeated experts of one token included


def test_plan_of_extreme_indices():
    check_plan(torch.full((700, 8), 5, dtype=torch.int32, device="cuda"), 9)      # all to one expert
    check_plan(torch.full((700, 8), -1, dtype=torch.int32, device="cuda"), 9)     # none anywhere
    check_plan(torch.tensor([[2**31 - 1, -(2**31), 0]], dtype=torch.int32, device="cuda"), 2)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("tokens,top_k,n", [(1, 1, 8), (16, 8, 2048), (33, 3, 1037), (130, 2, 264), (257, 2, 2056), (300, 5, 4096)])
@pytest.mark.parametrize("residual", [False, True])
def test_combine_and_its_gradient(tokens, top_k, n, residual, dtype):
    g = torch.Generator().manual_seed(n)
    indices = torch.randint(-1, 10, (tokens, top_k), generator=g, dtype=torch.int32).cuda()
    plan = og.expert_plan(indices, 10)
    y = torch.randn(plan.rows, n, generator=g).to(dtype).cuda()
    rows = int(plan.offsets[-1])
    y[rows:] = float("nan")  # nobody's rows
    weights = torch.rand(tokens, top_k, generator=g).cuda()
    weights[indices < 0] = float("nan")  # nor these pairs' weights
    add = torch.randn(tokens, n, generator=g).to(dtype).cuda() if residual else None
    there = (plan.positions >= 0)[..., None]
    by_pair = torch.where(there, y.double()[plan.positions.clamp(min=0).long()], 0.0)
    w = torch.where(there, weights.double()[..., None], 0.0)
    want = (w * by_pair).sum(1) + (0.0 if add is None else add.double())
    size = (w * by_pair).abs().sum(1) + want.abs()
    assert_within(og.expert_combine(y, weights, plan, residual=add), want, (top_k + 2) * 2.0**-24 * size)
    if add is not None:
        into = add.clone()
        assert og.expert_combine(y, weights, plan, residual=into, out=into) is into
        assert_within(into, want, (top_k + 2) * 2.0**-24 * size)

    grad = torch.randn(tokens, n, generator=g).to(dtype).cuda()
    grad_y, grad_weights = og.expert_combine_backward(grad, y, weights, plan)
    want_y = torch.zeros(plan.rows, n, dtype=torch.float64, device="cuda")
    want_y[plan.positions[plan.positions >= 0].long()] = (w * grad.double()[:, None])[plan.positions >= 0]
    assert_within(grad_y[:rows], want_y[:rows], 2.0**-24 * want_y[:rows].abs())
    terms = grad.double()[:, None] * by_pair
    assert_within(grad_weights, terms.sum(-1), (n / 8 + 16) * 2.0**-24 * terms.abs().sum(-1))


def test_refusals():
    x = torch.zeros(4, 16, device="cuda")
    for bad in (dict(top_k=0), dict(top_k=17), dict(top_k=2, groups=3), dict(top_k=2, groups=4, top_groups=5), dict(top_k=2, groups=4, group_top=3),
                dict(top_k=5, groups=4, top_groups=1)):
        with pytest.raises(RuntimeError):
            og.route(x, **bad)
    with pytest.raises(TypeError, match="scores"):
        og.route(x, 2, scores="tanh")
    with pytest.raises(TypeError, match="logits"):
        og.route(x.t(), 2)
    with pytest.raises(TypeError, match="logits"):
        og.route(x.double(), 2)
    with pytest.raises(TypeError, match="bias"):
        og.route(x, 2, bias=torch.zeros(16, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="1024"):
        og.route(torch.zeros(1, 1025, device="cuda"), 2)
    with pytest.raises(TypeError, match="indices"):
        og.expert_plan(torch.zeros(4, 2, device="cuda", dtype=torch.int64), 4)
    with pytest.raises(ValueError, match="1024"):
        og.expert_plan(torch.zeros(4, 2, device="cuda", dtype=torch.int32), 1025)
    weights, indices = og.route(x, 2)
    plan = og.expert_plan(indices, 16)
    y = torch.zeros(8, 64, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="y is"):
        og.expert_combine(y.float(), weights, plan)
    with pytest.raises(TypeError, match="y must"):
        og.expert_combine(y[:7], weights, plan)
    with pytest.raises(TypeError, match="weights"):
        og.expert_combine(y, weights[:, :1], plan)
    with pytest.raises(TypeError, match="residual"):
        og.expert_combine(y, weights, plan, residual=y)
    with pytest.raises(TypeError, match="grad_weights"):
        og.route_backward(weights[:2], x, indices)

"""`expert_gemm`, its gradients and `gemm_backward` against the definitions in 64 bits."""

import pytest
import torch

import opengemm_b200 as og
from opengemm_b200 import capi
from tests.feed_forward_util import HALF_STEP, act, act_error, act_gradient, assert_within, sum_error

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["native", "interpreter"], autouse=True)
def host_path(request):
    """Every test runs through the native host path and through the Python one."""
    before = capi.use_front(request.param == "native")
    assert (capi.front() is not None) == (request.param == "native")
    yield
    capi.use_front(before)


def routed(tokens, top_k, experts, seed=0, dropped=True):
    """Indices with repeats, empty experts and (with `dropped`) pairs that go nowhere."""
    g = torch.Generator().manual_seed(seed)
    busy = torch.randint(0, experts, (max(1, experts * 2 // 3),), generator=g)
    indices = busy[torch.randint(0, busy.numel(), (tokens, top_k), generator=g)].to(torch.int32)
    if dropped:
        indices[torch.rand(tokens, top_k, generator=g) < 0.1] = -1
    return indices.cuda()


def values(g, *shape, dtype, spread=1.0):
    return (torch.randn(*shape, generator=g) * spread).to(dtype).cuda()


def by_expert(plan):
    """(expert, slice of its rows) of every expert that has any."""
    offsets = plan.offsets.tolist()
    return [(e, slice(offsets[e], offsets[e + 1])) for e in range(plan.experts) if offsets[e + 1] > offsets[e]]


def reference(rows, w, plan, alpha):
    """(products, bound of the error of their float32 sums) of all rows, zeros behind the last."""
    z = torch.zeros(plan.rows, w.size(1), dtype=torch.float64, device="cuda")
    size = torch.zeros_like(z)
    for e, at in by_expert(plan):
        factor = 1.0 if alpha is None else alpha[e].item()
        z[at] = factor * (rows[at].double() @ w[e].double().T)
        size[at] = abs(factor) * (rows[at].double().abs() @ w[e].double().abs().T)
    return z, sum_error(size, rows.size(1)) + 2.0**-23 * z.abs()


def gated_error(name, z, z_error):
    """Bound of the error of act(gate) * up for errors of its two arguments."""
    gate, up = z.chunk(2, -1)
    gate_error, up_error = z_error.chunk(2, -1)
    value = act("silu" if name == "swiglu" else "gelu", gate)
    value_error = act_error(gate, gate_error)
    return value_error * (up.abs() + up_error) + value.abs() * up_error + 2.0**-23 * (value * up).abs()


def check(tokens, top_k, experts, n, k, dtype=torch.bfloat16, gather=True, activation=None, scaled=False, save=False, seed=0, indices=None):
    g = torch.Generator().manual_seed(seed)
    indices = routed(tokens, top_k, experts, seed) if indices is None else indices
    plan = og.expert_plan(indices, experts)
    last = int(plan.offsets[-1])
    x = values(g, tokens if gather else plan.rows, k, dtype=dtype)
    w = values(g, experts, n, k, dtype=dtype, spread=k**-0.5)
    alpha = (torch.rand(experts, generator=g) + 0.5).cuda() if scaled else None
    own = torch.bfloat16 if dtype is torch.float8_e4m3fn else dtype
    gated = activation in ("swiglu", "geglu")
    out = torch.full((plan.rows, n // 2 if gated else n), 7.0, device="cuda", dtype=own)
    z = torch.full((plan.rows, n), 7.0, device="cuda", dtype=own) if save else None
    assert og.expert_gemm(x, w, plan, gather=gather, activation=activation, alpha=alpha, out=out, preactivation=z) is out
    if save:
        z_too = torch.empty_like(z)
    again = og.expert_gemm(x, w, plan, gather=gather, activation=activation, alpha=alpha, preactivation=z_too if save else None)
    assert torch.equal(again[:last], out[:last]) and (not save or torch.equal(z_too[:last], z[:last]))
    rows = x[plan.tokens.clamp(0, tokens - 1).long()] if gather else x
    want_z, error = reference(rows, w, plan, alpha)
    if save:
        assert_within(z[:last], want_z[:last], error[:last], "pre-activation")
        assert (z[last:] == 7.0).all()
    want = act(activation, want_z)
    error = gated_error(activation, want_z, error) if gated else act_error(want_z, error) if activation else error
    assert_within(out[:last], want[:last], error[:last], "product")
    assert (out[last:] == 7.0).all()  # rows behind the last are left as they were


SHAPES = [(1, 1, 1, 8, 8), (1, 8, 64, 256, 512), (16, 8, 64, 384, 256), (33, 2, 5, 33, 72), (300, 4, 7, 520, 192), (1000, 2, 3, 264, 1032), (2500, 2, 4, 640, 128)]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("gather", [False, True])
def test_products(shape, dtype, gather):
    check(*shape, dtype=dtype, gather=gather)


@pytest.mark.parametrize("shape", [(1, 8, 64, 256, 512), (33, 2, 5, 33, 80), (700, 3, 6, 520, 208), (2500, 2, 4, 640, 1040)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("gather", [False, True])
def test_e4m3_products(shape, gather):
    check(*shape, dtype=torch.float8_e4m3fn, gather=gather, scaled=True, save=True)


@pytest.mark.parametrize("activation", ["relu", "gelu", "gelu_tanh", "silu", "swiglu", "geglu"])
@pytest.mark.parametrize("shape", [(40, 3, 9, 96, 64), (1500, 2, 3, 592, 128), (1, 2, 8, 2048, 128)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("save", [False, True])
def test_activations(shape, activation, save):
    check(*shape, activation=activation, save=save, scaled=save)
    check(*shape, dtype=torch.float16, gather=False, activation=activation, save=save)


def test_all_rows_to_one_expert_and_none_at_all():
    check(700, 2, 8, 200, 64, indices=torch.full((700, 2), 3, dtype=torch.int32, device="cuda"))
    check(700, 2, 8, 200, 64, indices=torch.full((700, 2), -1, dtype=torch.int32, device="cuda"))
    check(300, 1, 1024, 64, 64, indices=torch.arange(300, dtype=torch.int32, device="cuda")[:, None] * 3)


def test_values_of_other_experts_rows_do_not_leak():
    """A row of NaN reaches no other row, and in the weights' gradient no other expert."""
    indices = torch.tensor([[0], [1], [1], [2], [2], [2]], dtype=torch.int32, device="cuda")
    plan = og.expert_plan(indices, 4)
    x = torch.randn(6, 64, device="cuda").bfloat16()
    w = torch.randn(4, 128, 64, device="cuda").bfloat16()
    x[2] = float("nan")
    y = og.expert_gemm(x, w, plan, gather=True)
    assert y[2].isnan().all() and y[[0, 1, 3, 4, 5]].isfinite().all()
    for gather in (False, True):
        grad_x, grad_w = og.expert_gemm_backward(torch.randn(6, 128, device="cuda").bfloat16(), x, w, plan, gather=gather)
        assert grad_x.isfinite().all()
        assert grad_w[1].isnan().all() and grad_w[[0, 2, 3]].isfinite().all()
        assert (grad_w[3] == 0).all()


def check_gradients(tokens, top_k, experts, n, k, dtype=torch.bfloat16, gather=True, activation=None, out_dtype=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    plan = og.expert_plan(routed(tokens, top_k, experts, seed), experts)
    last = int(plan.offsets[-1])
    gated = activation in ("swiglu", "geglu")
    x = values(g, tokens if gather else plan.rows, k, dtype=dtype)
    w = values(g, experts, n, k, dtype=dtype, spread=k**-0.5)
    grad = values(g, plan.rows, n // 2 if gated else n, dtype=dtype)
    z = values(g, plan.rows, n, dtype=dtype) if activation else None
    grad[last:] = float("nan")
    if z is not None:
        z[last:] = float("nan")
    grad_x, grad_w = og.expert_gemm_backward(grad, x, w, plan, gather=gather, activation=activation, preactivation=z, out_dtype=out_dtype)
    dz = grad.double()[:last] if z is None else act_gradient(activation, z.double()[:last], grad.double()[:last])
    # dz is rounded to the operands' type before the products, after an evaluation in float32
    # whose error is a few units of the two factors
    dz_error = torch.zeros_like(dz)
    if z is not None:
        side = grad.double()[:last].repeat(1, 2 if gated else 1).abs()
        reach = z.double()[:last].abs().amax(-1, keepdim=True) + 2
        dz_error = HALF_STEP[dtype] * dz.abs() + 2e-6 * side * reach + torch.finfo(dtype).tiny
    rows = (x[plan.tokens[:last].long()] if gather else x[:last]).double()
    want_x = torch.zeros(plan.rows, k, dtype=torch.float64, device="cuda")
    x_error = torch.zeros_like(want_x)
    want_w = torch.zeros(w.shape, dtype=torch.float64, device="cuda")
    w_error = torch.zeros_like(want_w)
    for e, at in by_expert(plan):
        we = w[e].double()
        want_x[at], x_error[at] = dz[at] @ we, sum_error(dz[at].abs() @ we.abs(), n) + dz_error[at] @ we.abs()
        want_w[e] = dz[at].T @ rows[at]
        w_error[e] = sum_error(dz[at].abs().T @ rows[at].abs(), at.stop - at.start) + dz_error[at].T @ rows[at].abs()
    assert_within(grad_w, want_w, w_error, "weights' gradient")
    if gather:  # a token's rows are added in float32
        part_error = x_error + 2.0**-24 * want_x.abs()
        there = plan.positions >= 0
        at = plan.positions.clamp(min=0).long()
        total = (want_x[at] * there[..., None]).sum(1)
        error = ((part_error[at] + 2.0**-22 * want_x[at].abs()) * there[..., None]).sum(1)
        assert grad_x.dtype is dtype
        assert_within(grad_x, total, error, "tokens' gradient")
    else:
        assert_within(grad_x[:last], want_x[:last], x_error[:last], "rows' gradient")


@pytest.mark.parametrize("shape", [(1, 1, 1, 8, 8), (16, 8, 64, 128, 64), (33, 2, 5, 40, 72), (300, 4, 7, 520, 192), (1000, 2, 3, 264, 1032), (2500, 2, 2, 640, 384)],
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("out_dtype", [None, torch.float32], ids=str)
def test_gradients(shape, dtype, gather, out_dtype):
    check_gradients(*shape, dtype=dtype, gather=gather, out_dtype=out_dtype)


@pytest.mark.parametrize("activation", ["relu", "gelu", "gelu_tanh", "silu", "swiglu", "geglu"])
@pytest.mark.parametrize("gather", [False, True])
def test_gradients_through_activations(activation, gather):
    check_gradients(333, 2, 5, 592, 136, activation=activation, gather=gather)


def check_gemm_gradients(m, n, k, dtype, activation=None, alpha=None, out_dtype=None):
    g = torch.Generator().manual_seed(m)
    a, b = values(g, m, k, dtype=dtype), values(g, n, k, dtype=dtype, spread=k**-0.5)
    grad, z = values(g, m, n, dtype=dtype), values(g, m, n, dtype=dtype) if activation else None
    grad_a, grad_b, grad_bias = og.gemm_backward(grad, a, b, activation=activation, preactivation=z, alpha=alpha, want=("a", "b", "bias"), out_dtype=out_dtype)
    dz = grad.double() if z is None else act_gradient(activation, z.double(), grad.double())
    dz_error = torch.zeros_like(dz)
    eval_error = torch.zeros_like(dz)
    if z is not None:
        eval_error = 2e-6 * grad.double().abs() * (z.double().abs() + 2)
        dz_error = HALF_STEP[dtype] * dz.abs() + eval_error + torch.finfo(dtype).tiny
    f = 1.0 if alpha is None else alpha
    a64, b64 = a.double(), b.double()
    assert_within(grad_a, f * (dz @ b64), abs(f) * (sum_error(dz.abs() @ b64.abs(), n + 16) + dz_error @ b64.abs()), "a")
    assert_within(grad_b, f * (dz.T @ a64), abs(f) * (sum_error(dz.abs().T @ a64.abs(), m + 16) + dz_error.T @ a64.abs()), "b")
    # sums of at most 8 rows, of 8 row lanes, of blocks of 16 or 64 rows in eight lanes
    assert_within(grad_bias, dz.sum(0), (24 + m / 64) * 2.0**-24 * dz.abs().sum(0) + eval_error.sum(0), "bias")


@pytest.mark.parametrize("shape", [(1, 8, 8), (1, 4096, 256), (300, 520, 768), (77, 40, 128), (1001, 136, 264), (4100, 776, 512),
                                   (36, 4096, 264), (130, 2056, 128), (5001, 64, 72),  # cut along the reduction
                                   (16, 264, 64), (17, 264, 64), (128, 264, 64), (129, 264, 64), (1024, 264, 64), (9480, 512, 64)],  # the bias's sums
                         ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("out_dtype", [None, torch.float32], ids=str)
def test_gemm_gradients(shape, dtype, out_dtype):
    check_gemm_gradients(*shape, dtype, out_dtype=out_dtype, alpha=0.375)


@pytest.mark.parametrize("activation", ["relu", "gelu", "gelu_tanh", "silu"])
def test_gemm_gradients_through_activations(activation):
    check_gemm_gradients(333, 264, 136, torch.bfloat16, activation)
    check_gemm_gradients(130, 520, 72, torch.float16, activation)


def test_two_gradients_side_by_side_are_those_one_after_the_other():
    """The second product does not wait for the first: the same bits as when each is alone on the stream."""
    torch.manual_seed(6)
    sizes = [(300, 520, 768), (2048, 1024, 512), (1001, 136, 264), (64, 4096, 256), (4100, 776, 512)]
    sets, alone = [], []
    for m, n, k in sizes:
        a, b = torch.randn(m, k).bfloat16().cuda(), torch.randn(n, k).bfloat16().cuda()
        grad, z = torch.randn(m, n).bfloat16().cuda(), torch.randn(m, n).bfloat16().cuda()
        sets.append((grad, a, b))
        each = []
        for want in ("a", "b"):
            each.append([t for t in og.gemm_backward(*sets[-1], activation="gelu", preactivation=z, want=(want,)) if t is not None][0].clone())
            torch.cuda.synchronize()
        sets[-1] += (z,)
        alone.append(each)
    for _ in range(20):
        gots = [og.gemm_backward(grad, a, b, activation="gelu", preactivation=z, want=("a", "b", "bias")) for grad, a, b, z in sets]
        for got, want in zip(gots, alone):
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    plan = og.expert_plan(routed(900, 3, 7, seed=5), 7)
    x, w = torch.randn(900, 264).half().cuda(), torch.randn(7, 320, 264).half().cuda()
    grad, z = torch.randn(plan.rows, 160).half().cuda(), torch.randn(plan.rows, 320).half().cuda()
    run = lambda want: og.expert_gemm_backward(grad, x, w, plan, gather=True, activation="swiglu", preactivation=z, want=want)  # noqa: E731
    want_x, want_w = run(("x",))[0].clone(), run(("w",))[1].clone()
    torch.cuda.synchronize()
    for _ in range(20):
        grad_x, grad_w = run(("x", "w"))
        assert torch.equal(grad_x, want_x) and torch.equal(grad_w, want_w)


def test_gemm_gradients_against_differences_of_the_forward_call():
    torch.manual_seed(0)
    m, n, k = 24, 32, 16
    a, b, bias = torch.randn(m, k).cuda().half(), torch.randn(n, k).cuda().half(), torch.randn(n).cuda()
    residual = torch.randn(m, n).cuda().half()
    z = torch.empty(m, n, device="cuda", dtype=torch.float16)
    og.gemm(a, b, out_dtype=torch.float16, bias=bias, activation="gelu", residual=residual, preactivation=z)
    grad = torch.randn(m, n).cuda().half()
    grad_a, grad_b, grad_bias = og.gemm_backward(grad, a, b, activation="gelu", preactivation=z, want=("a", "b", "bias"))

    def loss(a, b, bias):  # the forward call's value before its last rounding
        return (act("gelu", a @ b.T + bias) * grad.double()).sum()

    for got, index in ((grad_a, 0), (grad_b, 1), (grad_bias, 2)):
        args = [a.double(), b.double(), bias.double()]
        for at in (0, 5, got.numel() - 1):
            up, down = [t.clone() for t in args], [t.clone() for t in args]
            up[index].view(-1)[at] += 2.0**-12
            down[index].view(-1)[at] -= 2.0**-12
            want = (loss(*up) - loss(*down)) / 2.0**-11
            # z and dz carry a rounding to float16 each: up to 32 terms of size 4
            assert abs(got.view(-1)[at].item() - want.item()) < 32 * 4 * 2.0**-10


def test_no_rows_at_all():
    plan = og.expert_plan(torch.zeros(0, 2, dtype=torch.int32, device="cuda"), 3)
    x, w = torch.zeros(0, 64, device="cuda", dtype=torch.bfloat16), torch.ones(3, 32, 64, device="cuda", dtype=torch.bfloat16)
    for gather in (False, True):
        assert og.expert_gemm(x, w, plan, gather=gather, activation="swiglu").shape == (0, 16)
        z = torch.zeros(0, 32, device="cuda", dtype=torch.bfloat16)
        grad_x, grad_w = og.expert_gemm_backward(z[:, :16].contiguous(), x, w, plan, gather=gather, activation="swiglu", preactivation=z)
        assert grad_x.shape == (0, 64) and grad_w.shape == w.shape and not grad_w.any()
    a, b = torch.zeros(0, 64, device="cuda", dtype=torch.float16), torch.ones(32, 64, device="cuda", dtype=torch.float16)
    z = torch.zeros(0, 32, device="cuda", dtype=torch.float16)
    grad_a, grad_b, grad_bias = og.gemm_backward(z, a, b, activation="gelu", preactivation=z, want=("a", "b", "bias"))
    assert grad_a.shape == (0, 64) and not grad_b.any() and not grad_bias.any()


def test_offsets_past_32_bits():
    """More than 2^31 values of output: the last rows are computed and stored in their place."""
    rows, n, k = 1_100_000, 2048, 64
    indices = torch.zeros(rows, 1, dtype=torch.int32, device="cuda")
    indices[-1000:] = 1
    plan = og.expert_plan(indices, 2)
    g = torch.Generator().manual_seed(0)
    x = torch.zeros(rows, k, device="cuda", dtype=torch.bfloat16)
    x[-1500:] = values(g, 1500, k, dtype=torch.bfloat16)
    w = values(g, 2, n, k, dtype=torch.bfloat16)
    y = og.expert_gemm(x, w, plan)
    for rows_of, e in ((slice(-1500, -1000), 0), (slice(-1000, None), 1)):
        want = x[rows_of].double() @ w[e].double().T
        assert_within(y[rows_of], want, sum_error(x[rows_of].double().abs() @ w[e].double().abs().T, k))
    assert not y[:-1500].any()
    out = og.expert_combine(y, torch.full((rows, 1), 2.0, device="cuda"), plan)
    assert torch.equal(out[-1500:], y[-1500:] * 2)
    del out
    residual = torch.zeros_like(y)
    residual[-700:] = 1
    c = og.gemm(x, w[1], out_dtype=torch.bfloat16, activation="relu", residual=residual)
    want = torch.relu(x[-1500:].double() @ w[1].double().T) + residual[-1500:].double()
    assert_within(c[-1500:], want, sum_error(x[-1500:].double().abs() @ w[1].double().abs().T, k) + 2.0**-23 * want.abs())
    assert not c[:-1500].any()


def layer(x, logits, w1, w2, top_k):
    """A mixture-of-experts layer; returns its output and what its gradient needs."""
    weights, indices = og.route(logits, top_k)
    plan = og.expert_plan(indices, w1.size(0))
    z = torch.empty(plan.rows, w1.size(1), device="cuda", dtype=x.dtype)
    h = og.expert_gemm(x, w1, plan, gather=True, activation="swiglu", preactivation=z)
    y = og.expert_gemm(h, w2, plan)
    return og.expert_combine(y, weights, plan, residual=x), (weights, indices, plan, z, h, y)


def layer_backward(grad, x, logits, w1, w2, saved):
    weights, indices, plan, z, h, y = saved
    grad_y, grad_weights = og.expert_combine_backward(grad, y, weights, plan)
    grad_h, grad_w2 = og.expert_gemm_backward(grad_y, h, w2, plan)
    grad_x, grad_w1 = og.expert_gemm_backward(grad_h, x, w1, plan, gather=True, activation="swiglu", preactivation=z)
    return grad_x + grad, og.route_backward(grad_weights, logits, indices), grad_w1, grad_w2


def test_a_layer_and_its_gradient_against_automatic_differentiation():
    torch.manual_seed(1)
    tokens, experts, top_k, hidden, inner = 200, 6, 2, 64, 48
    x = torch.randn(tokens, hidden).half().cuda()
    logits = torch.randn(tokens, experts).cuda()
    w1, w2 = (torch.randn(experts, 2 * inner, hidden) / 8).half().cuda(), (torch.randn(experts, hidden, inner) / 7).half().cuda()
    out, saved = layer(x, logits, w1, w2, top_k)
    grad = torch.randn(tokens, hidden).half().cuda()
    got = layer_backward(grad, x, logits, w1, w2, saved)
    leaves = [t.double().requires_grad_() for t in (x, logits, w1, w2)]
    x64, l64, w164, w264 = leaves
    s = torch.softmax(l64, -1)
    chosen = s.gather(1, saved[1].long())
    weight = chosen / chosen.sum(-1, keepdim=True)
    want = x64
    for j in range(top_k):
        e = saved[1][:, j].long()
        h = act("swiglu", torch.einsum("tk,tnk->tn", x64, w164[e]))
        want = want + weight[:, j:j + 1] * torch.einsum("tk,tnk->tn", h, w264[e])
    # roundings to float16 (2^-11 each) of h and y: relative to the sizes of what is added
    torch.testing.assert_close(out.double(), want, rtol=2.0**-9, atol=2.0**-9 * want.abs().max().item())
    wants = torch.autograd.grad((want * grad.double()).sum(), leaves)
    for name, g, w in zip(("x", "logits", "w1", "w2"), got, wants):
        # six roundings at most on the way, their errors spread over sums of many terms
        assert (g.double() - w).norm() < 6 * 2.0**-11 * w.norm(), name


def test_a_layer_in_a_graph_and_on_another_stream_gives_the_same_bits():
    torch.manual_seed(2)
    x = torch.randn(700, 128).bfloat16().cuda()
    logits = torch.randn(700, 8).cuda()
    w1, w2 = (torch.randn(8, 256, 128) / 11).bfloat16().cuda(), (torch.randn(8, 128, 128) / 11).bfloat16().cuda()
    grad = torch.randn(700, 128).bfloat16().cuda()

    def step():
        out, saved = layer(x, logits, w1, w2, 2)
        return (out, *layer_backward(grad, x, logits, w1, w2, saved))

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for got, w in zip(step(), want):
            assert torch.equal(got, w)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    logits.copy_(torch.randn(700, 8))  # another routing: the captured launches follow the new plan
    graph.replay()
    replayed = [t.clone() for t in captured]
    for got, w in zip(step(), replayed):
        assert torch.equal(got, w)


def test_two_layers_at_once_on_two_streams():
    torch.manual_seed(4)
    sets, streams, wants = [], [torch.cuda.Stream(), torch.cuda.Stream()], []
    for i in range(2):
        sets.append((torch.randn(900, 256).bfloat16().cuda(), torch.randn(900, 16).cuda(), (torch.randn(16, 512, 256) / 16).bfloat16().cuda(),
                     (torch.randn(16, 256, 256) / 16).bfloat16().cuda(), 4))
        wants.append(layer(*sets[i])[0].clone())
    torch.cuda.synchronize()
    gots = [[], []]
    for _ in range(10):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                gots[i].append(layer(*sets[i])[0])
    torch.cuda.synchronize()
    for i in range(2):
        for got in gots[i]:
            assert torch.equal(got, wants[i])


def test_refusals():
    indices = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    plan = og.expert_plan(indices, 3)
    x, w = torch.zeros(8, 64, device="cuda", dtype=torch.bfloat16), torch.zeros(3, 32, 64, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="x is"):
        og.expert_gemm(x.float(), w.float(), plan)
    with pytest.raises(TypeError, match="x must"):
        og.expert_gemm(x, w, plan, gather=True)  # eight rows, but four tokens
    with pytest.raises(TypeError, match="w must"):
        og.expert_gemm(x, w.half(), plan)
    with pytest.raises(ValueError, match="experts"):
        og.expert_gemm(x, w[:2], plan)
    with pytest.raises(ValueError, match="multiple of 8"):
        og.expert_gemm(x[:, :60].contiguous(), w[..., :60].contiguous(), plan)
    with pytest.raises(ValueError, match="16"):
        og.expert_gemm(x, w[:, :24].contiguous(), plan, activation="swiglu")
    with pytest.raises(TypeError, match="activation"):
        og.expert_gemm(x, w, plan, activation="tanh")
    with pytest.raises(TypeError, match="alpha"):
        og.expert_gemm(x, w, plan, alpha=torch.ones(2, device="cuda"))
    with pytest.raises(TypeError, match="out must"):
        og.expert_gemm(x, w, plan, out=torch.zeros(8, 32, device="cuda"))
    square = torch.zeros(3, 64, 64, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="share memory"):
        og.expert_gemm(x, square, plan, out=x)
    with pytest.raises(ValueError, match="share memory"):
        og.expert_gemm(x, square, plan, activation="relu", preactivation=x)
    with pytest.raises(ValueError, match="share memory"):
        og.expert_combine(x, torch.zeros(4, 2, device="cuda"), plan, out=x[:4])
    with pytest.raises(ValueError, match="16-byte"):
        og.expert_gemm(torch.zeros(8 * 64 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(8, 64), w, plan)
    grad = torch.zeros(8, 32, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="come together"):
        og.expert_gemm_backward(grad, x, w, plan, activation="relu")
    with pytest.raises(TypeError, match="want"):
        og.expert_gemm_backward(grad, x, w, plan, want=("a",))
    with pytest.raises(TypeError, match="grad must"):
        og.expert_gemm_backward(grad, x, w, plan, activation="swiglu", preactivation=grad)
    a, b = torch.zeros(16, 64, device="cuda", dtype=torch.bfloat16), torch.zeros(32, 64, device="cuda", dtype=torch.bfloat16)
    grad = torch.zeros(16, 32, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="16"):
        og.gemm_backward(grad.float(), a.float(), b.float())
    with pytest.raises(TypeError, match="grad must"):
        og.gemm_backward(grad.half(), a, b)
    with pytest.raises(TypeError, match="come together"):
        og.gemm_backward(grad, a, b, preactivation=grad)
    with pytest.raises(TypeError, match="leave as"):
        og.gemm_backward(grad, a, b, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="multiples of 8"):
        og.gemm_backward(grad[:, :30].contiguous(), a, b[:30])


def test_what_is_written_is_not_read():
    """Neither the factors and weights nor the plan may be written over by the call that reads them."""
    plan = og.expert_plan(torch.tensor([[0, 1], [2, 0], [1, 2], [0, 1]], device="cuda", dtype=torch.int32), 3)
    x, w = torch.zeros(8, 64, device="cuda", dtype=torch.bfloat16), torch.zeros(3, 64, 64, device="cuda", dtype=torch.bfloat16)
    store = torch.zeros(8 * 64, device="cuda")  # as bfloat16 twice the rows
    alpha, rows = store[:3], store.view(torch.bfloat16)[:8 * 64].view(8, 64)
    with pytest.raises(ValueError, match="out and alpha share memory"):
        og.expert_gemm(x, w, plan, alpha=alpha, out=rows)
    with pytest.raises(ValueError, match="preactivation and alpha share memory"):
        og.expert_gemm(x, w, plan, alpha=alpha, activation="relu", preactivation=rows)
    weights, tokens = store[:8].view(4, 2), store.view(torch.bfloat16)[:4 * 64].view(4, 64)
    with pytest.raises(ValueError, match="out and weights share memory"):
        og.expert_combine(x, weights, plan, out=tokens)
    with pytest.raises(ValueError, match="out and plan share memory"):
        og.expert_combine(x[:, :2].contiguous(), torch.zeros(4, 2, device="cuda"), plan, out=plan.offsets.view(torch.bfloat16).view(4, 2))
    assert not store.any()


def test_gradients_past_32_bits():
    """More than 2^31 values of gradients and pre-activations, and then of weights' gradients."""
    rows, n, k, tail = 1_100_000, 2048, 64, 700
    indices = torch.zeros(rows, 1, dtype=torch.int32, device="cuda")
    indices[-300:] = 1
    plan = og.expert_plan(indices, 2)
    g = torch.Generator().manual_seed(1)
    x = torch.ones(rows, k, device="cuda", dtype=torch.bfloat16)
    x[-tail:] = values(g, tail, k, dtype=torch.bfloat16)
    w = values(g, 2, n, k, dtype=torch.bfloat16)
    grad, z = (torch.zeros(rows, n, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    grad[-tail:], z[-tail:] = values(g, tail, n, dtype=torch.bfloat16), 1.0
    grad_x, grad_w = og.expert_gemm_backward(grad, x, w, plan, activation="relu", preactivation=z)
    dz, last = grad[-tail:].double(), x[-tail:].double()
    for e, at in ((0, slice(0, tail - 300)), (1, slice(tail - 300, tail))):
        we = w[e].double()
        assert_within(grad_x[-tail:][at], dz[at] @ we, sum_error(dz[at].abs() @ we.abs(), n), "rows")
        # the rows of zeros add nothing, and a sum of them loses nothing
        assert_within(grad_w[e], dz[at].T @ last[at], sum_error(dz[at].abs().T @ last[at].abs(), tail), "weights")
    assert not grad_x[:-tail].any()
    grad_a, grad_b, grad_bias = og.gemm_backward(grad, x, w[0], activation="relu", preactivation=z, want=("a", "b", "bias"))
    assert_within(grad_a[-tail:], dz @ w[0].double(), sum_error(dz.abs() @ w[0].double().abs(), n), "a")
    assert_within(grad_b, dz.T @ last, sum_error(dz.abs().T @ last.abs(), tail), "b")
    assert_within(grad_bias, dz.sum(0), (24 + tail / 64) * 2.0**-24 * dz.abs().sum(0), "bias")
    assert not grad_a[:-tail].any()
    del grad, z, grad_x, grad_a

    n = k = 33024  # two experts' weights
    plan = og.expert_plan(torch.tensor([[0], [1], [1]], dtype=torch.int32, device="cuda"), 2)
    grad, x = values(g, 3, n, dtype=torch.bfloat16), values(g, 3, k, dtype=torch.bfloat16)
    _, grad_w = og.expert_gemm_backward(grad, x, torch.empty(2, n, k, device="cuda", dtype=torch.bfloat16), plan, want=("w",))
    for part in (slice(0, 300), slice(n - 300, n)):
        for e, at in ((0, slice(0, 1)), (1, slice(1, 3))):
            dz, last = grad[at, part].double(), x[at].double()
            assert_within(grad_w[e, part], dz.T @ last, sum_error(dz.abs().T @ last.abs(), 2), f"weights of {e}")

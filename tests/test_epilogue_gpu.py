"""`gemm(..., activation=, residual=, preactivation=)`: C = act(alpha A.B^T + bias) + residual,
against the same formula in 64 bits on the operands' exact values."""

import pytest
import torch

import opengemm_b200 as og
from opengemm_b200 import capi
from opengemm_b200.configs import heuristic_config
from oracle import opengemm_oracle as ora
from tests.feed_forward_util import ACTIVATIONS, act, act_error, assert_within, sum_error
from tests.gemm_util import make_case, to_device

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["native", "interpreter"], autouse=True)
def host_path(request):
    """Every test runs through the native host path and through the Python one."""
    before = capi.use_front(request.param == "native")
    assert (capi.front() is not None) == (request.param == "native")
    yield
    capi.use_front(before)

PLANS = {
    "heuristic": None,
    "pair256": dict(use_2cta=True, output_n=256),
    "single96": dict(use_2cta=False, output_n=96),
    "single16": dict(use_2cta=False, output_n=16),
    "swap64": dict(use_2cta=False, output_n=64, swap_ab=True),
    "direct": dict(use_2cta=True, output_n=128, epi_direct=1),
    # schedules that a fused launch leaves for the static one
    "streamk": dict(use_2cta=True, output_n=128, split_k=2),
    "clc": dict(use_2cta=True, output_n=128, use_clc=True),
    "clusterk": dict(use_2cta=False, output_n=64, cluster_k=4),
}


def operands(name, m, n, k, seed=5):
    case = make_case(name, m, n, k, seed=seed)
    d = og.DTYPES[name]
    raw = [case.get("sfa_raw"), case.get("sfb_raw")]
    exact = [torch.from_numpy(ora.dequantize(name, case[s], raw[i], k, s).copy()).double().cuda() for i, s in enumerate("ab")]
    tensors = [to_device(case["a"], d.a), to_device(case["b"], d.b)]
    tensors += [to_device(case["sfa"], d.sf), to_device(case["sfb"], d.sf)] if d.impl == "smm" else [None, None]
    return tensors, exact


def reference(exact, k, alpha, bias, activation, residual):
    """(z, its error bound, C, its error bound) in 64 bits."""
    a, b = exact
    alpha = 1.0 if alpha is None else alpha
    z = alpha * (a @ b.T)
    error = sum_error(abs(alpha) * (a.abs() @ b.abs().T), k) + 2.0**-23 * z.abs()
    if bias is not None:
        z = z + bias.double()
        error = error + 2.0**-23 * (z.abs() + bias.double().abs())
    c, c_error = act(activation, z), act_error(z, error) if activation else error
    if residual is not None:
        c = c + residual.double()
        c_error = c_error + 2.0**-23 * c.abs()
    return z, error, c, c_error


def element_names(name):
    d = og.DTYPES[name]
    return dict(atype=d.elem_a, btype=d.elem_b) if d.a is torch.uint8 else {}


def check(name, m, n, k, out_dtype, activation, bias=True, residual=True, save=True, alpha=0.5, plan=None):
    (a, b, sfa, sfb), exact = operands(name, m, n, k)
    g = torch.Generator(device="cuda").manual_seed(m * 31 + n)
    bias = torch.randn(n, generator=g, device="cuda") if bias else None
    residual = torch.randn(m, n, generator=g, device="cuda").to(out_dtype) if residual else None
    z = torch.full((m, n), float("nan"), device="cuda", dtype=out_dtype) if save else None
    out = torch.full((m, n), float("nan"), device="cuda", dtype=out_dtype)
    if plan is None:
        fused = dict(alpha=alpha, bias=bias, activation=activation, residual=residual, preactivation=z, **element_names(name))
        og.gemm(a, b, sfa, sfb, out=out, **fused)
        for _ in range(2):  # the second call finds what the first one bound
            if save:
                z.fill_(float("nan"))
            again = og.gemm(a, b, sfa, sfb, out_dtype=out_dtype, **fused)
            assert torch.equal(again, out)
    else:
        config = heuristic_config(name, m, n, k)
        config.update(plan, cluster_m=2 if plan["use_2cta"] else 1)
        suffix = {torch.bfloat16: ".bf16", torch.float16: ".f16"}.get(out_dtype, "") if og.DTYPES[name].impl == "mm" else ""
        lib, bound = capi.bind(name + suffix, m, n, k, config)
        lib.launch_fused(bound, a, b, sfa, sfb, out, alpha, bias, activation, residual, z)
    want_z, z_error, want, error = reference(exact, k, alpha, bias, activation, residual)
    assert_within(out, want, error, "C")
    if save:
        assert_within(z, want_z, z_error, "pre-activation")


@pytest.mark.parametrize("activation", ACTIVATIONS + [None])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("shape", [(1, 8, 64), (300, 520, 768), (77, 33, 128)], ids=lambda s: "x".join(map(str, s)))
def test_bf16_activations_and_outputs(shape, out_dtype, activation):
    check("bf16", *shape, out_dtype, activation)


@pytest.mark.parametrize("name", ["f16", "tf32", "e4m3", "e4m3xe5m2", "e2m1", "e3m2"])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16], ids=str)
def test_dense_formats(name, out_dtype):
    check(name, 130, 264, 512, out_dtype, "gelu")


@pytest.mark.parametrize("name", ["nvfp4", "mxfp8", "mxfp4"])
@pytest.mark.parametrize("shape", [(1, 64, 128), (300, 520, 768), (515, 1031, 512)], ids=lambda s: "x".join(map(str, s)))
def test_block_scaled_formats(name, shape):
    check(name, *shape, torch.bfloat16, "silu")


@pytest.mark.parametrize("plan", list(PLANS))
@pytest.mark.parametrize("name,out_dtype", [("bf16", torch.bfloat16), ("e4m3", torch.float32), ("nvfp4", torch.bfloat16)], ids=str)
def test_every_plan(name, out_dtype, plan):
    check(name, 600, 776, 512, out_dtype, "gelu_tanh", plan=PLANS[plan])


@pytest.mark.parametrize("m", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("name", ["bf16", "f16"])
@pytest.mark.parametrize("n,k", [(1, 8), (53, 3616), (4735, 264), (4741, 72), (9001, 1032)])
def test_a_few_rows(m, name, n, k):
    """Up to four rows take another kernel than the tiled one."""
    check(name, m, n, k, torch.bfloat16 if name == "bf16" else torch.float16, "gelu")
    check(name, m, n, k, torch.float32, "silu", bias=False, save=False, alpha=None)
    check(name, m, n, k, torch.bfloat16, None, residual=True, save=False)


@pytest.mark.parametrize("parts", [dict(bias=False), dict(residual=False), dict(save=False), dict(bias=False, residual=False, save=False),
                                   dict(alpha=None, bias=False, save=False)], ids=str)
@pytest.mark.parametrize("shape", [(2304, 2560, 256), (64, 4096, 256)], ids=lambda s: "x".join(map(str, s)))
def test_parts_of_the_epilogue_and_several_tiles_a_cta(shape, parts):
    check("bf16", *shape, torch.bfloat16, "silu", **parts)
    check("bf16", *shape, torch.float32, None if parts.get("residual", True) else "relu", **parts)


def test_residual_may_be_the_output_and_start_anywhere():
    (a, b, _, _), exact = operands("bf16", 300, 520, 768)
    store = torch.randn(300 * 520 + 1, device="cuda").bfloat16()
    for residual in (store[1:].view(300, 520), store[:-1].view(300, 520)):
        before = residual.clone()
        _, _, want, error = reference(exact, 768, None, None, "silu", before)
        assert_within(og.gemm(a, b, out_dtype=torch.bfloat16, activation="silu", residual=residual), want, error, "any start")
    got = og.gemm(a, b, out=residual, activation="silu", residual=residual)
    assert got is residual
    assert_within(got, want, error, "in place")


def test_values_at_the_ends_of_the_range():
    """Activations of very large, infinite and NaN sums: one-hot rows pick bias values."""
    k, values = 64, [0.0, -0.0, 1e30, -1e30, 3e38, -3e38, float("inf"), float("nan"), 88.0, -88.0, 1e-30, -1e-30, 20.0, -20.0, 5.0, -5.0]
    a = torch.zeros(128, k, device="cuda", dtype=torch.bfloat16)
    b = torch.zeros(16, k, device="cuda", dtype=torch.bfloat16)
    bias = torch.tensor(values, device="cuda")
    for name in ACTIVATIONS:
        got = og.gemm(a, b, bias=bias, activation=name)
        want = act(name, bias.double())
        want[7] = float("nan")
        torch.testing.assert_close(got[5].double(), want.clamp(-3.5e38, 3.5e38).float().double(), rtol=2e-5, atol=1e-6, equal_nan=True)


@pytest.mark.parametrize("out_format", ["nvfp4", "mxfp8", "mxfp4"])
def test_activation_before_block_scaled_output(out_format):
    """The bytes are those of quantising the same call's bfloat16 output."""
    (a, b, _, _), _ = operands("e4m3", 300, 512, 256)
    bias = torch.randn(512, device="cuda")
    plain = og.gemm(a, b, out_dtype=torch.bfloat16, alpha=0.25, bias=bias, activation="gelu")
    packed, scales = og.gemm(a, b, alpha=0.25, bias=bias, activation="gelu", out_format=out_format)
    want, want_scales = og.quantize_blocked(plain, out_format)
    assert torch.equal(packed.view(torch.uint8), want.view(torch.uint8))
    assert torch.equal(scales.view(torch.uint8), want_scales.view(torch.uint8))
    scaled, _ = og.gemm(a, b, alpha=0.25, bias=bias, out_format=out_format)  # alpha and bias without an activation count too
    again, _ = og.quantize_blocked(og.gemm(a, b, out_dtype=torch.bfloat16, alpha=0.25, bias=bias), out_format)
    assert torch.equal(scaled.view(torch.uint8), again.view(torch.uint8))


def test_a_chain_of_fused_products_in_a_graph_and_on_another_stream():
    """Two layers, the second reading the first's output and adding the input: eager on a side
    stream and replayed from a graph, the same bits."""
    torch.manual_seed(3)
    x = torch.randn(200, 256, device="cuda").bfloat16()
    w1, w2 = torch.randn(512, 256, device="cuda").bfloat16() / 16, torch.randn(256, 512, device="cuda").bfloat16() / 23
    bias = torch.randn(512, device="cuda")

    def layer():
        h = og.gemm(x, w1, out_dtype=torch.bfloat16, bias=bias, activation="gelu")
        return og.gemm(h, w2, out_dtype=torch.bfloat16, residual=x)

    want = layer()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(layer(), want)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer()
    x.copy_(torch.randn(200, 256, device="cuda"))
    graph.replay()
    replayed = out.clone()
    assert torch.equal(replayed, layer())


def test_refusals():
    a, b = torch.zeros(64, 64, device="cuda", dtype=torch.bfloat16), torch.zeros(32, 64, device="cuda", dtype=torch.bfloat16)
    good = torch.zeros(64, 32, device="cuda")
    with pytest.raises(TypeError, match="activation"):
        og.gemm(a, b, activation="swish")
    with pytest.raises(TypeError, match="residual"):
        og.gemm(a, b, residual=good.bfloat16())
    with pytest.raises(TypeError, match="residual"):
        og.gemm(a, b, residual=good.t().contiguous().t())
    with pytest.raises(TypeError, match="residual"):
        og.gemm(a, b, residual=good[:32])
    with pytest.raises(TypeError, match="preactivation"):
        og.gemm(a, b, activation="relu", preactivation=torch.zeros(64, 32))
    with pytest.raises(ValueError, match="16-byte"):
        og.gemm(a, b, activation="relu", preactivation=torch.zeros(64 * 32 + 1, device="cuda")[1:].view(64, 32))
    with pytest.raises(ValueError, match="share memory"):
        og.gemm(a, b, out=good, activation="relu", preactivation=good)
    with pytest.raises(ValueError, match="overlap"):
        big = torch.zeros(65, 32, device="cuda")
        og.gemm(a, b, out=big[:64], activation="relu", residual=big[1:])
    with pytest.raises(TypeError, match="bias"):
        og.gemm(a, b, activation="relu", bias=torch.zeros(32, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(TypeError, match="block-scaled"):
        og.gemm(a, torch.zeros(64, 64, device="cuda", dtype=torch.bfloat16), out_format="nvfp4", residual=good)
    ints = torch.zeros(64, 64, device="cuda", dtype=torch.int8)
    with pytest.raises(TypeError, match="integers"):
        og.gemm(ints, ints, activation="relu")


def test_what_is_written_is_not_read():
    """Tiles still to come read the operands: a call may not write over them, not even where its residual is one."""
    a, b = torch.ones(64, 64, device="cuda"), torch.ones(64, 64, device="cuda")
    half_a, half_b = a.bfloat16(), b.bfloat16()
    bias = torch.zeros(64 * 64, device="cuda")
    for _ in range(2):  # as the first call of its shape, and as one known already
        with pytest.raises(ValueError, match="out and a share memory"):
            og.gemm(half_a, half_b, out=half_a, residual=half_a)
        with pytest.raises(ValueError, match="out and b share memory"):
            og.gemm(half_a, half_b, out=half_b, activation="relu")
        with pytest.raises(ValueError, match="out and bias share memory"):
            og.gemm(half_a, half_b, out=bias.view(64, 64), activation="relu", bias=bias[:64])
        for label, z in (("a", half_a), ("b", half_b)):
            with pytest.raises(ValueError, match=f"preactivation and {label} share memory"):
                og.gemm(half_a, half_b, out_dtype=torch.bfloat16, activation="relu", preactivation=z)
        with pytest.raises(ValueError, match="preactivation and bias share memory"):
            og.gemm(half_a, half_b, activation="relu", preactivation=bias.view(64, 64), bias=bias[64:128])
        assert (half_a == 1).all() and (half_b == 1).all() and not bias.any()
        c = og.gemm(half_a, half_b, out_dtype=torch.bfloat16, residual=half_a)  # a as its own residual, C elsewhere
        assert (c == 65).all()

"""The host paths of the feed-forward calls, native and in Python, and the switch that turns
dependent launches off."""

import ctypes
import os
import subprocess
import sys
import threading

import pytest
import torch

import opengemm_b200 as og
from opengemm_b200 import build, capi

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["native", "interpreter"])
def host_path(request):
    """The test runs through the native host path and through the Python one."""
    before = capi.use_front(request.param == "native")
    assert (capi.front() is not None) == (request.param == "native")
    yield request.param
    capi.use_front(before)


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("out_dtype", [None, torch.float32], ids=str)
def test_both_gradients_are_allocated_before_the_first_product(host_path, gather, out_dtype):
    """The weights' gradient starts beside the rows' and waits for nothing before it writes.  Memory
    handed out between the two launches could be what another thread freed there, under a launch of
    its own that still reads it; memory from before the first launch cannot."""
    lib = capi.library("mm")
    real, seen = lib._lib.og_b200_expert_product, []

    def record(product, device, stream):
        seen.append((product[0].mode, torch.cuda.memory_stats()["allocation.all.allocated"]))
        return real(product, device, stream)

    callback = ctypes.CFUNCTYPE(ctypes.c_int32, ctypes.POINTER(capi.OgExpertProduct), ctypes.c_int32, ctypes.c_void_p)(record)
    front = capi.front()
    if front is not None:
        addresses = {name: ctypes.cast(getattr(lib._lib, name), ctypes.c_void_p).value
                     for name in ["og_mm_error"] + ["og_b200_" + name for name in capi._FRONT_SYMBOLS]}
        front.bind({**addresses, "og_b200_expert_product": ctypes.cast(callback, ctypes.c_void_p).value})
    before = lib._expert_product
    lib._expert_product = lambda product, device, stream: callback(ctypes.pointer(product._obj), device, stream)
    try:
        plan = og.expert_plan(torch.tensor([[0, 1], [2, 0], [1, 2], [0, 1]], device="cuda", dtype=torch.int32), 3)
        x = torch.randn(4 if gather else 8, 64, device="cuda").bfloat16()
        w, grad = torch.randn(3, 32, 64, device="cuda").bfloat16(), torch.randn(8, 32, device="cuda").bfloat16()
        z = torch.randn(8, 32, device="cuda").bfloat16()
        og.expert_gemm_backward(grad, x, w, plan, gather=gather, activation="relu", preactivation=z, out_dtype=out_dtype)
    finally:
        lib._expert_product = before
        if front is not None:
            front.bind(addresses)
    assert [mode for mode, _ in seen] == [capi.ROWS_GRADIENT, capi.WEIGHTS_GRADIENT]
    assert seen[0][1] == seen[1][1]


def test_a_preactivation_over_the_plan_is_refused(host_path):
    """The launch would write over the table of rows that its other blocks still read."""
    plan = og.expert_plan(torch.tensor([[0, 1], [2, 0], [1, 2], [0, 1]], device="cuda", dtype=torch.int32), 3)
    x, w = torch.zeros(8, 64, device="cuda", dtype=torch.bfloat16), torch.zeros(3, 4, 64, device="cuda", dtype=torch.bfloat16)
    for part in (plan._store[:16], plan._store[4:]):  # from the offsets on, and from the tokens on
        over = part[:16].view(torch.bfloat16).view(8, 4)
        with pytest.raises(ValueError, match="preactivation and plan share memory"):
            og.expert_gemm(x, w, plan, activation="relu", preactivation=over)


def test_a_factor_past_the_floating_range_is_refused_alike(host_path):
    a, b = torch.zeros(8, 64, device="cuda", dtype=torch.bfloat16), torch.zeros(16, 64, device="cuda", dtype=torch.bfloat16)
    logits = torch.zeros(4, 8, device="cuda")
    og.gemm(a, b, activation="relu", alpha=1)
    weights, indices = og.route(logits, 2, scale=2)
    for call in (lambda f: og.gemm(a, b, activation="relu", alpha=f), lambda f: og.gemm_backward(og.gemm(a, b, out_dtype=torch.bfloat16), a, b, alpha=f),
                 lambda f: og.route(logits, 2, scale=f), lambda f: og.route_backward(weights, logits, indices, scale=f)):
        call(3)
        with pytest.raises(OverflowError):
            call(10**400)


PROGRAMMATIC_EDGES = """
import ctypes
import torch
import opengemm_b200 as og

def step():
    weights, indices = og.route(logits, 2)
    plan = og.expert_plan(indices, 6)
    z = torch.empty(plan.rows, 128, device="cuda", dtype=torch.bfloat16)
    h = og.expert_gemm(x, w, plan, gather=True, activation="swiglu", preactivation=z)
    y = og.expert_combine(h, weights, plan)
    grad_h, grad_weights = og.expert_combine_backward(y, h, weights, plan)
    grad_x, grad_w = og.expert_gemm_backward(grad_h, x, w, plan, gather=True, activation="swiglu", preactivation=z)
    kept = torch.empty(5000, 64, device="cuda", dtype=torch.bfloat16)
    c = og.gemm(tall, wide, out_dtype=torch.bfloat16, activation="gelu", preactivation=kept)
    few = og.gemm(tall[:2], wide, out_dtype=torch.bfloat16, activation="gelu")
    return og.route_backward(grad_weights, logits, indices), grad_x, grad_w, few, *og.gemm_backward(
        c, tall, wide, activation="gelu", preactivation=kept, want=("a", "b", "bias"))

torch.manual_seed(0)
x, logits = torch.randn(300, 64).bfloat16().cuda(), torch.randn(300, 6).cuda()
w, tall, wide = torch.randn(6, 128, 64).bfloat16().cuda(), torch.randn(5000, 72).bfloat16().cuda(), torch.randn(64, 72).bfloat16().cuda()
eager = [t.clone() for t in step()]
graph = torch.cuda.CUDAGraph(keep_graph=True)
with torch.cuda.graph(graph):
    captured = step()
edges_of = ctypes.CDLL("libcuda.so.1").cuGraphGetEdges_v2
handle, count = ctypes.c_void_p(graph.raw_cuda_graph()), ctypes.c_size_t(0)
assert edges_of(handle, None, None, None, ctypes.byref(count)) == 0
ends, data = [(ctypes.c_void_p * count.value)() for _ in range(2)], (ctypes.c_uint8 * (8 * count.value))()
assert edges_of(handle, *ends, data, ctypes.byref(count)) == 0
graph.instantiate()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(eager, captured))
print("programmatic", sum(data[8 * i + 2] == 1 for i in range(count.value)), "of", count.value)  # a type behind two ports
"""


@pytest.mark.parametrize("front", ["1", "0"])
def test_dependent_launches_can_be_turned_off(front):
    """OPENGEMM_PDL=0 leaves no launch that may start before its predecessor has ended, as a captured graph's edges show."""
    counts = {}
    for on in ("1", "0"):
        done = subprocess.run([sys.executable, "-c", PROGRAMMATIC_EDGES], cwd=build.ROOT, capture_output=True, text=True, timeout=300,
                              env={**os.environ, "OPENGEMM_PDL": on, "OPENGEMM_FRONT": front})
        assert done.returncode == 0, done.stderr[-2000:]
        words = done.stdout.split()
        counts[on] = int(words[1]), int(words[3])
    assert counts["1"][0] > counts["1"][1] // 2
    assert counts["0"][0] == 0 and counts["0"][1] >= 12


@pytest.mark.parametrize("m", [2, 200])
def test_a_weight_and_a_bias_that_the_launch_before_writes(m):
    """A launch starts while the one before still writes: its weight, its residual and its bias may be what that one writes."""
    g = torch.Generator().manual_seed(m)
    x = torch.randn(m, 512, generator=g).bfloat16().cuda()
    sources = [torch.randn(1024, 256, generator=g).bfloat16().cuda() for _ in range(8)]
    middle = torch.randn(512, 256, generator=g).bfloat16().cuda()
    one, bias = torch.ones(1, 256, device="cuda", dtype=torch.bfloat16), torch.empty(1, 1024, device="cuda")
    weight, residual = torch.empty(1024, 512, device="cuda", dtype=torch.bfloat16), torch.empty(m, 1024, device="cuda", dtype=torch.bfloat16)

    def step(source, wait):
        og.gemm(one, source, out=bias)
        wait()
        og.gemm(x[:, :256].contiguous(), source, out=residual)
        wait()
        og.gemm(source, middle, out=weight)
        wait()
        return og.gemm(x, weight, out_dtype=torch.bfloat16, bias=bias[0], activation="silu", residual=residual)

    wants = [step(source, torch.cuda.synchronize) for source in sources]
    torch.cuda.synchronize()
    for _ in range(20):
        gots = [step(source, lambda: None) for source in sources]
        for got, want in zip(gots, wants):
            assert torch.equal(got, want)


@pytest.mark.parametrize("out_dtype", [None, torch.float32], ids=str)
def test_two_threads_on_one_stream(host_path, out_dtype):
    """Gradients side by side in one thread, products whose operands are dropped at once in another: memory passes
    from one to the other in the order of the stream, which every launch has to keep."""
    torch.manual_seed(3)
    plan = og.expert_plan(torch.randint(0, 4, (600, 2), device="cuda", dtype=torch.int32), 4)
    x, w = torch.randn(600, 256, device="cuda").bfloat16(), torch.randn(4, 512, 256, device="cuda").bfloat16()
    grad, z = torch.randn(1200, 256, device="cuda").bfloat16(), torch.randn(1200, 512, device="cuda").bfloat16()
    a, b = torch.randn(2048 if out_dtype is None else 4096, 256, device="cuda").bfloat16(), torch.randn(512, 256, device="cuda").bfloat16()

    def gradients():
        return og.expert_gemm_backward(grad, x, w, plan, gather=True, activation="swiglu", preactivation=z, out_dtype=out_dtype)

    def product():
        dropped = a.clone()  # as large as the weights' gradient
        return (og.gemm(dropped, b, out_dtype=torch.bfloat16),)

    calls = {"gradients": gradients, "product": product}
    wants = {name: call() for name, call in calls.items()}
    torch.cuda.synchronize()
    wrong, failed = [], []

    def run(name):
        try:
            for _ in range(150):
                wrong.extend((got != want).any() for got, want in zip(calls[name](), wants[name]))
        except Exception as exc:  # a thread's failure is the test's
            failed.append(exc)

    threads = [threading.Thread(target=run, args=(name,)) for name in ("gradients", "product", "gradients", "product")]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not failed, failed
    assert not torch.stack(wrong).any()

"""The host paths of the feed-forward calls, native and in Python."""

import ctypes

import pytest
import torch

import opengemm_b200 as og
from opengemm_b200 import capi

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

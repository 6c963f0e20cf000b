"""Gradients of activations through the C entry point, and activations far from zero."""

import pytest
import torch

import opengemm_b200 as og
from opengemm_b200 import capi
from tests.feed_forward_util import HALF_STEP, act_gradient

pytestmark = pytest.mark.gpu

CODES = {None: 0, "relu": 1, "gelu": 2, "silu": 4}


@pytest.mark.parametrize("activation", list(CODES), ids=str)
@pytest.mark.parametrize("rows,limit", [(5000, 5000), (5000, 700), (5000, 704), (5000, 1), (5000, 0), (9, 4), (100, 17), (5000, 6000)])
def test_bias_gradient_of_some_of_the_rows(rows, limit, activation):
    """With a row limit on the device the column sums are those of the rows before it, whatever the workspace held."""
    lib, n = capi.library("mm"), 264
    g = torch.Generator().manual_seed(rows + limit)
    live, held = min(rows, limit), max(rows, limit)
    grad, z = (torch.randn(held, n, generator=g).bfloat16().cuda() for _ in range(2))
    grad[live:], z[live:] = float("nan"), float("nan")
    dz = torch.full_like(grad, 7.0)
    bias = torch.full((n,), float("nan"), device="cuda")
    workspace = torch.full((-(-rows // 16) * n,), float("nan"), device="cuda")
    at = torch.tensor([limit], dtype=torch.int32, device="cuda")
    lib.routing(lib._activation_gradient, 1, CODES[activation], grad.data_ptr(), z.data_ptr(), dz.data_ptr(), bias.data_ptr(),
                workspace.data_ptr(), at.data_ptr(), rows, n, 0)
    want = act_gradient(activation, z[:live].double(), grad[:live].double())
    # as the gradients of a whole product: sums of at most 8 rows, of 8 row lanes, of blocks in eight lanes
    error = (24 + rows / 64) * 2.0**-24 * want.abs().sum(0)
    if activation:
        error += (2e-6 * grad[:live].double().abs() * (z[:live].double().abs() + 2)).sum(0)
        assert (dz[live:] == 7.0).all()
        assert ((dz[:live].double() - want).abs() <= HALF_STEP[torch.bfloat16] * want.abs() + 3e-6 * grad[:live].double().abs() * (z[:live].double().abs() + 2)).all()
    assert ((bias.double() - want.sum(0)).abs() <= error + 1e-30).all()


# Phi(-|x|) = exp(-x^2 / 2) R(|x|), in units of 2^-24: x^2, its product with a rounded constant and that
# constant are three roundings of x^2 / 2; the exponential is good to 2 units of the last place (4), the
# reciprocal in R to one (2) of a value rounded once before, R's polynomial to 8, and three products.
def tail_error(x):
    return (1.5 * x * x + 20) * 2.0**-24


def far_values(dtype):
    """Every value of the type from -13 to 13, a multiple of 8 by 64 of them."""
    x = torch.arange(-2**15, 2**15, dtype=torch.int32).to(torch.int16).view(dtype)
    x = x[x.isfinite() & (x.abs() <= 13)]
    return torch.cat([x, x.new_zeros(-x.numel() % 512)]).view(-1, 64).cuda()


@pytest.mark.parametrize("rows", [4, None], ids=["few rows", "tiles"])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_gelu_keeps_its_digits_far_below_zero(dtype, out_dtype, rows):
    """gelu(x) for x < 0 is x Phi(x): as exact, relative to itself, as anywhere else."""
    x = far_values(dtype)
    one = torch.eye(64, device="cuda", dtype=dtype)
    parts = [x] if rows is None else list(x.split(rows))[::37]
    for part in parts:
        got = og.gemm(part, one, out_dtype=out_dtype, activation="gelu").double()
        z = part.double()
        want = z * 0.5 * torch.special.erfc(-z / 2**0.5)
        error = tail_error(z) * want.abs()
        step = 2.0**-24 if out_dtype is torch.float16 else 0.0  # of its subnormal values: half a step is 2^-25
        assert ((got - want).abs() <= error + HALF_STEP[out_dtype] * (want.abs() + error) + max(step / 2, 1e-36)).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_slope_of_gelu_keeps_its_digits_far_below_zero(dtype):
    """A gradient of ones over a single row: the bias's float32 sums are the slopes themselves."""
    z = far_values(dtype)[::5].contiguous().view(1, -1)
    n = z.numel()
    operand = torch.zeros(1, 8, device="cuda", dtype=dtype)
    b = torch.zeros(n, 8, device="cuda", dtype=dtype)
    got = og.gemm_backward(torch.ones_like(z), operand, b, activation="gelu", preactivation=z, want=("bias",))[2].double()
    x = z[0].double()
    cdf, density = 0.5 * torch.special.erfc(-x / 2**0.5), torch.exp(-x * x / 2) / (2 * torch.pi) ** 0.5
    # x times the density has three more products
    assert ((got - (cdf + x * density)).abs() <= (tail_error(x) + 4 * 2.0**-24) * (cdf + x.abs() * density) + 1e-36).all()

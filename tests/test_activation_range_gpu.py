"""Gradients of activations through the C entry point."""

import pytest
import torch

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

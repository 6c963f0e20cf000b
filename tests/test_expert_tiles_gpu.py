"""The experts' products through the C entry point: what the Python calls' sizes do not reach."""

from ctypes import byref

import pytest
import torch

from opengemm_b200 import capi
from tests.feed_forward_util import act, act_error, assert_within, sum_error
from tests.test_experts_gpu import gated_error

pytestmark = pytest.mark.gpu

# Rows of each expert: none, one, around the boxes of 64 and the tiles of 128 and 256 rows.
ROWS = [0, 1, 63, 64, 65, 0, 127, 128, 129, 255, 256, 257, 300, 520, 0]
BEHIND = 37  # rows behind the last expert's


def table(rows=ROWS):
    """(offsets, slices of the experts that have rows, rows in all)."""
    offsets = torch.tensor([0] + rows).cumsum(0)
    return offsets.int().cuda(), [(e, slice(int(offsets[e]), int(offsets[e + 1]))) for e in range(len(rows)) if rows[e]], int(offsets[-1])


def values(g, *shape, dtype, spread=1.0):
    return (torch.randn(*shape, generator=g) * spread).to(dtype).cuda()


def launch(mode, dtype, x, w, out, offsets, groups, rows, n, k, **more):
    name = {torch.bfloat16: b"bf16", torch.float16: b"f16", torch.float8_e4m3fn: b"e4m3"}[dtype]
    product = capi.OgExpertProduct(x=x.data_ptr(), w=w.data_ptr(), offsets=offsets.data_ptr(), out=out.data_ptr(), mode=mode, groups=groups, rows=rows, n=n, k=k,
                                   out_f32=out.dtype is torch.float32, factor=1.0, dtype=name, **more)
    lib = capi.library("mm")
    assert lib._expert_product(byref(product), 0, capi.raw_stream(0)) == capi.OG_OK, lib._experts_error().decode()


def check_forward(dtype, n, k, activation=None, gather=False, save=False, **more):
    g = torch.Generator().manual_seed(n + k)
    offsets, experts, last = table()
    rows, gated = last + BEHIND, activation in capi.GATED_ACTIVATIONS
    tokens = torch.randint(0, 400, (rows,), generator=g).int().cuda() if gather else None
    x, w = values(g, 400 if gather else rows, k, dtype=dtype), values(g, len(ROWS), n, k, dtype=dtype, spread=k**-0.5)
    alpha = (torch.rand(len(ROWS), generator=g) + 0.5).cuda()
    own = torch.bfloat16 if dtype is torch.float8_e4m3fn else dtype
    out, z = torch.full((rows, n // 2 if gated else n), 7.0, device="cuda", dtype=own), torch.full((rows, n), 7.0, device="cuda", dtype=own)
    if gather:
        tokens[last:] = 2**30  # not looked at
        more.update(tokens=tokens.data_ptr(), x_rows=400)
    launch(capi.FORWARD, dtype, x, w, out, offsets, len(ROWS), rows, n, k, alpha=alpha.data_ptr(), activation={**capi.ACTIVATIONS, **capi.GATED_ACTIVATIONS}[activation],
           preactivation=z.data_ptr() if save else 0, **more)
    for e, at in experts:
        mine = (x[tokens[at].long()] if gather else x[at]).double()
        want = alpha[e].double() * (mine @ w[e].double().T)
        error = sum_error(alpha[e].double() * (mine.abs() @ w[e].double().abs().T), k) + 2.0**-23 * want.abs()
        if save:
            assert_within(z[at], want, error, f"pre-activation of {e}")
        error = gated_error(activation, want, error) if gated else act_error(want, error) if activation else error
        assert_within(out[at], act(activation, want), error, f"product of {e}")
    assert (out[last:] == 7.0).all() and (z[last if save else 0:] == 7.0).all()


@pytest.mark.parametrize("activation", [None, "swiglu"], ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn], ids=str)
def test_many_gathered_rows(dtype, activation):
    """More rows an expert than the Python call gathers in the product."""
    check_forward(dtype, 592, 208, activation, gather=True)

"""The experts' products through the C entry point: every tile, whatever the sizes would choose, and
what the Python calls' sizes do not reach."""

from ctypes import byref

import pytest
import torch

from opengemm_b200 import capi
from tests.feed_forward_util import act, act_error, assert_within, sum_error
from tests.test_experts_gpu import check, check_gemm_gradients, check_gradients, gated_error

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


TILES = {"pair": 1, "256": 2, "128": 3, "64": 4}
# Columns and reduction: whole tiles, and neither whole tiles nor whole blocks of either.
SIZES = [(512, 128), (592, 208), (1040, 72)]


@pytest.fixture(params=list(TILES))
def tile(request):
    return TILES[request.param]


@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("activation", [None, "gelu", "swiglu", "geglu"], ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_forward(dtype, activation, size, tile):
    check_forward(dtype, *size, activation, tile=tile)
    check_forward(dtype, size[0] + 8 * (activation not in capi.GATED_ACTIVATIONS), size[1], activation, save=True, tile=tile)


@pytest.mark.parametrize("size", [(512, 128), (592, 208), (1040, 80)], ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("activation", [None, "relu", "gelu", "gelu_tanh", "silu", "swiglu", "geglu"], ids=str)
def test_forward_e4m3(activation, size, tile):
    for save in (False, True):
        check_forward(torch.float8_e4m3fn, *size, activation, save=save, tile=tile)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn], ids=str)
@pytest.mark.parametrize("activation", [None, "geglu"], ids=str)
@pytest.mark.parametrize("narrow", ["256", "128", "64"])
def test_forward_gathered(dtype, activation, narrow):
    check_forward(dtype, 592, 208, activation, gather=True, save=True, tile=TILES[narrow])


@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("out_dtype", [None, torch.float32], ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_rows_gradient(dtype, out_dtype, size, tile):
    k, n = size
    g = torch.Generator().manual_seed(n + k)
    offsets, experts, last = table()
    rows = last + BEHIND
    dz, w = values(g, rows, n, dtype=dtype), values(g, len(ROWS), n, k, dtype=dtype, spread=n**-0.5)
    dz[last:] = float("nan")
    out = torch.full((rows, k), 7.0, device="cuda", dtype=out_dtype or dtype)
    launch(capi.ROWS_GRADIENT, dtype, dz, w, out, offsets, len(ROWS), rows, n, k, tile=tile)
    for e, at in experts:
        mine, we = dz[at].double(), w[e].double()
        assert_within(out[at], mine @ we, sum_error(mine.abs() @ we.abs(), n), f"rows of {e}")
    assert (out[last:] == 7.0).all()


def check_weights_gradient(dtype, n, k, tile, out_dtype=None, rows_of=ROWS, poison=None):
    g = torch.Generator().manual_seed(n + k)
    offsets, experts, last = table(rows_of)
    rows = last + BEHIND
    dz, x = values(g, rows, n, dtype=dtype), values(g, rows, k, dtype=dtype)
    dz[last:], x[last:] = float("nan"), float("inf")
    if poison is not None:
        dz[dict(experts)[poison]] = float("nan")
    out = torch.full((len(rows_of), n, k), 7.0, device="cuda", dtype=out_dtype or dtype)
    launch(capi.WEIGHTS_GRADIENT, dtype, dz, x, out, offsets, len(rows_of), rows, n, k, tile=tile)
    for e in range(len(rows_of)):
        at = dict(experts).get(e, slice(0, 0))
        if e == poison:
            assert out[e].isnan().all()
            continue
        mine, xs = dz[at].double(), x[at].double()
        assert_within(out[e], mine.T @ xs, sum_error(mine.abs().T @ xs.abs(), rows_of[e]), f"weights of {e}, {rows_of[e]} rows")


@pytest.mark.parametrize("size", SIZES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("out_dtype", [None, torch.float32], ids=str)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_weights_gradient(dtype, out_dtype, size, tile):
    """Most groups end inside a block of 64 rows, whose rest belongs to the next expert or is no number at all."""
    check_weights_gradient(dtype, *size, tile, out_dtype)


def test_weights_gradient_beside_rows_of_nan(tile):
    """What is behind a group's end, whole boxes or single rows of it, reaches only its own expert."""
    for poison in (1, 3, 7, 12):
        check_weights_gradient(torch.bfloat16, 592, 208, tile, poison=poison)


def test_weights_gradient_of_one_group_without_a_table(tile):
    """The gradient of a plain product; reductions past a whole ring of stages, ended short by 1 to 63 rows."""
    g = torch.Generator().manual_seed(3)
    for rows in (1, 63, 1000, 1025, 4095, 4100):
        dz, x = values(g, rows, 264, dtype=torch.bfloat16), values(g, rows, 520, dtype=torch.bfloat16)
        out = torch.empty(264, 520, device="cuda", dtype=torch.float32)
        product = capi.OgExpertProduct(x=dz.data_ptr(), w=x.data_ptr(), out=out.data_ptr(), mode=capi.WEIGHTS_GRADIENT, groups=1, rows=rows, n=264, k=520, out_f32=1,
                                       factor=0.5, tile=tile, dtype=b"bf16")
        lib = capi.library("mm")
        assert lib._expert_product(byref(product), 0, capi.raw_stream(0)) == capi.OG_OK
        a, b = dz.double(), x.double()
        assert_within(out, 0.5 * (a.T @ b), 0.5 * sum_error(a.abs().T @ b.abs(), rows), f"{rows} rows")


def test_many_tiles_a_cluster(tile):
    """Accumulators, ring and barriers go round several times in every CTA, short blocks among whole ones."""
    rows = [700, 0, 65, 1300, 256, 1, 2111, 640] * 4
    check_weights_gradient(torch.bfloat16, 776, 520, tile, rows_of=rows)


@pytest.mark.parametrize("shape", [(4100, 4096, 4096), (2600, 2048, 1544)], ids=lambda s: "x".join(map(str, s)))
def test_gemm_gradients_of_training_sizes(shape):
    """As in training: the larger chooses pairs of CTAs for both gradients, the smaller for the weights', and both end inside a block of rows."""
    check_gemm_gradients(*shape, torch.bfloat16, "gelu_tanh", alpha=0.5)


@pytest.mark.parametrize("shape", [(3900, 2, 8, 2048, 1024)], ids=lambda s: "x".join(map(str, s)))
def test_a_prompt_of_experts(shape):
    """Some hundreds of rows an expert: the sizes that choose pairs of CTAs."""
    check(*shape, activation="swiglu", save=True)
    check(*shape, dtype=torch.float8_e4m3fn, activation="geglu", scaled=True)
    check(*shape, gather=False)
    check_gradients(*shape, activation="swiglu")

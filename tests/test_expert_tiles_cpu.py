"""Tiles that an experts' product refuses before it touches a device: needs no GPU."""

from ctypes import byref

import pytest

from opengemm_b200 import capi

SOME = 0x10000  # an address that is never followed


@pytest.mark.parametrize("fields", [dict(tile=-1), dict(tile=5), dict(tile=1, tokens=SOME)], ids=str)
def test_tiles_refused(fields):
    lib = capi.library("mm")
    product = capi.OgExpertProduct(x=SOME, w=SOME, offsets=SOME, out=SOME, groups=4, rows=8, x_rows=8, n=64, k=64, factor=1.0, dtype=b"bf16", **fields)
    assert lib._expert_product(byref(product), 0, 0) != capi.OG_OK
    assert "tile" in lib._experts_error().decode()

"""Null pointers that the feed-forward entry points refuse before they touch a device: needs no GPU."""

import pytest

from opengemm_b200 import capi

SOME = 0x10000  # an address that is never followed


def refused(code):
    assert code != capi.OG_OK
    assert "null" in capi.library("mm")._routing_error().decode()


def test_combine_refuses_null_rows():
    lib = capi.library("mm")
    for y_is_f32 in (0, 1):
        refused(lib._expert_combine(1, y_is_f32, 0, SOME, SOME, 0, SOME, 4, 2, 64, 0, 0))


@pytest.mark.parametrize("missing", ["grad", "y", "weights", "positions", "grad_y", "grad_weights"])
def test_combine_gradient_refuses_null(missing):
    args = [0 if name == missing else SOME for name in ("grad", "y", "weights", "positions", "grad_y", "grad_weights")]
    refused(capi.library("mm")._expert_combine_gradient(1, *args, 4, 2, 64, 0, 0))

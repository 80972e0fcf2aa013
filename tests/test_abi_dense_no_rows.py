"""No rows: an empty tensor's address is NULL, and there is nothing to read or write. Without a GPU:
nothing is launched."""

import ctypes

import pytest

from bux_amd import _lib


@pytest.mark.parametrize("twin", ["", "_f32"])
def test_slope(twin):
    lib = _lib.load()
    low = () if twin else (None,)  # bfloat16's low bytes
    plain = _lib.FfnStruct(0, 0, 0, 0.0, 0, 0.0, 0.0)
    for ffn in (ctypes.byref(plain), None):
        # dy, product and dz of no rows
        assert getattr(lib, "bux_dense_slope" + twin)(
            None, *low, None, ffn, 0, 64, None, None, None, 0, None) == 0, lib.bux_last_error()
    # what is wrong with rows is wrong without
    gated = _lib.FfnStruct(0, 1, 0, 0.0, 0, 0.0, 0.0)
    assert getattr(lib, "bux_dense_slope" + twin)(
        None, *low, None, ctypes.byref(gated), 0, 64, None, None, None, 0, None) == 1

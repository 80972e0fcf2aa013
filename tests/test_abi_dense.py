"""The dense products' and the clipping's host checks, without a GPU: every call is refused before
a launch."""

import ctypes

import pytest

from bux_amd import _lib

P = ctypes.c_void_p(16)  # never dereferenced


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _msg(lib):
    return lib.bux_last_error().decode()


def _ffn(activation=0, gated=1, clamped=0, limit=0.0, capped=0, cap=0.0):
    return _lib.FfnStruct(activation, gated, clamped, limit, capped, cap, 0.0)


@pytest.mark.parametrize("twin", ["", "_f32"])
def test_rows(lib, twin):
    def rows(x=P, w=P, m=4, n=64, k=64, ffn=None, residual=None, out=P, ws=None, nbytes=0,
             low=None):
        st = None if ffn is None else ctypes.byref(ffn)
        kept = (None,) if twin else (None, low)  # product, and bfloat16's low bytes
        return getattr(lib, "bux_dense_rows" + twin)(x, w, 0, m, n, k, None, st, residual, *kept,
                                                     out, ws, nbytes, None)

    for shape in (dict(m=-1), dict(n=0), dict(k=0), dict(n=-8)):
        assert rows(**shape) == 1 and "bad shape" in _msg(lib)
    for side in "mnk":
        assert rows(**{side: 1 << 31}) == 1 and "2^31" in _msg(lib)
    for missing in ("x", "w", "out"):
        assert rows(**{missing: None}) == 1 and "NULL" in _msg(lib)
    assert rows(ffn=_ffn(10)) == 1 and "activation 10" in _msg(lib)
    assert rows(ffn=_ffn(clamped=1, limit=-1.0)) == 1 and "limit" in _msg(lib)
    assert rows(ffn=_ffn(capped=1)) == 1 and "up_softcap" in _msg(lib)
    assert rows(ffn=_ffn(), n=63) == 1 and "even n" in _msg(lib)
    assert rows(ffn=_ffn(), residual=P) == 1 and "residual" in _msg(lib)
    # a long K of few tiles goes in parts, which need their workspace
    need = lib.bux_dense_workspace_size(4, 64, 65536)
    assert need >= 2 * 4 * 64 * 4
    assert rows(k=65536, ws=P, nbytes=8) == 2 and "workspace of 8 bytes" in _msg(lib)
    assert rows(k=65536) == 2
    assert rows(k=65536, ws=ctypes.c_void_p(8), nbytes=need) == 1 and "unaligned" in _msg(lib)
    if not twin:
        assert rows(low=P) == 1 and "low bytes" in _msg(lib)
    assert rows(m=0, x=None) == 0  # nothing to do


@pytest.mark.parametrize("twin", ["", "_f32"])
def test_units_backward(lib, twin):
    def backward(dy=P, m=4, f=64, d=64, ffn=_ffn(), nbytes=0, dp=P):
        st = None if ffn is None else ctypes.byref(ffn)
        kept, out = ((P,), (dp,)) if twin else ((P, None), (dp, None))  # and the low bytes
        return getattr(lib, "bux_dense_units_backward" + twin)(dy, P, m, f, d, *kept, st, *out, None,
                                                               nbytes, None)

    assert backward(f=0) == 1 and "bad shape" in _msg(lib)
    assert backward(ffn=None) == 1 and "NULL ffn" in _msg(lib)
    assert backward(ffn=_ffn(11)) == 1 and "activation 11" in _msg(lib)
    assert backward(dy=None) == 1 and "NULL" in _msg(lib)
    assert backward(dp=None) == 1 and "NULL" in _msg(lib)
    assert backward(d=65536) == 2 and "workspace" in _msg(lib)


@pytest.mark.parametrize("twin", ["", "_f32"])
def test_contract(lib, twin):
    def contract(x=P, m=4, k=64, n=64, dw=P):
        return getattr(lib, "bux_dense_contract" + twin)(x, P, m, k, n, dw, None, 0, None)

    assert contract(k=0) == 1 and "bad shape" in _msg(lib)
    assert contract(m=-1) == 1 and "bad shape" in _msg(lib)
    assert contract(x=None) == 1 and "NULL" in _msg(lib)
    assert contract(dw=None) == 1 and "NULL" in _msg(lib)
    assert contract(m=65536) == 2 and "workspace" in _msg(lib)


@pytest.mark.parametrize("twin", ["", "_f32"])
def test_slope(lib, twin):
    def slope(dy=P, product=P, ffn=_ffn(gated=0), m=4, n=64, dz=P, sums=None, low=None):
        st = None if ffn is None else ctypes.byref(ffn)
        given = (dy, product) if twin else (dy, low, product)
        return getattr(lib, "bux_dense_slope" + twin)(*given, st, m, n, dz, sums, None, 0, None)

    assert slope(n=0) == 1 and "bad shape" in _msg(lib)
    assert slope(ffn=_ffn()) == 1 and "gated" in _msg(lib)
    assert slope(product=None) == 1 and "product" in _msg(lib)
    assert slope(ffn=None) == 1 and "product" in _msg(lib)
    assert slope(dz=None) == 1 and "nothing" in _msg(lib)
    assert slope(dy=None) == 1 and "NULL" in _msg(lib)
    if not twin:
        assert slope(low=P) == 1 and "low bytes" in _msg(lib)
        assert slope(low=P, ffn=None, product=None) == 1 and "low bytes" in _msg(lib)
    assert slope(m=1 << 20, sums=P) == 2 and "workspace" in _msg(lib)


def test_clip(lib):
    def clip(*grads, max_norm=1.0, norm=P, ws=P, nbytes=1 << 20):
        table = (_lib.GradientStruct * max(1, len(grads)))(
            *(_lib.GradientStruct(*g) for g in grads))
        return lib.bux_clip(table, len(grads), max_norm, norm, ws, nbytes, None)

    assert clip() == 1 and "0 gradients" in _msg(lib)
    assert clip((16, 16, -1, 0)) == 1 and "-1 elements" in _msg(lib)
    assert clip((16, 16, 1 << 40, 0)) == 1 and "elements" in _msg(lib)
    assert clip((16, 16, 8, 2)) == 1 and "dtype 2" in _msg(lib)
    assert clip((None, 16, 8, 0)) == 1 and "gradient 0 is NULL" in _msg(lib)
    assert clip((16, 16, 8, 0), (16, None, 8, 0)) == 1 and "gradient 1 has no output" in _msg(lib)
    assert clip((16, None, 8, 0), (16, 16, 8, 0)) == 1 and "gradient 0 has no output" in _msg(lib)
    for most in (0.0, -1.0, float("nan")):
        assert clip((16, 16, 8, 0), max_norm=most) == 1 and "max_norm" in _msg(lib)
    assert clip((16, 16, 8, 0), norm=None) == 1 and "norm" in _msg(lib)
    assert clip((16, 16, 8, 0), ws=None) == 2 and "workspace" in _msg(lib)
    assert clip((16, 16, 8, 0), nbytes=lib.bux_clip_workspace_size(1) - 1) == 2
    assert clip((16, 16, 8, 0), ws=ctypes.c_void_p(4)) == 1 and "unaligned" in _msg(lib)
    # a list of more tensors takes more launches' sums
    assert lib.bux_clip_workspace_size(1000) > lib.bux_clip_workspace_size(1) > 0
    assert lib.bux_clip_workspace_size(0) == 0

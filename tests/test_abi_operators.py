"""The C-ABI of the operators around the experts without a GPU: the host-side checks turn bad
shapes, settings and workspaces into error codes and messages before any kernel launch."""

import ctypes
import os

import pytest

from bux_amd import _lib

P = ctypes.c_void_p(16)  # never dereferenced: the checks fail first


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.PATH):
        pytest.fail(f"{_lib.PATH} is not built: run python -m bux_amd.build")
    return _lib.load()


def _msg(lib) -> str:
    return lib.bux_last_error().decode()


def _norm(kind=0, affine=1, bias=1, eps=1e-6):
    return ctypes.byref(_lib.NormStruct(kind, affine, 0, 0, bias, eps))


@pytest.mark.parametrize("twin", ["", "_f32"])
def test_the_tokens_norm_rejects_bad_arguments(lib, twin):
    forward = getattr(lib, "bux_norm_forward" + twin)
    backward = getattr(lib, "bux_norm_backward" + twin)

    def fwd(m=4, d=64, norm=_norm(), residual=None, scale=P, bias=P, summed=None, x=P, out=P):
        return forward(x, residual, m, d, norm, scale, bias, summed, out, P, None)

    def bwd(m=4, d=64, norm=_norm(), dy=P, scale=P, d_scale=P, d_bias=P, ws=P, nbytes=1 << 20,
            stats=P):
        return backward(dy, P, stats, None, m, d, norm, scale, P, d_scale, d_bias, ws, nbytes, None)

    for call in (fwd, bwd):
        for bad in ({"d": 7}, {"d": 12289}, {"m": -1}, {"m": 1 << 31}):
            assert call(**bad) == 1 and "bad shape" in _msg(lib), bad
        assert call(norm=None) == 1 and "NULL norm" in _msg(lib)
        assert call(norm=_norm(kind=2)) == 1 and "kind 2" in _msg(lib)
        assert call(norm=_norm(eps=-1.0)) == 1 and "eps" in _msg(lib)
        assert call(norm=_norm(eps=float("nan"))) == 1 and "eps" in _msg(lib)
        assert call(scale=None) == 1 and "scale" in _msg(lib)
    assert fwd(bias=None) == 1 and "bias" in _msg(lib)
    assert fwd(residual=P) == 1 and "summed" in _msg(lib)
    assert fwd(summed=P) == 1 and "summed" in _msg(lib)
    assert fwd(x=None) == 1 and "NULL buffer" in _msg(lib)
    assert fwd(out=None) == 1 and "NULL buffer" in _msg(lib)
    assert fwd(m=0, x=None, out=None) == 0
    assert bwd(d_scale=None) == 1 and "d_scale" in _msg(lib)
    assert bwd(d_bias=None) == 1 and "d_bias" in _msg(lib)
    assert bwd(dy=None) == 1 and "NULL buffer" in _msg(lib)
    assert bwd(stats=None) == 1 and "NULL buffer" in _msg(lib)
    assert bwd(nbytes=2 * 4 * 64 * 4 - 1) == 2 and "workspace" in _msg(lib)
    assert bwd(ws=None) == 2 and "workspace" in _msg(lib)


def test_the_tokens_norms_workspace_never_falls_as_rows_grow(lib):
    size = lib.bux_norm_backward_workspace_size
    for d in (8, 1537, 2048, 12288):
        sizes = [size(m, d) for m in [*range(0, 1100), 4096, 70000, 1 << 30]]
        assert sizes == sorted(sizes) and sizes[0] == 0
        assert all(s <= 8 * m * d for m, s in enumerate(sizes[:1100]))
        assert sizes[-1] <= 8192 * d
    for m in (1, 513, 70000):
        sizes = [size(m, d) for d in range(8, 12289)]
        assert sizes == sorted(sizes)


def test_the_routers_backward_rejects_bad_arguments(lib):
    def call(t=8, d=64, n=32, router=0, scored=30, k=2, kernel=P, d_kernel=P, x=P, d_sinks=P,
             ws=P, nbytes=1 << 24):
        return lib.bux_route_backward(x, kernel, t, d, n, 1.0, router, scored, P, k, 1, 1.0, P, P,
                                      d_sinks, None, None, None, P, d_kernel, P, ws, nbytes, None)

    for bad, word in (({"t": -1}, "t=-1"), ({"d": 40}, "d=40"), ({"d": 0}, "d=0"),
                      ({"n": 0}, "n_logits=0"), ({"n": 1025}, "n_logits=1025"),
                      ({"scored": 0}, "scored=0"), ({"scored": 33}, "scored=33"),
                      ({"router": 3}, "router=3"), ({"k": 0}, "k=0"), ({"k": 17}, "k=17"),
                      ({"scored": 1, "k": 2}, "k=2"), ({"scored": 32}, "d_sinks"),
                      ({"kernel": None}, "NULL"), ({"d_kernel": None}, "NULL"), ({"x": None}, "NULL"),
                      ({"x": ctypes.c_void_p(18)}, "aligned"), ({"ws": ctypes.c_void_p(24)}, "aligned"),
                      ({"t": 1 << 30, "d": 4096}, "launch")):
        assert call(**bad) == 1 and word in _msg(lib), (bad, _msg(lib))
    need = lib.bux_route_backward_workspace_size(8, 64, 32)
    assert need >= 8 * 32 * 4 + 64 * 32 * 4
    assert call(nbytes=need - 1) == 2 and "workspace" in _msg(lib)
    assert call(ws=None) == 2 and "workspace" in _msg(lib)


@pytest.mark.parametrize("twin", ["", "_f32"])
def test_the_int8_quantizers_reject_bad_arguments(lib, twin):
    quantize = getattr(lib, "bux_int8_quantize" + twin)
    glu = getattr(lib, "bux_int8_glu" + twin)
    columns = getattr(lib, "bux_int8_quantize_columns" + twin)

    def rows(rows=8, cols=64, height=8, index=None, div=1, sources=8, x=P, values=P, ws=None,
             nbytes=0):
        return quantize(x, index, div, sources, rows, cols, height, None, values, P, ws, nbytes, None)

    for bad, word in (({"rows": -1}, "rows=-1"), ({"height": 7}, "height=7"),
                      ({"height": 1 << 26}, "height"), ({"height": (1 << 26) - 3}, "height"),
                      ({"cols": 0}, "cols=0"),
                      ({"cols": 131073}, "cols=131073"), ({"index": P, "div": 0}, "index_div=0"),
                      ({"index": P, "sources": -1}, "sources=-1"), ({"x": None}, "NULL"),
                      ({"values": None}, "NULL")):
        assert rows(**bad) == 1 and word in _msg(lib), (bad, _msg(lib))
    assert rows(rows=0, height=0, x=None, values=None) == 0
    # many rows of few tokens take room for the tokens' own codes
    size = lib.bux_int8_quantize_workspace_size
    assert size(8, 8, 64) == 0 and size(16384, 131072, 2048) >= 16384 * 2052
    big = {"rows": 131072, "height": 131072, "cols": 2048, "sources": 16384, "index": P, "div": 8}
    assert rows(**big) == 2 and "workspace" in _msg(lib)
    assert rows(ws=P, nbytes=size(16384, 131072, 2048) - 1, **big) == 2 and "workspace" in _msg(lib)

    odd = ctypes.c_void_p(24)
    assert rows(ws=odd, nbytes=1 << 30, **big) == 1 and "aligned" in _msg(lib)
    wide = {"rows": 1 << 25, "height": 1 << 25, "cols": 131072, "sources": 1 << 20, "index": P}
    assert rows(ws=P, nbytes=1 << 40, **wide) == 1 and "launch" in _msg(lib)

    def units(m=8, f=64, height=8, act=0, projected=P):
        ffn = _lib.FfnStruct(act, 1, 0, 0.0, 0, 0.0, 0.0)
        return glu(projected, P, None, m, f, ctypes.byref(ffn), height, P, P, None)

    for bad, word in (({"f": 66}, "f=66"), ({"f": 0}, "cols=0"), ({"height": 4}, "height=4"),
                      ({"act": 10}, "activation 10"), ({"projected": None}, "NULL")):
        assert units(**bad) == 1 and word in _msg(lib), (bad, _msg(lib))
    for g, k, n, w in ((-1, 64, 64, P), (1, 0, 64, P), (1, 64, 0, P), (1, 131073, 64, P),
                       (1, 64, 64, None)):
        assert columns(w, g, k, n, P, P, None) == 1, (g, k, n)


def test_the_int8_products_reject_bad_arguments(lib):
    def call(groups=4, m=128, n=64, k=128, height=128, out=0, a=P, y=P, llist=P, nbytes=1 << 20):
        return lib.bux_int8_grouped_rows_listed(a, P, P, P, llist, nbytes, groups, m, n, k, height,
                                                out, None, y, None)

    for bad, word in (({"groups": 0}, "groups=0"), ({"groups": 4097}, "groups=4097"),
                      ({"k": 64}, "k=64"), ({"k": 0}, "k=0"), ({"k": 131200}, "k=131200"),
                      ({"n": 66}, "n=66"), ({"n": 0}, "n=0"), ({"m": -1}, "m=-1"),
                      ({"m": 33_554_177, "nbytes": 1 << 40}, "33554176"), ({"out": 2}, "out_dtype"),
                      ({"a": None}, "NULL"), ({"y": None}, "NULL")):
        assert call(**bad) == 1 and word in _msg(lib), (bad, _msg(lib))
    need = lib.bux_mx_grouped_rows_workspace_size(4, 128, 128)
    assert call(nbytes=need - 1) == 2 and "list" in _msg(lib)
    assert call(llist=None) == 2 and "list" in _msg(lib)

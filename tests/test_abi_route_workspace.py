"""The router's backward: a workspace made for a batch holds every shorter one."""

import os

import pytest

from bux_amd import _lib


@pytest.mark.parametrize("d,n", [(16, 1), (16, 1024), (2048, 128), (2064, 130), (2880, 32), (7168, 256)])
def test_the_workspace_never_falls_as_tokens_grow(d, n):
    if not os.path.exists(_lib.PATH):
        pytest.fail(f"{_lib.PATH} is not built: run python -m bux_amd.build")
    size = _lib.load().bux_route_backward_workspace_size
    sizes = [size(t, d, n) for t in [*range(0, 5000), *range(5000, 70000, 16), 1 << 20, 1 << 27]]
    assert sizes == sorted(sizes)

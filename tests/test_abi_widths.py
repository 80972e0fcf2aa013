"""The grouped products refuse outputs so wide that a tile of them exceeds the stores' 32-bit
offsets (on the host: no kernel is launched)."""

import ctypes
import os

import pytest

from bux_amd import _lib

P = ctypes.c_void_p(16)  # never dereferenced: the checks fail first
N = 1 << 22  # 256 rows of it are 2 GiB of bfloat16
BIG = 1 << 40


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(_lib.PATH):
        pytest.fail(f"{_lib.PATH} is not built: run python -m bux_amd.build")
    return _lib.load()


def _refused(lib, rc):
    return rc == 1 and "exceed 2 GiB" in lib.bux_last_error().decode()


@pytest.mark.parametrize("dtype", [_lib.BF16, _lib.F32], ids=["bf16", "f32"])
@pytest.mark.parametrize("n,height", [(N, 256), (N, 4096), (33_554_176, 33), (33_554_176, 1 << 20),
                                      (8_388_608, 128)])
def test_rows_of_too_wide_outputs_are_refused(lib, n, height, dtype):
    m = max(height, 100)  # more than 16 rows a group
    assert _refused(lib, lib.bux_mx_grouped_rows(P, P, P, P, P, 2, m, n, 128, height, dtype, P, P, BIG, None))
    assert _refused(lib, lib.bux_mx_grouped_rows_started(P, P, P, P, P, P, 2, m, n, 128, height, dtype, P, P,
                                                         BIG, None))
    assert _refused(lib, lib.bux_mx_grouped_rows_noalloc(P, P, P, P, P, 2, m, n, 128, height, dtype, P, None))
    assert _refused(lib, lib.bux_mx_grouped_rows_listed(P, P, P, P, P, BIG, 2, m, n, 128, height, dtype, P,
                                                        None))
    assert _refused(lib, lib.bux_mx_grouped_rows_biased(P, P, P, P, P, BIG, 2, m, n, 128, height, dtype, P, P,
                                                        None))
    assert _refused(lib, lib.bux_int8_grouped_rows_listed(P, P, P, P, P, BIG, 2, m, n, 128, height, dtype,
                                                          None, P, None))


@pytest.mark.parametrize("dtype", [_lib.BF16, _lib.F32], ids=["bf16", "f32"])
def test_weight_gradients_of_too_wide_outputs_are_refused(lib, dtype):
    for d, f in ((256, N), (1000, N), (33, 33_554_176)):
        assert _refused(lib, lib.bux_mx_grouped_contract(P, P, P, P, P, 2, d, f, 128, dtype, P, P, BIG, None))
        assert _refused(lib, lib.bux_mx_grouped_contract_listed(P, P, P, P, P, BIG, 2, d, f, 128, dtype, P,
                                                                None))


def test_a_fused_product_of_too_wide_outputs_is_refused(lib):
    ffn = ctypes.byref(_lib.FfnStruct(0, 1, 0, 0.0, 0, 0.0, 0.0))
    assert _refused(lib, lib.bux_mx_grouped_glu(P, P, P, P, P, 2, 256, N, 128, 256, P, ffn, P, P, P, P, P, P,
                                                BIG, None))


def test_the_line_itself(lib):
    """The next shape below it passes the check (and fails the one after: no kernel is launched)."""
    for n, height in ((N - 4, 1 << 20), (33_554_172, 32)):
        rc = lib.bux_mx_grouped_rows(P, P, P, P, P, 2, 128, n, 128, height, 7, P, P, BIG, None)
        assert rc == 1 and "out_dtype" in lib.bux_last_error().decode()

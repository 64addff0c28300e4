"""CPU: extents so near 2^31 that the kernels' 32-bit counts of tiles and blocks would pass it are refused, the largest others are
not (a null tensor is what those calls are refused for). No device pointer is touched."""
import ctypes

import pytest

from muxi_race_b200 import _lib

F16, BF16, I32 = _lib.MOE_F16, _lib.MOE_BF16, _lib.MOE_I32
P = ctypes.c_void_p(256)
MOST = 2 ** 31 - 512  # a tile of up to 512 lanes or 256 rows, less 1, is added to an extent


def status(fn, *args):
    lib = _lib.lib()
    return getattr(lib, fn)(*args), lib.moe_last_error()


def rows_product(fn, R, N, K, x=P):
    return status(fn, x, max(N, K), P, P, I32, P, max(N, K), R, 2, N, K, F16, 1, None)


def weights_gradient(R, N, K, x=P):
    return status("moe_grouped_linear_dw", P, N, x, K, P, I32, P, F16, R, 2, N, K, F16, None)


def int8(M, N, K, x=P):
    return status("moe_int8_linear", x, K, P, P, P, None, P, N, BF16, M, N, K, None, 0, None)


CALLS = {"y": lambda *a: rows_product("moe_grouped_linear", *a), "dx": lambda *a: rows_product("moe_grouped_linear_dx", *a),
         "dw": weights_gradient}


@pytest.mark.parametrize("name", CALLS)
def test_grouped(name):
    call = CALLS[name]
    for sizes, msg in (((MOST + 1, 8, 8), b"row count"), ((2 ** 31 - 255, 8, 8), b"row count"), ((2 ** 31 - 1, 8, 8), b"row count"),
                       ((1, MOST + 8, 8), b"out_features"), ((1, 8, MOST + 8), b"in_features"), ((1, 2 ** 31 - 8, 8), b"out_features")):
        code, error = call(*sizes)
        assert code == -1 and msg in error, (sizes, code, error)
    # (a reduction has a bound of its own)
    for sizes in ((MOST, 8, 8), (1, MOST if call is not CALLS["dx"] else 8, 8), (1, 8, MOST if call is not CALLS["y"] else 8)):
        code, error = call(*sizes, None)
        assert code == -1 and b"null" in error, (sizes, code, error)


def test_long_reductions():
    """The kernels' waits give up after 2 s, and a tile's sums are waited for as one: 2^27 terms take 0.7 s."""
    most = 1 << 27
    for call, sizes, more in ((CALLS["y"], (1, 8, most), (1, 8, most + 8)), (CALLS["dx"], (1, most, 8), (1, most + 8, 8))):
        code, error = call(*more)
        assert code == -2 and b"2^27" in error, (more, code, error)
        code, error = call(*sizes, None)
        assert code == -1 and b"null" in error, (sizes, code, error)
    code, error = weights_gradient(most + 1, 8, 8)  # with a workspace, or in 32 bits, the rows are cut into parts
    assert code == -2 and b"moe_grouped_linear_dw_long" in error, (code, error)
    code, error = weights_gradient(most, 8, 8, None)
    assert code == -1 and b"null" in error


def test_int8():
    for sizes, msg in (((MOST + 1, 1, 16), b"row count"), ((2 ** 31 - 255, 1, 16), b"row count"), ((1, MOST + 1, 16), b"row count"),
                       ((1, 2 ** 31 - 1, 16), b"row count")):
        code, error = int8(*sizes)
        assert code == -1 and msg in error, (sizes, code, error)
    for sizes in ((MOST, 1, 16), (1, MOST, 16)):
        code, error = int8(*sizes, None)
        assert code == -1 and b"null" in error, (sizes, code, error)

"""CPU: the workspace of a 16-bit weights' gradient over many rows, and its checks (no device pointer is touched)."""
import ctypes

from muxi_race_b200 import _lib

F16, BF16, F32, I32 = _lib.MOE_F16, _lib.MOE_BF16, _lib.MOE_F32, _lib.MOE_I32
P = ctypes.c_void_p(256)


def call(R, dw_dtype=F16, x=P, dy=P, workspace=None, nbytes=0):
    lib = _lib.lib()
    code = lib.moe_grouped_linear_dw_long(dy, 32, x, 64, P, I32, P, dw_dtype, R, 2, 32, 64, F16, workspace, nbytes, None)
    return code, lib.moe_last_error()


def test_workspace():
    size = _lib.lib().moe_grouped_linear_dw_workspace_bytes
    # 74 pairs of CTAs, each with the fp32 sums of two halves of 128 lanes x 256 columns
    assert size(32769, F16) == size(1 << 30, BF16) == 148 * 2 * 128 * 256 * 4
    assert size(32768, F16) == size(0, BF16) == size(1 << 30, F32) == 0


def test_checks():
    need = _lib.lib().moe_grouped_linear_dw_workspace_bytes(40000, F16)
    for kw, code, msg in ((dict(), -5, str(need).encode()), (dict(workspace=P, nbytes=need - 1), -5, str(need).encode()),
                          (dict(workspace=ctypes.c_void_p(264), nbytes=need), -3, b"16-byte"),
                          (dict(workspace=P, nbytes=need, dw_dtype=BF16), -1, b"dw_dtype"),
                          (dict(workspace=P, nbytes=need, x=None), -1, b"null"), (dict(workspace=P, nbytes=need, dy=None), -1, b"null")):
        got, error = call(40000, **kw)
        assert got == code and msg in error, (kw, got, error)
    got, error = call(100, x=None)  # no workspace for few rows
    assert got == -1 and b"null" in error
    got, error = call(40000, dw_dtype=F32, x=None)  # nor for 32 bits
    assert got == -1 and b"null" in error

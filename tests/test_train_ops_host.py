"""CPU: argument checks of the grouped products, the activation, 8-bit rows and the dense int8 product (no device pointer
is touched), their sizes, and shape propagation of their torch operators."""
import ctypes

import pytest
import torch

import muxi_race_b200 as m
from muxi_race_b200 import _lib

F16, BF16, F32, I32, I64, I8, F8 = (_lib.MOE_F16, _lib.MOE_BF16, _lib.MOE_F32, _lib.MOE_I32, _lib.MOE_I64, _lib.MOE_I8,
                                    _lib.MOE_F8E4M3)
P = ctypes.c_void_p(256)


def refused(fn, *args, code=-1, msg=b""):
    lib = _lib.lib()
    assert getattr(lib, fn)(*args) == code, lib.moe_last_error()
    assert msg in lib.moe_last_error(), lib.moe_last_error()


def grouped(fn, x=P, ld=64, w=P, off=P, odt=I32, out=P, ld_out=32, R=4, E=2, N=32, K=64, dt=F16):
    return (x, ld, w, off, odt, out, ld_out, R, E, N, K, dt, 1, None)


def test_grouped_checks():
    for fn in ("moe_grouped_linear", "moe_grouped_linear_dx"):
        assert getattr(_lib.lib(), fn)(*grouped(fn, R=0)) == 0
        for kw, msg in ((dict(dt=F32), b"dtype"), (dict(odt=F32), b"offsets"), (dict(off=None), b"null"), (dict(E=0), b"num_experts"),
                        (dict(E=1025), b"1024"), (dict(N=12), b"multiples of 8"), (dict(K=0), b"multiples of 8"), (dict(R=-1), b"row count"),
                        (dict(x=None), b"null"), (dict(ld=8), b"pitches"), (dict(ld_out=8), b"pitches")):
            refused(fn, *grouped(fn, **kw), msg=msg)
    dw = (P, 32, P, 64, P, I32, P, F16, 4, 2, 32, 64, F16, None)
    refused("moe_grouped_linear_dw", *dw[:7], BF16, *dw[8:], msg=b"dw_dtype")
    refused("moe_grouped_linear_dw", *dw[:6], None, *dw[7:], msg=b"null")
    refused("moe_grouped_linear_dw", None, *dw[1:], msg=b"null")
    refused("moe_grouped_linear_dw", P, 16, *dw[2:], msg=b"pitches")


def test_rows8_checks():
    lib = _lib.lib()
    save = (P, 64, P, I8, P, 4, 64, 1, F16, None)
    assert lib.moe_save_rows8(*save[:5], 0, *save[6:]) == 0
    refused("moe_save_rows8", *save[:3], F16, *save[4:], msg=b"q_dtype")
    refused("moe_save_rows8", *save[:7], 3, *save[8:], msg=b"parts")
    refused("moe_save_rows8", *save[:8], F32, None, msg=b"dtype")
    refused("moe_save_rows8", P, 32, *save[2:], msg=b"pitch")
    refused("moe_save_rows8", *save[:4], None, *save[5:], msg=b"null")
    restore = (P, 64, I8, P, None, I32, 1, None, P, 4, 4, 64, 1, F16, None)
    refused("moe_restore_rows", P, 64, F32, *restore[3:], msg=b"src_dtype")
    refused("moe_restore_rows", *restore[:4], P, F32, *restore[6:], msg=b"index")
    refused("moe_restore_rows", *restore[:6], 0, *restore[7:], msg=b"index_div")
    refused("moe_restore_rows", *restore[:9], 5, *restore[10:], msg=b"more rows")
    refused("moe_restore_rows", *restore[:3], None, *restore[4:], msg=b"null")
    silu = (P, 64, None, 0, None, 0, None, P, None, 0, None, 4, 32, F16, None)
    refused("moe_silu_mul", P, 63, *silu[2:], msg=b"pitch")
    refused("moe_silu_mul", *silu[:2], P, I8, *silu[4:], msg=b"weights")
    refused("moe_silu_mul", *silu[:8], P, F16, P, *silu[11:], msg=b"q_dtype")
    refused("moe_silu_mul", *silu[:8], P, I8, None, *silu[11:], msg=b"null")
    refused("moe_silu_mul", *silu[:12], 0, F16, None, msg=b"row length")
    back = (P, 32, P, 64, F16, None, None, 0, None, 0, None, P, P, None, 4, 32, F16, None)
    refused("moe_silu_mul_backward", *back[:4], F32, *back[5:], msg=b"src_dtype")
    refused("moe_silu_mul_backward", *back[:4], I8, *back[5:], msg=b"null")
    refused("moe_silu_mul_backward", *back[:13], P, *back[14:], msg=b"needs weights")
    refused("moe_combine_rows", None, None, P, 4, 2, 8, 64, F16, None, msg=b"null")
    assert lib.moe_combine_rows(None, None, None, 0, 2, 8, 64, F16, None) == 0


def test_int8_checks_and_sizes():
    lib = _lib.lib()

    def args(x=P, ld=64, xs=P, w=P, ws=P, out=P, ld_out=32, dt=BF16, M=4, N=32, K=64, work=None, nbytes=0):
        return (x, ld, xs, w, ws, None, out, ld_out, dt, M, N, K, work, nbytes, None)

    assert lib.moe_int8_linear(*args(M=0)) == 0
    for kw, msg in ((dict(dt=I8), b"out_dtype"), (dict(K=24), b"multiple of 16"), (dict(K=131072), b"131072"), (dict(N=0), b"row count"),
                    (dict(ld=32), b"pitches"), (dict(ld_out=16), b"pitches"), (dict(xs=None), b"null"), (dict(w=None), b"null")):
        refused("moe_int8_linear", *args(**kw), msg=msg)
    refused("moe_int8_linear", *args(x=ctypes.c_void_p(8)), code=-3, msg=b"16 bytes")
    refused("moe_int8_linear", *args(ld=72), code=-3, msg=b"16 bytes")
    # few rows stream, many fill the SMs: neither cuts K; 64 rows of N = 4096, K = 14336 take 4 slices
    assert lib.moe_int8_linear_workspace_bytes(16, 4096, 14336) == 0
    assert lib.moe_int8_linear_workspace_bytes(4096, 4096, 14336) == 0
    assert lib.moe_int8_linear_workspace_bytes(64, 4096, 14336) == 4 * 64 * 4096 * 4
    refused("moe_int8_linear", *args(M=64, N=4096, K=14336, ld=14336, ld_out=4096), code=-5, msg=b"4194304")


def test_cpu_tensors_are_refused():
    h = torch.zeros(4, 64, dtype=torch.bfloat16)
    w = torch.zeros(2, 32, 64, dtype=torch.bfloat16)
    off = torch.zeros(3, dtype=torch.int32)
    for call in (lambda: m.grouped_linear(h, w, off), lambda: m.grouped_linear_backward(h[:, :32], h, w, off), lambda: m.silu_mul(h),
                 lambda: m.silu_mul_rows8(h), lambda: m.silu_mul_backward(h[:, :32], h), lambda: m.save_rows8(h),
                 lambda: m.restore_rows8(m.Rows8(torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4, 1), torch.bfloat16)),
                 lambda: m.int8_linear(h.to(torch.int8), torch.ones(4), w[0].to(torch.int8), torch.ones(32)),
                 lambda: m.moe_mlp(h, torch.zeros(2, 16, 64, dtype=torch.bfloat16), torch.zeros(2, 64, 8, dtype=torch.bfloat16),
                                   torch.zeros(4, 1, dtype=torch.int32), torch.ones(4, 1))):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_rows8_must_match():
    q = torch.zeros(4, 200, dtype=torch.int8)
    r = m.Rows8(q, torch.zeros(4, 2), torch.float16)
    assert r.shape == (4, 200) and r.nbytes() == 800 + 32
    m.Rows8(q, torch.zeros(4, 2), torch.float16, parts=2)
    for bad in ((q, torch.zeros(4, 3), torch.float16), (q, torch.zeros(4, 2).half(), torch.float16), (q.float(), torch.zeros(4, 2), torch.float16),
                (q, torch.zeros(4, 2), torch.float32), (q.t(), torch.zeros(200, 1), torch.float16), (q, torch.zeros(4, 3), torch.float16, 3)):
        with pytest.raises(ValueError):
            m.Rows8(*bad)


def test_shapes_of_the_torch_operators():
    import muxi_race_b200.torch_ops  # noqa: F401

    ops = torch.ops.muxi_race_b200
    meta = dict(device="meta")
    x, w = torch.empty(5, 64, dtype=torch.float16, **meta), torch.empty(3, 32, 64, dtype=torch.float16, **meta)
    off = torch.empty(4, dtype=torch.int32, **meta)
    assert ops.grouped_linear(x, w, off).shape == (5, 32)
    dx, dw = ops.grouped_linear_backward(torch.empty(5, 32, dtype=torch.float16, **meta), x, w, off)
    assert dx.shape == (5, 64) and dw.shape == (3, 32, 64)
    h = ops.silu_mul(x, None)
    assert h.shape == (5, 32) and h.dtype == torch.float16
    y = ops.int8_linear(torch.empty(5, 64, dtype=torch.int8, **meta), torch.empty(5, **meta), torch.empty(32, 64, dtype=torch.int8, **meta),
                        torch.empty(32, **meta), None, torch.bfloat16)
    assert y.shape == (5, 32) and y.dtype == torch.bfloat16

"""CPU: argument checks of the norm, routing and 4-bit entry points (no device pointer is touched), the
packed sizes, and shape propagation of their torch operators."""
import ctypes

import pytest
import torch

import muxi_race_b200 as m
from muxi_race_b200 import _lib

F16, BF16, F32 = _lib.MOE_F16, _lib.MOE_BF16, _lib.MOE_F32


def refused(fn, *args, code=-1, msg=b""):
    lib = _lib.lib()
    assert getattr(lib, fn)(*args) == code, lib.moe_last_error()
    assert msg in lib.moe_last_error(), lib.moe_last_error()


def norm_args(T=4, H=64, dtype=F16, wdtype=F16, out=F16, eps=1e-6, x=None, ld=64):
    return (x, ld, None, 0, x, wdtype, x, ld, out, None, None, 0, T, H, eps, dtype, None)


def test_norm_checks():
    p = ctypes.c_void_p(256)
    assert _lib.lib().moe_add_rms_norm(*norm_args(T=0)) == 0
    refused("moe_add_rms_norm", *norm_args(), msg=b"null")
    refused("moe_add_rms_norm", *norm_args(H=0), msg=b"hidden")
    refused("moe_add_rms_norm", *norm_args(H=16385), msg=b"hidden")
    refused("moe_add_rms_norm", *norm_args(dtype=_lib.MOE_I8), msg=b"dtype")
    refused("moe_add_rms_norm", *norm_args(wdtype=BF16), msg=b"weight_dtype")
    refused("moe_add_rms_norm", *norm_args(out=BF16), msg=b"out_dtype")
    refused("moe_add_rms_norm", *norm_args(dtype=F32, wdtype=F32, out=_lib.MOE_I8), code=-2, msg=b"8-bit rows")
    refused("moe_add_rms_norm", *norm_args(out=_lib.MOE_I8, x=p), msg=b"null")  # no scales
    refused("moe_add_rms_norm", *norm_args(x=p, ld=32), msg=b"pitches")
    refused("moe_add_rms_norm", *norm_args(eps=float("nan")), msg=b"eps")
    refused("moe_add_rms_norm", *norm_args(T=-1), msg=b"token count")
    lib = _lib.lib()
    assert lib.moe_add_rms_norm_backward_workspace_bytes(0, 64) == 0
    assert lib.moe_add_rms_norm_backward_workspace_bytes(7, 64) == 7 * 64 * 4
    back = (p, 64, p, 64, None, 0, p, F16, p, 64, p, 4, 64, 1e-6, F16)
    refused("moe_add_rms_norm_backward", *back[:10], None, *back[11:], None, 0, None, msg=b"null")
    refused("moe_add_rms_norm_backward", *back[:9], 63, *back[10:], None, 0, None, msg=b"pitches")


def test_route_checks():
    def args(dt=F32, T=4, E=64, k=4, scoring=0, ng=1, tg=1, top=2, ld=64):
        return (None, ld, dt, None, T, E, k, scoring, ng, tg, top, 1, 1.0, None, None, None, None)

    assert _lib.lib().moe_route_topk(*args(T=0)) == 0
    for kw, msg in ((dict(), b"null"), (dict(dt=_lib.MOE_I8), b"fp32"), (dict(E=0), b"num_experts"), (dict(E=1025), b"num_experts"),
                    (dict(k=0), b"topk"), (dict(k=33), b"topk"), (dict(E=3), b"topk"), (dict(scoring=2), b"scoring"),
                    (dict(ng=7), b"divide"), (dict(E=66, ng=33), b"num_groups"), (dict(ng=8, tg=9), b"topk_groups"),
                    (dict(ng=8, tg=0), b"topk_groups"), (dict(top=0), b"group_top"), (dict(ng=32, tg=1), b"within"),
                    (dict(T=-1), b"token count"), (dict(ld=-1), b"ld_logits")):
        refused("moe_route_topk", *args(**kw), msg=msg)
    refused("moe_route_topk_backward", None, None, 64, F32, None, 4, 64, 4, 0, 1, 1.0, None, None, msg=b"null")
    refused("moe_route_topk_backward", None, None, 64, F32, None, 4, 64, 65, 0, 1, 1.0, None, None, msg=b"topk")


def test_w4_sizes_and_checks():
    lib = _lib.lib()
    # 32 x 128 tiles: 2048 bytes of values, 64 of scales and 32 of zero points per group
    assert lib.moe_w4_packed_bytes(1, 32, 128, 128, 0, 0) == 2048 + 64
    assert lib.moe_w4_packed_bytes(3, 33, 129, 32, 1, 0) == 3 * 2 * 2 * (2048 + 4 * 96)
    assert lib.moe_w4_packed_bytes(1, 2 * 17, 128, 64, 0, 1) == 2 * (2048 + 2 * 64)  # 16 gate and 16 up rows a strip
    assert lib.moe_w4_packed_bytes(0, 32, 128, 128, 0, 0) == 0
    for bad in ((1, 32, 128, 48, 0, 0), (1, 0, 128, 64, 0, 0), (1, 33, 128, 64, 0, 1), (-1, 32, 128, 64, 0, 0)):
        assert lib.moe_w4_packed_bytes(*bad) == 0 and lib.moe_last_error()
    p = ctypes.c_void_p(256)
    refused("moe_w4_pack", p, p, None, 1, 32, 128, 128, 0, p, 100, None, code=-5, msg=b"2112")
    refused("moe_w4_pack", p, p, None, 1, 32, 128, 128, 0, ctypes.c_void_p(8), 4096, None, code=-3, msg=b"aligned")
    refused("moe_w4_quantize", p, F32, 4, 64, 32, p, p, None, None, msg=b"dtype")
    refused("moe_w4_linear", p, 64, p, p, 31, 4, 32, 64, 32, 0, F16, None, 0, None, msg=b"ld_out")
    refused("moe_w4_linear", None, 64, p, p, 32, 4, 32, 64, 32, 0, F16, None, 0, None, msg=b"null")
    assert lib.moe_w4_linear(p, 64, p, p, 32, 0, 32, 64, 32, 0, F16, None, 0, None) == 0
    # few rows of a short x fit in shared memory: no workspace; 16 rows of K = 14336 are cut
    assert lib.moe_w4_linear_workspace_bytes(8, 64, 4096, 128, F16) == 0
    assert lib.moe_w4_linear_workspace_bytes(16, 64, 14336, 128, F16) > 0
    moe = dict(T=4, H=128, I=64, E=8, k=2)

    def args(**kw):
        a = {**moe, "idt": _lib.MOE_I32, "wdt": F32, "dt": F16, "g": 64, **kw}
        return (p, a["H"], p, a["g"], 0, p, 64, 0, p, a["idt"], p, a["wdt"], p, a["T"], a["H"], a["I"], a["E"], a["k"], a["dt"],
                None, 0, None)

    refused("moe_fused_w4", *args(E=1025), msg=b"num_experts")
    refused("moe_fused_w4", *args(k=0), msg=b"topk")
    refused("moe_fused_w4", *args(g=96), msg=b"group")
    refused("moe_fused_w4", *args(idt=F32), msg=b"topk_ids")
    refused("moe_fused_w4", *args(wdt=_lib.MOE_I8), msg=b"topk_weights")
    refused("moe_fused_w4", *args(dt=F32), msg=b"dtype")
    assert lib.moe_fused_w4(*args(T=0)) == 0
    assert lib.moe_fused_w4_workspace_bytes(4, 2, 8, 128, 64, 64, 64, F16) >= 8 * 64 * 2 + 8 * 128 * 4


def test_q8_rows_checks():
    refused("moe_fused_q8_rows", None, None, F16, None, None, None, None, None, _lib.MOE_I32, None, F32, None, 4, 128, 64, 8, 2,
            F16, None, 0, None, msg=b"kind")
    refused("moe_fused_q8_rows", None, None, _lib.MOE_I8, None, None, None, None, None, _lib.MOE_I32, None, F32, None, 4, 128, 64,
            8, 2, F16, None, 0, None, msg=b"scales")


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 64)
    with pytest.raises(ValueError, match="CUDA"):
        m.add_rms_norm(x, torch.ones(64))
    with pytest.raises(ValueError, match="CUDA"):
        m.route_topk(x, 4)
    with pytest.raises(ValueError, match="CUDA"):
        m.pack_w4(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.float16), group_size=64)


def test_packed_weights_must_match_their_description():
    with pytest.raises(ValueError, match="2112 bytes"):
        m.W4Weights(torch.zeros(100, dtype=torch.uint8), (32, 128), torch.float16, 128, False, False)


def test_shapes_of_the_torch_operators():
    import muxi_race_b200.torch_ops  # noqa: F401

    ops = torch.ops.muxi_race_b200
    meta = dict(device="meta")
    x = torch.empty(5, 64, dtype=torch.float16, **meta)
    y, h = ops.add_rms_norm(x, torch.empty(64, **meta), x, 1e-6)
    assert y.shape == h.shape == (5, 64)
    dx, dw = ops.add_rms_norm_backward(x, x, torch.empty(64, **meta), None, 1e-6)
    assert dx.shape == (5, 64) and dw.shape == (64,)
    w, ids, counts = ops.route_topk(torch.empty(5, 16, **meta), 4, "softmax", None, 1, 1, 2, True, 1.0)
    assert w.shape == ids.shape == (5, 4) and counts.shape == (16,) and ids.dtype == torch.int32
    packed = torch.empty(2112, dtype=torch.uint8, **meta)
    assert ops.w4_linear(x, packed, 32, 128, False).shape == (5, 32)
    out = ops.fused_moe_w4(x, packed, packed, 8, 32, 128, False, 128, False, ids, w)
    assert out.shape == (5, 64)

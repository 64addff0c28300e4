"""GPU: the expert MLP on rows that are 8-bit already (hidden_scale) against the same call that
quantises the rows itself.

The rows that quantize_rows_int8 / _fp8 make of x are bit for bit the ones that fused_moe_int8 / _fp8
make of it inside (one scheme), so both calls compute the same products; the combine adds a token's k
routes in any order, each addition rounding to the output type: |difference| <= 2 k u sum|terms|,
bounded here by 2 k u max|out| + 2 k u (u = 2^-11 fp16, 2^-8 bf16).
"""
import pytest
import torch

from muxi_race_b200 import (add_rms_norm_quant, device_status, fused_moe_fp8, fused_moe_int8, quantize_rows_fp8,
                            quantize_rows_int8)

pytestmark = pytest.mark.gpu
KINDS = {"int8": (quantize_rows_int8, fused_moe_int8, torch.int8), "fp8": (quantize_rows_fp8, fused_moe_fp8, torch.float8_e4m3fn)}
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def inputs(T, H, I, E, k, dtype, kind):
    g = torch.Generator(device="cpu").manual_seed(T + H)
    quantize = KINDS[kind][0]
    x = torch.randn(T, H, generator=g).to(dtype).cuda()
    w13 = quantize((torch.randn(E, 2 * I, H, generator=g) * H ** -0.5).to(dtype).cuda())
    w2 = quantize((torch.randn(E, H, I, generator=g) * I ** -0.5).to(dtype).cuda())
    w, ids = torch.softmax(torch.randn(T, E, generator=g), -1).topk(k, -1)
    return x, (*w13, *w2), ids.int().cuda(), w.cuda()


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,H,I,E,k", [(1, 256, 128, 8, 2), (100, 512, 256, 16, 4), (300, 1024, 512, 8, 2)])
def test_same_as_quantising_inside(cuda_device, kind, dtype, T, H, I, E, k):
    quantize, fused, _ = KINDS[kind]
    x, w, ids, tw = inputs(T, H, I, E, k, dtype, kind)
    q, scale = quantize(x)
    got = fused(q, *w, ids, tw, hidden_scale=scale, out_dtype=dtype)
    want = fused(x, *w, ids, tw)
    assert device_status() == 0 and got.dtype == dtype
    tol = 2 * k * U[dtype] * (want.float().abs().amax() + 1)
    assert float((got.float() - want.float()).abs().amax()) <= float(tol)


@pytest.mark.parametrize("kind", ["int8", "fp8"])
def test_after_the_norm(cuda_device, kind):
    """Norm with 8-bit rows into the experts: near the experts on the unrounded norm. An 8-bit row is
    within 2^-8 (int8, of its largest value) or 2^-4 (e4m3, of each value) of y, so the output moves by at
    most a few percent of its size: 10 % bounds both."""
    _, fused, q_dtype = KINDS[kind]
    x, w, ids, tw = inputs(64, 512, 256, 8, 2, torch.bfloat16, kind)
    weight = torch.ones(512, device="cuda")
    res = x.flip(0)
    q, scale, h = add_rms_norm_quant(x, weight, res, q_dtype=q_dtype)
    got = fused(q, *w, ids, tw, hidden_scale=scale)
    y = (x.float() + res.float())
    y = (y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6)).bfloat16()
    want = fused(y, *w, ids, tw)
    assert device_status() == 0
    assert float((got.float() - want.float()).norm() / want.float().norm()) < 0.1


def test_refusals(cuda_device):
    x, w, ids, tw = inputs(4, 256, 128, 8, 2, torch.float16, "int8")
    q, scale = quantize_rows_int8(x)
    with pytest.raises(ValueError, match="int8"):
        fused_moe_int8(x, *w, ids, tw, hidden_scale=scale)
    with pytest.raises(ValueError, match="hidden_scale"):
        fused_moe_int8(q, *w, ids, tw, hidden_scale=scale[:2])
    with pytest.raises(ValueError, match="out_dtype"):
        fused_moe_int8(q, *w, ids, tw, hidden_scale=scale, out_dtype=torch.float32)
    with pytest.raises(ValueError, match="float8"):
        fused_moe_fp8(q, *w, ids, tw, hidden_scale=scale)

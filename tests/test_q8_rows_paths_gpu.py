"""GPU: rows that are 8-bit already (hidden_scale) on every way that Stage1 loads its rows, against the call that
quantises the rows itself.

Both compute the same products. With one route a token nothing is added up: the same bits. With k routes each
call adds a token's terms in any order, k additions that round to the output type, each by at most u of
the sum of the terms' magnitudes: |difference| <= 2 k u sum|terms| (u = 2^-11 fp16, 2^-8 bf16). The terms
come from calls with one route each; fp16 adds half its least spacing, 2^-25, for each addition."""
import pytest
import torch

from muxi_race_b200 import (_lib, device_status, fused_moe_fp8, fused_moe_int8, quantize_rows_fp8, quantize_rows_int8)

pytestmark = pytest.mark.gpu
KINDS = {"int8": (quantize_rows_int8, fused_moe_int8), "fp8": (quantize_rows_fp8, fused_moe_fp8)}
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(params=[("tma", "int8"), ("tma", "fp8"), ("gather", "int8"), ("gather", "fp8"), ("lsu", "int8")],
                ids=lambda p: "-".join(p))
def path(request):
    name, kind = request.param  # fp8 has no lsu path
    _lib.set_a_path(name)
    yield KINDS[kind]
    _lib.set_a_path(None)


def inputs(T, H, I, E, k, dtype, quantize):
    g = torch.Generator(device="cpu").manual_seed(T + H + k)
    x = torch.randn(T, H, generator=g).to(dtype).cuda()
    w13 = quantize((torch.randn(E, 2 * I, H, generator=g) * H ** -0.5).to(dtype).cuda())
    w2 = quantize((torch.randn(E, H, I, generator=g) * I ** -0.5).to(dtype).cuda())
    w, ids = torch.softmax(torch.randn(T, E, generator=g), -1).topk(k, -1)
    return x, (*w13, *w2), ids.int().cuda(), w.cuda()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,H,I,E,k", [(1, 256, 128, 8, 1), (333, 512, 256, 4, 1), (100, 512, 256, 16, 4), (300, 1024, 512, 8, 2)])
def test_same_products(cuda_device, path, dtype, T, H, I, E, k):
    quantize, fused = path
    x, w, ids, tw = inputs(T, H, I, E, k, dtype, quantize)
    q, scale = quantize(x)
    got = fused(q, *w, ids, tw, hidden_scale=scale, out_dtype=dtype)
    want = fused(x, *w, ids, tw)
    assert device_status() == 0 and got.dtype == dtype
    if k == 1:
        assert torch.equal(got, want)
        return
    terms = sum(fused(q, *w, ids[:, j:j + 1].contiguous(), tw[:, j:j + 1].contiguous(), hidden_scale=scale,
                      out_dtype=dtype).double().abs() for j in range(k))
    tol = 2 * k * (U[dtype] * terms * (1 + U[dtype]) + (2.0 ** -25 if dtype == torch.float16 else 0))
    assert bool(((got.double() - want.double()).abs() <= tol).all())


def test_skipped_ids_and_an_empty_row(cuda_device, path):
    quantize, fused = path
    x, w, ids, tw = inputs(50, 256, 128, 8, 2, torch.bfloat16, quantize)
    ids[3], ids[7, 1] = -1, 8
    x[9] = 0
    q, scale = quantize(x)
    got, want = fused(q, *w, ids, tw, hidden_scale=scale), fused(x, *w, ids, tw)
    assert bool((got[3] == 0).all()) and bool((got[9] == 0).all()) and torch.equal(got[7], want[7])
    assert device_status() == 0

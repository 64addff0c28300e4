"""GPU: outputs and scales of the expert calls that no kernel may touch are refused on the host."""
import pytest
import torch

import muxi_race_b200 as m

pytestmark = pytest.mark.gpu
T, H, I, E, K = 8, 256, 128, 4, 2


def calls(dtype=torch.float16):
    g = torch.Generator(device="cpu").manual_seed(0)
    x = torch.randn(T, H, generator=g).to(dtype).cuda()
    w13 = (torch.randn(E, 2 * I, H, generator=g) * H ** -0.5).to(dtype).cuda()
    w2 = (torch.randn(E, H, I, generator=g) * I ** -0.5).to(dtype).cuda()
    tw, ids = torch.softmax(torch.randn(T, E, generator=g), -1).topk(K, -1)
    tw, ids = tw.cuda(), ids.int().cuda()
    q8 = {n: (q(w13), q(w2), q(x)) for n, q in (("int8", m.quantize_rows_int8), ("fp8", m.quantize_rows_fp8))}
    packed = m.pack_weights(w13[:, :I].contiguous(), w13[:, I:].contiguous(), w2)
    fused = {"int8": m.fused_moe_int8, "fp8": m.fused_moe_fp8}
    by_name = {
        "fused_moe": lambda out, x=x: m.fused_moe(x, w13, w2, ids, tw, out=out),
        "ordered": lambda out, x=x: m.fused_moe(x, w13, w2, ids, tw, out=out, deterministic=True),
        "router": lambda out, x=x: m.fused_moe_router(x, w13, w2, torch.zeros(T, E, device="cuda"), K, out=out),
        "packed": lambda out, x=x: m.fused_moe_packed(x, packed, ids, tw, out=out)}
    for n, (a, b, xq) in q8.items():
        by_name[n] = lambda out, x=x, n=n, a=a, b=b: fused[n](x, *a, *b, ids, tw, out=out)
        by_name[n + " rows"] = lambda out, n=n, a=a, b=b, xq=xq: fused[n](xq[0], *a, *b, ids, tw, out=out, hidden_scale=xq[1],
                                                                         out_dtype=dtype)
    return x, by_name, q8, fused, ids, tw


def test_outputs(cuda_device):
    x, by_name, *_ = calls()
    for name, call in by_name.items():
        good = torch.empty_like(x)
        assert call(good) is good
        wide = torch.empty(T, 2 * H, dtype=x.dtype, device="cuda")
        for bad in (torch.empty(T, H, dtype=x.dtype), torch.empty(T - 1, H, dtype=x.dtype, device="cuda"),
                    torch.empty(T, H, dtype=torch.float32, device="cuda"), wide[:, :H]):
            with pytest.raises(ValueError):
                call(bad)
        if not name.endswith("rows"):
            big = torch.empty(T + 1, H, dtype=x.dtype, device="cuda")
            for shared in (x, big[1:]):
                with pytest.raises(ValueError, match="share memory"):
                    call(shared if shared is x else big[:-1], x=shared)


def test_scales(cuda_device):
    x, _, q8, fused, ids, tw = calls()
    for n, ((w13, s13), (w2, s2), (xq, sx)) in q8.items():
        for kw in (dict(), dict(hidden_scale=sx)):
            rows = xq if kw else x
            for a, b in ((s13.cpu(), s2), (s13, s2.cpu()), (s13[:1], s2), (s13, s2.half())):
                with pytest.raises(ValueError, match="scale must be fp32"):
                    fused[n](rows, w13, a, w2, b, ids, tw, **kw)
        with pytest.raises(ValueError, match="hidden_scale"):
            fused[n](xq, w13, s13, w2, s2, ids, tw, hidden_scale=sx.cpu())
    with pytest.raises(ValueError, match="logits' device"):
        m.grouped_topk(x, torch.zeros(T, 16, device="cuda"), 2, True, 4, 2, torch.zeros(16))

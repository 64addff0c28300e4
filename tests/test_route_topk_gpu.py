"""GPU: route_topk and its gradient against the definition in fp64.

Tolerances: expf is within 2 units in the last place, its argument l - m is rounded once (up to 20
units of 2^-24 for the logits here, 1.2e-6), the sum of at most 1024 terms is a tree of 37 additions
(2.2e-6): W = 5e-6 relative. Gradients: W on every term of a sum, whose magnitudes the test adds up,
then one rounding to the logits' type. Ids are exact wherever fp64 tells the candidates apart by
more than 1e-5 (two correct fp32 forms may differ below that); without bias and groups everywhere.
"""
import pytest
import torch

from muxi_race_b200 import fused_topk, grouped_topk, route_topk, route_topk_backward
from oracle.router_ref import route_scores64, route_topk_ref, route_weights64

pytestmark = pytest.mark.gpu
W = 5e-6
U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
NINF = float("-inf")


def logits_of(seed, T, E, dtype=torch.float32, masked=0.0, scale=1.5):
    g = torch.Generator(device="cpu").manual_seed(seed)
    l = torch.randn((T, E), generator=g) * scale
    if masked:
        l[torch.rand((T, E), generator=g) < masked] = NINF
        l[T // 2] = NINF
    return l.to(dtype).cuda()


def check(l, k, **how):
    bias = how.get("bias")
    w, ids, counts = route_topk(l, k, return_counts=True, **how)
    rw, rids, sure = route_topk_ref(l, k, how.get("scoring", "softmax"), bias, how.get("num_groups", 1),
                                    how.get("topk_groups", 1), how.get("group_top", 2), how.get("renormalize", True),
                                    how.get("scale", 1.0))
    assert w.dtype == torch.float32 and ids.dtype == torch.int32 and w.shape == ids.shape == (l.shape[0], k)
    assert float(sure.float().mean()) > 0.9, "the inputs leave too many rows undecided"
    assert torch.equal(ids[sure].long(), rids[sure])
    rw = route_weights64(l, ids, how.get("scoring", "softmax"), how.get("renormalize", True), how.get("scale", 1.0))
    assert bool(((w.double() - rw).abs() <= W * rw.abs() + 1e-37).all())
    there = ids[ids >= 0].long()
    assert torch.equal(counts.long(), torch.bincount(there, minlength=l.shape[1]))
    assert bool((w[ids < 0] == 0).all())
    for row in ids[:50].tolist():  # no expert twice
        row = [e for e in row if e >= 0]
        assert len(set(row)) == len(row)
    return w, ids


@pytest.mark.parametrize("T,E,k", [(1, 8, 2), (1, 256, 8), (7, 1, 1), (300, 60, 4), (1000, 256, 8), (129, 33, 3),
                                   (64, 130, 8), (50, 1024, 32), (40, 1000, 6), (70, 32, 32), (20, 62, 5)])
@pytest.mark.parametrize("scoring,renormalize", [("softmax", True), ("softmax", False), ("sigmoid", True),
                                                 ("sigmoid", False)])
@pytest.mark.parametrize("dtype,masked", [(torch.float32, 0.0), (torch.float32, 0.4), (torch.bfloat16, 0.0),
                                          (torch.float16, 0.95)])
def test_by_logits(cuda_device, T, E, k, scoring, renormalize, dtype, masked):
    check(logits_of(1, T, E, dtype, masked), k, scoring=scoring, renormalize=renormalize, scale=2.5)


@pytest.mark.parametrize("E,k", [(8, 2), (60, 8), (100, 9), (256, 8), (512, 10), (1024, 8)])
@pytest.mark.parametrize("T", [1, 8, 9, 16, 17, 63, 64, 65, 127, 128, 129, 257])
def test_counts_of_every_launch_form(cuda_device, T, E, k):
    """One block, one cluster of blocks, and many blocks add their counts up."""
    for seed in (2, 3):
        check(logits_of(seed, T, E, masked=0.1), k)


@pytest.mark.parametrize("T,E,k,groups,top_groups", [(200, 256, 8, 8, 4), (33, 256, 8, 8, 1), (100, 60, 6, 5, 3),
                                                     (100, 96, 2, 32, 7), (64, 12, 3, 3, 2), (50, 40, 4, 1, 1),
                                                     (30, 1024, 8, 16, 2), (30, 8, 4, 8, 5)])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias,group_top,masked", [(True, 2, 0.0), (False, 2, 0.0), (True, 1, 0.3), (False, 1, 0.3)])
def test_bias_and_groups(cuda_device, T, E, k, groups, top_groups, scoring, with_bias, group_top, masked):
    bias = None
    if with_bias:
        g = torch.Generator(device="cpu").manual_seed(3)
        bias = (torch.randint(-40, 41, (E,), generator=g) * 1e-3).cuda()
    check(logits_of(2, T, E, masked=masked), k, scoring=scoring, bias=bias, num_groups=groups, topk_groups=top_groups,
          group_top=group_top)


def test_agrees_with_the_fixed_forms(cuda_device):
    l = logits_of(4, 500, 256)
    w, ids = route_topk(l, 8)
    fw, fids = fused_topk(l, l, 8)
    assert torch.equal(ids, fids) and torch.allclose(w, fw, rtol=1e-5, atol=0)
    bias = (torch.randn(256) * 0.05).cuda()
    w, ids = route_topk(l, 8, scoring="sigmoid", bias=bias, num_groups=8, topk_groups=4, scale=2.5)
    fw, fids = grouped_topk(l, l, 8, True, 8, 4, bias, 2.5)
    _, _, sure = route_topk_ref(l, 8, "sigmoid", bias, 8, 4)
    assert torch.equal(ids[sure], fids[sure]) and torch.allclose(w[sure], fw[sure], rtol=1e-5, atol=0)


def test_ties_zeros_and_special_values(cuda_device):
    l = torch.zeros(6, 70).cuda()
    l[1, ::2] = -0.0
    l[2, 40] = float("inf")
    l[3, 5] = float("nan")
    l[4] = NINF
    l[4, 66] = -80.0
    l[5, :] = torch.arange(70).cuda() // 7
    w, ids = route_topk(l, 4)
    assert ids[0].tolist() == ids[1].tolist() == [0, 1, 2, 3]  # -0 is 0, equal logits by id
    assert ids[4].tolist() == [66, -1, -1, -1] and w[4].tolist() == [1, 0, 0, 0]
    assert ids[5].tolist() == [63, 64, 65, 66]
    assert int(ids[2, 0]) == 40 and bool(w[2].isnan().any())  # inf / inf, as torch.softmax
    assert int(ids[3, 0]) == 5 and bool(w[3].isnan().any())   # a spoilt row says so
    assert bool(w[[0, 1, 4, 5]].isfinite().all())
    w, ids = route_topk(l, 4, scoring="sigmoid")
    assert bool(w[3].isnan().any()) and w[4].tolist() == [1, 0, 0, 0]
    far = torch.full((1, 16), -200.0).cuda()  # every score rounds to 0
    w, _ = route_topk(far, 4, scoring="sigmoid")
    assert bool((w == 0).all())
    w, _ = route_topk(far, 4)
    assert bool((w == 0.25).all())


def test_pitches(cuda_device):
    big = logits_of(5, 50, 300)
    for off, E in ((0, 256), (3, 256), (8, 120), (1, 61)):
        check(big[:, off:off + E], 4, renormalize=False)
        check(big[:1, off:off + E].expand(50, E), 4)


def grad_ref(l, ids, dw, scoring, renormalize, scale):
    """fp64 gradient by autograd, and the sum of its terms' magnitudes."""
    x = l.double().requires_grad_()
    (route_weights64(x, ids, scoring, renormalize, scale) * dw.double()).sum().backward()
    s = route_scores64(l, scoring)
    g = torch.where(ids >= 0, dw.double().abs() * scale, 0.0)
    p = torch.where(ids >= 0, s.gather(1, ids.clamp_min(0).long()), 0.0)
    if renormalize:
        den = p.sum(-1, keepdim=True).clamp_min(1e-290)
        p = p / den
        spread = (g * p).sum(-1, keepdim=True)
        mag = torch.zeros_like(s).scatter_add_(1, ids.clamp_min(0).long(), p * (g + spread))
    else:
        mag = torch.zeros_like(s).scatter_add_(1, ids.clamp_min(0).long(), p * g)
        if scoring == "softmax":
            mag = mag + s * (g * p).sum(-1, keepdim=True)
    return x.grad, mag


@pytest.mark.parametrize("T,E,k", [(1, 8, 2), (300, 60, 4), (1000, 256, 8), (129, 33, 3), (50, 1024, 32)])
@pytest.mark.parametrize("scoring,renormalize", [("softmax", True), ("softmax", False), ("sigmoid", True),
                                                 ("sigmoid", False)])
@pytest.mark.parametrize("dtype,masked", [(torch.float32, 0.0), (torch.bfloat16, 0.5), (torch.float16, 0.0)])
def test_backward(cuda_device, T, E, k, scoring, renormalize, dtype, masked):
    l = logits_of(6, T, E, dtype, masked)
    _, ids = route_topk(l, k, scoring=scoring, renormalize=renormalize)
    dw = torch.randn(T, k, generator=torch.Generator(device="cpu").manual_seed(7)).cuda()
    got = route_topk_backward(dw, l, ids, scoring=scoring, renormalize=renormalize, scale=2.5)
    ref, mag = grad_ref(l, ids, dw, scoring, renormalize, 2.5)
    assert got.dtype == dtype and got.shape == l.shape
    tiny = 2.0 ** -25 if dtype == torch.float16 else 1e-37
    assert bool(((got.double() - ref).abs() <= U[dtype] * ref.abs() + 4 * W * mag + tiny).all())


def test_autograd_and_differences(cuda_device):
    """Through autograd, and against (L(l + e v) - L(l - e v)) / 2e along random directions: with e = 0.05
    the third-order term is at most e^2 / 6 of the second derivative's scale (4e-4 of sum |dw|), fp32
    rounding of the weights over e 20 * 6e-8 of it."""
    T, E, k = 40, 64, 6
    l = logits_of(8, T, E)
    dw = torch.randn(T, k, generator=torch.Generator(device="cpu").manual_seed(9)).cuda()
    for scoring in ("softmax", "sigmoid"):
        for renormalize in (True, False):
            x = l.clone().requires_grad_()
            w, ids, counts = route_topk(x, k, scoring=scoring, renormalize=renormalize, return_counts=True)
            assert not ids.requires_grad and int(counts.sum()) == T * k
            (w * dw).sum().backward()
            assert torch.equal(x.grad, route_topk_backward(dw, l, ids, scoring=scoring, renormalize=renormalize))
            v = torch.randn(T, E, generator=torch.Generator(device="cpu").manual_seed(10)).cuda()
            # the choice is held: its weights as functions of the logits, by the kernel's own weights
            e = 0.05
            order = ids.long()

            def weights(step):
                y = torch.full_like(l, NINF) if renormalize and scoring == "softmax" else l + step * v
                if renormalize and scoring == "softmax":
                    y.scatter_(1, order, (l + step * v).gather(1, order))
                    ww, ii = route_topk(y, k)
                else:
                    ww, ii = route_topk(y, E if E <= 32 else 32, scoring=scoring, renormalize=False)
                full = torch.zeros(T, E, device="cuda", dtype=torch.float64).scatter_(1, ii.long(), ww.double())
                ww = full.gather(1, order)
                if renormalize and scoring == "sigmoid":
                    ww = ww / ww.sum(-1, keepdim=True)
                return ww

            slope = ((weights(e) - weights(-e)) * dw.double()).sum(-1) / (2 * e)
            want = (x.grad.double() * v.double()).sum(-1)
            scale = (dw.double().abs().sum(-1) * v.abs().double().amax(-1) ** 3)
            assert bool(((slope - want).abs() <= 2e-3 * scale).all())


def test_empty_large_and_stream(cuda_device):
    w, ids, counts = route_topk(torch.empty(0, 16, device="cuda"), 4, return_counts=True)
    assert w.shape == (0, 4) and bool((counts == 0).all())
    assert route_topk_backward(w, torch.empty(0, 16, device="cuda"), ids).shape == (0, 16)
    l = logits_of(11, 40000, 64)
    _, _, counts = route_topk(l, 6, return_counts=True)
    assert int(counts.sum()) == 240000
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        w2, ids2 = route_topk(l, 6)
    side.synchronize()
    w1, ids1 = route_topk(l, 6)
    assert torch.equal(w1, w2) and torch.equal(ids1, ids2)


def test_refusals(cuda_device):
    l = logits_of(12, 4, 64)
    for kw, msg in ((dict(topk=33), "topk"), (dict(topk=4, num_groups=7), "divide"),
                    (dict(topk=4, num_groups=8, topk_groups=9), "topk_groups"),
                    (dict(topk=9, num_groups=8, topk_groups=1), "within"), (dict(topk=2, group_top=3), "group_top")):
        with pytest.raises(RuntimeError, match=msg):
            route_topk(l, **kw)
    with pytest.raises(RuntimeError, match="num_experts"):
        route_topk(torch.zeros(2, 1025, device="cuda"), 2)
    with pytest.raises(ValueError, match="scoring"):
        route_topk(l, 4, scoring="relu")
    with pytest.raises(ValueError, match="bias"):
        route_topk(l, 4, bias=torch.zeros(63, device="cuda"))
    with pytest.raises(ValueError, match="CUDA"):
        route_topk(l.cpu(), 4)
    with pytest.raises(ValueError, match="fp32, fp16 or bf16"):
        route_topk(l.double(), 4)
    _, ids = route_topk(l, 4)
    with pytest.raises(ValueError, match="dweights"):
        route_topk_backward(torch.zeros(4, 3, device="cuda"), l, ids)
    with pytest.raises(ValueError, match="topk_ids"):
        route_topk_backward(torch.zeros(4, 4, device="cuda"), l, ids.long())

"""CPU: the gradients of the norm and of the routing say that they cannot be differentiated again. The
kernels are replaced by CPU functions that, like them, return tensors without a graph."""
import pytest
import torch

from muxi_race_b200 import norm, route


def detached(fn):
    def call(*args, **kw):
        with torch.no_grad():
            return fn(*args, **kw)
    return call


@pytest.fixture
def cpu_kernels(monkeypatch):
    def norm_forward(x, weight, residual, eps, out, residual_out):
        h = x if residual is None else x + residual
        return h * torch.rsqrt(h.square().mean(-1, keepdim=True) + eps) * weight, None if residual is None else h

    def norm_backward(dy, h, weight, dh=None, eps=1e-6):
        with torch.enable_grad():
            h2, w2 = h.detach().requires_grad_(), weight.detach().requires_grad_()
            y = norm_forward(h2, w2, None, eps, None, None)[0]
            dx, dw = torch.autograd.grad(y, (h2, w2), dy.detach())
        return dx if dh is None else dx + dh.detach(), dw

    def route_forward(logits, topk, scoring, bias, num_groups, topk_groups, group_top, renormalize, scale, counts):
        w, ids = torch.softmax(logits, -1).topk(topk, -1)
        return w, ids.int(), None

    def route_backward(dweights, logits, ids, scoring="softmax", renormalize=True, scale=1.0):
        p = torch.softmax(logits.detach(), -1)
        d = torch.zeros_like(p).scatter_(1, ids.long(), dweights.detach())
        return p * (d - (p * d).sum(-1, keepdim=True))

    monkeypatch.setattr(norm, "_forward", detached(norm_forward))
    monkeypatch.setattr(norm, "add_rms_norm_backward", norm_backward)
    monkeypatch.setattr(route, "_forward", detached(route_forward))
    monkeypatch.setattr(route, "route_topk_backward", route_backward)


def second(loss, leaf):
    g, = torch.autograd.grad(loss, leaf, create_graph=True)
    return torch.autograd.grad(loss + g.square().sum(), leaf)


@pytest.mark.parametrize("power", [1, 2])  # 1: the gradient that reaches the operator is a constant
@pytest.mark.parametrize("with_residual", [False, True])
def test_norm(cpu_kernels, power, with_residual):
    x = torch.randn(3, 8, requires_grad=True)
    w = torch.randn(8, requires_grad=True)
    r = torch.randn(3, 8) if with_residual else None
    y = norm.add_rms_norm(x, w, r)
    y = y[0] if with_residual else y
    for leaf in (x, w):
        with pytest.raises(RuntimeError, match="add_rms_norm can be differentiated once"):
            second(y.pow(power).sum(), leaf)


@pytest.mark.parametrize("power", [1, 2])
def test_route(cpu_kernels, power):
    logits = torch.randn(5, 8, requires_grad=True)
    w, _ = route.route_topk(logits, 3)
    with pytest.raises(RuntimeError, match="route_topk can be differentiated once"):
        second((w * torch.arange(3)).pow(power).sum(), logits)


def test_first_derivatives_are_as_before(cpu_kernels):
    x, w = torch.randn(3, 8, requires_grad=True), torch.randn(8, requires_grad=True)
    res = torch.randn(3, 8, requires_grad=True)
    y, h = norm.add_rms_norm(x, w, res)
    plain = (x + res) * torch.rsqrt((x + res).square().mean(-1, keepdim=True) + 1e-6) * w
    for graph in (False, True):
        got = torch.autograd.grad(y.square().sum() + h.sum(), (x, w, res), create_graph=graph, retain_graph=True)
        want = torch.autograd.grad(plain.square().sum() + (x + res).sum(), (x, w, res), retain_graph=True)
        for a, b in zip(got, want):
            torch.testing.assert_close(a.detach(), b, rtol=1e-4, atol=1e-4)
    # the sum alone passes its gradient on as it is, to any order
    _, h = norm.add_rms_norm(x, w, res)
    g, = torch.autograd.grad(h.pow(3).sum(), x, create_graph=True)
    g2, = torch.autograd.grad(g.sum(), x)
    torch.testing.assert_close(g2, 6 * (x + res))

"""GPU: workspaces of calls from two threads on one stream, and of captured graphs.

The calls compared give the same bits on every run, so the results have to be equal."""
import gc
import threading

import pytest
import torch

from muxi_race_b200 import add_rms_norm_backward, device_status, fused_moe, fused_moe_w4, quantize_w4, w4_linear

pytestmark = pytest.mark.gpu


def randn(seed, *shape, dtype=torch.float16, scale=1.0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


def routing(seed, T, E, k):
    g = torch.Generator(device="cpu").manual_seed(seed)
    w, ids = torch.softmax(torch.randn(T, E, generator=g), -1).topk(k, -1)
    return ids.int().cuda(), w.cuda()


@pytest.fixture(scope="module")
def weights(cuda_device):
    E, H, I = 16, 1024, 512
    w13, w2 = randn(1, E, 2 * I, H, scale=H ** -0.5), randn(2, E, H, I, scale=I ** -0.5)
    return {"w13": w13, "w2": w2, "q13": quantize_w4(w13, gate_up=True), "q2": quantize_w4(w2),
            "lin": quantize_w4(randn(3, 256, 14336, scale=0.01))}


def calls(name, w):
    """Two calls of one operator on inputs of different sizes (T, and who gets which token)."""
    if name == "fused_moe_w4":
        return [lambda x=randn(s, T, 1024), r=routing(s, T, 16, 4): fused_moe_w4(x, w["q13"], w["q2"], *r)
                for s, T in ((10, 5), (11, 90))]
    if name == "fused_moe":
        return [lambda x=randn(s, T, 1024), r=routing(s, T, 16, 4): fused_moe(x, w["w13"], w["w2"], *r, deterministic=True)
                for s, T in ((10, 5), (11, 90))]
    if name == "w4_linear":  # K is cut into slices that meet in the workspace
        return [lambda x=randn(s, T, 14336): w4_linear(x, w["lin"]) for s, T in ((12, 16), (13, 30))]
    return [lambda dy=randn(s, T, 1000), h=randn(s + 1, T, 1000), g=randn(7, 1000): torch.cat(
        [t.flatten() for t in add_rms_norm_backward(dy, h, g)]) for s, T in ((14, 300), (16, 700))]


@pytest.mark.parametrize("name", ["fused_moe_w4", "fused_moe", "w4_linear", "add_rms_norm_backward"])
def test_two_threads_on_one_stream(weights, name):
    fns = calls(name, weights)
    refs = [f() for f in fns]
    torch.cuda.synchronize()
    wrong, start = [], threading.Barrier(2)

    def run(f, ref):
        start.wait()
        outs = [f() for _ in range(150)]  # no synchronisation between the calls
        torch.cuda.synchronize()
        wrong.append(sum(not torch.equal(o, ref) for o in outs))

    threads = [threading.Thread(target=run, args=a) for a in zip(fns, refs)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert wrong == [0, 0]
    assert device_status() == 0


@pytest.mark.parametrize("name", ["fused_moe_w4", "fused_moe", "w4_linear", "add_rms_norm_backward"])
def test_a_graph_after_larger_captures_and_the_first_graphs_end(weights, name):
    small, large = calls(name, weights)
    ref = small()
    large()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for f in (small, small, large):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(f())
        graphs.append(g)
    del g
    graphs[0].reset()
    del graphs[0], outs[0], outs[1]
    gc.collect()
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    filler = [torch.full((1 << 24,), 0xFF, dtype=torch.uint8, device="cuda") for _ in range(8)]  # takes freed memory
    for _ in range(3):
        outs[0].zero_()
        graphs[0].replay()
        large()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], ref)
    assert all(bool((t == 0xFF).all()) for t in filler)
    assert device_status() == 0

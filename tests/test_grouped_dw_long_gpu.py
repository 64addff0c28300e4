"""GPU: the 16-bit weights' gradient of experts with very many rows against sums in fp64.

The tensor core adds 16 products and the sum so far at a time and cuts the result towards zero, off by at most 2^-23 of it. The
rows are therefore taken in parts of at most 32768, 2048 such steps, whose sums are added in fp32 with rounding.
  Normal data: the sum so far is on average 2/3 of the part's, and the parts' errors add up like their values: 2/3 2048 2^-23 =
  1.63e-4 of dW's norm at most, and half a step u for the result. (In one piece 2^20 rows would be 16 to 32 times as far off.)
  Data of one sign: the sum so far is on average half of the part's: 1/2 2048 2^-23 = 1.23e-4 of each element, 2^-24 for each of the
  parts' sums, and u.
"""
import pytest
import torch

import muxi_race_b200 as m

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
U = {F16: 2.0 ** -11, BF16: 2.0 ** -8}


def randn(seed, *shape, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def dw_of(dy, x, ends, dw_dtype=None):
    w = torch.empty(len(ends) - 1, dy.shape[1], x.shape[1], dtype=x.dtype, device="cuda")
    offsets = torch.tensor(ends, dtype=torch.int32, device="cuda")
    return m.grouped_linear_backward(dy, x, w, offsets, dw_dtype=dw_dtype, need_dx=False)[1]


def exact(dy, x, a, b):
    total = torch.zeros(dy.shape[1], x.shape[1], dtype=torch.float64, device="cuda")
    for r in range(a, b, 1 << 17):
        at = slice(r, min(b, r + (1 << 17)))
        total += dy[at].double().T @ x[at].double()
    return total


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("sign", [False, True])
def test_one_expert(cuda_device, dtype, sign):
    R, N, K = (1 << 20) + 37, 72, 64
    x, dy = randn(1, R, K, dtype=dtype), randn(2, R, N, dtype=dtype) * (2.0 ** -6 if dtype == F16 else 1.0)
    if sign:
        x, dy = x.abs(), dy.abs() * 2.0 ** -4
    dw, ref = dw_of(dy, x, [0, R])[0].double(), exact(dy, x, 0, R)
    if sign:
        tol = U[dtype] + 0.5 * 2048 * 2.0 ** -23 + 33 * 2.0 ** -24
        assert bool(((dw - ref).abs() <= tol * ref.abs()).all()), float(((dw - ref) / ref).abs().max())
    else:
        assert float((dw - ref).norm() / ref.norm()) <= U[dtype] + 2 / 3 * 2048 * 2.0 ** -23


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_many_tiles_and_ragged_experts(cuda_device, dtype):
    """Tiles of 512 lanes in several rounds, a last round that is cut, lanes and columns that are no multiples of the tiles; experts of
    few rows beside the long ones, whose dW has the bits that it has in a short call."""
    ends, N, K = [0, 40003, 40003, 40100, 120000, 152768, 152800], 1032, 8200
    scale = 2.0 ** -6 if dtype == F16 else 1.0
    x, dy = randn(3, ends[-1], K, dtype=dtype), randn(4, ends[-1], N, dtype=dtype) * scale
    dw = dw_of(dy, x, ends)
    for e, (a, b) in enumerate(zip(ends, ends[1:])):
        if b - a > 32768:
            ref = exact(dy, x, a, b)
            assert float((dw[e].double() - ref).norm() / ref.norm()) <= U[dtype] + 2 / 3 * 2048 * 2.0 ** -23
            within = (dw[e].double() - ref).abs() <= U[dtype] * ref.abs() + 1e-2 * scale * (b - a) ** 0.5
            assert bool(within.all())  # no stray element: far above the sums' error, far below a value
        else:
            assert torch.equal(dw[e], dw_of(dy[a:b], x[a:b], [0, b - a])[0])
    assert torch.equal(dw, dw_of(dy, x, ends))
    assert m.device_status() == 0


def test_streams_and_graph(cuda_device):
    x, dy = randn(5, 70000, 512, dtype=BF16), randn(6, 70000, 264, dtype=BF16)
    ends = [0, 66000, 70000]
    want = dw_of(dy, x, ends)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:  # at once, each with its own workspace
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got += [dw_of(dy, x, ends) for _ in range(3)]
    torch.cuda.synchronize()
    assert all(torch.equal(want, t) for t in got)
    w, offsets = torch.empty(2, 264, 512, dtype=BF16, device="cuda"), torch.tensor(ends, dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m.grouped_linear_backward(dy, x, w, offsets, need_dx=False)[1]
    x.mul_(-1)
    for _ in range(2):
        graph.replay()
    assert torch.equal(out, -want)

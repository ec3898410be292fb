"""linear_cross_entropy with a gradient per row (reduction "none") in bf16: the products' common factors must not be rounded
into every row of s = softmax - onehot.

A gradient g that all rows share gives the bits that the same g gives through reduction "sum". Its errors against float64, as
a whole: an element of the result rounds by at most half a step of the binade that it lies in, evenly distributed, so
that the error's norm is at most v / sqrt(3) of the result's, v = 2^-8 (s's own rounding adds what the softmax beside the onehot
has of s's norm: under 2 % of the squares here); and in the direction of the result itself the N roundings, either way, cancel
but for v / sqrt(N), under 2^-16 here, and for the p that the target's -1 + p loses where it is below half a step, 2^-9: on
average 1 / V = 2^-12. A rounding shared by all rows would stand there with up to 2^-8."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

V8 = 2.0 ** -8


def _data(T, h, V, dev, ignored=0.0, seed=0):
    g = torch.Generator(device=dev).manual_seed(100 * seed + T + V)
    x = torch.randn(T, h, generator=g, device=dev).to(torch.bfloat16)
    w = (torch.randn(V, h, generator=g, device=dev) * 2 * h ** -0.5).to(torch.bfloat16)
    t = torch.randint(0, V, (T,), generator=g, device=dev)
    if ignored:
        t[torch.rand(T, generator=g, device=dev) < ignored] = -100
    return x, w, t


def _grads(x, w, t, g, reduction):
    from q38.hip import autograd
    x, w = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    return torch.autograd.grad(autograd.linear_cross_entropy(x, w, t, reduction=reduction), (x, w), g)


@pytest.mark.parametrize("T,h,V,ignored", [
    (1, 64, 300, 0.0),
    (65, 320, 129, 0.5),
    (1777, 256, 4099, 0.4),     # dx split over K, its parts joined
    (8192, 64, 70, 0.3),        # the last size whose list is made beside the copies
    (8193, 64, 70, 0.3),
    (8200, 64, 20001, 0.0),     # two pieces of the vocabulary
    (2100, 1024, 8200, 0.0),    # 256 x 256 tiles
])
def test_a_shared_gradient_gives_the_bits_of_the_sum(gpu, T, h, V, ignored):
    x, w, t = _data(T, h, V, gpu, ignored)
    for c in (1 / 1777, 0.5637, -0.37, 1.2e-12, 7.0e10, 0.0):  # (s times its power of two stays a normal number)
        print(f"shared gradient T={T} h={h} V={V} {c}", flush=True)
        one = torch.tensor(c, device=gpu)
        rows = torch.full((T,), c, device=gpu)
        rows[t == -100] = float("nan")  # those of ignored rows count for nothing
        for name, a, b in zip(("dx", "dw"), _grads(x, w, t, rows, "none"), _grads(x, w, t, one, "sum")):
            assert torch.equal(a, b), f"{name}: {int((a != b).sum())} of {a.numel()} differ"


@pytest.mark.parametrize("reduction", ["sum", "none"])
@pytest.mark.parametrize("c", [1 / 1777, 0.5637])
def test_the_errors_as_a_whole(gpu, reduction, c):
    T, h, V = 1777, 256, 4096
    x, w, t = _data(T, h, V, gpu)
    g = torch.full((T,) if reduction == "none" else (), c, device=gpu)
    print(f"errors {reduction} {c}", flush=True)
    dx, dw = _grads(x, w, t, g, reduction)
    xd, wd = x.double(), w.double()
    s = torch.softmax(xd @ wd.t().contiguous(), 1)
    s[torch.arange(T, device=gpu), t] -= 1.0
    s *= float(torch.tensor(c))
    for name, got, exact in (("dx", dx, s @ wd), ("dw", dw, s.t().contiguous() @ xd)):
        got = got.double()
        error = float((got - exact).norm() / exact.norm())
        along = float((got * exact).sum() / (exact * exact).sum()) - 1.0
        assert error <= V8 / math.sqrt(3) * 1.01, f"{name}: {error:.6f}"
        assert abs(along) <= 2.0 ** -11, f"{name}: {along:+.6f}"


def test_gradients_far_apart(gpu):
    """Rows whose gradients lie 2^200 apart: dx of each row is exact in itself (bounds of one rounding of s and one of the result)."""
    T, h, V = 300, 128, 700
    x, w, t = _data(T, h, V, gpu)
    g = 2.0 ** torch.linspace(-100, 100, T, device=gpu) * 1.37
    dx, _ = _grads(x, w, t, g, "none")
    xd, wd = x.double(), w.double()
    z = xd @ wd.t().contiguous()
    p = torch.softmax(z, 1)
    s = p.clone()
    s[torch.arange(T, device=gpu), t] -= 1.0
    u = 2.0 ** -24
    dz = 2 * (h + 1) * u * (xd.abs() @ wd.abs().t().contiguous()).amax(1, keepdim=True)
    e = (s.abs() * (V8 + 8 * u) + p * (2 * dz + (432 + V / 512) * u) + 2 * (V + 20) * u * s.abs()) @ wd.abs()
    exact, e = g.double()[:, None] * (s @ wd), g.double()[:, None] * e
    assert bool(((dx.double() - exact).abs() <= e + V8 * (exact.abs() + e)).all())


def test_a_row_whose_gradient_is_not_finite(gpu):
    """Its own dx takes it; the others' are what they are without it."""
    T, h, V = 200, 64, 500
    x, w, t = _data(T, h, V, gpu)
    g = torch.linspace(0.1, 1.3, T, device=gpu)
    g[7] = 0.0
    plain, _ = _grads(x, w, t, g, "none")
    for bad in (float("nan"), float("inf"), float("-inf")):
        g[7] = bad
        dx, _ = _grads(x, w, t, g, "none")
        rest = torch.arange(T, device=gpu) != 7
        assert torch.equal(dx[rest], plain[rest])
        assert not bool(torch.isfinite(dx[7]).any())


def test_captured(gpu):
    """Forward and backward in a graph, with a gradient per row that changes between the replays."""
    from q38.hip import ops
    x, w, t = _data(300, 128, 1000, gpu, ignored=0.2)
    g = torch.full((300,), 0.3, device=gpu)

    def step():
        loss, lse, _, _ = ops.linear_ce_forward(x, w, t)
        return (loss, *ops.linear_ce_backward(g, x, w, t, lse))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(4):
        g.copy_(torch.rand(300, device=gpu) * 3 ** i + 0.1)
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        for a, b in zip(got, step()):
            assert torch.equal(a, b), f"replay {i}"

"""grad_norm, clip_grads and clip_grad_norm_ (q38moe_clip.hip) against float64. Sums are in fp64, so the norm is off by its
rounding to fp32, 2^-24, and 1e-12; a clipped element by the norm's, the sum's, the quotient's and the product's
roundings (4 * 2^-24) and the output type's half step."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
SIZES = [1, 3, 7, 8, 9, 255, 256, 257, 2047, 2048, 8191, 8192, 16383, 16384, 16385, 40000, 100003]


def _grads(sizes, dtypes, dev, seed=0, std=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return [(torch.randn(n, generator=g, device=dev) * std).to(dtypes[i % len(dtypes)]) for i, n in enumerate(sizes)]


def _norm64(grads, p):
    flat = torch.cat([t.double().reshape(-1) for t in grads])
    return float(torch.linalg.vector_norm(flat, p))


def _check_scaled(before, after, norm64, max_norm):
    c = min(1.0, max_norm / (norm64 + 1e-6))
    for b, a in zip(before, after):
        want = b.double() * c
        tol = want.abs() * (torch.finfo(a.dtype).eps / 2 + 5 * U) + 1.5e-45
        assert bool(((a.double() - want).abs() <= tol).all()), tuple(b.shape)


@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("dtypes", [(torch.bfloat16,), (torch.float32,), (torch.bfloat16, torch.float32)])
def test_norm_and_clip(gpu, p, dtypes):
    from q38.hip import ops
    grads = _grads(SIZES, dtypes, gpu)
    n64 = _norm64(grads, p)
    assert abs(float(ops.grad_norm(grads, p)) - n64) <= n64 * (U + 1e-12)
    for max_norm in (0.25 * n64, 4 * n64, 0.0):
        out = [torch.full_like(t, 7.0) for t in grads]
        got = ops.clip_grads(grads, max_norm, p, out=out)
        assert abs(float(got) - n64) <= n64 * (U + 1e-12)
        _check_scaled(grads, out, n64, max_norm)
        here = [t.clone() for t in grads]
        assert torch.equal(ops.clip_grads(here, max_norm, p), got)
        assert all(torch.equal(a, b) for a, b in zip(here, out))


def test_other_types_out(gpu):
    """bf16 gradients clipped into fp32 tensors, and fp32 ones into bf16."""
    from q38.hip import ops
    for a, b in ((torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16)):
        grads = _grads(SIZES, (a,), gpu)
        out = [torch.empty_like(t, dtype=b) for t in grads]
        ops.clip_grads(grads, 1.0, out=out)
        _check_scaled(grads, out, _norm64(grads, 2), 1.0)


def test_unaligned_views(gpu):
    """Gradients that are views of one buffer, each off a 16-byte boundary by another amount; what lies between them
    stays."""
    from q38.hip import ops
    for dtype in (torch.bfloat16, torch.float32):
        flat = torch.full((sum(SIZES) + 16 * len(SIZES),), 3.0, dtype=dtype, device=gpu)
        views, at = [], 0
        for i, n in enumerate(SIZES):
            at += 1 + i % 9
            views.append(flat[at:at + n])
            at += n
        for v, t in zip(views, _grads(SIZES, (dtype,), gpu)):
            v.copy_(t)
        before = [v.clone() for v in views]
        n64 = _norm64(before, 2)
        ops.clip_grads(views, 1.0)
        _check_scaled(before, views, n64, 1.0)
        left = flat.clone()
        for v in views:
            s = v.storage_offset()
            left[s:s + v.numel()] = 3.0
        assert bool((left == 3.0).all())


@pytest.mark.parametrize("n", [1, 95, 96, 97, 300])
def test_many_tensors(gpu, n):
    """On both sides of the tensors that a launch takes; empty ones among them."""
    from q38.hip import ops
    sizes = [(37 * i) % 5000 for i in range(n)]
    sizes[-1] = max(sizes[-1], 5)
    grads = _grads(sizes, (torch.float32, torch.bfloat16), gpu, seed=n)
    for p in (1.0, 2.0, math.inf):
        n64 = _norm64(grads, p)
        here = [t.clone() for t in grads]
        got = ops.clip_grads(here, 0.5 * n64, p)
        assert abs(float(got) - n64) <= n64 * (U + 1e-12)
        _check_scaled(grads, here, n64, 0.5 * n64)


def test_one_large_tensor(gpu):
    from q38.hip import ops
    t = torch.randn(70_000_001, device=gpu)
    n64 = float(torch.linalg.vector_norm(t.double()))
    out = torch.empty_like(t)
    got = ops.clip_grads([t], 1.0, out=[out])
    assert abs(float(got) - n64) <= n64 * (U + 1e-12)
    _check_scaled([t], [out], n64, 1.0)


def test_extreme_values(gpu):
    """Squares that overflow or vanish in fp32; NaN and infinities as the formula has them."""
    from q38.hip import ops
    for size in (1e30, 1e-30):
        grads = [torch.full((1000,), size, device=gpu), torch.full((500,), -size, device=gpu).bfloat16()]
        n64 = _norm64(grads, 2)
        assert abs(float(ops.grad_norm(grads)) - n64) <= n64 * (U + 1e-12)
    for bad in (math.nan, math.inf, -math.inf):
        for p in (1.0, 2.0, math.inf):
            for dtype in (torch.float32, torch.bfloat16):
                grads = _grads([100, 5000], (dtype,), gpu)
                grads[1][4999] = bad
                want = torch.nn.utils.get_total_norm([t.float() for t in grads], p)
                got = ops.grad_norm(grads, p)
                assert torch.equal(torch.isnan(got), torch.isnan(want)) and (torch.isnan(got) or torch.equal(got, want))
                clipped = [t.clone() for t in grads]
                ops.clip_grads(clipped, 1.0, p)
                if math.isnan(bad):
                    assert all(torch.isnan(t).all() for t in clipped)
                else:  # max / inf = 0: finite gradients vanish, inf * 0 is NaN
                    assert torch.isnan(clipped[1][4999]) and not clipped[0].any() and not clipped[1][:4999].any()
    assert float(ops.grad_norm([torch.zeros(10, device=gpu)])) == 0.0
    empty = torch.zeros(0, device=gpu)
    assert float(ops.grad_norm([empty])) == 0.0 and float(ops.clip_grads([empty], 1.0)) == 0.0


def test_clip_grad_norm_matches_torch(gpu):
    from q38.hip import ops
    g = torch.Generator(device=gpu).manual_seed(1)
    shapes = [(64, 32), (7,), (3, 5, 9), (), (1000, 64)]
    for p in (1.0, 2.0, math.inf):
        ours = [torch.nn.Parameter(torch.zeros(s, device=gpu)) for s in shapes]
        theirs = [torch.nn.Parameter(torch.zeros(s, device=gpu)) for s in shapes]
        for a, b in zip(ours, theirs):
            a.grad = torch.randn(a.shape, generator=g, device=gpu)
            b.grad = a.grad.clone()
        ours[1].grad = theirs[1].grad = None
        ours[0].grad = ours[0].grad.t().contiguous().t()  # not contiguous
        a = ops.clip_grad_norm_((q for q in ours), 0.7, p)
        b = torch.nn.utils.clip_grad_norm_(theirs, 0.7, p)
        assert abs(float(a) - float(b)) <= 1e-5 * float(b)  # torch sums in fp32
        assert ours[1].grad is None
        for u, v in zip(ours, theirs):
            if u.grad is not None:
                assert torch.allclose(u.grad, v.grad, rtol=2e-5, atol=1e-9)
    assert float(ops.clip_grad_norm_([], 1.0)) == 0.0
    one = torch.nn.Parameter(torch.zeros(10, device=gpu))
    one.grad = torch.ones(10, device=gpu)
    assert abs(float(ops.clip_grad_norm_(one, 1.0)) - math.sqrt(10)) < 1e-6
    assert abs(float(one.grad.norm()) - 1.0) < 1e-5


def test_nonfinite_raises_before_a_change(gpu):
    from q38.hip import ops
    q = torch.nn.Parameter(torch.zeros(10, device=gpu))
    q.grad = torch.ones(10, device=gpu)
    q.grad[3] = math.inf
    before = q.grad.clone()
    with pytest.raises(RuntimeError, match="not finite"):
        ops.clip_grad_norm_([q], 1.0, error_if_nonfinite=True)
    assert torch.equal(q.grad, before)


def test_version_counter(gpu):
    """A clipped gradient counts as changed for autograd."""
    from q38.hip import ops
    t = torch.ones(10, device=gpu)
    v = t._version
    ops.clip_grads([t], 1.0)
    assert t._version > v


def test_overlaps_are_refused(gpu):
    from q38.hip import ops
    t = torch.ones(100, device=gpu)
    u = torch.ones(100, device=gpu)
    for grads, out in (([t, t], None), ([t[:60], t[50:]], None), ([t, u], [u, torch.empty_like(t)]),
                       ([t[:50]], [t[1:51]]), ([t, u], [torch.empty_like(t)] * 2)):
        with pytest.raises(RuntimeError, match="overlap"):
            ops.clip_grads(grads, 1.0, out=out)
    assert bool((t == 1).all()) and bool((u == 1).all())
    # read twice is no harm
    assert abs(float(ops.grad_norm([t, t])) - math.sqrt(200)) < 1e-5


def test_captured_and_on_another_stream(gpu):
    from q38.hip import ops
    grads = _grads(SIZES, (torch.float32, torch.bfloat16), gpu)
    out = [torch.empty_like(t) for t in grads]
    eager = ops.clip_grads(grads, 1.0, out=out).clone()
    want = [t.clone() for t in out]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = ops.clip_grads(grads, 1.0, out=out)
    torch.cuda.synchronize()
    assert torch.equal(other, eager) and all(torch.equal(a, b) for a, b in zip(out, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = ops.clip_grads(grads, 1.0, out=out)
    for i in range(3):
        for t in grads:
            t.mul_(1.5)
        graph.replay()
        torch.cuda.synchronize()
        got, clipped = norm.clone(), [t.clone() for t in out]
        assert torch.equal(got, ops.clip_grads(grads, 1.0, out=out))
        assert all(torch.equal(a, b) for a, b in zip(out, clipped))


def test_more_than_2_31_elements(gpu):
    from q38.hip import ops
    n = 2 ** 31 + 12345
    t = torch.zeros(n, dtype=torch.bfloat16, device=gpu)
    spots = [(0, 100_000), (2 ** 31 - 50_000, 2 ** 31 + 12345)]
    g = torch.Generator(device=gpu).manual_seed(1)
    for a, b in spots:
        t[a:b] = torch.randn(b - a, generator=g, device=gpu).to(torch.bfloat16)
    before = [t[a:b].clone() for a, b in spots]
    n64 = float(torch.cat([v.double() for v in before]).norm())
    got = ops.clip_grads([t], 1.0)
    assert abs(float(got) - n64) <= n64 * (U + 1e-12)
    _check_scaled(before, [t[a:b] for a, b in spots], n64, 1.0)
    assert not bool(t[200_000:2 ** 31 - 60_000].any())

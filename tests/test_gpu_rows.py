"""dispatch and combine (q38moe_rows.hip) against float64. Rows are copies (exact); a sum of at most 8 products in
fp32 is off by at most 10 * 2^-24 of the sum of its terms' sizes, a dot product of h by 2 (h + 8) 2^-24 (the 64 lanes'
sums in between add less), and one rounding to the output's type (finfo.eps / 2)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _inputs(T, h, E, k, dtype, dev, dropped=0.0, idx_dtype=torch.int64, w_dtype=None, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed + T)
    x = torch.randn(T, h, generator=g, device=dev).to(dtype)
    idx = torch.topk(torch.randn(T, E, generator=g, device=dev), k, dim=1).indices.to(idx_dtype)
    if dropped:
        out = torch.rand(T, k, generator=g, device=dev) < dropped
        idx[out] = E
        idx[out & (torch.rand(T, k, generator=g, device=dev) < 0.5)] = -1
    w = torch.rand(T, k, generator=g, device=dev).to(w_dtype or dtype)
    y = torch.randn(T * k, h, generator=g, device=dev).to(dtype)
    return x, idx, w, y, torch.randn(T * k, h, generator=g, device=dev).to(dtype), \
        torch.randn(T, h, generator=g, device=dev).to(dtype)


def _order(idx, E):
    """Pairs by expert, each expert's in ascending order (CPU list), and the counts."""
    flat = idx.reshape(-1).tolist()
    lists = [[p for p, e in enumerate(flat) if e == i] for i in range(E)]
    return [p for l in lists for p in l], [len(l) for l in lists]


def _near(got, exact, terms, sums, name):
    v = torch.finfo(got.dtype).eps / 2
    b = sums * U * terms
    b = b + v * (exact.abs() + b) + 1e-38
    err = (got.double() - exact).abs()
    assert bool((err <= b).all()), f"{name}: worst {float((err / b).max()):.3f} of the bound"


@pytest.mark.parametrize("dtype,w_dtype,idx_dtype", [(torch.bfloat16, torch.bfloat16, torch.int64),
                                                     (torch.bfloat16, torch.float32, torch.int32),
                                                     (torch.float32, torch.float32, torch.int64)])
@pytest.mark.parametrize("T,h,E,k,dropped", [
    (1, 64, 1, 1, 0.0),
    (1, 1024, 64, 5, 0.0),
    (3, 128, 8, 8, 0.3),
    (61, 1088, 60, 4, 0.0),
    (64, 256, 64, 8, 0.5),
    (333, 320, 16, 3, 0.1),
    (1000, 64, 64, 6, 0.95),
    (77, 192, 5, 2, 1.0),      # no pair has a row
    (50, 2048, 7, 7, 0.2),
    (512, 64, 16, 8, 0.1),     # the last pairs that one launch dispatches
    (513, 64, 16, 8, 0.1),     # the first that three do
    (1500, 320, 60, 5, 0.3),
    (900, 192, 9, 7, 1.0),
])
def test_rows(gpu, dtype, w_dtype, idx_dtype, T, h, E, k, dropped):
    from q38.hip import autograd
    x, idx, w, y, d_rows, d_out = _inputs(T, h, E, k, dtype, gpu, dropped, idx_dtype, w_dtype)
    print(f"rows T={T} h={h} E={E} k={k} {dtype} {w_dtype} dropped={dropped}", flush=True)
    order, counts = _order(idx, E)
    n = len(order)
    perm = torch.tensor(order, dtype=torch.int64, device=gpu)
    tok = perm // k
    leaves = [t.clone().requires_grad_(True) for t in (x, y, w)]
    rows, plan = autograd.dispatch(leaves[0], idx, E)
    out = autograd.combine(leaves[1], leaves[2], plan)
    dx, dy, dw = torch.autograd.grad((rows, out), leaves, (d_rows, d_out))
    torch.cuda.synchronize()
    assert plan.counts.tolist() == counts
    assert plan.starts.tolist() == [sum(counts[:e]) for e in range(E)]
    assert plan.perm[:n].tolist() == order and torch.equal(plan.inv[perm].long(), torch.arange(n, device=gpu))
    assert torch.equal(rows[:n], x[tok]) and not rows[n:].any()
    wd, yd = w.double().reshape(-1)[perm][:, None], y.double()[:n]
    zero = torch.zeros(T, h, dtype=torch.float64, device=gpu)
    _near(out, zero.clone().index_add_(0, tok, yd * wd), zero.clone().index_add_(0, tok, (yd * wd).abs()), 10, "out")
    dr = d_rows.double()[:n]
    _near(dx, zero.clone().index_add_(0, tok, dr), zero.clone().index_add_(0, tok, dr.abs()), 10, "dx")
    do = d_out.double()[tok]
    want = torch.zeros(T * k, h, dtype=torch.float64, device=gpu)
    want[:n] = do * wd
    _near(dy, want, want.abs(), 2, "dy")
    dots = torch.zeros(2, T * k, dtype=torch.float64, device=gpu)
    dots[0, perm], dots[1, perm] = (do * yd).sum(1), (do * yd).abs().sum(1)
    assert dw.dtype == w.dtype
    _near(dw, dots[0].view(T, k), dots[1].view(T, k), 2 * (h + 8), "dw")


def test_gradients_of_one_operand(gpu):
    from q38.hip import autograd
    x, idx, w, y, _, d_out = _inputs(100, 128, 8, 2, torch.bfloat16, gpu, 0.2)
    plan = autograd.dispatch(x, idx, 8)[1]
    yl, wl = y.clone().requires_grad_(True), w.clone().requires_grad_(True)
    dy, dw = torch.autograd.grad(autograd.combine(yl, wl, plan), (yl, wl), d_out)
    assert torch.equal(dy, torch.autograd.grad(autograd.combine(yl, w, plan), yl, d_out)[0])
    assert torch.equal(dw, torch.autograd.grad(autograd.combine(y, wl, plan), wl, d_out)[0])
    assert not autograd.combine(y, w, plan).requires_grad


def test_rows_without_a_pair_reach_nothing(gpu):
    """NaN in the rows behind the filled ones, and in the weights of dropped pairs, reaches no output."""
    from q38.hip import autograd
    x, idx, w, y, d_rows, d_out = _inputs(90, 64, 16, 4, torch.bfloat16, gpu, 0.4)
    plan = autograd.dispatch(x, idx, 16)[1]
    n = int(plan.counts.sum())
    y[n:], d_rows[n:] = float("nan"), float("nan")
    w[(idx < 0) | (idx >= 16)] = float("nan")
    leaves = [t.clone().requires_grad_(True) for t in (x, y, w)]
    rows, plan = autograd.dispatch(leaves[0], idx, 16)
    out = autograd.combine(leaves[1], leaves[2], plan)
    for t in (out, *torch.autograd.grad((rows, out), leaves, (d_rows, d_out))):
        assert torch.isfinite(t).all()


def test_the_same_expert_twice(gpu):
    """Both of a token's pairs at one expert are two rows."""
    from q38.hip import autograd
    x = torch.randn(5, 64, device=gpu)
    idx = torch.tensor([[1, 1], [0, 1], [1, 0], [0, 0], [1, 1]], device=gpu)
    rows, plan = autograd.dispatch(x, idx, 2)
    assert plan.counts.tolist() == [4, 6]
    back = autograd.combine(rows, torch.full((5, 2), 0.5, device=gpu), plan)
    assert torch.equal(back, x)


def test_strided_unaligned_and_empty(gpu):
    from q38.hip import autograd
    x, idx, w, y, _, _ = _inputs(40, 64, 8, 2, torch.bfloat16, gpu)
    rows, plan = autograd.dispatch(x, idx, 8)
    wide = torch.cat([x, x], 1)[:, :64]
    flat = torch.empty(x.numel() + 1, dtype=x.dtype, device=gpu)
    assert torch.equal(rows, autograd.dispatch(wide, idx.t().contiguous().t(), 8)[0])
    assert torch.equal(rows, autograd.dispatch(flat[1:].view_as(x).copy_(x), idx, 8)[0])
    out = autograd.combine(y, w, plan)
    assert torch.equal(out, autograd.combine(torch.cat([y, y], 1)[:, :64], w.t().contiguous().t(), plan))
    e = torch.empty(0, 64, device=gpu, requires_grad=True)
    rows, plan = autograd.dispatch(e, torch.empty(0, 2, dtype=torch.int64, device=gpu), 8)
    assert rows.shape == (0, 64) and plan.counts.tolist() == [0] * 8
    out = autograd.combine(rows, torch.empty(0, 2, device=gpu), plan)
    assert torch.autograd.grad(out.sum(), e)[0].shape == (0, 64)


def test_against_differences(gpu):
    """Both operators are linear in each operand: differences are exact up to fp32 roundings (the sums of h T k
    products of normals, each side within 1e-4 of its size)."""
    from q38.hip import autograd
    x, idx, w, y, _, d_out = _inputs(30, 64, 8, 3, torch.float32, gpu, 0.1)
    leaves = [t.clone().requires_grad_(True) for t in (x, w)]

    def f(a, b):
        rows, plan = autograd.dispatch(a, idx, 8)
        return (autograd.combine(rows, b, plan).double() * d_out.double()).sum()

    dx, dw = torch.autograd.grad(f(*leaves), leaves)
    ux, uw = torch.randn_like(x), torch.randn_like(w)
    for step, slope in (((ux, 0 * uw), (dx.double() * ux.double()).sum()), ((0 * ux, uw), (dw.double() * uw.double()).sum())):
        diff = (f(x + step[0], w + step[1]) - f(x - step[0], w - step[1])) / 2
        assert abs(float(diff) - float(slope)) <= 1e-4 * max(1.0, abs(float(slope)))


def test_captured_and_on_another_stream(gpu):
    from q38.hip import ops
    x, idx, w, y, _, d_out = _inputs(200, 128, 16, 4, torch.bfloat16, gpu, 0.1)

    def step():
        plan = ops.RowsPlan(idx, 16)
        return (ops.dispatch_rows(x, plan), ops.collect_rows(y, plan, w), plan.counts,
                *ops.spread_rows(d_out, plan, w, y))

    eager = [t.clone() for t in step()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(eager, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    g = torch.Generator(device=gpu).manual_seed(3)
    for _ in range(3):
        x.copy_(torch.randn(x.shape, generator=g, device=gpu))
        idx.copy_(torch.topk(torch.randn(200, 16, generator=g, device=gpu), 4, dim=1).indices)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs]
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_indices_may_change_after_dispatch(gpu):
    """Combine and the gradients follow the plan: indices overwritten since dispatch, dropped pairs made valid among them, reach
    nothing."""
    from q38.hip import autograd, ops
    x, idx, w, y, d_rows, d_out = _inputs(77, 128, 16, 4, torch.bfloat16, gpu, dropped=0.5)

    def run(spoil):
        mine = idx.clone()
        leaves = [a.clone().requires_grad_(True) for a in (x, w, y)]
        rows, plan = autograd.dispatch(leaves[0], mine, 16)
        assert bool(((plan.inv >= 0) == ((idx >= 0) & (idx < 16)).reshape(-1)).all())
        if spoil:
            mine.copy_(torch.arange(77 * 4, device=gpu).view(77, 4) % 16)
        out = autograd.combine(leaves[2], leaves[1], plan)
        return [rows, out, *torch.autograd.grad((rows, out), leaves, (d_rows, d_out))]

    for a, b in zip(run(False), run(True)):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError, match="plan is empty"):
        ops.collect_rows(y, ops.RowsPlan(idx, 16))
    with pytest.raises(RuntimeError, match="plan is empty"):
        ops.spread_rows(x, ops.RowsPlan(idx, 16))


def test_forward_mode_is_refused(gpu):
    """A tangent is not dropped silently."""
    import torch.autograd.forward_ad as fwad
    from q38.hip import autograd
    x, idx, w, y, _, _ = _inputs(8, 64, 4, 2, torch.float32, gpu)
    _, plan = autograd.dispatch(x, idx, 4)
    head, t = torch.randn(10, 64, device=gpu), torch.zeros(8, dtype=torch.int64, device=gpu)
    with fwad.dual_level():
        dual = fwad.make_dual(x, torch.ones_like(x))
        for f in (lambda: autograd.dispatch(dual, idx, 4), lambda: autograd.linear_cross_entropy(dual, head, t),
                  lambda: autograd.combine(fwad.make_dual(y, torch.ones_like(y)), w, plan)):
            with pytest.raises(Exception, match="jvp|forward mode"):
                f()


def test_offsets_past_32_bits(gpu):
    """Rows of more than 4 GiB: copies there and the sums back, checked in pieces."""
    from q38.hip import autograd
    T, h, E, k = 450_000, 1024, 64, 5
    g = torch.Generator(device=gpu).manual_seed(5)
    x = torch.empty(T, h, dtype=torch.bfloat16, device=gpu)
    for i in range(0, T, 50_000):
        x[i:i + 50_000] = torch.randn(50_000, h, generator=g, device=gpu).to(torch.bfloat16)
    idx = torch.topk(torch.rand(T, E, generator=g, device=gpu), k, dim=1).indices
    w = torch.rand(T, k, generator=g, device=gpu).to(torch.bfloat16)
    print("rows past 32 bits", flush=True)
    rows, plan = autograd.dispatch(x, idx, E)
    out = autograd.combine(rows, w, plan)
    inv = plan.inv.view(T, k).long()
    assert int(plan.counts.sum()) == T * k and bool((torch.sort(inv.reshape(-1)).values == torch.arange(T * k, device=gpu)).all())
    for i in range(0, T, 50_000):
        xd, wd = x[i:i + 50_000], w[i:i + 50_000].double()
        assert torch.equal(rows[inv[i:i + 50_000]], xd[:, None].expand(-1, k, -1))
        exact = xd.double() * wd.sum(1, keepdim=True)
        _near(out[i:i + 50_000], exact, xd.double().abs() * wd.sum(1, keepdim=True), 10, f"out {i}")

"""linear_cross_entropy (q38moe_loss.hip) against float64 on the same operands. Every bound is derived from the
roundings that the formulas allow, with u = 2^-24 for fp32 and v = the half step of the operands' type
(finfo.eps / 2: bf16 2^-8, fp32 2^-24):

* a logit is a sum of h exact (bf16) or rounded (fp32) products: off by dz <= 2 (h + 1) u sum |x w|;
* the log-sum-exp adds the roundings of sums of at most 128 terms, of joining the tiles (at most V / 64 of them over 16
  waves, then 16) and of exp and log: (400 + V / 512) u beside dz, and 4 u |.| for the last subtractions;
* s = exp(z - lse) - onehot has p's relative error d = 2 dz + (400 + V / 512 + 32) u (the exponent's own rounding, at most
  |z - lse| u where p matters, is in the 32) and one rounding v; the products sum K terms in fp32, 2 (K + 20) u, and
  round once to the output's type."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _data(T, h, V, dtype, dev, seed=0, ignored=0.0, std=2.0):
    g = torch.Generator(device=dev).manual_seed(1000 * seed + T + V)
    x = torch.randn(T, h, generator=g, device=dev).to(dtype)
    w = (torch.randn(V, h, generator=g, device=dev) * std * h ** -0.5).to(dtype)
    t = torch.randint(0, V, (T,), generator=g, device=dev)
    if ignored:
        t[torch.rand(T, generator=g, device=dev) < ignored] = -100
    return x, w, t, g


def _oracle(x, w, t, ignore=-100):
    """Rows' losses, softmax minus onehot, softmax, logit error dz per row, in float64; ignored rows are zero."""
    keep = t != ignore
    xd = torch.where(keep[:, None], x.double(), torch.zeros((), dtype=torch.float64, device=x.device))
    wd = w.double()
    z = xd @ wd.t().contiguous()
    lse = torch.logsumexp(z, 1)
    at = torch.where(keep, t, torch.zeros_like(t)).long()
    p = torch.exp(z - lse[:, None])
    zt = z.gather(1, at[:, None])[:, 0]
    s = p.clone()
    s.scatter_add_(1, at[:, None], -torch.ones_like(zt)[:, None])
    loss = (lse - zt) * keep
    mag = (xd.abs() @ wd.abs().t().contiguous()).amax(1) if x.shape[0] else zt
    dz = 2 * (x.shape[1] + 1) * U * mag
    return loss, lse, s * keep[:, None], p * keep[:, None], dz, xd, wd, keep


def _check(x, w, t, reduction, g, ignore=-100, what=""):
    """Loss and both gradients of one call against the bounds above."""
    from q38.hip import autograd
    T, h = x.shape
    V = w.shape[0]
    v = torch.finfo(x.dtype).eps / 2
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss = autograd.linear_cross_entropy(xl, wl, t, ignore_index=ignore, reduction=reduction)
    dx, dw = torch.autograd.grad(loss, (xl, wl), g)
    torch.cuda.synchronize()
    rows, lse, s, p, dz, xd, wd, keep = _oracle(x, w, t, ignore)
    n = max(int(keep.sum()), 1)
    rel = (400 + V / 512) * U
    e_rows = (2 * dz + rel + 4 * U * (rows.abs() + 2 * lse.abs())) * keep
    want, bound = rows, e_rows
    if reduction != "none":
        d = n if reduction == "mean" else 1
        want, bound = rows.sum() / d, e_rows.sum() / d + 2 * U * rows.sum().abs() / d
    assert loss.dtype == torch.float32 and loss.shape == want.shape
    err = (loss.double() - want).abs()
    assert bool((err <= bound).all()), f"{what} loss off by {float((err - bound).max()):.3e} more than the bound"
    G = g.double() * keep if reduction == "none" else g.double() / (n if reduction == "mean" else 1) * keep
    G = G[:, None]
    d = (2 * dz + rel + 32 * U)[:, None]
    e_s = s.abs() * (v + 8 * U) + p * d
    for name, got, exact, e in (
            ("dx", dx, (G * s) @ wd, ((G.abs() * (e_s + 2 * (V + 20) * U * s.abs())) @ wd.abs())),
            ("dw", dw, (G * s).t().contiguous() @ xd,
             (G.abs() * (e_s + 2 * (T + 20) * U * s.abs())).t().contiguous() @ xd.abs())):
        assert got.dtype == x.dtype
        b = e + v * (exact.abs() + e) + 1e-38
        err = (got.double() - exact).abs()
        assert bool((err <= b).all()), \
            f"{what} {name}: {int((err > b).sum())} of {err.numel()} off, worst {float((err / b).max()):.3f} of the bound"
    return loss, dx, dw


def _grad_of(reduction, T, gen, dev):
    return (torch.rand(T, generator=gen, device=dev) + 0.1 if reduction == "none"
            else torch.rand((), generator=gen, device=dev) + 0.5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,h,V,ignored", [
    (1, 64, 1, 0.0),         # one token, one word
    (1, 64, 300, 0.0),
    (2, 128, 64, 0.0),
    (63, 192, 127, 0.3),     # one row short of a wave, one word short of a tile
    (64, 256, 128, 0.0),
    (65, 320, 129, 0.5),     # one past both
    (128, 64, 1000, 0.0),
    (200, 1088, 513, 0.9),
    (256, 64, 256, 0.2),     # the last size whose rows the forward takes where they are
    (257, 64, 257, 0.2),     # the first whose rows are listed
    (515, 256, 777, 0.1),
    (1300, 128, 2049, 0.6),
    (100, 4096, 300, 0.1),   # 64 steps of K: the eight slots of small tiles go round
    (700, 1344, 200, 0.0),
    (2048, 64, 130, 0.3),    # the last size with 16 rows to a finishing block
    (2049, 64, 130, 0.3),
    (8192, 64, 70, 0.3),     # the last size whose list and copies are one launch
    (8193, 64, 70, 0.3),
])
def test_small(gpu, dtype, T, h, V, ignored):
    x, w, t, g = _data(T, h, V, dtype, gpu, ignored=ignored)
    for reduction in ("mean", "sum", "none"):
        print(f"loss T={T} h={h} V={V} {dtype} {reduction}", flush=True)
        _check(x, w, t, reduction, _grad_of(reduction, T, g, gpu), what=reduction)


@pytest.mark.parametrize("dtype,T,h,V,ignored,reduction", [
    (torch.bfloat16, 2100, 256, 4100, 0.0, "mean"),      # 256 x 256 tiles in the products over the vocabulary
    (torch.bfloat16, 8200, 1024, 8200, 0.1, "mean"),     # and in both gradients
    (torch.bfloat16, 8200, 64, 20001, 0.0, "none"),      # two pieces of the vocabulary
    (torch.bfloat16, 40, 1024, 10112, 0.0, "mean"),      # few tokens: the gradients split their sums
    (torch.bfloat16, 9000, 128, 70, 0.0, "sum"),
    (torch.float32, 2100, 256, 4100, 0.2, "mean"),
    (torch.float32, 4200, 64, 20001, 0.0, "none"),       # two pieces in fp32
])
def test_large(gpu, dtype, T, h, V, ignored, reduction):
    x, w, t, g = _data(T, h, V, dtype, gpu, ignored=ignored)
    print(f"loss T={T} h={h} V={V} {dtype} {reduction}", flush=True)
    _check(x, w, t, reduction, _grad_of(reduction, T, g, gpu))


def test_masked_rows_may_hold_anything(gpu):
    """NaN and infinities in rows whose target is ignored reach neither the loss nor a gradient."""
    for T in (100, 700):
        x, w, t, g = _data(T, 128, 500, torch.bfloat16, gpu, ignored=0.4)
        bad = x.clone()
        gone = t == -100
        bad[gone] = float("nan")
        bad[torch.nonzero(gone)[0, 0]] = float("inf")
        for reduction in ("mean", "none"):
            go = _grad_of(reduction, T, g, gpu)
            a = _check(x, w, t, reduction, go)
            b = _check(bad, w, t, reduction, go)
            assert all(torch.equal(u, v) for u, v in zip(a, b))
            assert not b[1][gone].any()


def test_all_ignored(gpu):
    from q38.hip import autograd
    for T in (1, 70, 400):
        x, w, t, _ = _data(T, 64, 200, torch.bfloat16, gpu)
        x[:] = float("nan")
        t[:] = -100
        for reduction in ("mean", "sum", "none"):
            xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
            loss = autograd.linear_cross_entropy(xl, wl, t, reduction=reduction)
            assert not loss.any()
            dx, dw = torch.autograd.grad(loss.sum(), (xl, wl))
            assert not dx.any() and not dw.any()


def test_no_rows(gpu):
    from q38.hip import autograd
    x = torch.empty(2, 0, 64, device=gpu, dtype=torch.bfloat16, requires_grad=True)
    w = torch.randn(10, 64, device=gpu, dtype=torch.bfloat16, requires_grad=True)
    t = torch.empty(2, 0, dtype=torch.int64, device=gpu)
    assert autograd.linear_cross_entropy(x, w, t, reduction="none").shape == (2, 0)
    loss = autograd.linear_cross_entropy(x, w, t)
    assert float(loss.detach()) == 0
    dx, dw = torch.autograd.grad(loss, (x, w))
    assert dx.shape == x.shape and not dw.any()


def test_other_ignore_index_types_and_shapes(gpu):
    """int32 targets, an ignore_index inside the vocabulary, leading dimensions, rows off 16-byte boundaries and
    strided operands give what the plain call gives."""
    from q38.hip import autograd
    x, w, t, g = _data(90, 64, 300, torch.bfloat16, gpu)
    base = autograd.linear_cross_entropy(x, w, t, ignore_index=7, reduction="none")
    assert torch.equal(base, autograd.linear_cross_entropy(x, w, t.int(), ignore_index=7, reduction="none"))
    assert bool((base[t == 7] == 0).all())
    assert torch.equal(base.view(3, 30), autograd.linear_cross_entropy(x.view(3, 30, 64), w, t.view(3, 30), 7, "none"))
    flat = torch.empty(x.numel() + 1, dtype=x.dtype, device=gpu)
    off = flat[1:].view_as(x).copy_(x)
    wide = torch.cat([w, w], 1)[:, :64]
    assert torch.equal(base, autograd.linear_cross_entropy(off, wide, t, 7, "none"))
    tall = torch.stack([t, t], 1)[:, 0]
    assert torch.equal(base, autograd.linear_cross_entropy(x, w, tall, 7, "none"))


def test_target_outside_the_vocabulary_is_nan(gpu):
    from q38.hip import autograd
    for T in (20, 300):
        x, w, t, _ = _data(T, 64, 100, torch.bfloat16, gpu)
        good = autograd.linear_cross_entropy(x, w, t, reduction="none")
        t[3], t[5] = 100, -1
        loss = autograd.linear_cross_entropy(x, w, t, reduction="none")
        bad = torch.isnan(loss)
        assert torch.nonzero(bad)[:, 0].tolist() == [3, 5]
        assert torch.equal(loss[~bad], good[~bad])


def test_large_logits(gpu):
    """Logits in the hundreds: nothing overflows, and the softmax of a certain row is a onehot."""
    x, w, t, g = _data(150, 128, 400, torch.float32, gpu, std=60.0)
    _check(x, w, t, "mean", torch.ones((), device=gpu))
    x, w, t, g = _data(150, 128, 400, torch.bfloat16, gpu, std=60.0)
    _check(x, w, t, "none", torch.ones(150, device=gpu))


def test_one_operand(gpu):
    """Only the gradients that are asked for, the same bits as together."""
    from q38.hip import autograd
    x, w, t, _ = _data(300, 128, 700, torch.bfloat16, gpu, ignored=0.2)
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    dx, dw = torch.autograd.grad(autograd.linear_cross_entropy(xl, wl, t), (xl, wl))
    assert torch.equal(dx, torch.autograd.grad(autograd.linear_cross_entropy(xl, w, t), xl)[0])
    assert torch.equal(dw, torch.autograd.grad(autograd.linear_cross_entropy(x, wl, t), wl)[0])
    assert not autograd.linear_cross_entropy(x, w, t).requires_grad


def test_autocast(gpu):
    """fp32 parameters under bf16 autocast: the bf16 call's loss, gradients in fp32."""
    from q38.hip import autograd
    x, w, t, _ = _data(100, 64, 300, torch.float32, gpu)
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = autograd.linear_cross_entropy(xl, wl, t)
    loss.backward()
    assert torch.equal(loss, autograd.linear_cross_entropy(x.bfloat16(), w.bfloat16(), t))
    assert xl.grad.dtype == wl.grad.dtype == torch.float32


def test_against_differences(gpu):
    """The gradient along a direction against central differences of the fp32 loss. With step e the differences are off
    by e^2 / 6 of the third derivative, at most the cube of the logits' largest change per unit step (a cumulant of a
    bounded variable), and by the losses' own bounds over e."""
    from q38.hip import autograd
    x, w, t, g = _data(40, 64, 300, torch.float32, gpu)
    dx_, dw_ = torch.randn(x.shape, generator=g, device=gpu) * 0.3, torch.randn(w.shape, generator=g, device=gpu) * 0.02
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    gx, gw = torch.autograd.grad(autograd.linear_cross_entropy(xl, wl, t, reduction="sum"), (xl, wl))
    e = 2.0 ** -6
    for along, slope in (((dx_, torch.zeros_like(w)), float((gx.double() * dx_.double()).sum())),
                         ((torch.zeros_like(x), dw_), float((gw.double() * dw_.double()).sum()))):
        up, down = (float(autograd.linear_cross_entropy(x + s * along[0], w + s * along[1], t, reduction="sum"))
                    for s in (e, -e))
        change = (along[0].double() @ w.double().t().contiguous() + x.double() @ along[1].double().t().contiguous())
        rows, lse, _, _, dz, _, _, _ = _oracle(x, w, t)
        noise = float((2 * dz + 500 * U + 8 * U * (rows.abs() + 2 * lse.abs())).sum()) / e
        # the operands' own roundings x + e d: half a step of |x| times the logits' sensitivity
        noise += float((x.abs().double() @ w.abs().double().t().contiguous()).amax(1).sum()) * 4 * U / e
        bound = e * e / 6 * 40 * float(change.abs().max()) ** 3 + noise + 1e-4 * abs(slope)
        assert abs((up - down) / (2 * e) - slope) <= bound, (up, down, slope, bound)


def test_same_bits_again_and_on_another_stream(gpu):
    from q38.hip import autograd
    x, w, t, _ = _data(700, 256, 3000, torch.bfloat16, gpu, ignored=0.1)
    xl, wl = x.clone().requires_grad_(True), w.clone().requires_grad_(True)

    def step():
        loss = autograd.linear_cross_entropy(xl, wl, t)
        return (loss.detach(), *torch.autograd.grad(loss, (xl, wl)))

    first = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = step()
        again = step()
    torch.cuda.synchronize()
    for a, b, c in zip(first, other, again):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_captured(gpu):
    """Forward and backward in a graph: every replay gives what the eager call on the present inputs gives."""
    from q38.hip import ops
    x, w, t, g = _data(300, 128, 1000, torch.bfloat16, gpu, ignored=0.2)
    one = torch.ones((), device=gpu)

    def step():
        loss, lse, red, scale = ops.linear_ce_forward(x, w, t, reduction="mean")
        return (loss, red, scale, *ops.linear_ce_backward(one, x, w, t, lse, row_scale=scale))

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
        x.copy_(torch.randn(x.shape, generator=g, device=gpu))
        t.copy_(torch.randint(0, 1000, t.shape, generator=g, device=gpu))
        t[:50 * i] = -100
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        for a, b in zip(got, step()):
            assert torch.equal(a, b), f"replay {i}"


def test_close_to_torch(gpu):
    """The same loss and gradients as torch's on materialised fp32 logits, to fp32 accuracy of the losses."""
    from q38.hip import autograd
    x, w, t, _ = _data(333, 256, 2000, torch.float32, gpu, ignored=0.1)
    leaves = [v.clone().requires_grad_(True) for v in (x, w, x, w)]
    ours = autograd.linear_cross_entropy(leaves[0], leaves[1], t)
    theirs = F.cross_entropy(F.linear(leaves[2], leaves[3]), t)
    assert abs(float(ours) - float(theirs)) <= 1e-5
    ours.backward()
    theirs.backward()
    for a, b in ((leaves[0], leaves[2]), (leaves[1], leaves[3])):
        assert float((a.grad - b.grad).norm() / b.grad.norm()) < 1e-5


def test_offsets_past_32_bits(gpu):
    """x, its copy and dx of more than 4 GiB. x is zero but for 3000 rows, at both ends and around element 2^31, so that dw
    sums (and rounds) 3000 terms."""
    from q38.hip import autograd
    T, h, V = 2_200_000, 1024, 70
    g = torch.Generator(device=gpu).manual_seed(3)
    x = torch.zeros(T, h, dtype=torch.bfloat16, device=gpu)
    for i in (0, 2 ** 31 // h - 500, T - 1000):
        x[i:i + 1000] = torch.randn(1000, h, generator=g, device=gpu).to(torch.bfloat16)
    w = (torch.randn(V, h, generator=g, device=gpu) * h ** -0.5).to(torch.bfloat16)
    t = torch.randint(0, V, (T,), generator=g, device=gpu)
    t[5] = t[T // 2] = t[T - 3] = -100  # a copy of x is made, and zeros are written
    x.requires_grad_(True)
    w.requires_grad_(True)
    print("loss past 32 bits", flush=True)
    loss = autograd.linear_cross_entropy(x, w, t, reduction="sum")
    dx, dw = torch.autograd.grad(loss, (x, w))
    x, w = x.detach(), w.detach()
    v, total, size = 2.0 ** -8, 0.0, 0.0
    want, bound = torch.zeros(V, h, dtype=torch.float64, device=gpu), torch.zeros(V, h, dtype=torch.float64, device=gpu)
    for i in range(0, T, 100_000):
        rows, _, s, p, dz, xd, wd, keep = _oracle(x[i:i + 100_000], w, t[i:i + 100_000])
        total, size = total + float(rows.sum()), size + float((2 * dz + 420 * U).sum())
        e = s.abs() * (v + 8 * U) + p * (2 * dz + 440 * U)[:, None]
        want += s.t().contiguous() @ xd
        bound += (e + 2 * (3000 + 20) * U * s.abs()).t().contiguous() @ xd.abs()
        exact, b = s @ wd, (e + 2 * (V + 20) * U * s.abs()) @ wd.abs()
        err = (dx[i:i + 100_000].double() - exact).abs()
        assert bool((err <= b + v * (exact.abs() + b) + 1e-38).all()), i
    assert abs(float(loss) - total) <= size + 2 * U * total
    assert bool(((dw.double() - want).abs() <= bound + v * (want.abs() + bound)).all())


@pytest.mark.parametrize("dtype,T,h,V,ignored,reduction", [
    # Sides of the gradients' tiles and ways of their last, partial round, on 256 CUs.
    (torch.bfloat16, 300, 1024, 8200, 0.0, "mean"),     # dw: 256, whole
    (torch.bfloat16, 4099, 2048, 300, 0.2, "mean"),     # dx: 256, whole
    (torch.bfloat16, 1500, 2048, 8200, 0.1, "sum"),     # dx: 256, equal parts
    (torch.bfloat16, 5000, 2048, 2049, 0.0, "none"),    # dw: 256, equal parts
    (torch.bfloat16, 3000, 2048, 20001, 0.0, "mean"),   # dx: 256, even runs
    (torch.bfloat16, 12000, 1024, 10112, 0.0, "mean"),  # dw: 256, even runs
    (torch.bfloat16, 16400, 256, 8200, 0.1, "mean"),    # dx: 256, equal parts, two pieces
    (torch.bfloat16, 3000, 512, 50021, 0.0, "mean"),    # dw: 256, whole, two pieces
    (torch.bfloat16, 16400, 64, 300, 0.0, "mean"),      # dx: 128, whole
    (torch.bfloat16, 12000, 64, 2049, 0.3, "none"),     # dx: 128, equal parts
    (torch.bfloat16, 20000, 256, 8200, 0.0, "sum"),     # dx: 128, whole, two pieces
    (torch.bfloat16, 6500, 64, 4100, 0.0, "mean"),      # dw: 128, equal parts
    (torch.bfloat16, 2100, 128, 50021, 0.0, "mean"),    # dx: 64, even runs
    (torch.bfloat16, 3000, 64, 50021, 0.1, "mean"),     # dx: 64, equal parts, two pieces
    (torch.float32, 2100, 128, 30011, 0.0, "mean"),     # dx: 64, even runs
    (torch.float32, 1500, 64, 50021, 0.0, "none"),      # dx: 64, equal parts, two pieces
    (torch.float32, 16400, 128, 8200, 0.1, "mean"),     # dw: 64, even runs, two pieces
    (torch.float32, 16400, 64, 300, 0.0, "mean"),       # dx: 128, whole
    (torch.float32, 1000, 512, 20001, 0.0, "mean"),     # dx: 128, even runs
    (torch.float32, 4099, 64, 30011, 0.1, "sum"),       # dx: 128, even runs, two pieces
    (torch.float32, 16400, 512, 1000, 0.0, "mean"),     # dw: 128, even runs
    (torch.float32, 300, 64, 20001, 0.0, "mean"),       # dw: 128, whole
])
def test_plans(gpu, dtype, T, h, V, ignored, reduction):
    x, w, t, g = _data(T, h, V, dtype, gpu, ignored=ignored)
    print(f"loss T={T} h={h} V={V} {dtype} {reduction}", flush=True)
    _check(x, w, t, reduction, _grad_of(reduction, T, g, gpu))

"""qk_norm_rope (q38moe_rope.hip) and linear attention (q38moe_linattn.hip) against float64.

u = 2^-24, v = the half step of the tensors' type. Rotation: a feature is a sum of two products of a normed value, whose norm is
a sum of d squares, a division and a reciprocal root, with a cosine that is off by 2 pi 2^-25 from the fraction of a turn and 2 u
from the function; (d + 40) u of the sizes covers all of it, and one rounding adds v of the result. Its gradients have a second
sum of d: 3 (d + 40) u of the sizes of their terms. An angle in 64 bits is itself off by 2^-53 of it for each product: one in
these references, and in the kernel position * inv_freq, times 1 / 2 pi and that constant's own rounding. Four together make
1e-11 at a position of 10^4 and 5e-4 at 2^40, where it is most of a bf16 rounding.

Linear attention: within a chunk of 64 tokens a bf16 call keeps the weighted scores in two parts (v^2 of each; v is counted) and
rounds the state that queries read once (v of each element), then the result (v). The fp32 sums have dk, 64 and, through the state, all earlier
tokens as terms: 2 (dk + 64 + n + 20) u of the sum of all terms' sizes, n the number of chunks (within a chunk 64 terms more; decays
are rounded once a chunk). States are not rounded to bf16 at all. The gradients are the same sums with the roles exchanged."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _randn(g, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g, device=g.device) * std).to(dtype)


def _within(got, exact, bound, name):
    err = (got.double() - exact).abs()
    bad = ~(err <= bound)
    assert not bool(bad.any()), f"{name}: worst {float((err / bound).nan_to_num(1e9).max()):.3f} of the bound"


# ---- norms and rotation -----------------------------------------------------------------------

def _turn(pos, inv, axes):
    at = pos.double()[..., None] if axes is None else pos.double()[axes.long()].movedim(0, -1)
    a = at * inv.double()
    return a.cos()[..., None, :], a.sin()[..., None, :]


def _rope64(x, w, cos, sin, eps, plus1, dy=None):
    """Result and its terms' sizes; with dy also (dx, sizes, dw, sizes)."""
    x, half = x.double(), cos.shape[-1]
    rstd = torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps) if w is not None else torch.ones_like(x[..., :1])
    ww = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if w is None else w.double() + (1.0 if plus1 else 0.0)

    def rotate(n, s, size=False):
        a, b = n[..., :half], n[..., half:2 * half]
        c, s = (cos.abs(), s.abs()) if size else (cos, s)
        # A turn's error is absolute: it counts whole, also where the cosine is small.
        lo = (a.abs() + b.abs()) if size else a * c - b * s
        hi = (a.abs() + b.abs()) if size else b * c + a * s
        return torch.cat([lo, hi, n[..., 2 * half:].abs() if size else n[..., 2 * half:]], -1)

    n = x * rstd * ww
    y, size = rotate(n, sin), rotate(n, sin, True)
    if dy is None:
        return y, size
    dy = dy.double()
    dn, dn_size = rotate(dy, -sin), rotate(dy, sin, True)
    if w is None:
        return y, size, dn, dn_size, None, None
    xh, gx, gx_size = x * rstd, dn * ww, dn_size * ww.abs()
    dot, dot_size = (gx * xh).mean(-1, keepdim=True), (gx_size * xh.abs()).mean(-1, keepdim=True)
    dx, dx_size = rstd * (gx - xh * dot), rstd * (gx_size + xh.abs() * dot_size)
    lead = tuple(range(x.dim() - 1))
    return y, size, dx, dx_size, (dn * xh).sum(lead), (dn_size * xh.abs()).sum(lead)


def _rope_inputs(dev, lead, H, KV, d, rot, dtype, axes, pos_dtype=torch.int64, far=5000, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed + d + H)
    q, k = _randn(g, *lead, H, d, dtype=dtype), _randn(g, *lead, KV, d, dtype=dtype)
    wq, wk = _randn(g, d, std=0.2, dtype=dtype), _randn(g, d, std=0.2, dtype=dtype)
    inv = (1e4 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1))).float().to(dev)
    pos = torch.randint(0, far, (*((axes,) if axes else ()), *lead), generator=g, device=dev).to(pos_dtype)
    am = torch.randint(0, axes, (rot // 2,), generator=g, device=dev).int() if axes else None
    return q, k, wq, wk, inv, pos, am, _randn(g, *lead, H, d, dtype=dtype), _randn(g, *lead, KV, d, dtype=dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lead,H,KV,d,rot,axes,norm,plus1,pos_dtype,far", [
    ((1,), 38, 2, 64, 16, 0, True, True, torch.int64, 1 << 20),
    ((2, 37), 5, 3, 64, 64, 3, True, False, torch.int32, 4096),
    ((61,), 16, 2, 256, 64, 3, True, True, torch.int64, 100),
    ((7, 1), 1, 1, 8, 8, 0, True, True, torch.int64, 50),
    ((33,), 3, 1, 96, 24, 2, True, True, torch.int32, 1 << 30),
    ((19,), 2, 2, 40, 0, 0, True, True, torch.int64, 10),       # norm alone
    ((129,), 13, 13, 128, 128, 4, False, True, torch.int64, 1 << 40),  # rotation alone
    ((300,), 33, 31, 24, 16, 0, True, False, torch.int64, 9999),
    ((2500,), 2, 1, 16, 8, 0, True, True, torch.int64, 9999),   # blocks with several groups of tokens
    ((0,), 2, 1, 64, 16, 0, True, True, torch.int64, 10),
])
def test_rope(gpu, dtype, lead, H, KV, d, rot, axes, norm, plus1, pos_dtype, far):
    from q38.hip import autograd
    print(f"rope {dtype} {lead} H={H} KV={KV} d={d} rot={rot} axes={axes}", flush=True)
    q, k, wq, wk, inv, pos, am, dq_o, dk_o = _rope_inputs(gpu, lead, H, KV, d, rot, dtype, axes, pos_dtype, far)
    if not norm:
        wq = wk = None
    leaves = [t.clone().requires_grad_(True) for t in (q, k, wq, wk) if t is not None]
    ws = leaves[2:] if norm else [None, None]
    qo, ko = autograd.qk_norm_rope(leaves[0], leaves[1], *ws, pos, inv, axes=am, eps=1e-5, unit_offset=plus1)
    grads = torch.autograd.grad((qo, ko), leaves, (dq_o, dk_o))
    torch.cuda.synchronize()
    assert qo.is_contiguous() and qo.shape == q.shape and ko.shape == k.shape
    with torch.no_grad():
        alone = autograd.qk_norm_rope(q, k, wq, wk, pos, inv, axes=am, eps=1e-5, unit_offset=plus1)
    assert torch.equal(alone[0], qo) and torch.equal(alone[1], ko)
    v = torch.finfo(dtype).eps / 2
    cos, sin = _turn(pos, inv, am)
    angle = 4 * 2.0 ** -53 * float(pos.abs().max() * inv.double().max()) if pos.numel() and rot else 0.0
    for i, (x, w, y, dy) in enumerate(((q, wq, qo, dq_o), (k, wk, ko, dk_o))):
        e, size, dx, dx_size, dw, dw_size = _rope64(x, w, cos, sin, 1e-5, plus1, dy)
        b = ((d + 40) * U + angle) * size
        _within(y.detach(), e, b + v * (e.abs() + b) + 1e-38, f"y{i}")
        b = (3 * (d + 40) * U + angle) * dx_size
        _within(grads[i], dx, b + v * (dx.abs() + b) + 1e-38, f"dx{i}")
        if w is not None:
            n = math.prod(lead) * (H, KV)[i]
            b = ((3 * (d + 40) + min(n, 2048) + 64) * U + angle) * dw_size
            _within(grads[2 + i], dw, b + v * (dw.abs() + b) + 1e-38, f"dw{i}")


def test_rope_differences(gpu):
    """The gradients along a direction against the difference of the float64 formula's results."""
    from q38.hip import autograd
    q, k, wq, wk, inv, pos, am, dq_o, dk_o = _rope_inputs(gpu, (23,), 4, 2, 64, 32, torch.float32, 3)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, wq, wk)]
    grads = torch.autograd.grad(autograd.qk_norm_rope(*leaves, pos, inv, axes=am), leaves, (dq_o, dk_o))
    cos, sin = _turn(pos, inv, am)
    g = torch.Generator(device=gpu).manual_seed(5)
    for at in range(4):
        way = torch.randn(leaves[at].shape, generator=g, device=gpu).double()

        def value(t):
            moved = [x.double() for x in (q, k, wq, wk)]
            moved[at] = moved[at] + t * way
            y = [_rope64(moved[i], moved[2 + i], cos, sin, 1e-6, True)[0] for i in range(2)]
            return float((y[0] * dq_o.double()).sum() + (y[1] * dk_o.double()).sum())

        slope = (value(1e-4) - value(-1e-4)) / 2e-4
        got = float((grads[at].double() * way).sum())
        # The difference is off by t^2 of the third derivative (1e-8, times some tens); the gradients by 400 u of their terms.
        assert abs(slope - got) <= 3e-5 * float((grads[at].double() * way).abs().sum()), at


def test_rope_views_and_copies(gpu):
    """Queries beside their gates and heads of a fused projection are taken where they lie; rows off 16-byte boundaries and
    transposed heads are copied: the same bits."""
    from q38.hip import autograd
    q, k, wq, wk, inv, pos, _, dq_o, dk_o = _rope_inputs(gpu, (3, 50), 6, 2, 64, 16, torch.bfloat16, 0)
    want = autograd.qk_norm_rope(q, k, wq, wk, pos, inv)
    fused = torch.cat([q.reshape(3, 50, -1), k.reshape(3, 50, -1), q.reshape(3, 50, -1)], -1)
    ways = {
        "gate": (torch.cat([q, q], -1)[..., :64], k),
        "fused": (fused[..., :384].unflatten(-1, (6, 64)), fused[..., 384:512].unflatten(-1, (2, 64))),
        "odd": (torch.cat([q[..., :1], q], -1)[..., 1:], torch.cat([k[..., :1], k], -1)[..., 1:]),
        "heads first": (q.transpose(1, 2).contiguous().transpose(1, 2), k.transpose(1, 2).contiguous().transpose(1, 2)),
        "rows": (torch.cat([q, q], 1)[:, :50], torch.cat([k, k], 1)[:, :50]),
        "broadcast": (q[:, :, :1].expand(3, 50, 6, 64), k),
    }
    for name, (a, b) in ways.items():
        a, b = a.detach().requires_grad_(True), b.detach().requires_grad_(True)
        got = autograd.qk_norm_rope(a, b, wq, wk, pos, inv)
        da, db = torch.autograd.grad(got, (a, b), (dq_o, dk_o))
        x = q[:, :, :1].expand(3, 50, 6, 64).contiguous() if name == "broadcast" else q
        x, y = x.clone().requires_grad_(True), k.clone().requires_grad_(True)
        want = autograd.qk_norm_rope(x, y, wq, wk, pos, inv)
        wa, wb = torch.autograd.grad(want, (x, y), (dq_o, dk_o))
        for one, two in zip((*got, da, db), (*want, wa, wb)):
            assert torch.equal(one, two), name


def test_rope_axis_outside(gpu):
    """An axis that the positions lack makes what turns by it NaN, and nothing else."""
    from q38.hip import ops
    q, k, wq, wk, inv, pos, am, _, _ = _rope_inputs(gpu, (9,), 2, 1, 64, 32, torch.float32, 3)
    am = torch.zeros_like(am)
    want = ops.qk_norm_rope(q, k, wq, wk, pos, inv, axes=am)
    am[5], am[7] = 3, -1
    got = ops.qk_norm_rope(q, k, wq, wk, pos, inv, axes=am)
    hit = torch.zeros(64, dtype=torch.bool, device=gpu)
    hit[[5, 7, 21, 23]] = True
    for a, b in zip(got, want):
        assert bool(a[..., hit].isnan().all()) and torch.equal(a[..., ~hit], b[..., ~hit])


# ---- linear attention -------------------------------------------------------------------------

def _sum64(q, k, v, g, S0, intra, inter, gain, lag):
    """One sequence, heads first [H,S,.], chunk by chunk: results, their sizes as rounded, their sizes with every term
    positive, the last state and its terms' sizes."""
    q, k, v, g = q.double(), k.double(), v.double(), g.double()[:, None, None]
    H, S, dk = q.shape
    dv = v.shape[-1]
    state = torch.zeros(H, dk, dv, dtype=torch.float64, device=q.device) if S0 is None else S0.double().clone()
    size = state.abs()
    out, rounded, terms = [], [], []
    for j0 in range(0, S, 64):
        a, b, c = q[:, j0:j0 + 64], k[:, j0:j0 + 64], v[:, j0:j0 + 64]
        n = a.shape[1]
        at = torch.arange(n, device=q.device)
        gap = at[:, None] - at[None, :]
        decay = torch.where(gap >= 0, torch.exp(g * gap.clamp(min=0)), torch.zeros((), dtype=torch.float64, device=q.device))
        s = (a @ b.transpose(1, 2)) * decay * intra
        read = torch.exp(g * (at[:, None] + 1 - lag)) * inter
        out.append(s @ c + read * (a @ state))
        rounded.append(s.abs() @ c.abs() + read.abs() * (a.abs() @ state.abs()))
        terms.append((a.abs() @ b.abs().transpose(1, 2) * decay * abs(intra)) @ c.abs() + read.abs() * (a.abs() @ size))
        put = torch.exp(g * (n - 1 - at[:, None] + lag)) * gain
        state = torch.exp(g * n) * state + (b * put).transpose(1, 2) @ c
        size = torch.exp(g * n) * size + (b.abs() * put.abs()).transpose(1, 2) @ c.abs()
    cat = lambda t, d: torch.cat(t, 1) if t else torch.zeros(H, 0, d, dtype=torch.float64, device=q.device)  # noqa: E731
    return cat(out, dv), cat(rounded, dv), cat(terms, dv), state, size


def _check(got, want, dtype, dk, name, group=1):
    """got [S,H/group,d] against _sum64's (out, rounded, terms) [H,S,d]."""
    out, rounded, terms = want
    H, S, d = out.shape
    v = torch.finfo(dtype).eps / 2
    n = 2 * (dk + 64 + S / 64 + 20 + group) * U
    bound = n * terms + (v * rounded * (1 + v) if dtype == torch.bfloat16 else 0)
    out, bound = (t.view(H // group, group, S, d).sum(1).transpose(0, 1) for t in (out, bound))
    _within(got, out, bound + v * (out.abs() + bound) + 1e-37, name)


def _check_state(got, state, size, dk, S, name):
    _within(got, state, 2 * (64 + S / 64 + 20) * U * size + 1e-37, name)


def _mix_inputs(dev, B, S, H, Hk, dk, dv, dtype, N=None, state=True, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed + S + 7 * dk + H)
    q, k, v = (_randn(g, B, S, h, d, dtype=dtype) for h, d in ((H, dk), (Hk, dk), (Hk, dv)))
    decay = -torch.rand(H, generator=g, device=dev) * torch.tensor([1.0, 0.1, 0.01, 1e-4], device=dev).repeat(-(-H // 4))[:H]
    decay[0] = 0.0  # one head that forgets nothing
    S0 = _randn(g, N or B, H, dk, dv) if state else None
    return q, k, v, decay, S0, _randn(g, B, S, H, dv, dtype=dtype), _randn(g, N or B, H, dk, dv)


def _heads(t, G=1):
    return t.transpose(0, 1).repeat_interleave(G, 0)


def _check_sequence(dtype, scale, q, k, v, g, S0, do, dS, got):
    """One sequence's tensors [S,.,.] and what the call gave for it: out, state, dq, dk, dv, ds."""
    S, H, dk = q.shape
    Hk, dv = v.shape[1:]
    G = H // Hk
    a, b, c = _heads(q), _heads(k, G), _heads(v, G)
    *want, state, size = _sum64(a, b, c, g, S0, scale, scale, 1.0, 0)
    _check(got["out"], want, dtype, dk, "out")
    _check_state(got["state"], state, size, dk, S, "state")
    if "dq" not in got:
        return
    d = _heads(do)
    t = lambda x: None if x is None else x.transpose(-1, -2)  # noqa: E731
    _check(got["dq"], _sum64(d, c, b, g, t(S0), scale, scale, 1.0, 0)[:3], dtype, dv, "dq")
    a, b, c, d = (x.flip(1) for x in (a, b, c, d))
    *want, _, _ = _sum64(c, d, a, g, t(dS), scale, 1.0, scale, 1)
    _check(got["dk"].flip(0), want, dtype, dv, "dk", G)
    *want, ds, size = _sum64(b, a, d, g, dS, scale, 1.0, scale, 1)
    _check(got["dv"].flip(0), want, dtype, dk, "dv", G)
    if S0 is not None:
        _check_state(got["ds"], ds, size, dk, S, "ds")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,S,H,Hk,dk,dv,state", [
    (1, 1, 1, 1, 64, 64, True),
    (2, 2, 4, 2, 8, 8, True),
    (1, 63, 2, 1, 128, 128, True),
    (3, 64, 2, 2, 64, 128, False),
    (1, 65, 4, 4, 128, 64, True),
    (2, 130, 5, 1, 48, 80, True),
    (1, 511, 3, 3, 96, 104, True),
    (1, 513, 2, 2, 128, 128, True),   # two segments, one token in the second
    (2, 1600, 4, 2, 64, 64, False),
    (1, 1777, 3, 1, 128, 128, True),
    (2, 0, 3, 1, 64, 64, True),
])
def test_linear_attention(gpu, dtype, B, S, H, Hk, dk, dv, state):
    from q38.hip import autograd
    print(f"linear attention {dtype} B={B} S={S} H={H} Hk={Hk} dk={dk} dv={dv} state={state}", flush=True)
    q, k, v, g, S0, do, dS = _mix_inputs(gpu, B, S, H, Hk, dk, dv, dtype, state=state)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v, S0) if t is not None]
    out, last = autograd.linear_attention(*leaves[:3], g, initial_state=leaves[3] if state else None, return_state=True)
    grads = torch.autograd.grad((out, last), leaves, (do, dS))
    with torch.no_grad():
        alone, none = autograd.linear_attention(q, k, v, g, initial_state=S0)
    torch.cuda.synchronize()
    assert none is None and torch.equal(alone, out)
    for b in range(B):
        got = dict(out=out[b].detach(), state=last[b].detach(), dq=grads[0][b], dk=grads[1][b], dv=grads[2][b])
        if state:
            got["ds"] = grads[3][b]
        _check_sequence(dtype, dk ** -0.5, q[b], k[b], v[b], g, S0[b] if state else None, do[b], dS[b], got)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens,tail,H,Hk,dk,dv,state", [
    ([1], 0, 2, 1, 64, 64, True),
    ([0, 5, 0, 64, 1, 0], 0, 4, 2, 64, 64, True),
    ([100, 600, 3, 64, 700], 37, 3, 3, 128, 128, True),
    ([65] * 40, 5, 2, 2, 48, 64, False),
    ([1] * 1500 + [300], 0, 1, 1, 64, 64, True),   # more sequences than one round of the plan holds
])
def test_linear_attention_packed(gpu, dtype, lens, tail, H, Hk, dk, dv, state):
    """Sequences of one row; tokens behind the last one come out zero, in the gradients too."""
    from q38.hip import autograd
    S, N = sum(lens) + tail, len(lens)
    print(f"packed {dtype} N={N} S={S} H={H} dk={dk} dv={dv}", flush=True)
    q, k, v, g, S0, do, dS = _mix_inputs(gpu, 1, S, H, Hk, dk, dv, dtype, N=N, state=state)
    if tail:
        for t in (q, k, v, do):
            t[:, S - tail:] = float("nan")
    cu = torch.tensor([0] + lens, dtype=torch.int32).cumsum(0).int().to(gpu)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v, S0) if t is not None]
    out, last = autograd.linear_attention(*leaves[:3], g, scale=0.3, initial_state=leaves[3] if state else None, cu_seqlens=cu,
                                          return_state=True)
    grads = torch.autograd.grad((out, last), leaves, (do, dS))
    torch.cuda.synchronize()
    if tail:
        for t in (out, *grads[:3]):
            assert not bool(t[:, S - tail:].any())
    at = cu.tolist()
    for n in range(N) if N < 100 else [0, 1, 700, N - 2, N - 1]:
        r = slice(at[n], at[n + 1])
        got = dict(out=out[0, r].detach(), state=last[n].detach(), dq=grads[0][0, r], dk=grads[1][0, r], dv=grads[2][0, r])
        if state:
            got["ds"] = grads[3][n]
        _check_sequence(dtype, 0.3, q[0, r], k[0, r], v[0, r], g, S0[n] if state else None, do[0, r], dS[n], got)


# Many heads make segments of several chunks: of the 256 CUs each has few of a head's.
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,S,H,Hk,dk,dv", [(1, 1500, 128, 64, 128, 128), (2, 2049, 64, 64, 64, 64), (1, 777, 96, 96, 64, 128),
                                            (1, 1100, 64, 16, 128, 64)])
def test_linear_attention_of_many_heads(gpu, dtype, B, S, H, Hk, dk, dv):
    print(f"many heads {dtype} B={B} S={S} H={H} Hk={Hk} dk={dk} dv={dv}", flush=True)
    test_linear_attention(gpu, dtype, B, S, H, Hk, dk, dv, True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens,tail,H,Hk,dk,dv", [
    ([700, 0, 1, 640, 65, 2], 9, 128, 128, 128, 128),                    # few sequences, and the rule for
    ([3, 900, 1, 128, 0, 257] + [31] * 20 + [384], 0, 96, 48, 64, 64),   # more of them than the CUs need
])
def test_linear_attention_packed_of_many_heads(gpu, dtype, lens, tail, H, Hk, dk, dv):
    test_linear_attention_packed(gpu, dtype, lens, tail, H, Hk, dk, dv, True)


def test_linear_attention_offsets_out_of_order(gpu):
    """Offsets past the row or out of order are brought in: each sequence what lies between the largest offset so far and the
    next, within the row; the rest zeros."""
    from q38.hip import ops
    q, k, v, g, _, _, _ = _mix_inputs(gpu, 1, 200, 2, 2, 64, 64, torch.float32)
    bad = torch.tensor([10, 90, 40, 150, 900], dtype=torch.int32, device=gpu)
    good = torch.tensor([10, 90, 90, 150, 200], dtype=torch.int32, device=gpu)
    a, s = ops.linear_attention(q, k, v, g, cu_seqlens=bad, return_state=True)
    b, t = ops.linear_attention(q, k, v, g, cu_seqlens=good, return_state=True)
    assert torch.equal(a, b) and torch.equal(s, t) and not bool(a[:, :10].any()) and not bool(s[1].any())
    c, _ = ops.linear_attention(q[:, 10:90], k[:, 10:90], v[:, 10:90], g)
    assert torch.equal(c, b[:, 10:90])


def test_linear_attention_differences(gpu):
    """The gradients along a direction against the difference of the float64 sums' results."""
    from q38.hip import autograd
    q, k, v, g, S0, do, dS = _mix_inputs(gpu, 1, 100, 4, 2, 64, 64, torch.float32)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v, S0)]
    out, last = autograd.linear_attention(*leaves[:3], g, initial_state=leaves[3], return_state=True)
    grads = torch.autograd.grad((out, last), leaves, (do, dS))
    r = torch.Generator(device=gpu).manual_seed(5)
    for at in range(4):
        way = torch.randn(leaves[at].shape, generator=r, device=gpu).double()

        def value(t):
            a, b, c, s = (x.double() + (t * way if i == at else 0.0) for i, x in enumerate((q, k, v, S0)))
            o, _, _, end, _ = _sum64(_heads(a[0]), _heads(b[0], 2), _heads(c[0], 2), g, s[0], 0.125, 0.125, 1.0, 0)
            return float((o.transpose(0, 1) * do[0].double()).sum() + (end * dS[0].double()).sum())

        # Linear in each operand: the difference is exact up to float64 roundings. The gradients are off by 320 u of their
        # terms' sizes, about (64 * 100)^1/2 times their own: random products of 64, random sums of 100.
        slope = (value(1.0) - value(-1.0)) / 2.0
        got = (grads[at].double() * way)
        assert abs(slope - float(got.sum())) <= 80 * 320 * U * float(got.abs().sum()), at


def test_linear_attention_views(gpu):
    """Heads of a fused projection, heads first, broadcast values: the same bits as contiguous copies, and their gradients."""
    from q38.hip import autograd
    q, k, v, g, S0, do, _ = _mix_inputs(gpu, 2, 100, 4, 2, 64, 64, torch.bfloat16)
    fused = torch.cat([t.reshape(2, 100, -1) for t in (q, k, v)], -1)
    ways = {
        "fused": (fused[..., :256].unflatten(-1, (4, 64)), fused[..., 256:384].unflatten(-1, (2, 64)),
                  fused[..., 384:].unflatten(-1, (2, 64))),
        "heads first": tuple(t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)),
        "odd": tuple(torch.cat([t[..., :1], t], -1)[..., 1:] for t in (q, k, v)),
        "broadcast": (q, k[:, :1].expand(2, 100, 2, 64), v[:, :, :1].expand(2, 100, 2, 64)),
    }
    for name, ops3 in ways.items():
        a = [t.detach().requires_grad_(True) for t in ops3]
        b = [t.detach().clone(memory_format=torch.contiguous_format).requires_grad_(True) for t in ops3]
        outs = [autograd.linear_attention(*x, g, initial_state=S0)[0] for x in (a, b)]
        assert torch.equal(*outs), name
        for one, two in zip(*(torch.autograd.grad(o, x, do) for o, x in zip(outs, (a, b)))):
            assert torch.equal(one, two), name


def test_linear_attention_partial_gradients(gpu):
    """Only the state's gradient given, only some operands asked for."""
    from q38.hip import autograd
    q, k, v, g, S0, do, dS = _mix_inputs(gpu, 2, 70, 2, 1, 64, 64, torch.float32)
    full = [t.clone().requires_grad_(True) for t in (q, k, v, S0)]
    out, last = autograd.linear_attention(*full[:3], g, initial_state=full[3], return_state=True)
    want = torch.autograd.grad((out, last), full, (torch.zeros_like(do), dS))
    out, last = autograd.linear_attention(*full[:3], g, initial_state=full[3], return_state=True)
    for a, b in zip(torch.autograd.grad(last, full, dS, allow_unused=True), want):
        assert torch.equal(a, b)
    kk = k.clone().requires_grad_(True)
    out, _ = autograd.linear_attention(q, kk, v, g, initial_state=S0)
    (a,) = torch.autograd.grad(out, kk, do)
    out, last = autograd.linear_attention(*full[:3], g, initial_state=full[3], return_state=True)
    assert torch.equal(a, torch.autograd.grad(out, full[1], do)[0])


# ---- the step, and all of it together ---------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,H,Hk,dk,dv,pool", [(1, 1, 1, 64, 64, 0), (5, 4, 2, 128, 128, 9), (3, 6, 1, 8, 104, 0),
                                               (61, 3, 3, 96, 40, 100), (0, 2, 2, 64, 64, 3)])
def test_step(gpu, dtype, B, H, Hk, dk, dv, pool):
    """Against float64: the state is two products and a sum (3 u of its terms), the output a sum of dk of its products; a slot
    outside the pool updates nothing and gives zero; states that no slot names keep their bits."""
    from q38.hip import ops
    r = torch.Generator(device=gpu).manual_seed(B + dk)
    q, k, v = (_randn(r, B, h, d, dtype=dtype) for h, d in ((H, dk), (Hk, dk), (Hk, dv)))
    state = _randn(r, pool or B, H, dk, dv)
    g = -torch.rand(H, generator=r, device=gpu)
    slots = torch.randperm(pool, generator=r, device=gpu)[:B].int() if pool else None
    if pool and B > 3:
        slots[1], slots[3] = -1, pool
    before = state.clone()
    out = ops.linear_attention_step(q, k, v, state, g, slots=slots)
    torch.cuda.synchronize()
    rows = list(range(B)) if slots is None else slots.tolist()
    kept = [n for n in range(state.shape[0]) if n not in rows]
    assert torch.equal(state[kept], before[kept])
    lam, vh = torch.exp(g.double())[:, None, None], torch.finfo(dtype).eps / 2
    for b, row in enumerate(rows):
        if not 0 <= row < state.shape[0]:
            assert not bool(out[b].any())
            continue
        kk, vv = (t[b].double().repeat_interleave(H // Hk, 0) for t in (k, v))
        add = kk[:, :, None] * vv[:, None, :]
        new, size = lam * before[row].double() + add, lam * before[row].double().abs() + add.abs()
        _within(state[row], new, 4 * U * size + 1e-37, "state")
        qq = q[b].double()[:, :, None]
        o = (qq * new).sum(1) * dk ** -0.5
        e = (dk + 12) * U * (qq.abs() * size).sum(1) * dk ** -0.5
        _within(out[b], o, e + vh * (o.abs() + e) + 1e-37, "out")


@pytest.mark.parametrize("B,again", [(2, (0, 1)), (301, (3, 300)), (301, (12, 13))])
def test_step_with_a_slot_twice(gpu, B, again):
    """The sequence that names a slot first has it; the other gets zero, and nothing else changes: bits as without the other."""
    from q38.hip import ops
    r = torch.Generator(device=gpu).manual_seed(B)
    q, k, v = (_randn(r, B, 2, 64, dtype=torch.bfloat16) for _ in range(3))
    state = _randn(r, B + 4, 2, 64, 64)
    g = -torch.rand(2, generator=r, device=gpu)
    slots = torch.randperm(B + 4, generator=r, device=gpu)[:B].int()
    twice, without = slots.clone(), slots.clone()
    twice[again[1]], without[again[1]] = slots[again[0]], -1
    a, b = state.clone(), state.clone()
    assert torch.equal(ops.linear_attention_step(q, k, v, a, g, slots=twice),
                       ops.linear_attention_step(q, k, v, b, g, slots=without))
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_prompt_then_tokens(gpu, dtype):
    """As they are used: a fused projection's heads normed and rotated, the prompts through linear attention, then token by token
    with the states in a pool; every output against float64 on the normed heads that the run had, over the whole length."""
    from q38.hip import autograd, ops
    B, S, more, H, Hk, d = 3, 150, 6, 4, 2, 64
    r = torch.Generator(device=gpu).manual_seed(3)
    qkv = _randn(r, B, S + more, (H + 2 * Hk) * d, dtype=dtype)
    wq, wk = _randn(r, d, std=0.1, dtype=dtype), _randn(r, d, std=0.1, dtype=dtype)
    inv = (1e4 ** (-torch.arange(0, 32, 2) / 32)).to(gpu)
    axes = ops.rope_axis_map([6, 5, 5], device=gpu)
    pos = torch.arange(S + more, device=gpu).expand(3, B, S + more).contiguous()
    g = -torch.rand(H, generator=r, device=gpu) * 0.1
    pool = _randn(r, 8, H, d, d)
    slots = torch.tensor([6, 0, 3], dtype=torch.int32, device=gpu)
    before = pool.clone()

    def heads(at):
        x = qkv[:, at]
        q, k, v = (x[..., a * d:b * d].unflatten(-1, (b - a, d)) for a, b in ((0, H), (H, H + Hk), (H + Hk, H + 2 * Hk)))
        return (*autograd.qk_norm_rope(q, k, wq, wk, pos[:, :, at], inv, axes=axes), v)

    q, k, v = heads(slice(0, S))
    out, last = autograd.linear_attention(q, k, v, g, return_state=True)
    pool[slots.long()] = last
    seen, outs = [(q, k, v)], [out]
    for t in range(S, S + more):
        q, k, v = heads(slice(t, t + 1))
        seen.append((q, k, v))
        outs.append(ops.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], pool, g, slots=slots)[:, None])
    torch.cuda.synchronize()
    q, k, v = (torch.cat([s[i] for s in seen], 1) for i in range(3))
    out = torch.cat(outs, 1)
    for b in range(B):
        got = dict(out=out[b], state=pool[int(slots[b])])
        _check_sequence(dtype, d ** -0.5, q[b], k[b], v[b], g, None, None, None, got)
    kept = [1, 2, 4, 5, 7]
    assert torch.equal(pool[kept], before[kept])


def test_captured_and_replayed(gpu):
    """The whole of it in a graph, forward, backward and a step: every replay the eager result, with eager work in between."""
    from q38.hip import autograd, ops
    H, Hk, d, S = 4, 2, 64, 700
    r = torch.Generator(device=gpu).manual_seed(3)
    q0, k0, v0 = (_randn(r, 1, S, h, d, dtype=torch.bfloat16).requires_grad_(True) for h in (H, Hk, Hk))
    wq, wk = (_randn(r, d, std=0.1, dtype=torch.bfloat16).requires_grad_(True) for _ in range(2))
    inv = (1e4 ** (-torch.arange(0, 16, 2) / 16)).to(gpu)
    pos = torch.arange(S, device=gpu)[None]
    g = -torch.rand(H, generator=r, device=gpu) * 0.1
    cu = torch.tensor([0, 3, 600, S], dtype=torch.int32, device=gpu)
    do = _randn(r, 1, S, H, d, dtype=torch.bfloat16)
    pool = torch.zeros(3, H, d, d, device=gpu)

    def run():
        q, k = autograd.qk_norm_rope(q0, k0, wq, wk, pos, inv)
        out, last = autograd.linear_attention(q, k, v0, g, cu_seqlens=cu, return_state=True)
        grads = torch.autograd.grad(out, (q0, k0, v0, wq, wk), do)
        pool.copy_(last.detach())
        step = ops.linear_attention_step(q[0, :3].detach(), k[0, :3].detach(), v0[0, :3].detach(), pool, g)
        return (out.detach(), last.detach(), step, pool, *grads)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for i in range(4):
        with torch.no_grad():
            for t in (q0, k0, v0):
                t.copy_(_randn(r, *t.shape, dtype=torch.bfloat16))
        cu.copy_(torch.tensor([0, 3 + 50 * i, 600, S - i], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        want = run()
        torch.cuda.synchronize()
        for n, (a, b) in enumerate(zip(got, want)):
            assert torch.equal(a, b), (i, n)


def test_two_streams(gpu):
    """Two calls at once on streams of their own give what each gives alone."""
    from q38.hip import autograd
    cases = []
    for seed in range(2):
        q, k, v, g, S0, do, _ = _mix_inputs(gpu, 2, 900, 4, 2, 64, 64, torch.bfloat16, seed=seed)
        cases.append(([t.requires_grad_(True) for t in (q, k, v)], g, S0, do))

    def run(c):
        out, last = autograd.linear_attention(*c[0], c[1], initial_state=c[2], return_state=True)
        return (out.detach(), last.detach(), *torch.autograd.grad(out, c[0], c[3]))

    want = [run(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run(cases[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for one in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(one, want[i]))


def test_gradients_are_taken_once(gpu):
    """With create_graph the gradients are the same bits and have no gradient themselves; forward-mode tangents are refused."""
    from q38.hip import autograd
    q, k, v, g, _, do, _ = _mix_inputs(gpu, 1, 70, 2, 2, 64, 64, torch.float32, state=False)
    pos, inv = torch.arange(70, device=gpu)[None], torch.rand(8, device=gpu)
    for call in (lambda q, k: autograd.qk_norm_rope(q, k, None, None, pos, inv)[0],
                 lambda q, k: autograd.linear_attention(q, k, v, g)[0]):
        leaves = [t.clone().requires_grad_(True) for t in (q, k)]
        once = torch.autograd.grad(call(*leaves), leaves, do)
        twice = torch.autograd.grad(call(*leaves), leaves, do, create_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(once, twice))
        with pytest.raises(RuntimeError):  # no graph of them
            torch.autograd.grad(twice[0].sum(), leaves, allow_unused=True)
        with torch.autograd.forward_ad.dual_level(), pytest.raises(RuntimeError):
            call(torch.autograd.forward_ad.make_dual(q, torch.ones_like(q)), k)


def test_saved_tensors_that_were_moved(gpu):
    """Under hooks that keep saved tensors elsewhere (other places and strides in the backward pass): the same bits."""
    from q38.hip import autograd
    g = torch.Generator(device=gpu).manual_seed(9)
    fused = _randn(g, 2, 100, 4 + 2 + 2, 64, dtype=torch.bfloat16)
    w = _randn(g, 2, 64, dtype=torch.bfloat16)
    pos, inv = torch.arange(100, device=gpu).repeat(2, 1), torch.rand(8, generator=g, device=gpu)
    decay = -torch.rand(4, generator=g, device=gpu)

    def run():
        x = fused.clone().requires_grad_(True)
        wq, wk = (t.clone().requires_grad_(True) for t in w)
        q, k = autograd.qk_norm_rope(x[..., :4, :], x[..., 4:6, :], wq, wk, pos, inv)
        out, _ = autograd.linear_attention(q, k, x[..., 6:, :], decay)
        return out, lambda: torch.autograd.grad(out, (x, wq, wk), torch.ones_like(out))

    want, grads = run()
    want = want, *grads()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (t.device, t.cpu()), lambda kept: kept[1].to(kept[0])):
        got, grads = run()
        junk = [_randn(g, 2, 100, n, 64, dtype=torch.bfloat16) for n in (2, 4, 8)]
        got = got, *grads()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    del junk


def test_autocast(gpu):
    from q38.hip import autograd
    q, k, v, g, _, do, _ = _mix_inputs(gpu, 1, 40, 2, 2, 64, 64, torch.float32)
    w = torch.zeros(64, device=gpu)
    inv, pos = torch.ones(8, device=gpu), torch.arange(40, device=gpu)[None]
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        a, b = autograd.qk_norm_rope(leaves[0], leaves[1], w, w, pos, inv)
        out, _ = autograd.linear_attention(a, b, leaves[2], g)
    assert a.dtype == b.dtype == out.dtype == torch.bfloat16
    grads = torch.autograd.grad(out, leaves, do.bfloat16())
    assert all(t.dtype == torch.float32 and bool(t.isfinite().all()) for t in grads)


# ---- values that are not finite, long offsets, other devices' streams -------------------------

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("dk,dv,S,H,Hk,places", [
    (64, 64, 200, 4, 2, (0, 15, 16, 77, 100, 127, 128, 199)), (128, 128, 200, 4, 2, (0, 15, 16, 77, 100, 127, 128, 199)),
    (64, 128, 200, 4, 2, (0, 15, 16, 77, 100, 127, 128, 199)), (128, 128, 700, 128, 64, (1, 130, 463)),
    (64, 64, 700, 128, 128, (77, 300))])   # many heads: segments of several chunks
def test_nothing_reaches_back(gpu, dtype, bad, dk, dv, S, H, Hk, places):
    """A NaN or infinity at a token changes no bit of what earlier tokens give, in its own chunk neither, and in the gradients of
    no later one; a value's stays in its column."""
    from q38.hip import autograd
    q, k, v, g, S0, do, _ = _mix_inputs(gpu, 1, S, H, Hk, dk, dv, dtype)

    def run(q, k, v, do):
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
        out, last = autograd.linear_attention(*leaves, g, initial_state=S0, return_state=True)
        return (out.detach(), last.detach(), *torch.autograd.grad(out, leaves, do))

    clean = run(q, k, v, do)
    for at in places:
        for i, name in enumerate("qkv"):
            ins = [t.clone() for t in (q, k, v)]
            ins[i][0, at, -1, 3] = bad  # of the last head
            got = run(*ins, do)
            before = got[0][:, :at], clean[0][:, :at]
            assert torch.equal(*before), (name, at)
            assert torch.equal(got[0][:, :, :1], clean[0][:, :, :1]), (name, at)  # another head
            if name == "q":
                assert torch.equal(got[0][:, at + 1:], clean[0][:, at + 1:]) and torch.equal(got[1], clean[1])
            if name == "v":
                rest = [c for c in range(dv) if c != 3]
                assert torch.equal(got[0][..., rest], clean[0][..., rest]) and torch.equal(got[1][..., rest], clean[1][..., rest])
                assert not bool(got[0][0, at, -1, 3].isfinite())
        d = do.clone()
        d[0, at, -1, 5] = bad
        got = run(q, k, v, d)
        assert torch.equal(got[2][:, :at], clean[2][:, :at]), at               # dq: its own token and the ones behind none
        assert torch.equal(got[2][:, at + 1:], clean[2][:, at + 1:]), at
        for j in (3, 4):                                                       # dk, dv: tokens at or before it
            assert torch.equal(got[j][:, at + 1:], clean[j][:, at + 1:]), (j, at)
        assert not bool(got[4][0, at, -1].isfinite().all())


def test_decays_at_the_ends(gpu):
    """log_decay 0 forgets nothing, -inf all but the token itself, -200 nearly so (e^-200 is a float's zero)."""
    from q38.hip import autograd, ops
    q, k, v, _, S0, _, _ = _mix_inputs(gpu, 1, 150, 4, 4, 64, 64, torch.float32)
    g = torch.tensor([0.0, float("-inf"), -200.0, -1e-7], device=gpu)
    out, last = autograd.linear_attention(q, k, v, g, initial_state=S0, return_state=True)
    own = (q * k).sum(-1, keepdim=True) * v / 8.0
    for h in (1, 2):
        torch.testing.assert_close(out[:, :, h], own[:, :, h], rtol=1e-5, atol=1e-5)
        torch.testing.assert_close(last[0, h], k[0, -1, h][:, None] * v[0, -1, h][None], rtol=1e-6, atol=1e-6)
    for h in (0, 3):
        *want, state, size = _sum64(_heads(q[0])[h:h + 1], _heads(k[0])[h:h + 1], _heads(v[0])[h:h + 1], g[h:h + 1],
                                    S0[0, h:h + 1], 0.125, 0.125, 1.0, 0)
        _check(out[0, :, h:h + 1], want, torch.float32, 64, f"head {h}")
        _check_state(last[0, h:h + 1], state, size, 64, 150, f"state {h}")
    state = S0.clone()
    o = ops.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], state, g)
    torch.testing.assert_close(o, out[:, 0], rtol=1e-5, atol=1e-5)


def test_slow_decay_over_a_long_sequence(gpu):
    """A decay of 1e-5 over 40000 tokens: the state remembers all of them, and is as near to float64 as sums of that many terms
    in fp32 are (64-token sums, one rounded decay a chunk: errors of both signs, so 16 u (n)^1/2 of the terms' size and
    not n u)."""
    from q38.hip import ops
    S = 40000
    q, k, v, _, _, _, _ = _mix_inputs(gpu, 1, S, 2, 2, 64, 64, torch.bfloat16, state=False)
    k, v = k.abs(), v.abs()  # no cancellation: a decay that is off in one direction would show
    g = torch.tensor([-1e-5, -3e-6], device=gpu)
    _, last = ops.linear_attention(q, k, v, g, return_state=True)
    w = torch.exp(g.double()[:, None] * torch.arange(S - 1, -1, -1, device=gpu).double())
    exact = torch.stack([(k[0, :, h].double() * w[h][:, None]).t().contiguous() @ v[0, :, h].double() for h in range(2)])
    err = float(((last[0].double() - exact) / exact).abs().max())
    assert err <= 16 * U * math.sqrt(S / 64), err


def test_offsets_past_32_bits(gpu):
    """Tokens 2^25 elements apart (5 GB from the first to the last), and outputs of more than 2^31 elements."""
    from q38.hip import ops
    far = torch.empty(70 << 25, dtype=torch.bfloat16, device=gpu)
    q, k, v, g, S0, _, _ = _mix_inputs(gpu, 1, 70, 2, 1, 64, 64, torch.bfloat16)
    parts = []
    for i, t in enumerate((q, k, v)):
        x = far.as_strided(t.shape, (0, 1 << 25, 64, 1), 256 * i)
        x.copy_(t)
        parts.append(x)
    for a, b in zip(ops.linear_attention(*parts, g, initial_state=S0, return_state=True),
                    ops.linear_attention(q, k, v, g, initial_state=S0, return_state=True)):
        assert torch.equal(a, b)
    w, inv, pos = torch.zeros(64, dtype=torch.bfloat16, device=gpu), torch.ones(8, device=gpu), torch.arange(70, device=gpu)
    for a, b in zip(ops.qk_norm_rope(parts[0][0], parts[1][0], w, w, pos, inv), ops.qk_norm_rope(q[0], k[0], w, w, pos, inv)):
        assert torch.equal(a, b)
    del far, parts
    T, H = (1 << 20) + 70, 32
    r = torch.Generator(device=gpu).manual_seed(1)
    q = torch.empty(T, H, 64, dtype=torch.bfloat16, device=gpu)
    q[-70:] = _randn(r, 70, H, 64, dtype=torch.bfloat16)
    q[:-70] = 0
    k = _randn(r, T, 1, 64, dtype=torch.bfloat16)
    pos = torch.arange(T, device=gpu)
    qo, ko = ops.qk_norm_rope(q, k, w, w, pos, inv)
    a, b = ops.qk_norm_rope(q[-70:], k[-70:], w, w, pos[-70:].contiguous(), inv)
    assert torch.equal(qo[-70:], a) and torch.equal(ko[-70:], b)
    del qo
    g = torch.full((H,), -0.5, device=gpu)
    out, last = ops.linear_attention(q[None], k[None], k[None], g, return_state=True)
    # e^-35 of what is before the last 70 tokens is left at their end, e^-0.5 .. at their start: from the state of the 500 before.
    _, S0 = ops.linear_attention(q[None, -570:-70], k[None, -570:-70], k[None, -570:-70], g, return_state=True)
    x = _heads(k[-70:], H)
    *want, state, size = _sum64(_heads(q[-70:]), x, x, g, S0[0], 0.125, 0.125, 1.0, 0)
    # The call's chunks lie otherwise than the reference's: a score rounded there is a state rounded here, of the same size.
    outs, rounded, terms = want
    bound = 2 * (64 + 64 + 20) * U * terms + 2.0 ** -8 * (terms + outs.abs()) * 1.01
    _within(out[0, -70:], outs.transpose(0, 1), bound.transpose(0, 1), "out")
    _check_state(last[0], state, size, 64, 570, "state")


def test_current_device_is_not_needed(gpu):
    """Tensors that another stream made are used in that order on the current one; a call inside torch.inference_mode."""
    from q38.hip import autograd, ops
    q, k, v, g, S0, _, _ = _mix_inputs(gpu, 1, 90, 2, 2, 64, 64, torch.bfloat16)
    want = ops.linear_attention(q, k, v, g, initial_state=S0)[0]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s), torch.inference_mode():
        q2, k2, v2 = q * 1, k * 1, v * 1
        got = autograd.linear_attention(q2, k2, v2, g, initial_state=S0)[0]
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)

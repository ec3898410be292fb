"""Timing cases of a token mixer with a carried state: its queries and keys normed and rotated, linear attention with a
decay for each head over prompts and in training, and its step for single tokens.

* ``rope``: ``autograd.qk_norm_rope``, the RMS norms of every query and key head and their rotation by position, on one axis
  of positions or on three (time, height, width). Forward alone (serving), or with every gradient.
* ``mix``: ``autograd.linear_attention``, S_t = e^g S_{t-1} + k_t v_t^T and o_t = scale S_t^T q_t for each head, over whole
  sequences or packed ones, with the state carried in and out. Forward alone (prompts), or with every gradient.
* ``step``: ``ops.linear_attention_step``, the same for one token of every sequence, the states updated in place in a
  pool that holds more sequences than the batch.

Shapes are the model's own (38 query and 2 key heads of 64, of which 16 features rotate; 13 key and 39 value heads of 64;
4 x 4096 tokens) and generic ones next to them (16 heads of 128; 256-wide heads). Outside ``own`` every operator runs in its
plain form: elementary torch operations in fp32, angles in float64, rounded once. ``exact`` restates them in float64, the
mixer token by token.
"""
import math
import sys
from pathlib import Path

import torch

own = False

_PKG = str(Path(__file__).resolve().parents[1] / "qwen35-moe-sparse_amd")
_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
_EPS = 1e-6
_THETA = 1e7


def _rope(name, T, H, KV, d, rot, dtype="bf16", train=False, axes=1, far=4096):
    case = dict(kind="rope", T=T, H=H, KV=KV, d=d, rot=rot, dtype=dtype, train=train, axes=axes, far=far)
    return dict(case, name=name) if name else case


def _mix(name, B, S, H, Hk, dk, dv, dtype="bf16", train=False, packed=0, state=False):
    """packed: 0, or the number of ragged sequences that the S tokens of one row hold; state: carried in and out."""
    case = dict(kind="mix", B=B, S=S, H=H, Hk=Hk, dk=dk, dv=dv, dtype=dtype, train=train, packed=packed, state=state)
    return dict(case, name=name) if name else case


def _step(name, B, H, Hk, dk, dv, dtype="bf16", pool=0):
    case = dict(kind="step", B=B, H=H, Hk=Hk, dk=dk, dv=dv, dtype=dtype, pool=pool)
    return dict(case, name=name) if name else case


def listed():
    return [
        # One decode step of 61 sequences, each at a far position of its own: latency.
        _rope("rope_decode_61", 61, 38, 2, 64, 16, far=131072),
        # The training step at the headline size, the model's own heads.
        _rope("rope_train_16384", 16384, 38, 2, 64, 16, train=True),
        # Images and video between text: three axes, wide heads, a ragged prompt.
        _rope("rope_axes_4097", 4097, 16, 2, 256, 64, axes=3),
        # An fp32 model's fine-tuning step.
        _rope("rope_fp32_515", 515, 38, 2, 64, 16, dtype="fp32", train=True),
        # One short prompt, whose state the steps go on from.
        _mix("prompt_777", 1, 777, 16, 16, 128, 128, state=True),
        # Prompts of many requests packed into one row, some of which go on from a state.
        _mix("packed_8191", 1, 8191, 16, 16, 128, 128, packed=23, state=True),
        # One very long prompt: few heads, all of the length to split.
        _mix("long_65536", 1, 65536, 16, 16, 128, 128, state=True),
        # The training step at the headline size.
        _mix("train_16384", 4, 4096, 16, 16, 128, 128, train=True),
        # The model's own head layout (39 heads that share 13), an odd length.
        _mix("grouped_2049", 2, 2049, 39, 13, 64, 64, train=True),
        # fp32, packed, with every gradient, the states' among them.
        _mix("fp32_1031", 1, 1031, 8, 4, 64, 64, dtype="fp32", train=True, packed=3, state=True),
        # One sequence's next token: latency.
        _step("step_1", 1, 16, 16, 128, 128),
        # A full decode batch, states spread over a pool.
        _step("step_256", 256, 16, 16, 128, 128, pool=320),
    ]


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def draw(rng):
    kind = rng.choice(["rope", "mix", "mix", "step"])
    if kind == "rope":
        H, KV = rng.choice([(38, 2), (16, 2), (8, 8), (13, 13), (24, 4)])
        d = rng.choice([64, 64, 96, 128, 256])
        rot = rng.choice([d // 4 // 8 * 8, d // 2 // 8 * 8, d])
        axes = rng.choice([1, 1, 3])
        T = _log_uniform(rng, 1, min(16384, 16384 * 40 * 64 // ((H + KV) * d)))
        return _rope(None, T, H, KV, d, rot, dtype=rng.choice(["bf16", "bf16", "fp32"]), train=rng.random() < 0.6,
                     axes=axes, far=_log_uniform(rng, 4096, 1000000))
    H, Hk = rng.choice([(16, 16), (39, 13), (8, 2), (12, 12), (5, 1)])
    dk, dv = rng.choice([(64, 64), (128, 128), (128, 128), (64, 128), (96, 96), (48, 80)])
    if kind == "step":
        B = _log_uniform(rng, 1, max(1, 256 * 16 * 128 * 128 // (H * dk * dv)))
        return _step(None, B, H, Hk, dk, dv, dtype=rng.choice(["bf16", "bf16", "fp32"]),
                     pool=rng.choice([0, B + rng.randint(1, 40)]))
    dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
    T = _log_uniform(rng, 1, 16384 if dtype == "bf16" and H <= 16 else 4096)
    train, state = rng.random() < 0.5, rng.random() < 0.5
    packed = rng.choice([0, 0, rng.randint(2, 12)]) if T >= 24 else 0
    B = 1 if packed else rng.choice([b for b in (1, 2, 3, 4) if T // b >= 1])
    return _mix(None, B, T // B, H, Hk, dk, dv, dtype=dtype, train=train, packed=packed, state=state)


# ---- inputs -----------------------------------------------------------------------------------

def _lengths(case, seed):
    """Lengths of a packed row's sequences: ragged, one of them a single token."""
    n = case["packed"]
    g = torch.Generator().manual_seed(seed)
    cuts = torch.randperm(case["S"] - 2, generator=g)[:n - 2].add(2).sort().values.tolist()
    at = [0, 1] + cuts + [case["S"]]
    return [b - a for a, b in zip(at, at[1:])]


def _axis_map(half, axes):
    """The axis of each frequency: all the first, or three interleaved with the first axis taking what is left."""
    if axes == 1:
        return torch.zeros(half, dtype=torch.int32)
    at = torch.arange(half)
    third = half // 3
    return torch.where((at % 3 == 1) & (at < 3 * third), 1, torch.where((at % 3 == 2) & (at < 3 * third), 2, 0)).int()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[case["dtype"]]

    def normal(shape, std, dtype=dt):
        return torch.randn(shape, generator=g, device="cuda").mul_(std).to(dtype)

    s = dict(case=case)
    if case["kind"] == "rope":
        T, H, KV, d, rot, axes = (case[n] for n in ("T", "H", "KV", "d", "rot", "axes"))
        # Queries lie beside their gates in the projection's output, as the model's do.
        s["q"] = normal((T, H, 2 * d), 1.0)[..., :d]
        s["k"] = normal((T, KV, d), 1.0)
        s["wq"], s["wk"] = normal((d,), 0.05), normal((d,), 0.05)
        s["inv_freq"] = (1.0 / _THETA ** (torch.arange(0, rot, 2, dtype=torch.float32) / rot)).cuda()
        s["pos"] = torch.randint(0, case["far"], (axes, T) if axes > 1 else (T,), generator=g, device="cuda")
        s["axes"] = _axis_map(rot // 2, axes).cuda() if axes > 1 else None
        if case["train"]:
            for n in ("q", "k", "wq", "wk"):
                s[n].requires_grad_(True)
            s["dq"], s["dk"] = normal((T, H, d), 0.1), normal((T, KV, d), 0.1)
        return s
    H, Hk, dk, dv = (case[n] for n in ("H", "Hk", "dk", "dv"))
    # A decay for each head from fast to slow, none of them alike in two models.
    slope = 2.0 ** (-8.0 * torch.arange(1, H + 1, device="cuda") / H)
    s["g"] = -slope * (0.75 + 0.5 * torch.rand(H, generator=g, device="cuda"))
    if case["kind"] == "step":
        B, pool = case["B"], case["pool"]
        s["q"], s["k"], s["v"] = normal((B, H, dk), 1.0), normal((B, Hk, dk), 1.0), normal((B, Hk, dv), 1.0)
        s["state"] = normal((pool or B, H, dk, dv), 1.0, torch.float32)
        s["slots"] = torch.randperm(pool, generator=g, device="cuda")[:B].int() if pool else None
        return s
    B, S, packed = case["B"], case["S"], case["packed"]
    s["q"], s["k"], s["v"] = normal((B, S, H, dk), 1.0), normal((B, S, Hk, dk), 1.0), normal((B, S, Hk, dv), 1.0)
    s["cu"] = s["index"] = None
    n = B
    if packed:
        n = packed
        lens = _lengths(case, seed)
        s["cu"] = torch.tensor([0] + lens, dtype=torch.int32).cumsum(0).int().cuda()
        s["longest"] = max(lens)
    s["state"] = normal((n, H, dk, dv), 0.5, torch.float32) if case["state"] else None
    if case["train"]:
        for name in ("q", "k", "v"):
            s[name].requires_grad_(True)
        s["do"] = normal((B, S, H, dv), 0.1)
        if case["state"]:
            s["state"].requires_grad_(True)
            s["dstate"] = normal((n, H, dk, dv), 0.05, torch.float32)
    return s


# ---- the calls --------------------------------------------------------------------------------

def _hip():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    from q38.hip import autograd, ops

    return autograd, ops


def run(s):
    case = s["case"]
    return {"rope": _run_rope, "mix": _run_mix, "step": _run_step}[case["kind"]](s, case)


def _run_rope(s, case):
    rot, d = case["rot"], case["d"]
    if own:
        autograd, _ = _hip()
        q, k = autograd.qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["pos"], s["inv_freq"], axes=s["axes"], eps=_EPS)
        if not case["train"]:
            return {"q": q, "k": k}
        dq, dk, dwq, dwk = torch.autograd.grad((q, k), (s["q"], s["k"], s["wq"], s["wk"]), (s["dq"], s["dk"]))
        return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk, "dwq": dwq, "dwk": dwk}
    pos = s["pos"].double()
    at = pos[s["axes"].long()].t() if case["axes"] > 1 else pos[:, None]
    angle = at * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    half = rot // 2

    def normed(x):
        x = x.detach().float()
        r = torch.rsqrt(x.square().mean(-1, keepdim=True) + _EPS)
        return x * r, r

    def turned(n):
        a, b = n[..., :half], n[..., half:rot]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, n[..., rot:]], -1)

    def back(dy, x, r, w):
        dy = dy.float()
        a, b = dy[..., :half], dy[..., half:rot]
        dn = torch.cat([a * cos + b * sin, b * cos - a * sin, dy[..., rot:]], -1)
        gx = dn * (1.0 + w.float())
        return r * (gx - x * (gx * x).mean(-1, keepdim=True)), (dn * x).sum((0, 1), dtype=torch.float64)

    out, dt = {}, s["q"].dtype
    for n, dn in (("q", "dq"), ("k", "dk")):
        w = s["w" + n].detach()
        x, r = normed(s[n])
        out[n] = turned(x * (1.0 + w.float())).to(dt)
        if case["train"]:
            dx, dw = back(s[dn], x, r, w)
            out[dn], out["dw" + n] = dx.to(dt), dw.to(dt)
    return out


_C = 128  # tokens of a chunk in the plain form


def _mixed(q, k, v, g):
    """sum_{j <= i} e^{g (i - j)} (q_i . k_j) v_j over [N, H, S, .] in fp32: inside chunks by their scores, from chunk to chunk
    by their states, which a product with the decays between chunks carries on."""
    N, H, S, _ = q.shape
    n = -(-S // _C)
    q, k, v = (torch.nn.functional.pad(t, (0, 0, 0, n * _C - S)).view(N, H, n, _C, t.shape[-1]) for t in (q, k, v))
    at = torch.arange(_C, device=q.device)
    g = g.double().view(H, 1, 1)
    between = at[:, None] - at[None, :]
    decay = torch.where(between >= 0, torch.exp(g * between.clamp(min=0)), torch.zeros((), device=q.device)).float()
    o = (q @ k.transpose(-1, -2) * decay[:, None]) @ v
    to_end, from_start = torch.exp(g * (_C - 1 - at)[:, None]).float(), torch.exp(g * (at + 1)[:, None]).float()
    local = (k * to_end[:, None]).transpose(-1, -2) @ v
    ci = torch.arange(n, device=q.device)
    ahead = ci[:, None] - ci[None, :] - 1
    carry = torch.where(ahead >= 0, torch.exp(g * _C * ahead.clamp(min=0)), torch.zeros((), device=q.device)).float()
    state = (carry @ local.reshape(N, H, n, -1)).view(local.shape)
    o = o + (q * from_start[:, None]) @ state
    return o.reshape(N, H, n * _C, -1)[:, :, :S]


def _run_mix(s, case):
    if own:
        autograd, _ = _hip()
        o, state = autograd.linear_attention(s["q"], s["k"], s["v"], s["g"], initial_state=s["state"], cu_seqlens=s["cu"],
                                             return_state=case["state"])
        if not case["train"]:
            return {"o": o, "state": state} if case["state"] else {"o": o}
        if not case["state"]:
            dq, dk, dv = torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])
            return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv}
        dq, dk, dv, ds = torch.autograd.grad((o, state), (s["q"], s["k"], s["v"], s["state"]), (s["do"], s["dstate"]))
        return {"o": o.detach(), "state": state.detach(), "dq": dq, "dk": dk, "dv": dv, "ds": ds}
    B, S, H, Hk, dk, dv = (case[n] for n in ("B", "S", "H", "Hk", "dk", "dv"))
    dt, dev, g, scale = s["q"].dtype, s["q"].device, s["g"], case["dk"] ** -0.5
    if s["cu"] is None:
        N, L = B, S
        lens = torch.full((N,), S, device=dev)
        token = torch.arange(B * S, device=dev).view(N, L)
        there = torch.ones(N, L, dtype=torch.bool, device=dev)
    else:
        N, L = case["packed"], s["longest"]
        lens = (s["cu"][1:] - s["cu"][:-1]).long()
        at = torch.arange(L, device=dev)
        there = at < lens[:, None]
        token = torch.where(there, s["cu"][:-1, None].long() + at, torch.zeros_like(at))
    mask = there[:, None, :, None]

    def sequences(t):
        """[N, H, L, .] fp32, zero behind each sequence's end, shared heads repeated."""
        t = t.detach().reshape(B * S, t.shape[2], t.shape[3])[token].float().transpose(1, 2) * mask
        return t.repeat_interleave(H // t.shape[1], dim=1)

    def tokens(t, heads):
        """Back to [B, S, heads, .], the heads that share one added."""
        t = t.reshape(N, heads, -1, L, t.shape[-1]).sum(2).transpose(1, 2)
        return t[there].view(B, S, heads, -1).to(dt)

    q, k, v = sequences(s["q"]), sequences(s["k"]), sequences(s["v"])
    pos = torch.arange(L, device=dev)
    gd = g.double()[:, None]
    o = _mixed(q, k, v, g)
    left = (lens[:, None] - 1 - pos).clamp(min=0)  # tokens that follow
    to_end = torch.exp(gd * left[:, None]).float()[..., None]
    from_start = torch.exp(gd * (pos + 1)).float()[..., None]
    if case["state"]:
        S0 = s["state"].detach()
        o = o + (q * from_start) @ S0
        whole = torch.exp(gd * lens[:, None, None]).float()[..., None]
        state = S0 * whole + (k * to_end).transpose(-1, -2) @ v
    out = {"o": tokens(o * scale, H)}
    if case["state"]:
        out["state"] = state
    if not case["train"]:
        return out
    do = sequences(s["do"])
    dq = _mixed(do, v, k, g)
    back = [t.flip(2) for t in (q, k, v, do)]
    dk_ = _mixed(back[2], back[3], back[0], g).flip(2) * scale
    dv_ = _mixed(back[1], back[0], back[3], g).flip(2) * scale
    if case["state"]:
        dS = s["dstate"]
        dq = dq + (do * from_start) @ S0.transpose(-1, -2)
        dk_ = dk_ + (v * to_end) @ dS.transpose(-1, -2)
        dv_ = dv_ + (k * to_end) @ dS
        out["ds"] = scale * ((q * from_start).transpose(-1, -2) @ do) + dS * whole
    return dict(out, dq=tokens(dq * scale, H), dk=tokens(dk_ * mask, Hk), dv=tokens(dv_ * mask, Hk))


def _run_step(s, case):
    if own:
        _, ops = _hip()
        o = ops.linear_attention_step(s["q"], s["k"], s["v"], s["state"], s["g"], slots=s["slots"])
        return {"o": o, "state": s["state"]}
    H, Hk = case["H"], case["Hk"]
    k, v = (s[n].float().repeat_interleave(H // Hk, dim=1) for n in ("k", "v"))
    old = s["state"] if s["slots"] is None else s["state"][s["slots"].long()]
    new = torch.exp(s["g"])[:, None, None] * old + k[..., :, None] * v[..., None, :]
    if s["slots"] is None:
        s["state"].copy_(new)
    else:
        s["state"][s["slots"].long()] = new
    o = (s["q"].float()[..., None] * new).sum(2) * case["dk"] ** -0.5
    return {"o": o.to(s["q"].dtype), "state": s["state"]}


# ---- the work, and the values in float64 ------------------------------------------------------

def work(case):
    b = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "rope":
        T, H, KV, d, rot, axes = (case[n] for n in ("T", "H", "KV", "d", "rot", "axes"))
        x, small = b * T * (H + KV) * d, 8 * axes * T + 4 * rot + 2 * b * d
        if not case["train"]:
            return {"bytes": 2 * x + small, "flops": 8 * T * (H + KV) * d}
        return {"bytes": 4 * x + small + 2 * b * d, "flops": 24 * T * (H + KV) * d}
    H, Hk, dk, dv = (case[n] for n in ("H", "Hk", "dk", "dv"))
    if case["kind"] == "step":
        B = case["B"]
        return {"bytes": 8 * B * H * dk * dv + b * B * (H * dk + Hk * (dk + dv) + H * dv) + 4 * H,
                "flops": 5 * B * H * dk * dv}
    T = case["B"] * case["S"]
    states = 4 * (case["packed"] or case["B"]) * H * dk * dv if case["state"] else 0
    inputs, out = b * T * (H * dk + Hk * (dk + dv)), b * T * H * dv
    if not case["train"]:
        return {"bytes": inputs + out + 2 * states, "flops": 4 * T * H * dk * dv}
    return {"bytes": 2 * inputs + 2 * out + 4 * states, "flops": 12 * T * H * dk * dv}


def exact(case, seed):
    s = prepare(case, seed)
    s = {n: v.detach() if isinstance(v, torch.Tensor) else v for n, v in s.items()}
    return {"rope": _exact_rope, "mix": _exact_mix, "step": _exact_step}[case["kind"]](s, case)


def _exact_rope(s, case):
    rot, T = case["rot"], case["T"]
    half, out = rot // 2, {}
    pos = s["pos"].reshape(-1, T).double()
    axis = s["axes"].long().tolist() if case["axes"] > 1 else [0] * half
    angle = torch.stack([pos[a] * s["inv_freq"][i].double() for i, a in enumerate(axis)], 1)
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]  # a pair of features as a complex number
    for n in ("q", "k"):
        x, w = s[n].double(), 1.0 + s["w" + n].double()
        rstd = (x.pow(2).sum(-1, keepdim=True) / case["d"] + _EPS).pow(-0.5)
        y = x * rstd * w
        z = torch.complex(y[..., :half], y[..., half:rot]) * turn
        out[n] = torch.cat([z.real, z.imag, y[..., rot:]], -1)
        if case["train"]:
            dy = s["d" + n].double()
            z = torch.complex(dy[..., :half], dy[..., half:rot]) * turn.conj()
            dn = torch.cat([z.real, z.imag, dy[..., rot:]], -1)
            out["dw" + n] = (dn * x * rstd).sum(0).sum(0)
            dn = dn * w
            out["d" + n] = rstd * dn - x * rstd.pow(3) * (dn * x).sum(-1, keepdim=True) / case["d"]
    return out


def _exact_mix(s, case):
    """Token by token: the state forwards for o and dq, its gradient backwards for dk and dv."""
    B, S, H, Hk, dk, dv = (case[n] for n in ("B", "S", "H", "Hk", "dk", "dv"))
    dev, G, scale = s["q"].device, H // Hk, dk ** -0.5
    lam = torch.exp(s["g"].double())[:, None, None]
    starts = list(range(0, B * S, S)) if s["cu"] is None else s["cu"].tolist()[:-1]
    lens = [S] * B if s["cu"] is None else (s["cu"][1:] - s["cu"][:-1]).tolist()
    N = len(starts)
    train, carried = case["train"], case["state"]
    q, k, v = (s[n].double().reshape(B * S, -1, s[n].shape[-1]) for n in "qkv")
    k, v = k.repeat_interleave(G, dim=1), v.repeat_interleave(G, dim=1)
    do = s["do"].double().reshape(B * S, H, dv) if train else None
    o, dq = torch.zeros_like(q[..., :1]).expand(-1, -1, dv).clone(), torch.zeros_like(q)
    order = sorted(range(N), key=lambda i: -lens[i])  # longest first: those still going are a prefix
    first = torch.tensor([starts[i] for i in order], device=dev)
    count = [sum(n > t for n in lens) for t in range(max(lens))]
    state = (s["state"].double()[order] if carried else torch.zeros(N, H, dk, dv, dtype=torch.float64, device=dev))
    for t, n in enumerate(count):
        at, now = first[:n] + t, state[:n]
        now.mul_(lam).addcmul_(k[at][..., None], v[at][..., None, :])
        o[at] = (q[at][..., None, :] @ now)[..., 0, :] * scale
        if train:
            dq[at] = (now @ do[at][..., None])[..., 0] * scale
    back = torch.empty_like(state)
    back[order] = state
    out = {"o": o.view(B, S, H, dv)}
    if carried:
        out["state"] = back
    if not train:
        return out
    dks, dvs = torch.zeros_like(k), torch.zeros_like(v)
    grad = s["dstate"].double()[order] if carried else torch.zeros_like(state)
    for t in range(len(count) - 1, -1, -1):
        n = count[t]
        at, now = first[:n] + t, grad[:n]
        now.addcmul_(q[at][..., None], do[at][..., None, :], value=scale)
        dks[at] = (now @ v[at][..., None])[..., 0]
        dvs[at] = (k[at][..., None, :] @ now)[..., 0, :]
        now.mul_(lam)
    if carried:
        back = torch.empty_like(grad)
        back[order] = grad
        out["ds"] = back
    return dict(out, dq=dq.view(B, S, H, dk), dk=dks.view(B, S, Hk, G, dk).sum(3), dv=dvs.view(B, S, Hk, G, dv).sum(3))


def _exact_step(s, case):
    G = case["H"] // case["Hk"]
    rows = range(case["B"]) if s["slots"] is None else s["slots"].tolist()
    state, lam = s["state"].double(), torch.exp(s["g"].double())
    o = torch.empty(case["B"], case["H"], case["dv"], dtype=torch.float64, device=state.device)
    for b, row in enumerate(rows):
        k, v = (s[n][b].double().repeat_interleave(G, dim=0) for n in "kv")
        state[row] = lam[:, None, None] * state[row] + torch.einsum("hk,hv->hkv", k, v)
        o[b] = torch.einsum("hk,hkv->hv", s["q"][b].double(), state[row]) * case["dk"] ** -0.5
    return {"o": o, "state": state}

"""How exact the token mixer is where its results are not: the roundings that test_gpu_mixer.py's bounds leave room for.

bf16: the weighted scores and the state that queries read are operands in two bf16 parts. The first leaves at most v of a
value (v = 2^-8, half a step), the second v of that: v^2 of every score and of every element of the state, beside the fp32 sums
and v for the rounding of the result. An operand of one part is v off: most where a result is small beside its terms."""
import pytest
import torch

import test_gpu_mixer as mixer
from test_gpu_mixer import U, _sum64, _within

V = 2.0 ** -8


def _sharp(got, want, dtype, dk, name, group=1):
    """mixer._check with v^2 of each score and element of the state in the place of v."""
    out, rounded, terms = want
    H, S, d = out.shape
    v = torch.finfo(dtype).eps / 2
    bound = 2 * (dk + 64 + S / 64 + 20 + group) * U * terms + (v * v * rounded * (1 + v) if dtype == torch.bfloat16 else 0)
    out, bound = (t.view(H // group, group, S, d).sum(1).transpose(0, 1) for t in (out, bound))
    _within(got, out, bound + v * (out.abs() + bound) + 1e-37, name)


def _parts(x, n):
    """x as the sum of n bf16 numbers."""
    got = torch.zeros_like(x)
    for _ in range(n):
        got = got + (x - got).bfloat16().double()
    return got


def _emulated(q, k, v, g, S0, scale, of_scores, of_state):
    """The chunked sums in float64 with operands of so many parts, rounded to bf16; [S,H,.] in, [S,H,dv] out."""
    q, k, v = (t.double().transpose(0, 1) for t in (q, k, v))
    g, state, outs = g.double()[:, None, None], S0.double(), []
    for j0 in range(0, q.shape[1], 64):
        a, b, c = (t[:, j0:j0 + 64] for t in (q, k, v))
        n = a.shape[1]
        at = torch.arange(n)
        gap = at[:, None] - at[None, :]
        s = a @ b.transpose(1, 2) * torch.where(gap >= 0, torch.exp(g * gap.clamp(min=0)), torch.zeros((), dtype=torch.float64))
        outs.append(_parts(s * scale, of_scores) @ c + torch.exp(g * (at[:, None] + 1)) * scale * (a @ _parts(state, of_state)))
        state = torch.exp(g * n) * state + (b * torch.exp(g * (n - 1 - at[:, None]))).transpose(1, 2) @ c
    return torch.cat(outs, 1).transpose(0, 1).bfloat16()


@pytest.mark.parametrize("dk,dv", [(8, 8), (64, 64), (128, 128)])
def test_the_bound_sees_a_part_less(dk, dv):
    """On the CPU: sums with operands of two parts are within the bound, with one part of either they are not."""
    q, k, v, g, S0, _, _ = mixer._mix_inputs(torch.device("cpu"), 1, 200, 4, 4, dk, dv, torch.bfloat16)
    scale = dk ** -0.5
    want = _sum64(*(t[0].transpose(0, 1) for t in (q, k, v)), g, S0[0], scale, scale, 1.0, 0)[:3]
    args = q[0], k[0], v[0], g, S0[0], scale
    _sharp(_emulated(*args, 2, 2), want, torch.bfloat16, dk, "two parts")
    for parts in ((1, 2), (2, 1)):
        with pytest.raises(AssertionError, match="of the bound"):
            _sharp(_emulated(*args, *parts), want, torch.bfloat16, dk, "one part")


@pytest.mark.gpu
@pytest.mark.parametrize("B,S,H,Hk,dk,dv,state", [
    (2, 1, 2, 1, 64, 64, True), (1, 70, 4, 4, 8, 8, True), (2, 300, 4, 2, 64, 64, True), (1, 300, 4, 2, 64, 128, True),
    (1, 300, 4, 2, 128, 64, True), (2, 300, 4, 4, 128, 128, True), (1, 640, 4, 1, 48, 80, False), (1, 1500, 128, 64, 128, 128, True),
])
def test_operands_in_two_parts(gpu, monkeypatch, B, S, H, Hk, dk, dv, state):
    """Outputs and every gradient."""
    monkeypatch.setattr(mixer, "_check", _sharp)
    mixer.test_linear_attention(gpu, torch.bfloat16, B, S, H, Hk, dk, dv, state)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,tail,H,Hk,dk,dv", [([100, 600, 3, 64, 0, 200], 37, 4, 2, 64, 64),
                                                  ([700, 0, 1, 640, 65, 2], 9, 128, 128, 128, 128)])
def test_operands_in_two_parts_packed(gpu, monkeypatch, lens, tail, H, Hk, dk, dv):
    monkeypatch.setattr(mixer, "_check", _sharp)
    mixer.test_linear_attention_packed(gpu, torch.bfloat16, lens, tail, H, Hk, dk, dv, True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_many_steps_of_a_slow_decay(gpu, dtype):
    """20000 single tokens with decays next to 1, everything positive, against float64. A step rounds the state twice (u of it
    each, one sign or the other: a walk of at most 2 u (n/3)^1/2 as a standard deviation, 5 of them make 6 u n^1/2). A decay in one float
    is off the same way every time, which makes 25 u n^1/2 or more of each of these."""
    from q38.hip import ops
    n, d = 20000, 32
    decay = torch.tensor([-1e-5, -3e-6, -1e-7, -2e-8], device=gpu)
    r = torch.Generator(device=gpu).manual_seed(4)
    q, k, v = (torch.randn(n, 4, d, generator=r, device=gpu).abs().to(dtype) for _ in range(3))
    state = 1e4 * (0.5 + torch.rand(1, 4, d, d, generator=r, device=gpu))
    exact = torch.exp(decay.double() * n)[:, None, None] * state[0].double()
    left = torch.exp(decay.double()[:, None] * torch.arange(n - 1, -1, -1, device=gpu))[..., None]
    exact += (k.double().transpose(0, 1) * left).transpose(1, 2).contiguous() @ v.double().transpose(0, 1).contiguous()
    for t in range(n):
        out = ops.linear_attention_step(q[t:t + 1], k[t:t + 1], v[t:t + 1], state, decay)
    torch.cuda.synchronize()
    bound = 6 * U * n ** 0.5
    _within(state[0], exact, bound * exact, "state")
    o = (q[-1].double()[:, None] @ exact)[:, 0] * d ** -0.5
    half = torch.finfo(dtype).eps / 2
    _within(out[0], o, (bound + (d + 12) * U + half) * (1 + half) * o, "out")


# ---- decays over many chunks and segments -------------------------------------------------------

def _midway(tokens):
    """A log_decay near -1e-5 whose e^{g tokens} lies next to the middle between two floats."""
    g = (-1e-5 * (1 + 1e-4 * torch.arange(2000, dtype=torch.float64))).float().double()
    x = torch.exp(g * tokens)
    return float(g[(x - x.float().double()).abs().argmax()])


def _decayed(S, g, tokens, times, low):
    """S e^{g tokens times} with a rounding to fp32 each time, the decay in two floats or (not low) in one."""
    x = torch.exp(torch.tensor(g, dtype=torch.float64) * tokens)
    hi = x.float().double()
    lo = (x - hi).float().double() if low else 0.0
    for _ in range(times):
        S = (S.double() * hi + (S.double() * lo).float().double()).float()
    return S


# A rounding (u of the state, either sign) each time: 5 standard deviations of the walk, u (n/3)^1/2, are 3 u n^1/2. What
# test_decay_alone_over_many_chunks runs is rounded up to 260 times: by 256 segments and 4 chunks of the last, or by 256 chunks.
DECAY_BOUND = 3 * U * 260 ** 0.5


@pytest.mark.parametrize("tokens,times", [(64, 256), (256, 256), (512, 128)])
def test_the_bound_sees_a_decay_in_one_float(tokens, times):
    """On the CPU, for every length of segments that the next test runs and its number of them: what that allows is more than two
    floats leave and less than one does."""
    g, S = _midway(tokens), 1.0 + torch.rand(64, 64, generator=torch.Generator().manual_seed(1))
    exact = S.double() * torch.exp(torch.tensor(g, dtype=torch.float64) * tokens * times)
    off = [float(((_decayed(S, g, tokens, times, low).double() - exact) / exact).abs().max()) for low in (True, False)]
    assert off[0] < 0.8 * DECAY_BOUND and DECAY_BOUND < 0.8 * off[1], (off[0] / U, off[1] / U, DECAY_BOUND / U)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("S,H,d", [(65536, 4, 64),                        # 256 segments of 256 tokens or 128 of 512
                                   (16384, 1024, 8), (16384, 512, 128)])  # so many heads that a segment has all 256 chunks
def test_decay_alone_over_many_chunks(gpu, dtype, S, H, d):
    """Keys and values of zero: the last state is e^{gS} of the first, and the gradients' likewise, through every chunk's and every
    segment's decay and nothing else, with decays that one float rounds by half a step."""
    from q38.hip import ops
    g = torch.tensor([_midway(n) for n in (64, 128, 256, 512)], device=gpu).repeat(H // 4)
    r = torch.Generator(device=gpu).manual_seed(2)
    S0, dS = (1.0 + torch.rand(1, H, d, d, generator=r, device=gpu) for _ in range(2))
    x = torch.zeros(1, S, 1, d, dtype=dtype, device=gpu).expand(1, S, H, d)
    out, last = ops.linear_attention(x, x, x, g, initial_state=S0, return_state=True)
    assert not bool(out[0, :, :4].any())
    left = torch.exp(g.double() * S)[:, None, None]
    _within(last[0], S0[0].double() * left, DECAY_BOUND * S0[0].double() * left, "state")
    ds = ops.linear_attention_backward(out.zero_(), dS, x, x, x, g, initial_state=S0, need_state=True)[3]
    _within(ds[0], dS[0].double() * left, DECAY_BOUND * dS[0].double() * left, "ds")


# ---- rotation -----------------------------------------------------------------------------------

@pytest.mark.gpu
def test_turns_near_their_zeros(gpu):
    """Sines and cosines themselves, as the rotation of (1, 0) in fp32, at angles next to multiples of a quarter turn, where one of the
    two is all that the angle's rounding leaves. The functions' 2 ulp (4 u), what the angle adds to them (u, and u for the product), and
    the rotation's own rounding (u) of each; the angle's four roundings in 64 bits are absolute."""
    from q38.hip import ops
    # Whole numbers next to n quarter turns: numerators of convergents of pi / 2 and multiples of them.
    at = [1, 2, 3, 11, 22, 33, 44, 355, 710, 1065, 52174, 104348, 260515, 521030, 1042060]
    pos = torch.tensor(at + [5, 17, 100, 4097], device=gpu)
    T, d = pos.numel(), 64
    inv = torch.ones(d // 2, device=gpu)
    inv[1:] = 0.5 ** torch.arange(1, d // 2, device=gpu)  # exact fractions of them
    x = torch.zeros(T, 1, d, device=gpu)
    x[..., :d // 2] = 1.0
    q, k = ops.qk_norm_rope(x, x, None, None, pos, inv)
    angle = pos.double()[:, None] * inv.double()
    exact = torch.cat([angle.cos(), angle.sin()], -1)[:, None]
    _within(q, exact, 7 * U * exact.abs() + 4 * 2.0 ** -53 * torch.cat([angle, angle], -1)[:, None], "turn")
    assert torch.equal(q, k)

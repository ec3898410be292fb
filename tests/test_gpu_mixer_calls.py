"""Calls of the token mixer that lie at the edges of what it takes: large batches of single tokens, nothing at all, gradients that
are broadcast or taken twice, graphs replayed in turn."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,again", [(3000, ((0, 2999), (1023, 1024))), (1030, ((255, 1029), (256, 1025), (2, 767))),
                                     (2500, ((1024, 1800), (769, 2048), (7, 2304)))])
def test_step_of_many_sequences_with_slots_twice(gpu, B, again):
    """The first to name a slot has it, wherever in the batch the two are: bits as where the others name none, and as in batches of
    a few sequences."""
    from q38.hip import ops
    r = torch.Generator(device=gpu).manual_seed(B)
    q, k, v = (torch.randn(B, 2, 16, generator=r, device=gpu).bfloat16() for _ in range(3))
    state = torch.randn(B + 4, 2, 16, 16, generator=r, device=gpu)
    g = -torch.rand(2, generator=r, device=gpu)
    slots = torch.randperm(B + 4, generator=r, device=gpu)[:B].int()
    twice, without = slots.clone(), slots.clone()
    for first, second in again:
        twice[second], without[second] = slots[first], -1
    a, b, c = state.clone(), state.clone(), state.clone()
    got = ops.linear_attention_step(q, k, v, a, g, slots=twice)
    assert torch.equal(got, ops.linear_attention_step(q, k, v, b, g, slots=without)) and torch.equal(a, b)
    for n in range(0, B, 100):
        part = slice(n, n + 100)
        assert torch.equal(got[part], ops.linear_attention_step(q[part], k[part], v[part], c, g, slots=without[part])), n
    assert torch.equal(a, c)
    for _, second in again:
        assert not bool(got[second].any())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_nothing_to_do(gpu, dtype):
    """No tokens, no sequences, packed sequences without tokens, no states: states pass through, gradients too."""
    from q38.hip import autograd, ops
    g = torch.full((2,), -0.1, device=gpu)
    for B, S, N, cu in ((0, 5, 0, None), (3, 0, 3, None), (1, 0, 4, torch.zeros(5, dtype=torch.int32, device=gpu))):
        q, k, v = (torch.zeros(B, S, h, d, dtype=dtype, device=gpu, requires_grad=True) for h, d in ((2, 64), (1, 64), (1, 128)))
        S0 = torch.randn(N, 2, 64, 128, device=gpu, requires_grad=True)
        out, last = autograd.linear_attention(q, k, v, g, initial_state=S0, cu_seqlens=cu, return_state=True)
        assert out.shape == (B, S, 2, 128) and torch.equal(last, S0)
        dS = torch.randn_like(S0)
        grads = torch.autograd.grad((out, last), (q, k, v, S0), (torch.zeros_like(out), dS))
        assert torch.equal(grads[3], dS) and [t.shape for t in grads[:3]] == [t.shape for t in (q, k, v)]
    q, k, v = (torch.randn(3, 2, 64, device=gpu).to(dtype) for _ in range(3))
    slots = torch.tensor([0, -1, 7], dtype=torch.int32, device=gpu)
    out = ops.linear_attention_step(q, k, v, torch.zeros(0, 2, 64, 64, device=gpu), g, slots=slots)
    assert not bool(out.any())
    state = torch.randn(2, 2, 64, 64, device=gpu)
    kept = state.clone()
    out = ops.linear_attention_step(q, k, v, state, g, slots=torch.full_like(slots, -1))
    assert not bool(out.any()) and torch.equal(state, kept)


def test_gradients_broadcast_and_taken_twice(gpu):
    """A loss that sums (its gradient is one number, expanded), a graph that is kept and gone through again, recomputation in the
    backward pass, the state's gradient alone asked for: the same bits as by themselves."""
    from torch.utils.checkpoint import checkpoint
    from q38.hip import autograd
    r = torch.Generator(device=gpu).manual_seed(6)
    q, k, v = (torch.randn(2, 150, h, 64, generator=r, device=gpu).bfloat16() for h in (4, 2, 2))
    w = torch.randn(64, generator=r, device=gpu).bfloat16()
    S0 = torch.randn(2, 4, 64, 64, generator=r, device=gpu)
    pos, inv, g = torch.arange(150, device=gpu).expand(2, 150), torch.rand(8, device=gpu), -torch.rand(4, device=gpu)

    def run(q, k, v, w, S0):
        q, k = autograd.qk_norm_rope(q, k, w, w, pos, inv)
        return autograd.linear_attention(q, k, v, g, initial_state=S0)[0]

    def leaves():
        return [t.clone().requires_grad_(True) for t in (q, k, v, w, S0)]

    a = leaves()
    out = run(*a)
    want = torch.autograd.grad(out, a, torch.ones_like(out), retain_graph=True)
    for got in (torch.autograd.grad(out.sum(), a, retain_graph=True), torch.autograd.grad(out.sum(), a)):
        assert all(torch.equal(x, y) for x, y in zip(got, want))
    b = leaves()
    got = torch.autograd.grad(checkpoint(run, *b, use_reentrant=False).sum(), b)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    c = S0.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(run(q, k, v, w, c).sum(), c)[0], want[4])


def test_graphs_replayed_in_turn(gpu):
    """Two captured graphs of packed prompts and a step of each, replayed in turn and on new inputs: each the eager result."""
    from q38.hip import ops
    r = torch.Generator(device=gpu).manual_seed(8)
    graphs = []
    for S, cuts in ((900, (0, 100, 700, 900)), (333, (0, 0, 333, 333))):
        x = [torch.randn(1, S, 4, 64, generator=r, device=gpu).bfloat16() for _ in range(3)]
        cu = torch.tensor(cuts, dtype=torch.int32, device=gpu)
        slots = torch.tensor([2, 0, 2], dtype=torch.int32, device=gpu)
        g = -torch.rand(4, generator=r, device=gpu)

        def run(x=x, cu=cu, slots=slots, g=g):
            out, pool = ops.linear_attention(*x, g, cu_seqlens=cu, return_state=True)
            token = ops.linear_attention_step(*(t[0, :3] for t in x), pool, g, slots=slots)
            return out, pool, token

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = run()
        graphs.append((graph, held, run, x))
    for _ in range(3):
        for graph, _, _, x in graphs:
            for t in x:
                t.copy_(torch.randn(t.shape, generator=r, device=gpu))
            graph.replay()
        torch.cuda.synchronize()
        for _, held, run, _ in graphs:
            for a, b in zip(held, run()):
                assert torch.equal(a, b)

"""Calls of the token mixer that lie at the edges of what it takes: large batches of single tokens."""
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

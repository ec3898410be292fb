"""Refusals of the training step's operators, before any launch (no GPU): the torch front end's checks and the C
ABI's."""
import ctypes
import math

import pytest
import torch


def _lib():
    from q38.hip import _lib
    return _lib


def test_loss_refusals():
    from q38.hip import autograd, ops
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(10, 64, dtype=torch.bfloat16)
    t = torch.zeros(4, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA/HIP tensor"):
        autograd.linear_cross_entropy(x, w, t)
    with pytest.raises(TypeError, match="bf16 or fp32"):
        autograd.linear_cross_entropy(x.half(), w.half(), t)
    with pytest.raises(ValueError, match="reduction"):
        autograd.linear_cross_entropy(x, w, t, reduction="batchmean")
    with pytest.raises(ValueError, match="do not match"):
        autograd.linear_cross_entropy(x, w, t[:3])
    with pytest.raises(TypeError, match="bf16 or fp32"):
        ops.linear_ce_forward(x.double(), w, t)


@pytest.mark.parametrize("T,h,V,dtype,msg", [
    (-1, 64, 10, 1, "T must be"), ((1 << 24) + 1, 64, 10, 1, "T must be"), (4, 100, 10, 1, "h must be"),
    (4, 65600, 10, 1, "h must be"), (4, 64, 0, 1, "V must be"), (4, 64, 1 << 21, 1, "V must be"),
    (4, 64, 10, 3, "dtype"),
])
def test_loss_shapes(T, h, V, dtype, msg):
    m = _lib()
    n = ctypes.c_size_t()
    assert m.lib.q38moe_linear_ce_workspace_bytes(T, h, V, 0, dtype, ctypes.byref(n)) == -1
    assert msg in m.lib.q38moe_last_error().decode()


def test_loss_abi_arguments():
    m = _lib()
    lib, p = m.lib, ctypes.c_void_p(1 << 20)
    fwd = lambda x, t, ws, n, T=4: lib.q38moe_linear_ce_forward(x, p, t, 1, -100, p, p, None, None, 0, T, 64, 10,  # noqa: E731
                                                                ws, n, 1, None)
    assert fwd(None, p, p, 1 << 30) == -1 and "x must not be NULL" in lib.q38moe_last_error().decode()
    assert fwd(ctypes.c_void_p(8), p, p, 1 << 30) == -1 and "aligned" in lib.q38moe_last_error().decode()
    assert fwd(p, None, p, 1 << 30) == -1 and "targets" in lib.q38moe_last_error().decode()
    assert fwd(p, p, p, 16) == -2 and "workspace needs" in lib.q38moe_last_error().decode()
    assert fwd(None, None, None, 0, T=0) == 0
    bwd = lambda g, dx, dw, n, T=4: lib.q38moe_linear_ce_backward(g, 0, None, p, p, p, 1, -100, p, dx, dw, T, 64, 10,  # noqa: E731
                                                                  p, n, 1, None)
    assert bwd(None, p, None, 1 << 30) == -1 and "must not be NULL" in lib.q38moe_last_error().decode()
    assert bwd(p, p, None, 16) == -2
    assert bwd(None, None, None, 0) == 0
    assert bwd(p, p, None, 1 << 30, T=0) == -1


def test_loss_workspace_is_bounded():
    """The workspace of the backward pass does not grow with the vocabulary beyond a piece of it and what is left
    over of the gradients' partial sums."""
    m = _lib()
    sizes = []
    for V in (20000, 40000, 160000, 640000):
        n = ctypes.c_size_t()
        assert m.lib.q38moe_linear_ce_workspace_bytes(16384, 1024, V, 1, 1, ctypes.byref(n)) == 0
        sizes.append(n.value)
    logits = 2 * 16384 * 640000
    assert max(sizes) < (1 << 30) < logits // 16
    assert max(sizes) <= 2 * min(sizes)


def test_clip_refusals():
    from q38.hip import ops
    t = torch.zeros(4)
    with pytest.raises(RuntimeError, match="CUDA/HIP"):
        ops.grad_norm([t])
    with pytest.raises(ValueError, match="norm_type"):
        ops.grad_norm([t], 3.0)
    with pytest.raises(ValueError, match="norm_type"):
        ops.grad_norm([], 0.5)
    with pytest.raises(TypeError, match="bf16 or fp32"):
        ops.grad_norm([t.half()])
    with pytest.raises(TypeError, match="bf16 or fp32"):
        ops.clip_grads([3.0], 1.0)
    with pytest.raises(ValueError, match="max_norm"):
        ops.clip_grads([t], -1.0)
    with pytest.raises(ValueError, match="max_norm"):
        ops.clip_grads([t], math.nan)
    with pytest.raises(ValueError, match="out must hold"):
        ops.clip_grads([t], 1.0, out=[])
    assert float(ops.grad_norm([])) == 0.0 and float(ops.clip_grad_norm_([], 1.0)) == 0.0


def test_clip_abi_arguments():
    m = _lib()
    lib = m.lib

    def call(src, dst, sizes, dts=None, odts=None, norm=2, max_norm=1.0, ws=1 << 20, nbytes=1 << 30):
        n = len(src)
        dts = dts or [2] * n
        return lib.q38moe_clip_grads((ctypes.c_void_p * n)(*src), (ctypes.c_void_p * n)(*dst),
                                     (ctypes.c_int64 * n)(*sizes), (ctypes.c_int32 * n)(*dts),
                                     (ctypes.c_int32 * n)(*(odts or dts)), n, norm, max_norm, ctypes.c_void_p(1 << 20),
                                     ctypes.c_void_p(ws), nbytes, None)

    def says(text):
        return text in lib.q38moe_last_error().decode()

    a, b = 1 << 24, 1 << 25
    assert call([a], [a], [4], norm=7) == -1 and says("norm")
    assert call([a], [a], [4], dts=[5]) == -1 and says("dtype")
    assert call([a], [a], [-4]) == -1 and says("size")
    assert call([a + 2], [a], [4]) == -1 and says("aligned")
    assert call([a], [None], [4]) == -1 and says("output")
    assert call([a], [a], [4], max_norm=-1.0) == -1 and says("max_norm")
    assert call([a], [a], [4], max_norm=math.nan) == -1 and says("max_norm")
    assert call([a], [a], [4], nbytes=16) == -2 and says("workspace needs")
    assert call([a], [a], [4], dts=[2], odts=[1]) == -1 and says("in place")
    assert call([a, a], [a, a], [4, 4]) == -1 and says("overlap")
    assert call([a, a + 8], [a, a + 8], [4, 4]) == -1 and says("overlap")
    assert call([a, b], [b, a], [4, 4]) == -1 and says("overlap")
    assert call([a], [a + 4], [4]) == -1 and says("overlap")
    n = ctypes.c_size_t()
    assert lib.q38moe_grad_norm_workspace_bytes(-1, ctypes.byref(n)) == -1
    assert lib.q38moe_grad_norm_workspace_bytes(97, ctypes.byref(n)) == 0 and n.value > 0


def test_rows_refusals():
    from q38.hip import autograd
    x, idx = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(4, 2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="CUDA/HIP tensor"):
        autograd.dispatch(x, idx, 8)
    with pytest.raises(TypeError, match="bf16 or fp32"):
        autograd.dispatch(x.half(), idx, 8)
    with pytest.raises(ValueError, match="topk_idx"):
        autograd.dispatch(x, idx[:3], 8)
    with pytest.raises(ValueError, match="topk_idx"):
        autograd.dispatch(x[None], idx, 8)


def test_rows_abi_arguments():
    m = _lib()
    lib, p = m.lib, ctypes.c_void_p(1 << 20)

    def spread(src=p, w=None, w_dtype=1, y=None, plan=p, dst=p, dw=None, T=4, h=64, E=8, k=2, dtype=1):
        return lib.q38moe_spread_rows(src, w, w_dtype, y, plan, dst, dw, T, h, E, k, dtype, None)

    def says(text):
        return text in lib.q38moe_last_error().decode()

    assert spread(dtype=5) == -1 and says("dtype")
    assert spread(E=65) == -1 and says("E must be")
    assert spread(k=9) == -1 and says("k must be")
    assert spread(h=100) == -1 and says("h must be")
    assert spread(w=p, w_dtype=1, dtype=2) == -1 and says("weights")
    assert spread(dw=p) == -1 and says("dw needs")
    assert spread(src=None) == -1 and says("src")
    assert spread(plan=None) == -1 and says("plan")
    assert lib.q38moe_rows_plan_ints(5, 6, 3) == 2 * 8 + 2 * 16 + 6 and lib.q38moe_rows_plan_ints(5, 65, 3) == -1
    assert lib.q38moe_dispatch_rows(p, p, 1, None, p, 4, 64, 8, 2, 1, None) == -1 and says("plan")
    assert lib.q38moe_dispatch_rows(None, p, 1, p, p, 4, 64, 8, 2, 1, None) == -1 and says("x must not")
    assert lib.q38moe_dispatch_rows(p, p, 1, p, p, 4, 100, 8, 2, 1, None) == -1 and says("h must be")
    assert spread(T=0) == 0 and spread(dst=None) == 0
    assert lib.q38moe_dispatch_rows(p, None, 1, p, p, 4, 64, 8, 2, 1, None) == -1 and says("topk_idx")
    assert lib.q38moe_collect_rows(None, None, 1, p, p, 4, 64, 8, 2, 1, None) == -1 and says("src")
    assert lib.q38moe_collect_rows(p, None, 1, None, p, 4, 64, 8, 2, 1, None) == -1 and says("plan")
    assert lib.q38moe_collect_rows(None, None, 1, None, None, 0, 64, 8, 2, 1, None) == 0


def test_model_loss_refuses_other_labels():
    """Before the trunk runs (it could not: the blocks have no CPU path)."""
    from q38 import prefill as P
    from q38.models.qwen3_8_moe import Qwen3_8MoeForCausalLM, Qwen3_8MoeTextConfig
    ids = torch.zeros(2, 8, dtype=torch.long)
    with torch.device("meta"):
        model = Qwen3_8MoeForCausalLM(Qwen3_8MoeTextConfig())
    with pytest.raises(ValueError, match="labels"):
        model(input_ids=ids, labels=ids[:, 1:])
    with pytest.raises(ValueError, match="labels"):
        P.Q38Prefill(P.PrefillConfig()).loss(ids, ids[:1])
    with pytest.raises(ValueError, match="labels"):
        P.next_token_loss(torch.zeros(2, 8, 64), torch.zeros(10, 64), ids[:, 1:])

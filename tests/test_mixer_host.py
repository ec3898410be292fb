"""Refusals of the token mixer's operators, before any launch (no GPU): the torch front end's checks and the C ABI's; the
axes of a rotation's frequencies."""
import ctypes

import pytest
import torch


def _lib():
    from q38.hip import _lib
    return _lib


def test_axis_map():
    from q38.hip import ops
    assert ops.rope_axis_map([4]).tolist() == [0, 0, 0, 0]
    assert ops.rope_axis_map([4, 2, 2]).tolist() == [0, 1, 2, 0, 1, 2, 0, 0]
    assert ops.rope_axis_map([2, 1, 1], interleaved=False).tolist() == [0, 0, 1, 2]
    sections = [11, 11, 10]
    found = ops.rope_axis_map(sections).tolist()
    assert [found.count(a) for a in range(3)] == sections and found[:6] == [0, 1, 2, 0, 1, 2]
    for bad in ([], [1, -1], [1, 2, 3, 4, 5], [0, 4]):
        with pytest.raises(ValueError, match="sections"):
            ops.rope_axis_map(bad)


def test_front_end_refusals():
    from q38.hip import autograd, ops
    q, k = torch.zeros(4, 2, 64), torch.zeros(4, 1, 64)
    w, pos, inv = torch.zeros(64), torch.arange(4), torch.ones(8)
    with pytest.raises(RuntimeError, match="CUDA/HIP tensor"):
        autograd.qk_norm_rope(q, k, w, w, pos, inv)
    with pytest.raises(TypeError, match="bf16 or fp32"):
        autograd.qk_norm_rope(q.half(), k.half(), w, w, pos, inv)
    x, g = torch.zeros(1, 4, 2, 64), torch.zeros(2)
    with pytest.raises(RuntimeError, match="CUDA/HIP tensor"):
        autograd.linear_attention(x, x, x, g)
    with pytest.raises(TypeError, match="bf16 or fp32"):
        autograd.linear_attention(x.double(), x, x, g)
    with pytest.raises(ValueError, match="log_decay has no gradient"):
        autograd.linear_attention(x, x, x, g.requires_grad_(True))
    with pytest.raises(RuntimeError, match="CUDA/HIP tensor"):
        ops.linear_attention_step(x[0], x[0], x[0], torch.zeros(4, 2, 64, 64), g)


def test_rope_abi_arguments():
    m = _lib()
    lib, p = m.lib, ctypes.c_void_p(1 << 20)

    def call(q=p, k=p, strides=(128, 64, 64, 64), wq=p, pos=p, n_axes=1, inv=p, qo=p, T=4, H=2, KV=1, d=64, rot=16, dtype=1):
        s = None if strides is None else (ctypes.c_int64 * 4)(*strides)
        return lib.q38moe_qk_norm_rope(q, k, s, wq, p, 1, pos, 1, None, n_axes, inv, qo, p, T, H, KV, d, rot, 1e-6, dtype, None)

    def says(text):
        return text in lib.q38moe_last_error().decode()

    assert call(dtype=5) == -1 and says("dtype")
    assert call(T=-1) == -1 and says("T must be")
    assert call(H=0) == -1 and says("H and KV")
    assert call(KV=5000) == -1 and says("H and KV")
    assert call(d=60) == -1 and says("d must be") and call(d=264) == -1 and call(d=0) == -1
    assert call(rot=12) == -1 and says("rot must be") and call(rot=72) == -1
    assert call(n_axes=5) == -1 and says("n_axes")
    assert call(strides=None) == -1 and says("strides")
    assert call(strides=(128, 60, 64, 64)) == -1 and says("stride 1")
    assert call(strides=(128, 64, -64, 64)) == -1 and says("stride 2")
    assert call(q=None) == -1 and says("q must not")
    assert call(qo=ctypes.c_void_p(8)) == -1 and says("q_out must be 16-byte aligned")
    assert call(wq=ctypes.c_void_p(8)) == -1 and says("q_norm")
    assert call(pos=None) == -1 and says("positions")
    assert call(inv=None) == -1 and says("inv_freq")

    def back(dy=p, wq=p, dwq=p, ws=p, n=1 << 30):
        s = (ctypes.c_int64 * 4)(128, 64, 64, 64)
        return lib.q38moe_qk_norm_rope_backward(dy, p, p, p, s, wq, p, 1, p, 1, None, 1, p, p, p, dwq, None, 4, 2, 1, 64, 16, 1e-6,
                                                ws, n, 1, None)

    assert back(dy=None) == -1 and says("d_q_out")
    assert back(wq=None) == -1 and says("needs the weight")
    assert back(ws=None) == -1 and says("workspace must")
    assert back(n=16) == -2 and says("workspace needs")
    n = ctypes.c_size_t()
    assert lib.q38moe_qk_norm_rope_workspace_bytes(4, 2, 1, 64, 16, ctypes.byref(n)) == 0 and n.value >= 2 * 64 * 4
    assert lib.q38moe_qk_norm_rope_workspace_bytes(4, 2, 1, 63, 16, ctypes.byref(n)) == -1


def test_linear_attention_abi_arguments():
    m = _lib()
    lib, p = m.lib, ctypes.c_void_p(1 << 20)

    def says(text):
        return text in lib.q38moe_last_error().decode()

    def shape(N=2, S=100, H=4, Hk=2, dk=64, dv=64, packed=0, backward=0):
        n = ctypes.c_size_t()
        rc = lib.q38moe_linear_attention_workspace_bytes(N, S, H, Hk, dk, dv, packed, backward, 1, ctypes.byref(n), None)
        return rc if rc else n.value

    assert shape(N=-1) == -1 and says("N must be")
    assert shape(S=-1) == -1 and says("S must be") and shape(S=(1 << 30) + 1) == -1
    assert shape(H=3) == -1 and says("H must be") and shape(Hk=0) == -1
    assert shape(dk=60) == -1 and says("dk must be") and shape(dk=136) == -1 and shape(dk=0) == -1
    assert shape(dv=4) == -1 and says("dv must be")
    assert shape(N=1 << 24, S=1, H=128, Hk=1) == -1 and says("too many")
    assert shape(S=64) == 0                                # one segment each: nothing to keep
    assert shape(packed=1) >= 4 * 7                        # the plan
    assert shape(S=65536, N=1) > 0
    assert shape(backward=1) >= 2 * 100 * 4 * 64 * 4       # a gradient for each head that shares
    # Many short sequences keep no states, however many they are.
    assert shape(N=10000, S=10000, packed=1) < (1 << 20) + shape(N=2, S=10000, packed=1)

    nine = (ctypes.c_int64 * 9)(25600, 256, 64, 12800, 128, 64, 12800, 128, 64)

    def fwd(q=p, v=p, strides=nine, g=p, cu=None, out=p, N=2, S=100, H=4, ws=p, n=1 << 40, dtype=1, saved=None,
            sn=0):
        return lib.q38moe_linear_attention_forward(q, p, v, strides, g, 1.0, None, cu, out, None, saved, sn, N, S, H, 2, 64,
                                                   64, ws, n, dtype, None)

    assert fwd(dtype=7) == -1
    assert fwd(strides=None) == -1 and says("strides")
    assert fwd(strides=(ctypes.c_int64 * 9)(*([64] * 8), 63)) == -1 and says("stride 8")
    assert fwd(q=None) == -1 and says("q must not")
    assert fwd(out=ctypes.c_void_p(8)) == -1 and says("out must be 16-byte")
    assert fwd(g=None) == -1 and says("log_decay")
    assert fwd(N=0, S=8, cu=p) == -1 and says("need a sequence")
    assert fwd(N=1, S=65536, ws=None) == -1 and says("workspace must")
    assert fwd(N=1, S=65536, n=16) == -2 and says("workspace needs")
    assert fwd(N=1, S=65536, saved=ctypes.c_void_p(8), sn=1 << 40) == -1 and says("saved must be 16-byte")
    assert fwd(N=1, S=65536, saved=p, sn=16) == -2 and says("saved needs")
    assert fwd(N=0) == 0

    def back(do=p, dv=p, ds=None):
        return lib.q38moe_linear_attention_backward(do, None, p, p, p, nine, p, 1.0, None, None, None, 0, None, None, dv, ds,
                                                    2, 100, 4, 2, 64,
                                                    64, p, 1 << 40, 1, None)

    assert back(do=None) == -1 and says("d_out")
    assert back(dv=ctypes.c_void_p(8)) == -1 and says("dv must be 16-byte")
    assert back(dv=None, ds=p) == -1 and says("comes with dv")
    assert back(dv=None) == 0

    six = (ctypes.c_int64 * 6)(256, 64, 128, 64, 128, 64)

    def step(q=p, strides=six, state=p, slots=p, out=p, B=2, pool=3, H=4, g=p):
        return lib.q38moe_linear_attention_step(q, p, p, strides, g, 1.0, state, slots, out, B, pool, H, 2, 64, 64, 1, None)

    assert step(B=-1) == -1 and says("N must be")
    assert step(H=5) == -1 and says("H must be")
    assert step(strides=None) == -1 and says("strides")
    assert step(pool=-1) == -1 and says("pool")
    assert step(pool=1, slots=None) == -1 and says("pool must hold")
    assert step(state=None) == -1 and says("state must not")
    assert step(q=None) == -1 and says("q must not")
    assert step(g=None) == -1 and says("log_decay")
    assert step(B=0) == 0


def test_step_refuses_gradients(monkeypatch):
    """Operands that want a gradient or carry a tangent are refused; not under no_grad."""
    from q38.hip import ops
    names = ("q", "k", "v", "state", "log_decay")

    def operands():
        x = torch.zeros(4, 2, 64)
        return dict(q=x, k=x.clone(), v=x.clone(), state=torch.zeros(4, 2, 64, 64), log_decay=torch.zeros(2))

    def refused(args, text):
        with monkeypatch.context() as m:  # as if the tensors were on a GPU
            m.setattr(ops, "_one_gpu", lambda *tensors: tensors[0].device)
            with pytest.raises(ValueError, match=text):
                ops.linear_attention_step(**args)

    def passed_on(args):
        with pytest.raises(RuntimeError, match="CUDA/HIP tensor"):
            ops.linear_attention_step(**args)

    for name in names:
        args = operands()
        args[name].requires_grad_(True)
        refused(args, "has no gradient")
        with torch.no_grad():
            passed_on(args)
        args[name] = args[name] * 1.0  # a state that a prompt has left, say
        refused(args, "has no gradient")
        args = operands()
        with torch.autograd.forward_ad.dual_level():
            passed_on(args)
            args[name] = torch.autograd.forward_ad.make_dual(args[name], torch.ones_like(args[name]))
            refused(args, "forward-mode")


def test_rope_refuses_a_gradient_of_the_frequencies():
    from q38.hip import autograd
    q, k = torch.zeros(4, 2, 64), torch.zeros(4, 1, 64)
    args = q, k, None, None, torch.arange(4), torch.ones(8, requires_grad=True)
    with pytest.raises(ValueError, match="inv_freq has no gradient"):
        autograd.qk_norm_rope(*args)
    with pytest.raises(ValueError, match="inv_freq has no gradient"):
        autograd.qk_norm_rope(*args[:5], args[5] * 1.0)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA/HIP tensor"):
        autograd.qk_norm_rope(*args)


def test_as_many_workgroups_as_a_launch_takes():
    """A launch's thread ids have 32 bits: workgroups of 4 threads for each column of a padded state (64 or 128), of both dk and dv
    backwards in bf16, of 256 in a step. Refused from there on, before anything is launched, and not below."""
    m = _lib()
    lib, n = m.lib, ctypes.c_size_t()

    def query(N, H, dk, dv, dtype, backward, packed=0):
        S = N if packed else 1
        return lib.q38moe_linear_attention_workspace_bytes(N, S, H, H, dk, dv, packed, backward, dtype, ctypes.byref(n), None)

    for dk, dv, dtype, backward, threads in [(128, 128, m.BF16, 0, 512), (64, 64, m.BF16, 0, 256), (128, 64, m.BF16, 0, 256),
                                             (64, 128, m.FP32, 0, 512), (128, 128, m.BF16, 1, 1024), (64, 64, m.BF16, 1, 512),
                                             (128, 64, m.BF16, 1, 768), (128, 64, m.FP32, 1, 512), (64, 64, m.FP32, 1, 256)]:
        for H in (16, 3):
            most = (1 << 32) // threads // H  # one-token sequences
            assert query(most + 1, H, dk, dv, dtype, backward) == -1, (dk, dv, dtype, backward, H)
            assert b"too many" in lib.q38moe_last_error()
            assert query(most - 64, H, dk, dv, dtype, backward) == 0, (dk, dv, dtype, backward, H)
    for H in (1 << 20, 1 << 29, 1 << 30, (1 << 31) - 1):  # nor where the product passes 64 bits
        assert query(1 << 24, H, 128, 128, m.BF16, 1) == -1 and b"too many" in lib.q38moe_last_error(), H
    assert lib.q38moe_linear_attention_workspace_bytes(1 << 24, 1 << 30, (1 << 31) - 1, 1, 128, 128, 0, 0, m.BF16, ctypes.byref(n),
                                                       None) == -1 and b"too many" in lib.q38moe_last_error()
    assert query(1 << 19, 16, 128, 128, 1, 0, packed=1) == -1 and query(1 << 18, 16, 128, 128, 1, 0, packed=1) == 0

    six, p = (ctypes.c_int64 * 6)(*([64] * 6)), ctypes.c_void_p(1 << 20)
    assert lib.q38moe_linear_attention_step(p, p, p, six, p, 1.0, p, p, p, 1 << 20, 1 << 20, 8, 8, 64, 64, 1, None) == -1
    assert b"too many" in lib.q38moe_last_error()

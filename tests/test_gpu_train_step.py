"""A training step's operators in one run: router, dispatch, experts of the caller's own (torch products per expert over
plan.counts), combine, residual, linear_cross_entropy, backward, clip_grad_norm_; and the model's loss without logits.

Every stage is held against float64 on the tensors that the stage before it gave in this very run, so the bounds are those
of one stage. u = 2^-24, v = the half step of the tensors' type. A product of K terms summed in fp32 is off by 2 (K + 20) u
of the sum of its terms' sizes; each stored tensor adds v of its value. The router's logits, which have tests of their own,
are taken as the kernel gave them."""
import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def _params(dtype, dev, T=150, h=128, E=8, k=2, V=777, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)

    def r(*s, std=1.0):
        return (torch.randn(*s, generator=g, device=dev) * std).to(dtype)

    x, w_r = r(T, h), r(E, h, std=h ** -0.5)
    up = r(E, h, h, std=0.5 * h ** -0.5)
    head = r(V, h, std=0.5 * h ** -0.5)
    t = torch.randint(0, V, (T,), generator=g, device=dev)
    t[torch.rand(T, generator=g, device=dev) < 0.2] = -100
    return x, w_r, up, head, t, k


def _step(x, w_r, up, head, t, k):
    """The step as a user writes it. The leaves' gradients are in .grad, and those of the tensors between that are given back."""
    from q38.hip import autograd
    E = up.shape[0]
    logits, w, idx = autograd.router(x, w_r, k)
    rows, plan = autograd.dispatch(x, idx, E)
    y = torch.cat([part @ up[e].t() for e, part in enumerate(rows.split(plan.counts.tolist()))])
    hidden = x + autograd.combine(y, w, plan)
    loss = autograd.linear_cross_entropy(hidden, head, t)
    mid = dict(logits=logits, w=w, rows=rows, y=y, hidden=hidden)
    for name in ("w", "rows", "y", "hidden"):
        mid[name].retain_grad()
    loss.backward()
    return loss.detach(), idx.detach(), mid


def _store(exact, e, v):
    return exact, e + v * (exact.abs() + e)


def _mm(a, b, v, ea=None):
    """a @ b, and its error where a is off by ea: the operand's, the sum's and the store's."""
    size = a.abs() if ea is None else a.abs() + ea
    e = 2 * (a.shape[1] + 20) * U * (size @ b.abs())
    return _store(a @ b, e if ea is None else e + ea @ b.abs(), v)


def _stages(leaves, t, k, loss, idx, mid):
    """(name, got, exact, bound) of every stage of one step."""
    v = torch.finfo(leaves[0].dtype).eps / 2
    x, w_r, up, head = (a.detach().double() for a in leaves)
    g = {n: mid[n].grad.double() for n in ("w", "rows", "y", "hidden")}
    lg, w, rows, y, hid = (mid[n].detach().double() for n in ("logits", "w", "rows", "y", "hidden"))
    T, E, V = x.shape[0], up.shape[0], head.shape[0]
    idx = idx.long()
    flat = idx.reshape(-1).cpu()
    perm = torch.sort(flat, stable=True).indices.to(x.device)     # row -> pair, experts in order
    inv = torch.empty_like(perm).scatter_(0, perm, torch.arange(T * k, device=x.device)).view(T, k)
    tok = perm // k
    counts = torch.bincount(flat, minlength=E).tolist()
    zero = torch.zeros((), dtype=torch.float64, device=x.device)
    yield "rows", rows, x[tok], zero
    # Routing weights: a softmax over the chosen logits, about 16 roundings in fp32, one store.
    p = torch.softmax(lg, 1)
    pv = p.gather(1, idx)
    s = pv.sum(1, keepdim=True)
    yield "w", w, *_store(pv / s, 64 * U * pv / s, v)
    parts = [_mm(r, up[e].t().contiguous(), v) for e, r in enumerate(rows.split(counts))]
    yield "y", y, torch.cat([a for a, _ in parts]), torch.cat([e for _, e in parts])
    wy = w[..., None] * y[inv]
    o, eo = _store(wy.sum(1), 20 * U * wy.abs().sum(1), v)
    yield "hidden", hid, *_store(x + o, eo, v)
    # The loss: logits off by dz; the log-sum-exp's and the subtractions' roundings.
    keep = t != -100
    n = int(keep.sum())
    z = hid @ head.t().contiguous()
    dz = 2 * (x.shape[1] + 1) * U * (hid.abs() @ head.abs().t().contiguous()).amax(1)
    lse = torch.logsumexp(z, 1)
    at = torch.where(keep, t, torch.zeros_like(t))
    per = (lse - z.gather(1, at[:, None])[:, 0]) * keep
    rel = (400 + V / 512) * U
    eper = (2 * dz + rel + 4 * U * (per.abs() + 2 * lse.abs())) * keep
    yield "loss", loss.double(), per.sum() / n, eper.sum() / n + 2 * U * per.sum() / n
    P = torch.exp(z - lse[:, None])
    ds = P.clone()
    ds.scatter_add_(1, at[:, None], -torch.ones_like(lse)[:, None])
    eds = (ds.abs() * (v + 8 * U) + P * (2 * dz + rel + 32 * U)[:, None]) * keep[:, None] / n
    ds = ds * keep[:, None] / n
    yield "d hidden", g["hidden"], *_mm(ds, head, v, eds)
    yield "d head", leaves[3].grad.double(), *_mm(ds.t().contiguous(), hid, v, eds.t().contiguous())
    # combine's backward from hidden's gradient: rows' w dh, weights' <dh, y>.
    dh = g["hidden"]
    dy = w.reshape(-1)[perm][:, None] * dh[tok]
    yield "d y", g["y"], *_store(dy, 4 * U * dy.abs(), v)
    terms = dh[:, None] * y[inv]
    yield "d w", g["w"], *_store(terms.sum(2), 2 * (x.shape[1] + 20) * U * terms.abs().sum(2), v)
    parts = [(_mm(a, up[e], v), _mm(a.t().contiguous(), r, v))
             for e, (a, r) in enumerate(zip(g["y"].split(counts), rows.split(counts)))]
    yield "d rows", g["rows"], torch.cat([a[0] for a, _ in parts]), torch.cat([a[1] for a, _ in parts])
    yield "d experts", leaves[2].grad.double(), torch.stack([a[0] for _, a in parts]), torch.stack([a[1] for _, a in parts])
    # The router's backward: dv = (dw - <dw, w>) / s, dz = p (dp - <dp, p>). p <= s for each expert, so with G the largest
    # |dw| of a row the roundings of each bracket add less than 64 u G to dz.
    dv = (g["w"] - (g["w"] * (pv / s)).sum(1, keepdim=True)) / s
    dp = torch.zeros_like(p).scatter_(1, idx, dv)
    dlg = p * (dp - (dp * p).sum(1, keepdim=True))
    dlg, edlg = _store(dlg, 128 * U * g["w"].abs().amax(1, keepdim=True).expand_as(dlg), v)
    yield "d router", leaves[1].grad.double(), *_mm(dlg.t().contiguous(), x, v, edlg.t().contiguous())
    # Three paths reach x (dispatch's sums k rows first); their sum is stored twice on the way.
    back = g["rows"][inv]
    a, ea = _store(back.sum(1), 20 * U * back.abs().sum(1), v)
    b, eb = _mm(dlg, w_r, v, edlg)
    exact, e = dh + a + b, ea + eb
    yield "d x", leaves[0].grad.double(), exact, e + 2 * v * (dh.abs() + a.abs() + b.abs() + e)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_step(gpu, dtype):
    from q38.hip import ops
    x, w_r, up, head, t, k = _params(dtype, gpu)
    leaves = [a.requires_grad_(True) for a in (x, w_r, up, head)]
    print(f"step {dtype}", flush=True)
    loss, idx, mid = _step(x, w_r, up, head, t, k)
    for name, got, exact, e in _stages(leaves, t, k, loss, idx, mid):
        assert got.shape == exact.shape
        err = (got - exact).abs()
        assert bool((err <= e + 1e-38).all()), f"{name}: worst {float((err / (e + 1e-38)).max()):.3f} of the bound"
        # The bound is small beside the whole, or it would say nothing.
        assert float(e.norm()) < (1e-3 if dtype == torch.float32 else 0.1) * float(exact.norm()), name
    before = [a.grad.clone() for a in leaves]
    norm64 = float(torch.cat([b.double().reshape(-1) for b in before]).norm())
    got = ops.clip_grad_norm_(leaves, 0.5 * norm64)
    assert abs(float(got) - norm64) <= norm64 * (U + 1e-12)
    c = 0.5 * norm64 / (norm64 + 1e-6)
    for b, a in zip(before, leaves):
        exact = b.double() * c
        assert bool(((a.grad.double() - exact).abs() <= exact.abs() * (torch.finfo(dtype).eps / 2 + 5 * U) + 1.5e-45).all())


def test_step_again_and_on_another_stream(gpu):
    """The same bits from a second run, and from one on another stream."""
    from q38.hip import ops
    x, w_r, up, head, t, k = _params(torch.bfloat16, gpu, seed=1)
    leaves = [a.requires_grad_(True) for a in (x, w_r, up, head)]

    def run():
        for a in leaves:
            a.grad = None
        loss = _step(x, w_r, up, head, t, k)[0]
        norm = ops.clip_grad_norm_(leaves, 0.1)
        return [loss, norm] + [a.grad for a in leaves]

    first = run()
    again = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        there = run()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for a, b, c in zip(first, again, there):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_two_captured_steps(gpu):
    """The step's calls below autograd in two graphs, replayed in turn: neither sees the other's workspaces, and a
    replay reads the inputs as they are then."""
    from q38.hip import ops

    def calls(x, idx, w, head, t, g):
        plan = ops.RowsPlan(idx, 8)
        rows = ops.dispatch_rows(x, plan)
        hid = ops.collect_rows(rows, plan, w)
        loss, lse, mean, scale = ops.linear_ce_forward(hid, head, t, -100, "mean")
        dx, dw = ops.linear_ce_backward(g, hid, head, t, lse, -100, scale, True, True)
        d_rows, d_w = ops.spread_rows(dx, plan, w, rows, True)
        norm = ops.clip_grads([dw, d_rows], 0.01, 2.0)
        return mean, dw, d_rows, d_w, norm

    args = []
    for seed in range(2):
        x, w_r, up, head, t, k = _params(torch.bfloat16, gpu, T=300 + 7 * seed, seed=seed)
        idx = torch.topk(x.float() @ w_r.float().t().contiguous(), k, dim=1).indices
        w = torch.softmax(idx.float(), 1).to(torch.bfloat16)
        args.append((x, idx, w, head, t, torch.ones((), device=gpu)))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for a in args:
            calls(*a)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for a in args:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(calls(*a))
        graphs.append(graph)
    for turn in range(3):
        for a in args:
            a[0].mul_(0.75)       # new inputs for every replay
            a[4].copy_(a[4].roll(1))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for i, a in enumerate(args):
            for name, got, want in zip(("loss", "dw", "d_rows", "d_w", "norm"), outs[i], calls(*a)):
                assert torch.equal(got, want), (turn, i, name)


def _tiny(gpu, dtype):
    from q38 import prefill as P
    cfg = P.PrefillConfig(vocab=300, hidden=128, layers=2, heads=4, kv_heads=2, lin_k_heads=2, lin_v_heads=4, experts=8,
                          topk=2, moe_ffn=64, shared_ffn=64, ngram_rows=512,
                          layer_types=("linear_attention", "full_attention"))
    model = P.Q38Prefill(cfg).load_params(P.init_params(cfg, 3)).to(device=gpu, dtype=dtype)
    return model, P.make_ids(2, 200, cfg, seed=9, eos_every=64).to(gpu)


def _near_logits_loss(loss, hs, head, labels, reduction):
    """loss against float64 over the hidden states it was made from."""
    z = hs.double() @ head.double().t().contiguous()
    nxt = F.pad(labels[:, 1:], (0, 1), value=-100)
    want = F.cross_entropy(z.view(-1, z.shape[-1]), nxt.reshape(-1), ignore_index=-100, reduction=reduction)
    dz = 2 * (hs.shape[-1] + 20) * U * float((hs.double().abs() @ head.double().abs().t().contiguous()).max())
    rows = 1 if reduction != "sum" else int((nxt != -100).sum())
    lim = rows * (2 * dz + (500 + 16 * float(z.abs().max()) + 12 * z.shape[-1]) * U)
    assert loss.dtype == torch.float32
    assert bool(((loss.double().reshape(-1) - want).abs() <= lim).all())


def test_prefill_loss(gpu):
    """Q38Prefill.loss against float64 over the same hidden states; the forward's results stay."""
    from q38 import prefill as P
    model, ids = _tiny(gpu, torch.bfloat16)
    before = model(ids)
    head = model.model.embed_tokens.weight
    with torch.no_grad():
        hs = P.trunk_forward(model.model, model.cfg, ids, model._moe)
    for reduction in ("mean", "sum", "none"):
        loss = model.loss(ids, reduction=reduction)
        assert loss.shape == (ids.shape if reduction == "none" else ())
        _near_logits_loss(loss, hs, head, ids, reduction)
    labels = ids.clone()
    labels[0, :150] = -100
    labels[1] = -100
    _near_logits_loss(model.loss(ids, labels), hs, head, labels, "mean")
    assert float(model.loss(ids, torch.full_like(ids, -100))) == 0.0
    assert float(model.loss(ids[:, :1])) == 0.0  # one token has no next one
    assert torch.equal(model(ids), before)
    with pytest.raises(ValueError, match="labels"):
        model.loss(ids, labels[:, 1:])


def test_causal_lm_labels(gpu):
    """labels add the loss and change nothing else; without logits the loss is the same."""
    from q38.models.qwen3_8_moe import Qwen3_8MoeForCausalLM, Qwen3_8MoeTextConfig
    torch.manual_seed(0)
    cfg = Qwen3_8MoeTextConfig(vocab_size=300, hidden_size=128, num_hidden_layers=4, num_attention_heads=4,
                               num_key_value_heads=2, linear_num_key_heads=2, linear_num_value_heads=4, num_experts=8,
                               num_experts_per_tok=2, moe_intermediate_size=64, shared_expert_intermediate_size=64,
                               ngram_rows=512, router_aux_loss_coef=0.25)
    model = Qwen3_8MoeForCausalLM(cfg).eval().to(device=gpu, dtype=torch.bfloat16)
    ids = torch.randint(0, 299, (2, 130), device=gpu)
    labels = ids.clone()
    labels[:, :40] = -100
    plain = model(input_ids=ids)
    out = model(input_ids=ids, labels=labels)
    assert plain.loss is None and torch.equal(out.logits, plain.logits)
    last = model(input_ids=ids, labels=labels, logits_to_keep=1)
    assert torch.equal(last.loss, out.loss) and last.logits.shape[1] == 1
    # The same rows of the same product, but for the order of its sums over 128 terms and its rounding.
    z = plain.logits[:, -1:].float()
    assert bool(((last.logits.float() - z).abs() <= 2 * 2.0 ** -8 * z.abs() + 1e-3).all())
    none = model(input_ids=ids, labels=labels, logits_to_keep=None)
    assert none.logits is None and torch.equal(none.loss, out.loss)
    aux = model(input_ids=ids, labels=labels.cpu(), output_router_logits=True)
    assert torch.equal(aux.loss, out.loss + 0.25 * aux.aux_loss)
    with torch.no_grad():
        z = plain.logits.double()  # logits rounded to bf16: each off by at most 2^-8 of its size
    want = F.cross_entropy(z[:, :-1].reshape(-1, 300), labels[:, 1:].reshape(-1), ignore_index=-100)
    assert abs(float(out.loss) - float(want)) <= 2 * 2.0 ** -8 * float(z.abs().max()) * 1.01 + 1e-5
    with pytest.raises(ValueError, match="labels"):
        model(input_ids=ids, labels=labels[:, 1:])


def test_two_streams_at_once(gpu):
    """Steps under way on two streams at the same time give the bits that they give alone."""
    from q38.hip import ops
    sets = [[a.requires_grad_(a.is_floating_point()) if isinstance(a, torch.Tensor) else a
             for a in _params(torch.bfloat16, gpu, T=400 + 9 * s, seed=s)] for s in range(2)]

    def run(args):
        x, w_r, up, head, t, k = args
        from q38.hip import autograd
        logits, w, idx = autograd.router(x, w_r, k)
        rows, plan = autograd.dispatch(x, idx, up.shape[0])
        hidden = x + autograd.combine(rows, w, plan)
        loss = autograd.linear_cross_entropy(hidden, head, t)
        grads = torch.autograd.grad(loss, (x, w_r, head))
        return [loss.detach(), ops.clip_grads(list(grads), 0.1), *grads]

    alone = [run(a) for a in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(run(sets[i]))
    torch.cuda.synchronize()
    for want, many in zip(alone, got):
        for one in many:
            assert all(torch.equal(a, b) for a, b in zip(want, one))

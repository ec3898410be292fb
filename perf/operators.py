"""Timing cases of the operators around the MoE block in a training step, over the sizes they are called at.

* ``loss``: ``autograd.linear_cross_entropy``, the softmax cross entropy of the tied head from hidden states,
  the head's weight and target ids, without the logits. Forward alone (evaluation), or with the gradients of
  both operands for a given gradient of the loss (training).
* ``clip``: ``ops.clip_grads``, the global norm of many gradients and the gradients scaled to a largest norm. The
  gradients are views of one flat buffer, as a data-parallel wrapper's buckets are; the scaled ones go to views of
  another, which the optimizer reads.
* ``rows``: ``autograd.dispatch`` and ``autograd.combine``, tokens sorted by expert and the experts' outputs brought back
  with the routing weights, for experts that are the user's own. Forward alone, or with every gradient.

Shapes are those of the benchmark configurations (hidden 1024, vocabulary 10112, 64 experts of which each token takes
5; hidden 256 in fp32; hidden 2048) and generic ones next to them. Outside ``own`` every operator runs in its plain form:
elementary torch operations in fp32, rounded once. ``exact`` restates them in float64.
"""
import math
import sys
from pathlib import Path

import torch

own = False

_PKG = str(Path(__file__).resolve().parents[1] / "qwen35-moe-sparse_amd")
_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
_IGNORE = -100


def _loss(name, T, h, V, dtype="bf16", train=True, reduction="mean", ignored=0.0):
    case = dict(kind="loss", T=T, h=h, V=V, dtype=dtype, train=train, reduction=reduction, ignored=ignored)
    return dict(case, name=name) if name else case


def _clip(name, layers, h, V, dtype, p=2.0, ngram=0, small=False):
    case = dict(kind="clip", layers=layers, h=h, V=V, dtype=dtype, p=p, ngram=ngram, small=small)
    return dict(case, name=name) if name else case


def _rows(name, T, h, dtype="bf16", train=True, E=64, k=5, dropped=0.0):
    case = dict(kind="rows", T=T, h=h, E=E, k=k, dtype=dtype, train=train, dropped=dropped)
    return dict(case, name=name) if name else case


def listed():
    return [
        # Scoring the continuation tokens of a prompt, each apart: the head's weight is read for almost no work.
        _loss("score_61", 61, 1024, 10112, train=False, reduction="none"),
        # Evaluation of a packed batch, every token's loss: 4 x 4096 tokens, forward only.
        _loss("eval_16384", 16384, 1024, 10112, train=False, reduction="none"),
        # A ragged micro-batch of a fine-tuning run: prompts' targets ignored, forward and gradients.
        _loss("tune_1777", 1777, 1024, 10112, ignored=0.4),
        # The training step's loss at the headline size.
        _loss("train_16384", 16384, 1024, 10112),
        # A wide model with a large, odd vocabulary.
        _loss("wide_4099", 4099, 2048, 50021),
        # An fp32 model; the loss of each token apart, weighted by the caller.
        _loss("fp32_515", 515, 256, 10112, dtype="fp32", reduction="none", ignored=0.05),
        # The gradients of one layer's small parameters (norms, router, decays): latency.
        _clip("clip_small", 1, 1024, 0, "bf16", small=True),
        # One layer of the 12-layer model, bf16.
        _clip("clip_layer", 1, 1024, 0, "bf16"),
        # The whole model with fp32 gradients: 12 layers, embedding and N-gram tables, about 300 tensors.
        _clip("clip_model", 12, 1024, 10112, "fp32", ngram=131072),
        # A decode step of a batch through the user's own experts.
        _rows("rows_61", 61, 1024, train=False),
        # The training step at the headline size.
        _rows("rows_16384", 16384, 1024),
        # fp32, with pairs that an expert's capacity dropped.
        _rows("rows_fp32_2047", 2047, 256, dtype="fp32", dropped=0.1),
    ]


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def draw(rng):
    kind = rng.choice(["loss"] * 3 + ["clip", "rows", "rows"])
    if kind == "loss":
        dtype = "fp32" if rng.random() < 0.2 else "bf16"
        h = rng.choice([64, 256, 512, 768, 1024, 1024, 1344, 2048])
        V = _log_uniform(rng, 300, 50021)
        most = 1.0e11 if dtype == "bf16" else 2.0e9  # T h V of the largest cases of the type
        T = _log_uniform(rng, 1, max(1, min(16384, int(most / (h * V)))))
        return _loss(None, T, h, V, dtype=dtype, train=rng.random() < 0.7,
                     reduction=rng.choice(["mean", "sum", "none"]), ignored=rng.choice([0.0, 0.0, 0.1, 0.7]))
    if kind == "clip":
        return _clip(None, rng.randint(1, 6), rng.choice([256, 320, 512, 1024]), _log_uniform(rng, 100, 20000),
                     rng.choice(["bf16", "fp32"]), p=rng.choice([1.0, 2.0, 2.0, math.inf]), small=rng.random() < 0.3)
    E, k = rng.choice([(64, 5), (64, 8), (60, 4), (8, 2), (16, 1)])
    return _rows(None, _log_uniform(rng, 1, 16384), rng.choice([64, 256, 512, 1024, 1088, 2048]),
                 dtype=rng.choice(["bf16", "bf16", "fp32"]), train=rng.random() < 0.7, E=E, k=k,
                 dropped=rng.choice([0.0, 0.0, 0.15]))


# ---- inputs -----------------------------------------------------------------------------------

def _clip_shapes(case):
    """Shapes of the gradients: the parameters of ``layers`` layers at hidden h (the 12-layer model's widths at
    1024), the embedding and the N-gram tables where asked for."""
    h, I, E = case["h"], case["h"] // 4, 64
    heads = max(1, round(1.2 * h / 64)) * 2
    nk = max(1, round(0.8 * h / 64))
    kd, vd = nk * 64, 3 * nk * 64
    shapes = []
    for i in range(case["layers"]):
        shapes += [(h,), (h,), (E, h), (1, h), (24, h // 8), (4,), (4,), (4, 4), (3,)]
        if i % 4 == 3:
            shapes += [(64,), (64,)]
            if not case["small"]:
                shapes += [(heads * 128, h), (128, h), (128, h), (h, heads * 64)]
        else:
            shapes += [(3 * nk,), (3 * nk,), (64,), (3 * nk, h), (3 * nk, h), (2 * kd + vd, 1, 4)]
            if not case["small"]:
                shapes += [(2 * kd + vd, h), (vd, h), (h, vd)]
        if not case["small"]:
            shapes += [(E, 2 * I, h), (E, h, I), (I, h), (I, h), (h, I), (h // 8, 4 * h), (h // 8, 4 * h)]
    if case["V"]:
        shapes += [(case["V"], h), (h,)]
    if case["ngram"]:
        shapes += [(case["ngram"], h), (case["ngram"], h), (h, h), (h,)]
    return shapes


def _views(flat, shapes):
    """Views of the flat buffer, each on a 16-byte boundary."""
    out, at = [], 0
    for s in shapes:
        n = math.prod(s)
        out.append(flat[at:at + n].view(s))
        at += -(-n // 8) * 8
    return out


def _flat_size(shapes):
    return sum(-(-math.prod(s) // 8) * 8 for s in shapes)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[case["dtype"]]

    def normal(shape, std, dtype=dt):
        return torch.randn(shape, generator=g, device="cuda").mul_(std).to(dtype)

    s = dict(case=case)
    if case["kind"] == "loss":
        T, h, V = case["T"], case["h"], case["V"]
        s["x"], s["w"] = normal((T, h), 1.0), normal((V, h), 2.0 / math.sqrt(h))
        s["targets"] = torch.randint(0, V, (T,), generator=g, device="cuda")
        at = torch.randperm(T, generator=g, device="cuda")[:int(T * case["ignored"])]
        s["targets"][at] = _IGNORE
        if case["train"]:
            s["x"].requires_grad_(True)
            s["w"].requires_grad_(True)
            s["g"] = (torch.rand(T, generator=g, device="cuda") if case["reduction"] == "none"
                      else torch.rand((), generator=g, device="cuda") + 0.5)
    elif case["kind"] == "clip":
        shapes = _clip_shapes(case)
        flat = torch.zeros(_flat_size(shapes), device="cuda", dtype=dt)
        s["grads"] = _views(flat, shapes)
        for t in s["grads"]:  # each parameter's gradients have a size of their own
            t.copy_(torch.randn(t.shape, generator=g, device="cuda").mul_(float(t.numel()) ** -0.5))
        s["out_flat"] = torch.zeros_like(flat)
        s["out"] = _views(s["out_flat"], shapes)
    else:
        T, h, E, k = (case[n] for n in ("T", "h", "E", "k"))
        s["x"] = normal((T, h), 1.0)
        s["idx"] = torch.topk(torch.randn(T, E, generator=g, device="cuda"), k, dim=1).indices
        w = torch.rand(T, k, generator=g, device="cuda") + 0.05
        s["w"] = (w / w.sum(1, keepdim=True)).to(dt)
        if case["dropped"]:  # the sentinel that routing with a capacity leaves
            s["idx"][torch.rand(T, k, generator=g, device="cuda") < case["dropped"]] = E
        s["y"] = normal((T * k, h), 0.5)
        if case["train"]:
            for n in ("x", "w", "y"):
                s[n].requires_grad_(True)
            s["d_rows"], s["d_out"] = normal((T * k, h), 0.1), normal((T, h), 0.1)
    return s


# ---- the calls --------------------------------------------------------------------------------

def _hip():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    from q38.hip import autograd, ops

    return autograd, ops


def run(s):
    case = s["case"]
    return {"loss": _run_loss, "clip": _run_clip, "rows": _run_rows}[case["kind"]](s, case)


def _run_loss(s, case):
    if own:
        autograd, _ = _hip()
        loss = autograd.linear_cross_entropy(s["x"], s["w"], s["targets"], ignore_index=_IGNORE,
                                             reduction=case["reduction"])
        if not case["train"]:
            return {"loss": loss}
        dx, dw = torch.autograd.grad(loss, (s["x"], s["w"]), s["g"])
        return {"loss": loss.detach(), "dx": dx, "dw": dw}
    x, w = s["x"].detach().float(), s["w"].detach().float()
    kept = s["targets"] != _IGNORE
    at = torch.where(kept, s["targets"], torch.zeros_like(s["targets"]))[:, None]
    z = x @ w.t()
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    each = torch.where(kept, (top + torch.log(total) - z.gather(1, at))[:, 0], torch.zeros_like(top[:, 0]))
    count = kept.sum().clamp(min=1)
    loss = {"none": lambda: each, "sum": lambda: each.double().sum().float(),
            "mean": lambda: (each.double().sum() / count).float()}[case["reduction"]]()
    if not case["train"]:
        return {"loss": loss}
    g = s["g"] / count if case["reduction"] == "mean" else s["g"]
    g = (g * kept)[:, None]
    dz = e.div_(total).mul_(g)
    dz.scatter_add_(1, at, -g)
    return {"loss": loss, "dx": (dz @ w).to(s["x"].dtype), "dw": (dz.t() @ x).to(s["w"].dtype)}


_MAX_NORM = 1.0


def _run_clip(s, case):
    if own:
        _, ops = _hip()
        norm = ops.clip_grads(s["grads"], _MAX_NORM, norm_type=case["p"], out=s["out"])
        return {"norm": norm, "grads": s["out_flat"]}
    p = case["p"]
    if p == math.inf:
        norm = torch.stack([t.abs().amax().float() for t in s["grads"]]).amax()
    else:
        parts = [(t.float().abs() if p == 1 else t.float().square()).sum(dtype=torch.float64) for t in s["grads"]]
        norm = torch.stack(parts).sum().pow(1.0 / p).float()
    scale = (_MAX_NORM / (norm + 1e-6)).clamp(max=1.0)
    for t, o in zip(s["grads"], s["out"]):
        o.copy_(t.float() * scale)
    return {"norm": norm, "grads": s["out_flat"]}


def _run_rows(s, case):
    T, h, E, k = (case[n] for n in ("T", "h", "E", "k"))
    if own:
        autograd, _ = _hip()
        rows, plan = autograd.dispatch(s["x"], s["idx"], E)
        out = autograd.combine(s["y"], s["w"], plan)
        if not case["train"]:
            return {"rows": rows, "counts": plan.counts, "out": out}
        dx, dw, dy = torch.autograd.grad((rows, out), (s["x"], s["w"], s["y"]), (s["d_rows"], s["d_out"]))
        return {"rows": rows.detach(), "counts": plan.counts, "out": out.detach(), "dx": dx, "dw": dw, "dy": dy}
    x, w, y = s["x"].detach(), s["w"].detach().float(), s["y"].detach().float()
    dt = x.dtype
    pairs = s["idx"].reshape(-1)
    pairs = torch.where((pairs >= 0) & (pairs < E), pairs, torch.full_like(pairs, E))
    perm = torch.argsort(pairs, stable=True)
    filled = (pairs[perm] < E)[:, None]
    counts = (pairs[:, None] == torch.arange(E, device=x.device)).sum(0).to(torch.int32)
    token = perm // k
    rows = torch.where(filled, x[token], torch.zeros((), dtype=dt, device=x.device))
    inv = torch.empty_like(perm).scatter_(0, perm, torch.arange(T * k, device=x.device))
    kept = (pairs < E).view(T, k)
    zero = torch.zeros((), device=x.device)
    back = torch.where(kept[..., None], y[inv].view(T, k, h), zero)
    out = (back * w[..., None]).sum(1).to(dt)
    if not case["train"]:
        return {"rows": rows, "counts": counts, "out": out}
    d_out = s["d_out"].float()
    dx = torch.where(kept[..., None], s["d_rows"].float()[inv].view(T, k, h), zero).sum(1)
    dw = (back * d_out[:, None]).sum(2)
    dy = torch.where(filled, d_out[token] * w.reshape(-1)[perm][:, None], zero)
    return {"rows": rows, "counts": counts, "out": out, "dx": dx.to(dt), "dw": dw.to(dt), "dy": dy.to(dt)}


# ---- the work, and the values in float64 ------------------------------------------------------

def work(case):
    b = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] == "loss":
        T, h, V = case["T"], case["h"], case["V"]
        n = T - int(T * case["ignored"])
        product, operands = 2 * n * h * V, b * (n * h + V * h)
        rows = 8 * T + (4 * T if case["reduction"] == "none" else 4)
        if not case["train"]:
            return {"bytes": operands + rows, "flops": product}
        return {"bytes": operands + rows + b * (T * h + V * h), "flops": 3 * product}
    if case["kind"] == "clip":
        n = sum(math.prod(s) for s in _clip_shapes(case))
        return {"bytes": 2 * b * n, "flops": 3 * n}
    T, h, k = case["T"], case["h"], case["k"]
    few, many, pairs = b * T * h, b * T * k * h, T * k
    forward = few + many + many + few + (8 + b) * pairs
    if not case["train"]:
        return {"bytes": forward, "flops": 2 * pairs * h}
    return {"bytes": forward + many + few + few + many + b * pairs, "flops": 6 * pairs * h}


def exact(case, seed):
    s = prepare(case, seed)
    s = {n: v.detach() if isinstance(v, torch.Tensor) else v for n, v in s.items()}
    return {"loss": _exact_loss, "clip": _exact_clip, "rows": _exact_rows}[case["kind"]](s, case)


def _exact_loss(s, case):
    x, w, targets = s["x"].double(), s["w"].double(), s["targets"]
    keep = torch.nonzero(targets != _IGNORE)[:, 0]
    n, V = keep.numel(), case["V"]
    xk, tk = x[keep], targets[keep]
    logp = torch.log_softmax(xk @ w.t().contiguous(), dim=1)
    rows = torch.zeros(case["T"], dtype=torch.float64, device=x.device)
    rows[keep] = -logp[torch.arange(n, device=x.device), tk]
    loss = rows if case["reduction"] == "none" else rows.sum()
    if case["reduction"] == "mean":
        loss = loss / max(n, 1)
    if not case["train"]:
        return {"loss": loss}
    g = s["g"].double()
    if case["reduction"] == "none":
        g = g[keep]
    else:
        g = (g / max(n, 1) if case["reduction"] == "mean" else g).expand(n)
    d = logp.exp_()
    d[torch.arange(n, device=x.device), tk] -= 1.0
    d *= g[:, None]
    dx = torch.zeros_like(x)
    dx[keep] = d @ w
    return {"loss": loss, "dx": dx, "dw": d.t().contiguous() @ xk}


def _exact_clip(s, case):
    p = case["p"]
    norms = torch.stack([torch.linalg.vector_norm(t.double(), p) for t in s["grads"]])
    norm = torch.linalg.vector_norm(norms, p)
    scale = min(1.0, _MAX_NORM / (float(norm) + 1e-6))
    shapes = _clip_shapes(case)
    flat = torch.zeros(_flat_size(shapes), dtype=torch.float64, device="cuda")
    for t, o in zip(s["grads"], _views(flat, shapes)):
        o.copy_(t.double() * scale)
    return {"norm": norm, "grads": flat}


def _exact_rows(s, case):
    T, h, E, k = (case[n] for n in ("T", "h", "E", "k"))
    idx = s["idx"].cpu().reshape(-1)
    order = [torch.nonzero(idx == e)[:, 0] for e in range(E)]
    perm = torch.cat(order).to(s["x"].device)  # pairs by expert, ascending within one; dropped pairs nowhere
    n = perm.numel()
    token = perm // k
    x, w, y = s["x"].double(), s["w"].double().reshape(-1), s["y"].double()
    rows = torch.zeros(T * k, h, dtype=torch.float64, device=x.device)
    rows[:n] = x[token]
    out = torch.zeros(T, h, dtype=torch.float64, device=x.device)
    out.index_add_(0, token, y[:n] * w[perm][:, None])
    found = {"rows": rows, "counts": None, "out": out}
    if not case["train"]:
        return found
    d_out, d_rows = s["d_out"].double(), s["d_rows"].double()
    dx = torch.zeros_like(out).index_add_(0, token, d_rows[:n])
    dw = torch.zeros(T * k, dtype=torch.float64, device=x.device)
    dw[perm] = (d_out[token] * y[:n]).sum(1)
    dy = torch.zeros_like(rows)
    dy[:n] = d_out[token] * w[perm][:, None]
    return dict(found, dx=dx, dw=dw.view(T, k), dy=dy)

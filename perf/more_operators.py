"""What a student model's training step needs around the optimizer, as cases that can be timed and compared: layer norm, the gated
feed-forward block and distillation from a teacher's top logits.

A case names an operator, its sizes, the type of what it works on and the form of the call.  One pass is the forward and the
backward pass through the operator as autograd makes them, or a forward pass alone where the case says ``train=False``.
"""

import math
import random

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-5

# ---------------------------------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------------------------------


def listed():
    norm = dict(op="layer_norm", train=True, weight="same", bias=True)
    ffn = dict(op="gated_ffn", train=True, act="silu")
    distil = dict(op="distillation", form="autograd", masked=True, padded=True, temperature=2.0)
    return [
        # a batch of 128 through a perceptron of width 128: all latency
        dict(name="norm mlp fp32", **norm, dtype="fp32", rows=128, width=128),
        # GPT-2-medium's rows, 8 sequences of 1024, in fp32 as learned optimizers train them
        dict(name="norm gpt fp32", **norm, dtype="fp32", rows=8192, width=1024),
        # sizes that are multiples of nothing: no row but the first begins on a boundary; fp32 weights beside fp16
        dict(name="norm ragged fp16", **{**norm, "weight": "fp32"}, dtype="fp16", rows=12289, width=1001),
        # Llama-3-8B's width, 32 K tokens
        dict(name="norm llama bf16", **norm, dtype="bf16", rows=32768, width=4096),
        # a classifier of ten classes and its teacher: K = V
        dict(name="distil classes fp32", **{**distil, "padded": False, "masked": False}, dtype="fp32", rows=256, vocab=10, top=10),
        # GPT-2's vocabulary, odd: through autograd, with padding tokens and teachers that gave fewer than 64 entries
        dict(name="distil gpt bf16", **distil, dtype="bf16", rows=8192, vocab=50257, top=64),
        # a large vocabulary, loss and gradient in one call
        dict(name="distil llama bf16", **{**distil, "form": "grad", "temperature": 1.0}, dtype="bf16", rows=4096, vocab=128256, top=128),
        # one token through a Llama-3-8B block's feed-forward: the weights' bytes
        dict(name="ffn token bf16", **{**ffn, "train": False}, dtype="bf16", rows=1, width=4096, hidden=14336),
        # few tokens of a small model, sizes that are multiples of nothing
        dict(name="ffn ragged fp16", **{**ffn, "act": "gelu"}, dtype="fp16", rows=203, width=1001, hidden=2731),
        # GPT-2-medium's width, 8 sequences of 1024
        dict(name="ffn gpt bf16", **ffn, dtype="bf16", rows=8192, width=1024, hidden=4096),
        # a Llama-3-8B block's feed-forward over 8 K tokens
        dict(name="ffn llama bf16", **ffn, dtype="bf16", rows=8192, width=4096, hidden=14336),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _round(rng, x):
    """Most models have widths that are multiples of 64 or 8; some do not care."""
    m = rng.choice((64, 64, 8, 1))
    return max(m, x // m * m)


def draw(rng: random.Random):
    """One more case: any of the operators, in any of the types and forms, sizes spread over their logarithm."""
    op = rng.choice(("layer_norm", "gated_ffn", "distillation"))
    c = dict(op=op, dtype=rng.choice(("fp32", "bf16", "fp16") if op != "gated_ffn" else ("bf16", "fp16")))
    while True:
        if op == "layer_norm":
            c.update(rows=_log(rng, 1, 65536), width=_round(rng, _log(rng, 16, 16384)), train=rng.random() < 0.75)
            c.update(weight=rng.choice(("same", "same", "fp32", "none")))
            c.update(bias=c["weight"] != "none" and rng.random() < 0.7)
            if c["rows"] * c["width"] <= 1 << 27:
                return c
        elif op == "distillation":
            c.update(rows=_log(rng, 1, 8192), vocab=_round(rng, _log(rng, 8, 131072)), form=rng.choice(("autograd", "grad")))
            c.update(top=_log(rng, 1, min(256, c["vocab"])), masked=rng.random() < 0.5, padded=rng.random() < 0.5)
            c.update(temperature=rng.choice((1.0, 2.0, 4.0)))
            if c["rows"] * c["vocab"] <= 400_000_000:
                return c
        else:
            c.update(rows=_log(rng, 1, 8192), width=_round(rng, _log(rng, 64, 4096)), hidden=_round(rng, _log(rng, 64, 14336)))
            c.update(train=rng.random() < 0.75, act=rng.choice(("silu", "silu", "gelu")))
            return c


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt, n = TYPES[case["dtype"]], case["rows"]
    randn = lambda *shape: torch.randn(shape, generator=gen, device="cuda")  # noqa: E731
    rand = lambda *shape: torch.rand(shape, generator=gen, device="cuda")  # noqa: E731
    s = {"case": dict(case)}
    if case["op"] == "layer_norm":
        d = case["width"]
        # rows of very different size, off centre, as a residual stream's are
        s["x"] = ((randn(n, d) + 0.5 * randn(n, 1)) * 10.0 ** (2 * rand(n, 1) - 1)).to(dt)
        wt = {"same": dt, "fp32": torch.float32, "none": None}[case["weight"]]
        if wt is not None:
            s["weight"] = (1 + 0.2 * randn(d)).to(wt)
            if case["bias"]:
                s["bias"] = (0.2 * randn(d)).to(wt)
        if case["train"]:
            s["dy"] = randn(n, d).to(dt)
        names = ("x", "weight", "bias")
    elif case["op"] == "gated_ffn":
        d, f = case["width"], case["hidden"]
        s["x"] = randn(n, d).to(dt)  # rows behind a norm
        s["w_gate"], s["w_up"] = (randn(f, d) * d ** -0.5).to(dt), (randn(f, d) * d ** -0.5).to(dt)
        s["w_down"] = (randn(d, f) * f ** -0.5).to(dt)
        if case["train"]:
            s["dy"] = (0.1 * randn(n, d)).to(dt)
        names = ("x", "w_gate", "w_up", "w_down")
    else:
        v, k = case["vocab"], case["top"]
        logits = 2.5 * randn(n, v)
        # a teacher that agrees in part: its largest logits, in order
        s["teacher"], s["ids"] = (logits + 2.0 * randn(n, v)).topk(k, dim=1)
        s["teacher"] = s["teacher"].to(dt)
        s["logits"] = logits.to(dt)
        if case["padded"]:  # behind them, nothing: one row in four has fewer than K entries
            left = torch.where(rand(n) < 0.25, (rand(n) * k).long() + 1, k)
            s["ids"] = torch.where(torch.arange(k, device="cuda") < left[:, None], s["ids"], -1)
        if case["masked"]:  # one token in eight is a prompt's or a batch's padding; the last one stays
            s["weights"] = (rand(n) >= 0.125).float()
            s["weights"][-1] = 1.0
        names = ("logits",)
    if case.get("train") or case.get("form") == "autograd":
        s["leaves"] = [s[k].requires_grad_() for k in names if k in s]
        s["names"] = ["d" + k for k in names if k in s]
    return s


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------


def run(s):
    case = s["case"]
    if case["op"] == "layer_norm":
        y = _own_norm(s) if own else _norm(s["x"].float(), _float(s.get("weight")), _float(s.get("bias"))).to(s["x"].dtype)
    elif case["op"] == "gated_ffn":
        y = _own_ffn(s) if own else _ffn(*(s[k].float() for k in ("x", "w_gate", "w_up", "w_down")), case["act"]).to(s["x"].dtype)
    elif case["form"] == "grad":
        return _own_distil_grad(s) if own else _distil_grad(s)
    else:
        loss = _own_distil(s) if own else _distil(s["logits"].float(), s)
        return {"loss": loss.detach(), **dict(zip(s["names"], torch.autograd.grad(loss, s["leaves"])))}
    if not case["train"]:
        return {"y": y}
    return {"y": y.detach(), **dict(zip(s["names"], torch.autograd.grad(y, s["leaves"], s["dy"])))}


def _own_norm(s):
    from pylo_b200 import layers

    return layers.layer_norm(s["x"], s.get("weight"), s.get("bias"), eps=EPS)


def _own_ffn(s):
    from pylo_b200 import layers

    return layers.gated_ffn(s["x"], s["w_gate"], s["w_up"], s["w_down"], activation=s["case"]["act"])


def _own_distil(s):
    from pylo_b200 import layers

    return layers.distillation_loss(s["logits"], s["teacher"], s["ids"], temperature=s["case"]["temperature"], weights=s.get("weights"))


def _own_distil_grad(s):
    from pylo_b200 import layers

    loss, grad = layers.distillation_loss_and_grad(s["logits"], s["teacher"], s["ids"], temperature=s["case"]["temperature"], weights=s.get("weights"))
    return {"loss": loss, "dlogits": grad}


def _float(x):
    return None if x is None else x.float()


def _norm(x, weight, bias):
    mean = x.mean(1, keepdim=True)
    xc = x - mean
    y = xc * torch.rsqrt((xc * xc).mean(1, keepdim=True) + EPS)
    if weight is not None:
        y = y * weight
    return y if bias is None else y + bias


def _ffn(x, w_gate, w_up, w_down, act):
    g, u = x @ w_gate.t(), x @ w_up.t()
    a = g * torch.sigmoid(g) if act == "silu" else 0.5 * g * (1 + torch.erf(g * math.sqrt(0.5)))
    return (a * u) @ w_down.t()


def _teacher(s, t):
    """The teacher's probabilities over its entries, the ids with something harmless for padding, and the rows' weights."""
    there = s["ids"] >= 0
    z = torch.where(there, t / s["case"]["temperature"], -math.inf)
    e = torch.exp(z - z.amax(1, keepdim=True))
    p = e / e.sum(1, keepdim=True)
    w = s["weights"] if "weights" in s else torch.ones_like(p[:, 0])
    return p, s["ids"].clamp(min=0), w.to(t.dtype)


def _distil(x, s):
    T = s["case"]["temperature"]
    p, ids, w = _teacher(s, s["teacher"].float())
    x = x / T
    x = x - x.detach().amax(1, keepdim=True)
    lse = torch.log(torch.exp(x).sum(1))
    log_p = torch.log(torch.where(p > 0, p, 1.0))
    rows = (p * (log_p - x.gather(1, ids) + lse[:, None])).sum(1)
    return T * T * (rows * w).sum() / w.sum()


def _distil_grad(s):
    T = s["case"]["temperature"]
    p, ids, w = _teacher(s, s["teacher"].float())
    x = s["logits"].float() / T
    x -= x.amax(1, keepdim=True)
    picked = x.gather(1, ids)
    e = torch.exp(x)
    total = e.sum(1, keepdim=True)
    log_p = torch.log(torch.where(p > 0, p, 1.0))
    rows = (p * (log_p - picked + torch.log(total))).sum(1)
    grad = (e / total).scatter_add_(1, ids, -p) * (T * w / w.sum())[:, None]
    return {"loss": T * T * (rows * w).sum() / w.sum(), "dlogits": grad.to(s["logits"].dtype)}


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without, and its result in 64 bits
# ---------------------------------------------------------------------------------------------------------------------


def work(case):
    e, n = (4 if case["dtype"] == "fp32" else 2), case["rows"]
    if case["op"] == "layer_norm":
        d = case["width"]
        vectors = (0 if case["weight"] == "none" else 1 + case["bias"]) * d * (4 if case["weight"] == "fp32" else e)
        if not case["train"]:
            return {"bytes": 2 * n * d * e + vectors, "flops": 8 * n * d}
        return {"bytes": 4 * n * d * e + 2 * vectors, "flops": 22 * n * d}  # x, dy; y, dx
    if case["op"] == "gated_ffn":
        d, f = case["width"], case["hidden"]
        one = (2 * n * d + 3 * d * f) * e
        return {"bytes": one * (2 if case["train"] else 1), "flops": 6 * n * d * f * (3 if case["train"] else 1)}
    v, k = case["vocab"], case["top"]
    return {"bytes": 2 * n * v * e + n * k * (e + 8) + (4 * n if case["masked"] else 0), "flops": 8 * n * v + 8 * n * k}


def exact(case, seed):
    """The operators' formulas and those of their gradients, in 64 bits."""
    s = prepare(case, seed)
    d = {k: v.detach().double() for k, v in s.items() if isinstance(v, torch.Tensor) and v.is_floating_point()}
    if case["op"] == "layer_norm":
        x, w, b = d["x"], d.get("weight"), d.get("bias")
        var, mean = torch.var_mean(x, dim=1, unbiased=False, keepdim=True)
        r = (var + EPS) ** -0.5
        xh = (x - mean) * r
        out = {"y": xh * (1.0 if w is None else w) + (0.0 if b is None else b)}
        if case["train"]:
            dy = d["dy"]
            q = dy if w is None else dy * w
            out["dx"] = r * (q - q.mean(1, keepdim=True) - xh * (q * xh).mean(1, keepdim=True))
            if w is not None:
                out["dweight"] = torch.einsum("nd,nd->d", dy, xh)
            if b is not None:
                out["dbias"] = dy.sum(0)
        return out
    if case["op"] == "gated_ffn":
        x, wg, wu, wd = (d[k] for k in ("x", "w_gate", "w_up", "w_down"))
        g, u = torch.einsum("nd,fd->nf", x, wg), torch.einsum("nd,fd->nf", x, wu)
        if case["act"] == "silu":
            slope = 1 / (1 + torch.exp(-g))
            a = g * slope
            slope = slope + a * (1 - slope)
        else:
            slope = 0.5 * torch.special.erfc(-g * 0.5 ** 0.5)
            a = g * slope
            slope = slope + g * torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
        h = a * u
        out = {"y": torch.einsum("nf,df->nd", h, wd)}
        if case["train"]:
            dy = d["dy"]
            out["dw_down"] = torch.einsum("nd,nf->df", dy, h)
            dh = torch.einsum("nd,df->nf", dy, wd)
            dg, du = dh * u * slope, dh * a
            out["dx"] = torch.einsum("nf,fd->nd", dg, wg) + torch.einsum("nf,fd->nd", du, wu)
            out["dw_gate"], out["dw_up"] = torch.einsum("nf,nd->fd", dg, x), torch.einsum("nf,nd->fd", du, x)
        return out
    T, n, v = case["temperature"], case["rows"], case["vocab"]
    w = d["weights"] if "weights" in d else torch.ones(n, dtype=torch.float64, device="cuda")
    loss, grads = 0.0, []
    for a in range(0, n, 512):  # some rows at a time
        rows = slice(a, min(n, a + 512))
        there = s["ids"][rows] >= 0
        log_p = torch.log_softmax(d["teacher"][rows].div(T).masked_fill(~there, -math.inf), dim=1)
        log_q = torch.log_softmax(d["logits"][rows] / T, dim=1)
        p = log_p.exp()
        ids = s["ids"][rows].where(there, 0)
        kl = (p * (log_p.masked_fill(~there, 0) - log_q.gather(1, ids))).sum(1)
        loss = loss + T * T * (kl * w[rows]).sum() / w.sum()
        full = torch.zeros_like(log_q).scatter_add_(1, ids, p)
        grads.append((log_q.exp() - full) * (w[rows] * T / w.sum())[:, None])
    return {"loss": loss, "dlogits": torch.cat(grads)}

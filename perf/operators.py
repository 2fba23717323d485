"""The steps beside the learned optimizers, as cases that can be timed and compared: AdamW over many tensors with states in
32 bits and in 8, and the clipping of many gradients by their global norm.

A case names an operator, a family of parameter shapes with its sizes, the types of parameters and gradients and the options of
the run.  One pass is one ``step()`` (or one clipping) in the middle of a training run: the states exist, the gradients are in
device memory.

All parameters of a model are views into one flat buffer, and so are its gradients and every kind of state, as sharded training
lays them out; the whole result of a step is then a few tensors.  Every tensor begins on a multiple of 256 elements with zeros up
to the next, or, in a ``packed`` case, parameters and gradients lie one behind the other as they come, which leaves most of them
on no boundary at all (the states, which the optimizer allocates, are never packed).
"""

import math
import random

import torch

own = False

BLOCK = 256  # elements of a tensor that share a scale in the 8-bit states, and what a tensor begins on a multiple of
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
LR, BETAS, EPS, WD = 3e-4, (0.9, 0.95), 1e-8, 0.1
SEED = 5  # of the stochastic rounding

# ---------------------------------------------------------------------------------------------------------------------
# parameter shapes
# ---------------------------------------------------------------------------------------------------------------------


def shapes_of(case):
    net, d, ff, layers = case["net"], case["width"], case.get("ff", 0), case["layers"]
    if net == "mlp":  # inputs -> width -> ... -> width -> outputs
        s, fan_in = [], case["inputs"]
        for out in [d] * layers + [case["outputs"]]:
            s += [(out, fan_in), (out,)]
            fan_in = out
        return s
    if net == "conv":  # 3x3 convolutions with batch-norm vectors, channels doubling at every stage, a linear classifier
        s, fan_in, out = [(d, 3, 7, 7), (d,), (d,)], d, d
        for stage in range(layers):
            for k in range(2):
                s += [(out, fan_in, 3, 3), (out,), (out,)]
                fan_in = out
            out *= 2
        return s + [(case["outputs"], fan_in), (case["outputs"],)]
    if net == "gpt":  # biases and layer norms everywhere, one matrix for each of queries, keys and values
        s = [(case["outputs"], d), (case["context"], d)]
        for _ in range(layers):
            s += [(d,), (d,)] + [(d, d), (d,)] * 4 + [(d,), (d,), (d, ff), (ff,), (ff, d), (d,)]
        return s + [(d,), (d,)]
    s = [(case["outputs"], d)] if case["outputs"] else []  # "llama": gated feed-forward, grouped keys and values, no biases
    for _ in range(layers):
        s += [(d, d), (d // 4, d), (d // 4, d), (d, d), (ff, d), (ff, d), (d, ff), (d,), (d,)]
    return s + [(d,)] + ([(case["outputs"], d)] if case["outputs"] else [])


def sizes_of(case):
    return [math.prod(s) for s in shapes_of(case)]


# ---------------------------------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------------------------------


def listed():
    mlp = dict(net="mlp", inputs=784, width=128, layers=2, outputs=10)
    ragged = dict(net="mlp", inputs=1433, width=1001, layers=3, outputs=7)
    conv = dict(net="conv", width=64, layers=4, outputs=1000)
    gpt = dict(net="gpt", width=1024, ff=4096, layers=24, context=1024, outputs=50257)
    llama = dict(net="llama", width=4096, ff=14336, layers=2, outputs=0)
    return [
        # the 784-128-128-10 perceptron of the learned optimizers' own tasks: all latency, thousands of steps in a row
        dict(name="adamw mlp", op="adamw", p="fp32", g="fp32", **mlp),
        # sizes that are multiples of nothing, in one flat buffer without gaps
        dict(name="adamw ragged packed", op="adamw", p="fp32", g="fp32", packed=True, **ragged),
        # GPT-2-medium's sizes (350 M, almost 400 tensors) in mixed precision: bf16 weights, an fp32 copy in the state, clipping
        dict(name="adamw gpt bf16 master", op="adamw", p="bf16", g="bf16", master=True, clip=True, **gpt),
        # two Llama-3-8B blocks (436 M parameters), what one of many ranks owns of the whole model, all in fp32
        dict(name="adamw llama", op="adamw", p="fp32", g="fp32", **llama),
        # the perceptron with 8-bit states, clipped
        dict(name="adamw8 mlp clip", op="adamw8", p="fp32", g="fp32", clip=True, **mlp),
        # an image classifier of four stages: four-dimensional weights and many vectors
        dict(name="adamw8 conv", op="adamw8", p="fp32", g="fp32", **conv),
        # fp16 weights with a master copy, blocks that end inside of tensors, nothing aligned
        dict(name="adamw8 ragged fp16 packed", op="adamw8", p="fp16", g="fp16", master=True, packed=True, **ragged),
        # the least memory there is: bf16 weights without a copy, 8-bit states
        dict(name="adamw8 gpt bf16", op="adamw8", p="bf16", g="bf16", clip=True, **gpt),
        # bf16 weights with a master copy, gradients accumulated in fp32
        dict(name="adamw8 llama master", op="adamw8", p="bf16", g="fp32", master=True, **llama),
        # clipping before a learned optimizer's step: the perceptron, a language model in bf16, two Llama-3-8B blocks in fp32
        dict(name="clip mlp", op="clip", p="fp32", g="fp32", **mlp),
        dict(name="clip gpt bf16", op="clip", p="bf16", g="bf16", **gpt),
        dict(name="clip llama", op="clip", p="fp32", g="fp32", **llama),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _round(rng, x):
    """Most models have widths that are multiples of 64 or 8; some do not care."""
    m = rng.choice((64, 64, 8, 4, 1))
    return max(m, x // m * m)


def draw(rng: random.Random):
    """One more case: any operator over any of the shape families, in any of the types, sizes spread over their logarithm."""
    op = rng.choice(("adamw", "adamw", "adamw8", "adamw8", "clip"))
    while True:
        net = rng.choice(("mlp", "conv", "gpt", "llama"))
        if net == "mlp":
            c = dict(net=net, inputs=_log(rng, 16, 4000), width=_round(rng, _log(rng, 24, 4096)), layers=rng.randint(1, 6), outputs=_log(rng, 2, 1000))
        elif net == "conv":
            c = dict(net=net, width=_round(rng, _log(rng, 8, 160)), layers=rng.randint(2, 4), outputs=_log(rng, 10, 1000))
        elif net == "gpt":
            d = _round(rng, _log(rng, 64, 1600))
            c = dict(net=net, width=d, ff=rng.choice((2, 4)) * d, layers=rng.randint(1, 24), context=_log(rng, 64, 2048), outputs=_log(rng, 256, 50257))
        else:
            d = max(64, _log(rng, 96, 4096) // 32 * 32)
            c = dict(net=net, width=d, ff=_round(rng, d * 7 // 2), layers=rng.randint(1, 8), outputs=rng.choice((0, _log(rng, 256, 32000))))
        if sum(sizes_of(c)) <= 300_000_000:
            break
    p = rng.choice(("fp32", "fp32", "bf16", "fp16"))
    c.update(op=op, p=p, g=p if op == "clip" else rng.choice((p, p, "fp32")), packed=rng.random() < 0.25)
    if op != "clip":
        c.update(master=p != "fp32" and rng.random() < 0.6, clip=rng.random() < 0.5)
    return c


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------


def _layout(case):
    """What a program that owns the flat buffers knows of them: sizes, where each tensor begins in the buffers with gaps and in those
    without, and how long both are."""
    sizes = sizes_of(case)
    at, packed_at, n, packed = [], [], 0, 0
    for k in sizes:
        at.append(n)
        packed_at.append(packed)
        n += -(-k // BLOCK) * BLOCK
        packed += k
    if not case.get("packed"):
        packed_at, packed = at, n
    return sizes, at, packed_at, n, packed


def _decoded(codes, scales):
    return (codes.float().view(-1, BLOCK) * scales.float().view(-1, 1)).view(-1)


def _nearest(x):
    """Codes and scales of values >= 0 or of either sign, rounded to nearest: how the states of the run begin."""
    b = x.view(-1, BLOCK)
    e = (b.abs().amax(1).view(torch.int32) >> 23).clamp(min=8)
    scale = ((e - 7) << 23).view(torch.float32)
    return (b / scale[:, None]).to(torch.float8_e4m3fn).view(-1), (e - 7).to(torch.uint8).view(torch.float8_e8m0fnu)


def prepare(case, seed):
    sizes, at, packed_at, n, packed = _layout(case)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dev = dict(device="cuda")
    length = torch.tensor(sizes, **dev)
    first = torch.tensor(at, **dev)
    gaps = torch.tensor([b - a for a, b in zip(at, at[1:] + [n])], **dev)
    index = torch.arange(n, **dev) - torch.repeat_interleave(first, gaps)  # an element's number in its tensor
    real = index < torch.repeat_interleave(length, gaps)  # where a tensor's elements are, not the zeros behind them
    where = torch.nonzero(real).view(-1) if case.get("packed") else None
    # gradients of very different size from block to block, and one block in sixteen that had none in this step or ever (rows of an
    # embedding whose token did not occur)
    size = 10.0 ** (-4 + 2 * torch.rand(n // BLOCK, generator=gen, **dev))
    size *= torch.rand(n // BLOCK, generator=gen, **dev) > 1 / 16
    size = size[:, None]
    draw_ = lambda f: f((n // BLOCK, BLOCK), generator=gen, **dev)  # noqa: E731
    flat = lambda x: torch.where(real, x.view(-1), 0.0)  # noqa: E731
    lay = lambda x, t: (x if where is None else x[where]).to(TYPES[t])  # noqa: E731
    s = {"case": dict(case), "g": lay(flat(draw_(torch.randn) * size), case["g"])}
    del index
    if case["op"] == "clip":
        s["max_norm"] = 0.3 * float(torch.linalg.vector_norm(s["g"].double()))
        if own:
            s["params"] = [torch.nn.Parameter(torch.empty(shape, dtype=s["g"].dtype, **dev)) for shape in shapes_of(case)]
            for p, a, k in zip(s["params"], packed_at, sizes):
                p.grad = s["g"][a:a + k].view(p.shape)
        return s
    p = flat(draw_(torch.randn) * 0.02)
    m, v = flat(draw_(torch.randn) * size * 0.3), flat((0.5 + draw_(torch.rand)) * size ** 2)
    s["p"] = lay(p, case["p"])
    if case.get("master"):
        s["master"] = p
    if case["op"] == "adamw8":
        s["exp_avg"], s["exp_avg_scale"] = _nearest(m)
        s["exp_avg_sq_root"], s["exp_avg_sq_root_scale"] = _nearest(v.sqrt())
    else:
        s["exp_avg"], s["exp_avg_sq"] = m, v
    s["step"] = 10 + seed % 1000
    # half of what the norm is, so that the gradients are clipped
    s["clip"] = 0.5 * float(torch.linalg.vector_norm(s["g"].double())) if case.get("clip") else 0.0
    s["where"], s["tensors"] = where, (first, gaps)
    if own:
        _optimizer(s, sizes, at, packed_at)
    return s


def _optimizer(s, sizes, at, packed_at):
    from pylo_b200 import optim

    case = s["case"]
    params = []
    for shape, a, k in zip(shapes_of(case), packed_at, sizes):
        p = torch.nn.Parameter(s["p"][a:a + k].view(shape))
        p.grad_dtype = s["g"].dtype
        p.grad = s["g"][a:a + k].view(shape)
        params.append(p)
    kw = dict(lr=LR, betas=BETAS, eps=EPS, weight_decay=WD, master_weights=bool(case.get("master")))
    if s["clip"]:
        kw.update(clip_grad=True, clip_norm=s["clip"])
    s["opt"] = optim.AdamW8bit_CUDA(params, seed=SEED, **kw) if case["op"] == "adamw8" else optim.AdamW_CUDA(params, **kw)
    for p, a, k in zip(params, at, sizes):
        st = {"step": torch.tensor(float(s["step"]), dtype=torch.float64)}
        for name in ("master", "exp_avg", "exp_avg_sq", "exp_avg_sq_root"):
            if name in s:
                st[name] = s[name][a:a + k].view(p.shape)
        for name in ("exp_avg_scale", "exp_avg_sq_root_scale"):
            if name in s:
                st[name] = s[name][a // BLOCK:a // BLOCK + -(-k // BLOCK)]
        s["opt"].state[p] = st


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------


def run(s):
    if s["case"]["op"] == "clip":
        s["max_norm"] *= 0.9999  # clipped gradients are clipped again by the next pass
        if own:
            from pylo_b200 import optim

            norm = optim.clip_grad_norm_(s["params"], s["max_norm"])
        else:
            norm = torch.sqrt(torch.sum(s["g"].double() ** 2)).float()
            s["g"].copy_(s["g"].float() * torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0))
        return {"norm": norm, "g": s["g"]}
    if own:
        s["opt"].step()
    else:
        _plain_step(s)
    return {k: s[k] for k in OUTPUTS if k in s}


OUTPUTS = ("p", "master", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_root", "exp_avg_sq_root_scale")


def _plain_step(s):
    where, eight = s["where"], s["case"]["op"] == "adamw8"
    s["step"] += 1
    t, (b1, b2) = s["step"], BETAS
    g = s["g"].float()
    if s["clip"]:
        norm = torch.sqrt(torch.sum(g.double() ** 2)).float()
        g = g * (s["clip"] / torch.clamp(norm, min=s["clip"]))
    m = _decoded(s["exp_avg"], s["exp_avg_scale"]) if eight else s["exp_avg"]
    v = _decoded(s["exp_avg_sq_root"], s["exp_avg_sq_root_scale"]) ** 2 if eight else s["exp_avg_sq"]
    if where is not None:
        g = torch.zeros_like(m).index_put_((where,), g)
    p = s["master"] if "master" in s else s["p"].float() if where is None else torch.zeros_like(m).index_put_((where,), s["p"].float())
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * (g * g)
    root = torch.sqrt(v)
    p = p * (1 - LR * WD) - LR / (1 - b1 ** t) * (m / (root / math.sqrt(1 - b2 ** t) + EPS))
    if eight:
        random_m, random_u = _random(s, t)
        _encode(m, random_m, s["exp_avg"], s["exp_avg_scale"])
        _encode(root, random_u, s["exp_avg_sq_root"], s["exp_avg_sq_root_scale"], least=1)
    else:
        s["exp_avg"].copy_(m)
        s["exp_avg_sq"].copy_(v)
    if "master" in s:
        s["master"].copy_(p)
    s["p"].copy_(p if where is None else p[where])


#: the first 32 bits behind the point of the square roots of the first sixteen primes, made odd
ROOTS = [(math.isqrt(q << 64) & 0xFFFFFFFF) | 1 for q in (2, 3, 5, 7, 11, 13, 17, 19, 23, 29, 31, 37, 41, 43, 47, 53)]


def _mixed(x):
    x = x ^ (x >> 16)
    x = (x * ROOTS[0]) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * ROOTS[1]) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _random(s, step):
    """24 random bits for every element of both states: a hash of seed, step and the number of the element's group of eight in its
    tensor, times a factor for each place in the group."""
    first, gaps = s["tensors"]
    group = (torch.arange(s["exp_avg"].numel() // 8, device="cuda") - torch.repeat_interleave(first // 8, gaps // 8)) & 0xFFFFFFFF
    base = _mixed((group * ROOTS[2] + _mixed((SEED * ROOTS[3] + step) & 0xFFFFFFFF)) & 0xFFFFFFFF)
    factors = torch.tensor(ROOTS, device="cuda")
    bits = lambda f: ((base[:, None] * f & 0xFFFFFFFF) >> 8).to(torch.int32).view(-1)  # noqa: E731
    return bits(factors[8:]), bits(factors[:8])


def _encode(x, random_bits, codes, scales, least=0):
    """Into e4m3 with a power of two for every block, rounded up with the probability of what is cut off; a value that is not zero
    gets at least the code `least`."""
    b = x.view(-1, BLOCK)
    e = (b.abs().amax(1).view(torch.int32) >> 23).clamp(min=8)
    # over the power of two of the largest (two to the -127 has no exponent of its own), then down to where a float's top seven bits
    # behind the sign are the code: exponent 14 of e4m3 for the largest
    over = ((254 - e) << 23).clamp(min=1 << 22).view(torch.float32)
    t = (b.abs() * over[:, None]) * 2.0 ** -113
    code = ((t.view(torch.int32) << 4) + random_bits.view(-1, BLOCK)) >> 24
    code = torch.maximum(code, (b != 0).int() * least) | torch.where(b < 0, 128, 0)
    codes.copy_(code.to(torch.uint8).view(torch.float8_e4m3fn).view(-1))
    scales.copy_((e - 7).to(torch.uint8).view(torch.float8_e8m0fnu))


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without, and its result in 64 bits
# ---------------------------------------------------------------------------------------------------------------------


def work(case):
    n = sum(sizes_of(case))
    wide = {"fp32": 4, "bf16": 2, "fp16": 2}
    if case["op"] == "clip":
        return {"bytes": 2 * wide[case["g"]] * n, "flops": 3 * n}
    # parameters are read and written, or written only where a master copy is read and written instead; gradients are read
    bytes_ = wide[case["g"]] + (wide[case["p"]] + 8 if case.get("master") else 2 * wide[case["p"]])
    bytes_ += 4 * (1 + 1 / BLOCK) if case["op"] == "adamw8" else 16
    return {"bytes": bytes_ * n, "flops": (16 if case["op"] == "adamw" else 30) * n}


def exact(case, seed):
    """The unrounded values of all outputs.  A code stands for a value that was rounded up or down at random: here it is the value
    over the block's power of two, which the codes are off from by that rounding.  The power of two itself jumps where the largest
    value passes one, and so has none in 64 bits that another could be held to."""
    s = prepare(case, seed)
    g = s["g"].double()
    norm = torch.linalg.vector_norm(g)
    if case["op"] == "clip":
        return {"norm": norm, "g": g * min(1.0, s["max_norm"] * 0.9999 / (float(norm) + 1e-6))}
    n = s["exp_avg"].numel()
    spread = lambda x: x if s["where"] is None else torch.zeros(n, dtype=torch.float64, device="cuda").scatter_(0, s["where"], x)  # noqa: E731
    if s["clip"]:
        g *= s["clip"] / max(float(norm), s["clip"])
    g = spread(g)
    (b1, b2), t = BETAS, s["step"] + 1
    p = s["master"].double() if "master" in s else spread(s["p"].double())
    per_element = lambda x: x.double().repeat_interleave(BLOCK)  # noqa: E731
    eight = case["op"] == "adamw8"
    m, v = s["exp_avg"].double(), s["exp_avg_sq_root" if eight else "exp_avg_sq"].double()
    if eight:
        m *= per_element(s["exp_avg_scale"])
        v = (v * per_element(s["exp_avg_sq_root_scale"])).square()
    m = torch.lerp(g, m, b1)
    v = torch.lerp(g.square(), v, b2)
    m_hat, v_hat = m / (1 - b1 ** t), v / (1 - b2 ** t)
    p = p - LR * WD * p - LR * m_hat / (v_hat.sqrt() + EPS)
    out = {"p": p if s["where"] is None else p[s["where"]], "master": p if "master" in s else None}
    if not eight:
        return {**out, "exp_avg": m, "exp_avg_sq": v}
    for name, x in (("exp_avg", m), ("exp_avg_sq_root", v.sqrt())):
        most = x.view(-1, BLOCK).abs().amax(1)
        scale = torch.exp2(torch.floor(torch.log2(most)).clamp(min=8 - 127) - 7)
        out[name], out[name + "_scale"] = x / scale.repeat_interleave(BLOCK), None
    return out

"""Layer norm, the gated feed-forward block and distillation against their formulas in 64 bits.

Tolerances are bounds: u = eps / 2 of the type for every rounding to it, 2^-24 for every fp32 operation on the way (2^-23 where the tensor core adds,
which cuts off), each times the magnitudes that it acts on."""

import ctypes as C
import math

import pytest
import torch

from pylo_b200 import _lib as L
from pylo_b200 import layers, workloads

gpu = pytest.mark.gpu
F32, BF16, FP16 = torch.float32, torch.bfloat16, torch.float16
E = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
    """Half the step between the smallest numbers of a type."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def near(got, want, slack, what=""):
    """|got - want| <= a rounding of got's type + slack (of the arithmetic before it), element by element."""
    bound = half_step(got.dtype) * (want.abs() + slack) + least(got.dtype) + slack
    over = (got.double() - want).abs() - bound
    assert got.shape == want.shape, what
    assert bool((over <= 0).all()), (what, float(over.max()), float((over / bound).max()))


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(*shape, seed=0, dtype=F32, scale=1.0):
    return (torch.randn(shape, generator=gen(seed), device="cuda") * scale).to(dtype)


# ---------------------------------------------------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------------------------------------------------


def norm64(x, weight, bias, dy, eps):
    """{name: (value, slack)} of the outputs in 64 bits."""
    x, w = x.double(), (1.0 if weight is None else weight.double())
    b = 0.0 if bias is None else bias.double()
    mean = x.mean(-1, keepdim=True)
    r = ((x - mean).square().mean(-1, keepdim=True) + eps).rsqrt()
    xh = (x - mean) * r
    width, rows = x.shape[-1], x[..., 0].numel()
    # a sum of a row: 32 elements of a thread, 5 + 5 levels; then the square root, quotient and products
    k = 64 * E
    off = x.abs().mean(-1, keepdim=True) * r          # what an error of the mean does to xh
    exh = k * (xh.abs() + off)
    ww = w if isinstance(w, float) else w.abs()
    bb = b if isinstance(b, float) else b.abs()
    out = {"y": (xh * w + b, exh * ww + k * (xh.abs() * ww + bb))}
    if dy is not None:
        dy = dy.double()
        q = dy * w
        s1, s2 = q.mean(-1, keepdim=True), (q * xh).mean(-1, keepdim=True)
        a1 = q.abs().mean(-1, keepdim=True)
        a2 = (q.abs() * (xh.abs() + off)).mean(-1, keepdim=True)
        out["dx"] = (r * (q - s1 - xh * s2), 2 * k * r * (q.abs() + a1 + (xh.abs() + off) * a2))
        flat = lambda t: t.reshape(rows, width)
        seq = (rows + 64) * E                          # a column's sum: at most all rows in a line
        out["dweight"] = (flat(dy * xh).sum(0), flat(dy.abs() * (exh + seq * (xh.abs() + exh))).sum(0))
        out["dbias"] = (flat(dy).sum(0), seq * flat(dy.abs()).sum(0))
    return out


def check_norm(x, weight=None, bias=None, dy=None, eps=1e-5):
    want = norm64(x.detach(), weight, bias, dy, eps)
    leaves = [t.detach().requires_grad_() if i else t.requires_grad_() for i, t in enumerate((x, weight, bias)) if t is not None]
    y = layers.layer_norm(*leaves, eps=eps)
    near(y.detach(), *want["y"], "y")
    with torch.no_grad():
        assert torch.equal(layers.layer_norm(*leaves, eps=eps), y)
    if dy is None:
        return
    for leaf, got, name in zip(leaves, torch.autograd.grad(y, leaves, dy), ("dx", "dweight", "dbias")):
        assert got.dtype == leaf.dtype
        near(got, *want[name], name)


SHAPES = [(1, 1), (3, 7), (5, 8), (2, 128), (7, 129), (300, 33), (33, 1000), (9, 1001), (130, 256), (9, 1024), (6, 1025), (700, 768), (11, 4096), (5, 8192), (3, 8200), (2, 12001),
          (2, 16384), (500, 2050), (200, 5001)]


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, FP16])
@pytest.mark.parametrize("rows,width", SHAPES)
def test_norm(rows, width, dtype):
    x = (randn(rows, width, seed=1) + 3 * randn(rows, 1, seed=2)).mul(10.0 ** (randn(rows, 1, seed=3).clamp(-2, 2))).to(dtype)
    check_norm(x, 1 + 0.3 * randn(width, seed=4).to(dtype), 0.3 * randn(width, seed=5).to(dtype), randn(rows, width, seed=6, dtype=dtype))


@gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("width", [64, 77, 1024, 2048])
def test_norm_with_fp32_weights(width, dtype):
    check_norm(randn(37, width, seed=1, dtype=dtype), 1 + 0.3 * randn(width, seed=4), 0.3 * randn(width, seed=5), randn(37, width, seed=6, dtype=dtype))


@gpu
@pytest.mark.parametrize("width", [96, 99, 3000])
def test_norm_without_weight_or_bias(width):
    x, dy = randn(21, width, seed=1, dtype=BF16), randn(21, width, seed=2, dtype=BF16)
    check_norm(x, dy=dy)
    check_norm(x.detach(), 1 + 0.1 * randn(width, seed=3, dtype=BF16), dy=dy)


@gpu
def test_norm_of_strided_and_expanded_rows():
    big = randn(40, 3, 200, seed=1, dtype=BF16)
    for x in (big[:, 1, 8:136], big[:, 1, 3:131], big[::2, :, :64], big[:, 2, :128].t(), big[:1, 0, :128].expand(9, 128)):
        w = randn(x.shape[-1], seed=2, dtype=BF16)
        want = norm64(x, w, None, torch.ones_like(x), 1e-5)
        x = x.detach().requires_grad_()
        y = layers.layer_norm(x, w)
        near(y.detach(), *want["y"], "y")
        y.sum().backward()   # an expanded gradient
        near(x.grad, *want["dx"], "dx")


@gpu
def test_norm_of_one_value_repeated_and_of_no_rows():
    check_norm(torch.full((4, 300), 7.25, device="cuda"), randn(300, seed=1), randn(300, seed=2), randn(4, 300, seed=3), eps=1e-3)
    x, w = torch.empty(0, 16, device="cuda", requires_grad=True), torch.ones(16, device="cuda", requires_grad=True)
    layers.layer_norm(x, w).sum().backward()
    assert x.grad.shape == (0, 16) and torch.equal(w.grad, torch.zeros_like(w))


@gpu
def test_norm_keeps_rows_apart():
    """A row of NaN or infinities spoils itself alone."""
    x = randn(50, 136, seed=1)
    x[7], x[9, 3] = float("nan"), float("inf")
    y = layers.layer_norm(x)
    bad = y.isnan().all(1)
    assert bad.nonzero().view(-1).tolist() == [7, 9] and bool(y[~bad].isfinite().all())


@gpu
def test_norm_gradients_are_those_of_differences():
    """Along a direction v: (L(x + h v) - L(x - h v)) / 2h with L = sum(c y).  Its truncation is of order h^2, its rounding that of the
    two sums of 960 fp32 values of about 1 (960 roots of 2^-24 squared, over h)."""
    x, c, v = (randn(6, 160, seed=k).double() for k in (1, 2, 3))
    w = 1 + 0.2 * randn(160, seed=4)
    h = 2.0 ** -7
    value = lambda t: float((c * layers.layer_norm(t.float(), w).double()).sum())
    leaf = x.float().requires_grad_()
    (g,) = torch.autograd.grad(layers.layer_norm(leaf, w), leaf, c.float())
    want = (value(x + h * v) - value(x - h * v)) / (2 * h)
    scale = float((c.abs() * v.abs()).sum())
    assert abs(float((g.double() * v).sum()) - want) < scale * (10 * h * h + 64 * E / h)


# ---------------------------------------------------------------------------------------------------------------------
# the gated feed-forward block
# ---------------------------------------------------------------------------------------------------------------------


def act64(name, g):
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if name == "gelu":
        phi = 0.5 * torch.special.erfc(-g * 0.5 ** 0.5)
        return g * phi, phi + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        k = math.sqrt(2 / math.pi)
        t = torch.tanh(k * (g + 0.044715 * g ** 3))
        return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * k * (1 + 3 * 0.044715 * g * g)
    return g.clamp(min=0), (g > 0).double()


def ffn64(x, wg, wu, wd, dy, act, operands=None):
    """{name: (value, slack)}: slack without the last rounding.  operands: how far h, dg and du are off, relative to their size: half a step of the type,
    or what is given."""
    u_ = half_step(x.dtype) if operands is None else operands
    tiny = least(x.dtype)
    x, wg, wu, wd = (t.double() for t in (x, wg, wu, wd))
    rows, width = x.shape
    hidden, out = wg.shape[0], wd.shape[0]
    add = lambda k: (k + 16) * 2.0 ** -23    # a sum of k products
    g, u = x @ wg.t(), x @ wu.t()
    eg, eu = add(width) * (x.abs() @ wg.abs().t()), add(width) * (x.abs() @ wu.abs().t())
    a, s = act64(act, g)
    ea = 1.2 * eg + 2.0 ** -18 * g.abs()     # slopes are 1.13 at most; fast exponentials
    jump = (g.abs() <= eg) if act == "relu" else torch.zeros_like(g, dtype=torch.bool)
    es = 1.0 * eg + 2.0 ** -18 * (1 + g.abs()) + jump   # and their slopes' 0.8
    h = a * u
    eh = ea * (u.abs() + eu) + a.abs() * eu + 8 * E * h.abs()
    eh = eh + u_ * (h.abs() + eh) + tiny
    out_ = {"y": (h @ wd.t(), eh @ wd.abs().t() + add(hidden) * ((h.abs() + eh) @ wd.abs().t()))}
    if dy is None:
        return out_
    dy = dy.double()
    p, q = u * s, a
    ep = es * (u.abs() + eu) + s.abs() * eu
    ep, eq = ep + 2.0 ** -16 * (p.abs() + ep), ea + 2.0 ** -16 * (q.abs() + ea)
    dh = dy @ wd
    edh = add(out) * (dy.abs() @ wd.abs())
    rounded = lambda v, e: e + u_ * (v.abs() + e) + 4 * E * v.abs() + tiny
    dg, du = dh * p, dh * q
    edg = rounded(dg, edh * (p.abs() + ep) + dh.abs() * ep)
    edu = rounded(du, edh * (q.abs() + eq) + dh.abs() * eq)
    mag_g, mag_u = dg.abs() + edg, du.abs() + edu
    out_["dx"] = (dg @ wg + du @ wu, edg @ wg.abs() + edu @ wu.abs() + add(2 * hidden) * (mag_g @ wg.abs() + mag_u @ wu.abs()))
    for name, v, e, m in (("dw_gate", dg, edg, mag_g), ("dw_up", du, edu, mag_u)):
        out_[name] = (v.t() @ x, e.t() @ x.abs() + add(rows) * (m.t() @ x.abs()))
    out_["dw_down"] = (dy.t() @ h, dy.abs().t() @ eh + add(rows) * (dy.abs().t() @ (h.abs() + eh)))
    return out_


def ffn_inputs(rows, width, hidden, out, dtype, seed=0):
    return (randn(rows, width, seed=seed, dtype=dtype), randn(hidden, width, seed=seed + 1, dtype=dtype, scale=width ** -0.5),
            randn(hidden, width, seed=seed + 2, dtype=dtype, scale=width ** -0.5), randn(out, hidden, seed=seed + 3, dtype=dtype, scale=hidden ** -0.5),
            randn(rows, out, seed=seed + 4, dtype=dtype, scale=0.3))


def check_ffn(x, wg, wu, wd, dy, act="silu"):
    want = ffn64(x, wg, wu, wd, dy, act)
    leaves = [t.detach().requires_grad_() for t in (x, wg, wu, wd)]
    y = layers.gated_ffn(*leaves, activation=act)
    results = {"y": y.detach(), **dict(zip(("dx", "dw_gate", "dw_up", "dw_down"), torch.autograd.grad(y, leaves, dy)))}
    layers.check_status()
    for name, got in results.items():
        near(got, *want[name], name)
        if got.numel() >= 1000:
            # the result's rounding and that of the operand before it: each u / sqrt(3) of the result at most, in the root mean square
            rel = float((got.double() - want[name][0]).norm() / want[name][0].norm())
            assert rel < half_step(x.dtype), (name, rel)
    with torch.no_grad():
        assert torch.equal(layers.gated_ffn(*leaves, activation=act), results["y"])
    return results


@gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("rows,width,hidden,out", [
    (1, 64, 64, 64), (1, 8, 8, 8), (1, 1, 1, 1), (2, 3, 5, 7), (64, 64, 128, 64), (130, 72, 200, 136), (257, 128, 64, 264), (100, 1001, 333, 77), (33, 512, 2000, 512), (1, 2048, 1024, 2048),
    (300, 264, 136, 8), (520, 520, 1032, 520)])
def test_ffn(rows, width, hidden, out, dtype):
    check_ffn(*ffn_inputs(rows, width, hidden, out, dtype))


@gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("rows,width,hidden,out", [(1, 64, 64, 64), (2, 3, 5, 7), (1, 40, 64, 1200), (5, 1001, 333, 77), (16, 136, 200, 72), (16, 512, 2000, 512)])
def test_ffn_of_few_rows_rounds_only_results(rows, width, hidden, out, dtype):
    """Up to 16 rows, h, dg and du are two numbers of the type each: what the second leaves is half a step of half a step."""
    x, wg, wu, wd, dy = ffn_inputs(rows, width, hidden, out, dtype, seed=11)
    want = ffn64(x, wg, wu, wd, dy, "silu", operands=half_step(dtype) ** 2)
    leaves = [t.detach().requires_grad_() for t in (x, wg, wu, wd)]
    y = layers.gated_ffn(*leaves)
    for name, got in {"y": y.detach(), **dict(zip(("dx", "dw_gate", "dw_up", "dw_down"), torch.autograd.grad(y, leaves, dy)))}.items():
        near(got, *want[name], name)
    layers.check_status()


@gpu
def test_ffn_of_few_rows_beyond_the_type():
    """A hidden value that rounds to infinity leaves nothing behind that a second number could hold."""
    one = torch.ones(1, 1, device="cuda", dtype=FP16)
    with torch.no_grad():
        assert layers.gated_ffn(300 * one, one, one, one, "relu").item() == math.inf


@gpu
@pytest.mark.parametrize("act", sorted(layers.ACTIVATIONS))
def test_ffn_activations(act):
    x, *rest = ffn_inputs(140, 96, 160, 96, BF16, seed=5)
    check_ffn(x * 3, *rest, act=act)


@gpu
def test_ffn_of_large_values():
    """Gates far beyond where exponentials overflow."""
    for act in ("silu", "gelu", "gelu_tanh"):
        x, wg, wu, wd, dy = ffn_inputs(40, 64, 128, 64, BF16, seed=9)
        for name, got in check_ffn(x * 16, wg * 16, wu, wd, dy, act=act).items():
            assert bool(got.isfinite().all()), name
        for v in (1e25, -1e25):   # whose squares are infinite
            x1 = torch.full((2, 8), v, device="cuda", dtype=BF16).requires_grad_()
            w = torch.eye(8, device="cuda", dtype=BF16)
            y = layers.gated_ffn(x1, w, w * 0, w, activation=act)
            (g,) = torch.autograd.grad(y, x1, torch.ones_like(y))
            assert not bool(y.any()) and not bool(g.any()), act


@gpu
def test_ffn_of_many_tiles():
    """More tiles than run at once, of rows and columns that end inside of them."""
    check_ffn(*ffn_inputs(2100, 328, 2600, 328, BF16, seed=2))


@gpu
def test_ffn_of_strided_operands():
    big = randn(70, 3, 144, seed=1, dtype=BF16)
    _, wg, wu, wd, dy = ffn_inputs(70, 128, 96, 128, BF16, seed=3)
    wide = randn(96, 400, seed=8, dtype=BF16, scale=0.1)
    for x in (big[:, 1, :128], big[:, 1, 3:131], big[:, 0, :140:1][:, 8:136]):
        for gate in (wg, wide[:, 16:144], wide[:, 5:133], wg.t().contiguous().t()):
            check_ffn(x, gate, wu, wd, dy)
    x = randn(7, 10, 128, seed=4, dtype=BF16).requires_grad_()
    y = layers.gated_ffn(x, wg, wu, wd)
    assert y.shape == (7, 10, 128)
    y.sum().backward()
    want = ffn64(x.detach().view(70, 128), wg, wu, wd, torch.ones(70, 128, device="cuda"), "silu")
    near(x.grad.view(70, 128), *want["dx"])


@gpu
def test_ffn_gradients_of_some_inputs_and_of_no_rows():
    x, wg, wu, wd, dy = ffn_inputs(50, 64, 96, 64, BF16, seed=6)
    want = ffn64(x, wg, wu, wd, dy, "silu")
    names = ("dx", "dw_gate", "dw_up", "dw_down")
    for which in range(1, 16):
        leaves = [t.detach().requires_grad_(bool(which >> k & 1)) for k, t in enumerate((x, wg, wu, wd))]
        asked = [(n, t) for n, t in zip(names, leaves) if t.requires_grad]
        for (name, _), got in zip(asked, torch.autograd.grad(layers.gated_ffn(*leaves), [t for _, t in asked], dy)):
            near(got, *want[name], name)
    leaves = [t.detach().requires_grad_() for t in (x[:0], wg, wu, wd)]
    layers.gated_ffn(*leaves).sum().backward()
    assert leaves[0].grad.shape == (0, 64) and all(not bool(t.grad.any()) for t in leaves[1:])


def test_ffn_gradient_formulas_are_those_of_differences():
    """The formulas that the kernels are held to, in 64 bits on the CPU: (L(t + h v) - L(t - h v)) / 2h, error of order h^2 and 2^-52 / h."""
    make = lambda *shape: torch.randn(shape, generator=torch.Generator().manual_seed(sum(shape)), dtype=torch.float64)
    x, wg, wu, wd, dy = make(5, 6), make(7, 6), make(7, 6) + 0.5, make(4, 7), make(5, 4)
    h = 1e-4
    for act in ("silu", "gelu", "gelu_tanh"):
        value = lambda *t: float((ffn64_y(*t, act) * dy).sum())
        got = grads64(x, wg, wu, wd, dy, act)
        for k, t in enumerate((x, wg, wu, wd)):
            v = make(*t.shape).flip(0)
            at = lambda s: [t + s * v if i == k else o for i, o in enumerate((x, wg, wu, wd))]
            assert abs((value(*at(h)) - value(*at(-h))) / (2 * h) - float((got[k] * v).sum())) < 1e-5


def ffn64_y(x, wg, wu, wd, act):
    return (act64(act, x @ wg.t())[0] * (x @ wu.t())) @ wd.t()


def grads64(x, wg, wu, wd, dy, act):
    g, u = x @ wg.t(), x @ wu.t()
    a, s = act64(act, g)
    dh = dy @ wd
    dg, du = dh * u * s, dh * a
    return dg @ wg + du @ wu, dg.t() @ x, du.t() @ x, dy.t() @ (a * u)


# ---------------------------------------------------------------------------------------------------------------------
# distillation
# ---------------------------------------------------------------------------------------------------------------------


def distill64(logits, teacher, ids, T, weights=None):
    """(rows' losses, weights that count, the rows' gradients, slack of a loss, slack of a gradient), unweighted."""
    n, v = logits.shape
    c = 1.4426950408889634 / T
    s = logits.double() / T
    there = (ids >= 0) & (ids < v) & ~(teacher.double() == -math.inf)
    z = torch.where(there, teacher.double() / T, -math.inf)
    has = there.any(1)
    w = (torch.ones(n, device=logits.device) if weights is None else weights).double() * has
    log_p = torch.where(has[:, None], z - torch.where(has[:, None], z, 0.0).logsumexp(1, keepdim=True), -math.inf)
    p = log_p.exp()
    log_q = s - s.logsumexp(1, keepdim=True)
    at = torch.where(there, ids.long(), 0)
    loss = T * T * torch.where(there & (p > 0), p * (log_p - log_q.gather(1, at)), 0.0).sum(1)
    q = log_q.exp()
    full = torch.zeros_like(q).scatter_add_(1, at, torch.where(there, p, 0.0))
    finite = lambda t: torch.where(t.isfinite(), t.abs(), 0.0).amax(1)
    big, big_t = finite(logits.double()) * c, finite(torch.where(there, teacher.double(), 0.0)) * c   # magnitudes of the exponents
    # each exponent is off by a rounding or two of its magnitude; sums of V / threads elements, K / threads, and the levels above
    per = 64 + v / 32
    slack_loss = T * T * E * (8 * (big + big_t) + per + 8 * loss.abs() / T / T)
    slack_grad = T * E * ((4 * big + per)[:, None] * q + (4 * big_t + per)[:, None] * full)
    return loss, w, T * (q - full), slack_loss, slack_grad


def check_distill(logits, teacher, ids, T=1.0, weights=None, upstream=1.0):
    loss, w, grad, slack_loss, slack_grad = distill64(logits, teacher, ids, T, weights)
    on = w != 0
    zero = lambda t: torch.where(on.view(-1, *[1] * (t.dim() - 1)), t, 0.0)
    total = w.sum()
    # weighted rows
    leaf = logits.detach().requires_grad_()
    rows = layers.distillation_loss(leaf, teacher, ids, T, weights, "none")
    near(rows.detach(), zero(loss * w), zero(slack_loss * w.abs()), "rows")
    up = torch.linspace(-1, 2, len(w), device="cuda")
    (g,) = torch.autograd.grad(rows, leaf, up)
    f = (up.double() * w)[:, None]
    near(g, zero(grad * f), zero((slack_grad + 8 * E * grad.abs()) * f.abs()), "gradient of rows")
    for reduction in ("sum", "mean"):
        by = 1.0 if reduction == "sum" else (1 / total if total != 0 else torch.zeros_like(total))
        value, slack = zero(loss * w).sum() * by, zero((slack_loss + 4 * E * loss.abs()) * w.abs()).sum() * by
        leaf = logits.detach().requires_grad_()
        got = layers.distillation_loss(leaf, teacher, ids, T, weights, reduction)
        near(got.detach(), value, slack, reduction)
        (g,) = torch.autograd.grad(got * upstream, leaf)
        f = (w * by * upstream)[:, None]
        near(g, zero(grad * f), zero((slack_grad + 8 * E * grad.abs()) * f.abs()), "gradient, " + reduction)
        assert not bool(g[~on].any())
        both = layers.distillation_loss_and_grad(logits, teacher, ids, T, weights, reduction, scale=upstream)
        near(both[0], value, slack, reduction + " of both")
        near(both[1], zero(grad * f), zero((slack_grad + 8 * E * grad.abs()) * f.abs()), "gradient of both, " + reduction)
        with torch.no_grad():
            assert torch.equal(layers.distillation_loss(leaf, teacher, ids, T, weights, reduction), got)


def distill_inputs(rows, vocab, top, dtype, seed=0):
    logits = randn(rows, vocab, seed=seed, scale=2.5)
    t, ids = (logits + randn(rows, vocab, seed=seed + 1, scale=2.0)).topk(top, dim=1)
    return logits.to(dtype), t.to(dtype), ids


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, FP16])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (4, 2, 1), (256, 10, 10), (5, 7, 3), (37, 100, 100), (9, 1000, 17), (3, 1024, 64), (6, 1025, 64), (5, 5003, 128), (4, 32768, 1024),
                                            (3, 50257, 64), (2, 128256, 128), (2, 400001, 16), (700, 2500, 7)])
def test_distill(rows, vocab, top, dtype):
    logits, teacher, ids = distill_inputs(rows, vocab, top, dtype)
    check_distill(logits, teacher, ids, T=2.0, upstream=0.5)


@gpu
@pytest.mark.parametrize("vocab", [50, 4099])
@pytest.mark.parametrize("T", [0.5, 1, 7.3])
def test_distill_of_padded_masked_and_repeated_entries(T, vocab):
    logits, teacher, ids = distill_inputs(24, vocab, 12, BF16, seed=3)
    ids = ids.clone()
    ids[1, 5:] = -1
    ids[2] = -1                                    # a row without a teacher
    ids[3, 2], ids[3, 4] = vocab, vocab + 10 ** 9  # beyond the classes: padding too
    ids[4, 7] = ids[4, 0]                          # the same class twice, three times
    ids[4, 9] = ids[4, 0]
    ids[5, :] = ids[5, 0]
    ids[12], ids[13] = -1, -1                      # padding before and between class 0
    ids[12, 3], ids[13, 2], ids[13, 5], ids[13, 6] = 0, 0, 0, 1
    ids[14, :6] = torch.arange(6, device="cuda") * 64 % vocab   # neighbours in a table
    teacher[6, 3:] = -math.inf
    teacher[7] = -math.inf
    teacher[1, 5:] = math.nan                      # beside padding: not looked at
    weights = torch.rand(24, generator=gen(1), device="cuda") + 0.5
    weights[8:11] = 0
    logits[8] = math.nan                           # in rows of weight 0: not looked at
    logits[9, 3] = math.inf
    logits[2] = -math.inf
    clean = logits.clone()
    clean[[2, 8, 9]] = 0
    for w in (weights, None):
        if w is None:
            logits = clean
        check_distill(logits, teacher, ids, T, w)
        check_distill(logits, teacher, ids.int(), T, w)
    mask = weights > 0
    a = layers.distillation_loss(clean, teacher, ids, T, mask)
    assert torch.equal(a, layers.distillation_loss(clean, teacher, ids, T, mask.float()))
    check_distill(logits, teacher, ids, T, torch.zeros(24, device="cuda"))   # nothing counts


@gpu
@pytest.mark.parametrize("vocab", [40, 3001])
def test_distill_of_infinite_logits(vocab):
    """-inf is a class that is left out: probability and gradient 0, a loss of +inf only where the teacher asks for it."""
    logits, teacher, ids = distill_inputs(8, vocab, 5, F32, seed=4)
    out = torch.rand(8, vocab, generator=gen(2), device="cuda") < 0.3
    out.scatter_(1, ids, False)
    logits[out] = -math.inf
    check_distill(logits, teacher, ids, 2.0)
    (g,) = torch.autograd.grad(layers.distillation_loss(logits.requires_grad_(), teacher, ids), logits)
    assert not bool(g[out].any())
    logits = logits.detach().clone()
    logits[3, ids[3, 0]] = -math.inf
    rows = layers.distillation_loss(logits, teacher, ids, reduction="none")
    assert rows[3] == math.inf and bool(rows[[0, 1, 2, 4, 5, 6, 7]].isfinite().all())
    logits[4], logits[5, 1], logits[6, 0] = -math.inf, math.inf, math.nan
    assert layers.distillation_loss(logits, teacher, ids, reduction="none").isnan().tolist() == [False] * 4 + [True] * 3 + [False]


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, FP16])
@pytest.mark.parametrize("vocab", [60, 5001])
def test_distill_beside_masks_of_the_lowest_value(vocab, dtype):
    """Classes that are masked with the type's lowest number, among others, have no probability and no gradient."""
    logits, teacher, ids = distill_inputs(7, vocab, 6, dtype, seed=5)
    out = torch.rand(7, vocab, generator=gen(3), device="cuda") < 0.9
    out.scatter_(1, ids, False)
    for value, T in ((torch.finfo(dtype).min, 1.0), (torch.finfo(dtype).min, 4.0), (-1e4, 1.0), (-1e30 if dtype != FP16 else -3e4, 1.0), (-1e38 if dtype != FP16 else -6e4, 0.5)):
        logits[out] = value
        rows = layers.distillation_loss(logits, teacher, ids, T, reduction="none")
        want, *_ = distill64(logits.double().masked_fill(out, -math.inf), teacher, ids, T)
        # the magnitudes of the exponents: those of the logits that are left
        slack = T * T * E * (16 * float(logits[~out].abs().max()) * 1.45 / T + 64 + vocab / 32 + 8 * want / T / T)
        near(rows, want, slack, "rows")
        _, g = layers.distillation_loss_and_grad(logits, teacher, ids, T)
        assert bool(g.isfinite().all()) and not bool(g[out].any())
    # nothing but such values: all classes are alike
    logits[:] = torch.finfo(dtype).min
    for T in (1.0, 2.0):
        for t in (torch.zeros_like(teacher), torch.full_like(teacher, torch.finfo(dtype).min)):
            loss, g = layers.distillation_loss_and_grad(logits, t, ids, T, reduction="sum")
            want = T * T * math.log(vocab / 6) * 7   # uniform over the classes, and over the six entries
            assert abs(float(loss) - want) < want * 64 * E
            full = torch.full((7, vocab), T / vocab, device="cuda", dtype=torch.float64).scatter_add_(1, ids, torch.full((7, 6), -T / 6, device="cuda", dtype=torch.float64))
            near(g, full, 64 * E * full.abs(), "uniform")
    # far off centre: as exact as the logits
    near_one = (torch.randn(7, vocab, generator=gen(4), device="cuda") + 1e3).to(dtype)
    rows = layers.distillation_loss(near_one, teacher, ids, reduction="none")
    want, *_ = distill64(near_one - 1e3 if dtype == F32 else near_one.double() - 1e3, teacher, ids, 1.0)
    near(rows, want, E * (16 * 8 * 1.45 + 64 + vocab / 32 + 8 * want + 16 * float(teacher.abs().max())), "off centre")


@gpu
def test_distill_of_strided_logits_and_other_types_of_teacher():
    big = randn(12, 3, 1200, seed=1, dtype=BF16, scale=2.0)
    for logits in (big[:, 1, 8:1108], big[:, 1, 3:1104], big[:, 0, :30], big[:, 0, ::3]):
        _, teacher, ids = distill_inputs(12, logits.shape[1], 9, F32, seed=2)
        for t in (teacher, teacher.half(), teacher.bfloat16()):
            check_distill(logits, t, ids, 1.5)
    logits, teacher, ids = distill_inputs(30, 200, 4, F32, seed=7)
    a = layers.distillation_loss(logits.view(5, 6, 200), teacher.view(5, 6, 4), ids.view(5, 6, 4), weights=torch.ones(5, 6, device="cuda"))
    assert torch.equal(a, layers.distillation_loss(logits, teacher, ids))


@gpu
def test_distill_of_many_and_of_no_rows():
    logits, teacher, ids = distill_inputs(40_001, 13, 5, F32, seed=2)
    check_distill(logits, teacher, ids, 1.0, (torch.rand(40_001, generator=gen(5), device="cuda") < 0.8).float())
    for reduction in ("mean", "sum"):
        leaf = torch.empty(0, 9, device="cuda", requires_grad=True)
        loss = layers.distillation_loss(leaf, torch.empty(0, 3, device="cuda"), torch.empty(0, 3, device="cuda", dtype=torch.int64), reduction=reduction)
        loss.backward()
        assert float(loss.detach()) == 0 and leaf.grad.shape == (0, 9)


@gpu
def test_distill_gradient_is_that_of_differences():
    """Error of order h^2 of the difference, and the loss's rounding (64 of 2^-24) over h."""
    logits, teacher, ids = distill_inputs(5, 300, 20, F32, seed=8)
    v = randn(5, 300, seed=9)
    h, T = 2.0 ** -6, 2.0
    value = lambda t: float(layers.distillation_loss(t, teacher, ids, T, reduction="sum"))
    leaf = logits.clone().requires_grad_()
    (g,) = torch.autograd.grad(layers.distillation_loss(leaf, teacher, ids, T, reduction="sum"), leaf)
    loss = value(logits)
    assert abs((value(logits + h * v) - value(logits - h * v)) / (2 * h) - float((g * v).sum())) < 10 * h * h * 5 + 64 * E * (loss + 100) / h


@gpu
def test_distill_scale_on_the_device():
    logits, teacher, ids = distill_inputs(6, 700, 8, FP16, seed=1)
    scale = torch.tensor([1024.0], device="cuda")
    a, b = (layers.distillation_loss_and_grad(logits, teacher, ids, scale=s) for s in (scale, 1024.0))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


# ---------------------------------------------------------------------------------------------------------------------
# refusals
# ---------------------------------------------------------------------------------------------------------------------


def test_library_refuses_before_it_launches():
    """Arguments out of range get a negative code on the host (no GPU is asked)."""
    norm = dict(x=16, y=16, rows=4, width=8, x_stride=8, type=L.FP32, weight_type=L.FP32, eps=1e-5)
    for bad in (dict(x=None), dict(y=None), dict(width=0), dict(width=L.NORM_MOST + 1), dict(rows=-1), dict(type=3), dict(eps=-1.0), dict(bias=16), dict(mean=16),
                dict(eps=float("nan"))):
        assert L.lib.pylo_b200_layer_norm(C.byref(L.Norm(**{**norm, **bad})), None) < 0, bad
    back = dict(x=16, dy=16, dx=16, mean=16, rstd=16, rows=4, width=8, x_stride=8, dy_stride=8, type=L.FP32, weight_type=L.FP32)
    for bad in (dict(mean=None), dict(dy=None), dict(dweight=16), dict(dweight=16, work=16, work_floats=1)):
        assert L.lib.pylo_b200_layer_norm_backward(C.byref(L.Norm(**{**back, **bad})), None) < 0, bad
    distill = dict(logits=16, teacher=16, ids=16, loss=16, work=16, work_bytes=1 << 20, rows=4, stride=10, vocab=10, top=3, type=L.FP32, teacher_type=L.FP32,
                   ids_bytes=8, reduction=L.REDUCE_MEAN, temperature=1.0, scale=1.0)
    for bad in (dict(logits=None), dict(ids=None), dict(vocab=0), dict(top=0), dict(top=L.DISTILL_MOST_TOP + 1), dict(ids_bytes=2), dict(temperature=0.0), dict(stride=9),
                dict(work=None), dict(work_bytes=8), dict(type=5), dict(teacher_type=-1), dict(logits=18), dict(work=24), dict(temperature=float("nan"))):
        assert L.lib.pylo_b200_distill(C.byref(L.Distill(**{**distill, **bad})), L.DISTILL_LOSS, None) < 0, bad
    assert L.lib.pylo_b200_distill(C.byref(L.Distill(**distill)), L.DISTILL_GRAD, None) < 0      # no grad
    assert L.lib.pylo_b200_distill(C.byref(L.Distill(**distill)), 4, None) < 0
    ffn = dict(x=256, w_gate=256, w_up=256, w_down=256, y=256, kept=256, rows=4, ld_x=8, ld_gate=8, ld_up=8, ld_down=16, width=8, hidden=16, out=8, type=L.BF16)
    for bad in (dict(x=None), dict(x=264), dict(ld_x=7), dict(ld_x=12), dict(ld_down=8), dict(kept=16), dict(kept=None), dict(type=L.FP32), dict(activation=4), dict(width=0),
                dict(hidden=0), dict(out=0), dict(rows=-1), dict(rows=1 << 31), dict(y=None)):
        assert L.lib.pylo_b200_gated_ffn(C.byref(L.Ffn(**{**ffn, **bad})), None) < 0, bad
    back = {**ffn, "dy": 256, "ld_dy": 8, "work": 256, "dx": 256}
    for bad in (dict(dy=None), dict(ld_dy=4), dict(work=None), dict(work=16), dict(rows=0), dict(w_up=None), dict(kept=None)):
        assert L.lib.pylo_b200_gated_ffn_backward(C.byref(L.Ffn(**{**back, **bad})), None) < 0, bad
    pad = dict(src=16, dst=16, rows=4, cols=5, row_stride=5, col_stride=1, ld=8)
    for bad in (dict(src=None), dict(dst=None), dict(dst=24), dict(src=17), dict(ld=4), dict(ld=12), dict(rows=-1)):
        assert L.lib.pylo_b200_pad_rows((L.Pad * 1)(L.Pad(**{**pad, **bad})), 1, None) < 0, bad
    assert L.lib.pylo_b200_pad_rows((L.Pad * 5)(), 5, None) < 0
    for call in (L.lib.pylo_b200_layer_norm, L.lib.pylo_b200_layer_norm_backward, L.lib.pylo_b200_gated_ffn, L.lib.pylo_b200_gated_ffn_backward):
        assert call(None, None) < 0


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 8)
    with pytest.raises(ValueError, match="CUDA"):
        layers.layer_norm(x)
    with pytest.raises(ValueError, match="CUDA"):
        layers.gated_ffn(x.bfloat16(), *[torch.zeros(8, 8, dtype=BF16)] * 3)
    with pytest.raises(ValueError, match="CUDA"):
        layers.distillation_loss(x, x, torch.zeros(2, 8, dtype=torch.int64))
    with pytest.raises(TypeError, match="tensor"):
        layers.layer_norm([1.0])
    with pytest.raises(ValueError, match="activation"):
        layers.gated_ffn(x, x, x, x, activation="tanh")
    with pytest.raises(ValueError, match="activation"):
        layers.GatedFFN(8, 8, activation="tanh")


@gpu
def test_refusals():
    x, v = torch.zeros(3, 8, device="cuda"), torch.zeros(8, device="cuda")
    for error, args in ((TypeError, (x.double(),)), (ValueError, (x[0, 0],)), (ValueError, (x[:, :0],)), (ValueError, (torch.zeros(1, 40000, device="cuda"),)), (ValueError, (x, None, v)),
                        (ValueError, (x, v[:7])), (TypeError, (x.half(), v.bfloat16())), (TypeError, (x, v.half())), (TypeError, (x.half(), v, v.half())), (ValueError, (x, v.cpu())),
                        (ValueError, (x, v, v, -1.0)), (ValueError, (x, v, v, math.nan))):
        with pytest.raises(error):
            layers.layer_norm(*args)
    x, w = torch.zeros(3, 8, device="cuda", dtype=BF16), torch.zeros(16, 8, device="cuda", dtype=BF16)
    for error, args in ((TypeError, (x.float(), w.float(), w.float(), w.t().float())), (TypeError, (x, w.half(), w, w.t())), (ValueError, (x, w, w, w)), (ValueError, (x, w, w[:8], w.t())),
                        (ValueError, (x, w[0], w[0], w.t())), (ValueError, (x, w, w.cpu(), w.t())), (ValueError, (x[:, :0], w[:, :0], w[:, :0], w.t()))):
        with pytest.raises(error):
            layers.gated_ffn(*args)
    s, t, i = torch.zeros(3, 8, device="cuda"), torch.zeros(3, 4, device="cuda"), torch.zeros(3, 4, device="cuda", dtype=torch.int64)
    for error, args in ((TypeError, (s.double(), t, i)), (TypeError, (s, t, i.float())), (ValueError, (s, t, i[:, :2])), (ValueError, (s[:2], t, i)), (ValueError, (s, t, i, 0.0)),
                        (ValueError, (s, t, i, math.inf)), (ValueError, (s, t, i, 1.0, torch.ones(2, device="cuda"))), (ValueError, (s, t, i, 1.0, None, "median")), (ValueError, (s, t[:, :0], i[:, :0])),
                        (ValueError, (s, t.clone().requires_grad_(), i)), (ValueError, (s, torch.zeros(3, 1025, device="cuda"), torch.zeros(3, 1025, device="cuda", dtype=torch.int64))),
                        (ValueError, (s, t.cpu(), i)), (TypeError, (s, t, i, 1.0, torch.ones(3, device="cuda", dtype=torch.int32)))):
        with pytest.raises(error):
            layers.distillation_loss(*args)
    with pytest.raises(ValueError):
        layers.distillation_loss_and_grad(s, t, i, reduction="none")
    with pytest.raises(ValueError):
        layers.distillation_loss_and_grad(s, t, i, scale=torch.ones(2, device="cuda"))


@gpu
def test_a_reported_wait_stops_the_next_call(monkeypatch):
    x, wg, wu, wd, _ = ffn_inputs(4, 8, 8, 8, BF16)
    layers.gated_ffn(x, wg, wu, wd)
    layers.check_status()
    layers._reported[1][0] = 16
    for call in (lambda: layers.gated_ffn(x, wg, wu, wd), layers.check_status):
        with pytest.raises(L.PyloLibError, match="ran out"):
            call()
    layers.clear_status()
    layers.gated_ffn(x, wg, wu, wd)
    layers.check_status()


# ---------------------------------------------------------------------------------------------------------------------
# together, on streams and in graphs
# ---------------------------------------------------------------------------------------------------------------------


def student_step(student, x, teacher, ids, weights):
    loss = layers.distillation_loss(student(x), teacher, ids, 2.0, weights)
    loss.backward()
    return loss.detach()


def student_and_batch(seed=0, classes=1003):
    torch.manual_seed(seed)
    student = workloads.student(72, 136, 2, classes)
    x = randn(5, 31, 72, seed=seed + 1, dtype=BF16)
    _, teacher, ids = distill_inputs(155, classes, 16, BF16, seed=seed + 2)
    return student, (x, teacher.view(5, 31, 16), ids.view(5, 31, 16), (torch.rand(5, 31, generator=gen(seed), device="cuda") < 0.9))


@gpu
@pytest.mark.parametrize("name", ["AdamW_CUDA", "AdafacLO_CUDA"])
def test_a_student_trains_on_them(name):
    """Gradients of the whole model against 64 bits, a step of an optimizer of this package, the next pass."""
    from pylo_b200 import models, optim

    student, batch = student_and_batch()
    student_step(student, *batch)
    twin = {k: p.detach().double().requires_grad_() for k, p in student.named_parameters()}

    def norm(x, k):
        return torch.nn.functional.layer_norm(x, x.shape[-1:], twin[f"norms.{k}.weight"], twin[f"norms.{k}.bias"])

    x, teacher, ids, weights = batch
    h = x.double()
    for k in range(2):
        z = norm(h, k)
        g, u = z @ twin[f"blocks.{k}.w_gate"].t(), z @ twin[f"blocks.{k}.w_up"].t()
        h = h + (torch.nn.functional.silu(g) * u) @ twin[f"blocks.{k}.w_down"].t()
    s = norm(h, 2) @ twin["head.weight"].t()
    p = torch.softmax(teacher.double() / 2, -1)
    kl = (p * (p.log() - torch.log_softmax(s / 2, -1).gather(-1, ids))).sum(-1) * 4
    ((kl * weights).sum() / weights.sum()).backward()
    for k, q in student.named_parameters():
        rel = float((q.grad.double() - twin[k].grad).norm() / twin[k].grad.norm())
        # about twenty roundings lie between a gradient and the input, each of half a step at most, amplified by the norms' and blocks' slopes
        assert rel < 40 * half_step(BF16), (k, rel)
    params = list(student.parameters())
    before = [p.detach().clone() for p in params]
    if name == "AdamW_CUDA":
        opt = optim.AdamW_CUDA(params, lr=1e-2, clip_grad=True, clip_norm=1.0)
    else:   # fp32 parameters of its own, which the student's follow
        masters = [torch.nn.Parameter(p.detach().float()) for p in params]
        for m, p in zip(masters, params):
            m.grad = p.grad.float()
        torch.manual_seed(0)
        opt = optim.AdafacLO_CUDA(masters, lr=1e-2, network=models.MetaMLP(39, 32, 1))
    opt.step()
    if name == "AdafacLO_CUDA":
        with torch.no_grad():
            for m, p in zip(masters, params):
                p.copy_(m)
    assert any(not torch.equal(a, p) for a, p in zip(before, params))
    for p in params:
        p.grad = None
    assert bool(torch.isfinite(student_step(student, *batch)))


@gpu
def test_the_same_inputs_give_the_same_bits():
    results = []
    for _ in range(2):
        student, batch = student_and_batch(seed=3)
        results.append([student_step(student, *batch)] + [p.grad for p in student.parameters()])
    assert all(torch.equal(a, b) for a, b in zip(*results))


@gpu
def test_on_another_stream():
    student, batch = student_and_batch(seed=5)
    want = [student_step(student, *batch)] + [p.grad.clone() for p in student.parameters()]
    side = torch.cuda.Stream()
    for _ in range(3):
        for p in student.parameters():
            p.grad = None
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = [student_step(student, *batch)] + [p.grad for p in student.parameters()]
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@gpu
def test_two_streams_at_once():
    """Calls that run beside one another have nothing in common."""
    batches = [student_and_batch(seed=k) for k in (11, 12)]
    want = []
    for student, batch in batches:
        want.append([student_step(student, *batch)] + [p.grad.clone() for p in student.parameters()])
    streams = [torch.cuda.Stream() for _ in batches]
    for _ in range(5):
        got = []
        for student, _ in batches:
            for p in student.parameters():
                p.grad = None
        for stream, (student, batch) in zip(streams, batches):
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                got.append([student_step(student, *batch)] + [p.grad for p in student.parameters()])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))


@gpu
def test_on_another_device_than_the_current_one():
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU visible")
    student, batch = student_and_batch(seed=5)
    want = [student_step(student, *batch)] + [p.grad.clone() for p in student.parameters()]
    for p in student.parameters():
        p.grad = None
    student, batch = student.to("cuda:1"), [t.to("cuda:1") for t in batch]
    got = [student_step(student, *batch)] + [p.grad for p in student.parameters()]
    assert all(torch.equal(a.cpu(), b.cpu()) for a, b in zip(got, want))


@gpu
def test_norm_beyond_32_bits():
    """More than 2^31 elements: the last rows are those of a small call; the columns' sums hold for gradients that are equal."""
    rows, width = 2_100_003, 1024
    x, dy = randn(1, width, seed=1, dtype=BF16).repeat(rows, 1), randn(1, width, seed=2, dtype=BF16).repeat(rows, 1)
    x[-3:], dy[-3:] = randn(3, width, seed=3, dtype=BF16), randn(3, width, seed=4, dtype=BF16)
    w, b = randn(width, seed=5).requires_grad_(), randn(width, seed=6).requires_grad_()
    y = layers.layer_norm(x.requires_grad_(), w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    few = [t[-5:].detach().clone() for t in (x, dy)]
    small = few[0].requires_grad_()
    z = layers.layer_norm(small, w, b)
    assert torch.equal(y[-5:], z) and torch.equal(dx[-5:], torch.autograd.grad(z, small, few[1])[0])
    assert torch.equal(y[0], z[0]) and torch.equal(dx[0], dx[1000])
    want = norm64(small.detach()[:1], w.detach(), b.detach(), few[1][:1], 1e-5)
    # a column's sum of equal terms: rows / 592 / 4 in a line per warp, then those
    for got, name in ((dw, "dweight"), (db, "dbias")):
        value, slack = (v * (rows - 3) for v in want[name])
        near(got, value, slack + 6e3 * E * value.abs() + 50, name)   # (three rows of other terms, of 5 at most each)


@gpu
def test_distill_beyond_32_bits():
    rows, vocab = 43_000, 50_257
    logits, teacher, ids = distill_inputs(5, vocab, 8, BF16)
    many = torch.empty(rows, vocab, device="cuda", dtype=BF16)
    many[:-5] = logits[:1]
    many[-5:] = logits
    t, i = (torch.cat([v[:1].expand(rows - 5, 8), v]) for v in (teacher, ids))
    got = layers.distillation_loss(many.requires_grad_(), t, i, reduction="none")
    (g,) = torch.autograd.grad(got, many, torch.ones_like(got))
    small = logits.requires_grad_()
    want = layers.distillation_loss(small, teacher, ids, reduction="none")
    (h,) = torch.autograd.grad(want, small, torch.ones_like(want))
    # (few rows are shared by several CTAs, whose sums are added up in another order)
    assert torch.allclose(got[-5:], want, rtol=64 * E, atol=64 * E)
    assert bool((got[:-5] == got[0]).all()) and torch.equal(g[0], g[-6])
    near(g[-5:], h.double(), 2 * half_step(BF16) * h.double().abs() + 1e-9)


@gpu
def test_ffn_beyond_32_bits():
    """More than 2^31 hidden values: the last rows are those of a small call."""
    rows, width, hidden = 270_003, 64, 8008
    x, wg, wu, wd, dy = ffn_inputs(300, width, hidden, 8, BF16, seed=3)
    many, many_dy = torch.empty(rows, width, device="cuda", dtype=BF16), torch.empty(rows, 8, device="cuda", dtype=BF16)
    for a, b in ((many, x), (many_dy, dy)):
        a[:-300] = b[:1]
        a[-300:] = b
    many.requires_grad_()
    (dx,) = torch.autograd.grad(layers.gated_ffn(many, wg, wu, wd), many, many_dy)
    want = ffn64(x, wg, wu, wd, dy, "silu")
    near(dx[-300:], *want["dx"], "dx")
    assert torch.equal(dx[0], dx[-301])
    layers.check_status()


@gpu
def test_ffn_of_a_contraction_of_many_stages():
    """The weights' gradients of 2^28 rows, of which the last 300 are not zero: no wait for a whole tile runs out, and every row counts."""
    rows, width, hidden = (1 << 28) + 5, 8, 8
    x, wg, wu, wd, dy = ffn_inputs(300, width, hidden, 8, BF16, seed=4)
    many, many_dy = torch.zeros(rows, width, device="cuda", dtype=BF16), torch.zeros(rows, 8, device="cuda", dtype=BF16)
    many_dy[:] = dy[:1]
    many[-300:], many_dy[-300:] = x, dy
    weights = [w.clone().requires_grad_() for w in (wg, wu, wd)]
    grads = torch.autograd.grad(layers.gated_ffn(many, *weights), weights, many_dy)
    layers.check_status()
    want = ffn64(x, wg, wu, wd, dy, "silu")
    for name, g in zip(("dw_gate", "dw_up", "dw_down"), grads):
        near(g, *want[name], name)


@gpu
def test_captured_into_graphs():
    """Forward and backward of a student in a graph; two graphs that are replayed in turn, with new inputs."""
    graphs = []
    for seed in (7, 8):
        student, batch = student_and_batch(seed=seed)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            student_step(student, *batch)
        torch.cuda.current_stream().wait_stream(side)
        for p in student.parameters():
            p.grad = None
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            loss = student_step(student, *batch)
        graphs.append((graph, student, batch, loss, [p.grad for p in student.parameters()]))
    for round_ in range(3):
        for k, (graph, student, batch, loss, grads) in enumerate(graphs):
            batch[0].copy_(randn(5, 31, 72, seed=100 + 10 * round_ + k, dtype=BF16))
            graph.replay()
        for graph, student, batch, loss, grads in graphs:
            for p in student.parameters():
                p.grad = None
            want = student_step(student, *batch)
            assert torch.equal(want, loss)
            assert all(torch.equal(p.grad, g) for p, g in zip(student.parameters(), grads))
            for p in student.parameters():
                p.grad = None


@gpu
def test_twice_through_one_graph_of_autograd():
    """retain_graph: a second backward pass gives the same; a second derivative is refused."""
    logits, teacher, ids = distill_inputs(6, 50, 4, F32)
    x, wg, wu, wd, dy = ffn_inputs(20, 32, 48, 32, BF16)
    for leaf, call in ((logits, lambda t: layers.distillation_loss(t, teacher, ids)), (x, lambda t: layers.gated_ffn(t, wg, wu, wd)), (x, lambda t: layers.layer_norm(t))):
        leaf = leaf.clone().requires_grad_()
        out = call(leaf)
        up = torch.ones_like(out)
        (a,), (b,) = (torch.autograd.grad(out, leaf, up, retain_graph=True) for _ in range(2))
        assert torch.equal(a, b)
        (g,) = torch.autograd.grad(out, leaf, up, create_graph=True)
        with pytest.raises(RuntimeError):
            g.float().sum().backward()


@gpu
def test_a_saved_input_that_is_changed_is_noticed():
    x = randn(8, 64, seed=1).requires_grad_()
    z = x * 2
    y = layers.layer_norm(z)
    z.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()


@gpu
def test_the_benchmark_runs_a_student(monkeypatch):
    import bench

    lines = []
    monkeypatch.setattr(bench, "emit", lines.append)
    bench.run_student(bench.parse(["--workload", "student_small", "--steps", "2", "--warmup", "3"]))
    (line,) = lines
    assert line["value"] > 0 and line["e2e"]["value"] > 0 and line["gpu_launches"] > 0 and line["gpu_launches"] % 2 == 0

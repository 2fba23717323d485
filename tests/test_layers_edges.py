"""Layer norm, the gated feed-forward block and distillation where calls leave the ordinary: values that are no numbers, tensors that come back
from autograd's hooks, forward-mode derivatives, first calls of several threads."""

import concurrent.futures
import ctypes as C
import contextlib
import math
import threading
import time

import pytest
import torch
import torch.autograd.forward_ad as forward

from pylo_b200 import _lib as L
from pylo_b200 import layers
from test_layers import BF16, F32, FP16, E, check_ffn, distill64, distill_inputs, ffn_inputs, near, norm64, randn

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, FP16])
@pytest.mark.parametrize("vocab,top", [(50, 12), (1024, 200), (4099, 12), (5003, 300), (400_001, 12)])
def test_distill_of_teachers_that_are_no_numbers(vocab, top, dtype):
    """A counted entry of NaN or +inf, in rows that hold padding too: the row's loss is NaN, as is its gradient where the teacher has entries, and no
    other row knows of it.  Padding has no class: nothing is read for it."""
    logits, teacher, ids = distill_inputs(12, vocab, top, dtype, seed=21)
    ids = ids.clone()
    ids[:, 3], ids[4:, 7:] = -1, vocab + 5
    ids[2, 0] = -1
    clean = teacher.clone()
    bad = {1: math.nan, 2: math.inf, 4: math.nan, 6: math.inf, 9: math.nan}
    for row, value in bad.items():
        teacher[row, 1] = value
    ids[6, 0], ids[6, 2:] = -1, -1           # nothing but padding beside it
    ids[9, 5] = ids[9, 1]                    # its class twice
    off = torch.tensor([row in bad for row in range(12)], device="cuda")
    want = distill64(logits, clean, ids, 2.0)
    for reduction in ("none", "sum", "mean"):
        leaf = logits.clone().requires_grad_()
        loss = layers.distillation_loss(leaf, teacher, ids, 2.0, reduction=reduction)
        (g,) = torch.autograd.grad(loss, leaf, torch.ones_like(loss))
        if reduction == "none":
            assert torch.equal(loss.isnan(), off)
            near(loss.detach()[~off], want[0][~off], want[3][~off], "rows")
        else:
            assert bool(loss.isnan())
        by = 1 / 12 if reduction == "mean" else 1.0
        near(g[~off], want[2][~off] * by, (want[4][~off] + 8 * E * want[2][~off].abs()) * by, "gradient of the other rows")
        there = torch.zeros_like(g, dtype=torch.bool).scatter_(1, torch.where((ids >= 0) & (ids < vocab), ids, ids[:, 1:2]), True)
        assert torch.equal(g.isnan(), there & off[:, None])
        if reduction != "none":
            both = layers.distillation_loss_and_grad(logits, teacher, ids, 2.0, reduction=reduction)
            assert bool(both[0].isnan()) and torch.equal(both[1].isnan(), there & off[:, None])
            near(both[1][~off], want[2][~off] * by, (want[4][~off] + 8 * E * want[2][~off].abs()) * by, "of both")


# ---------------------------------------------------------------------------------------------------------------------
# hooks on what autograd saves
# ---------------------------------------------------------------------------------------------------------------------


def elsewhere(t, gap=3):
    """The same matrix, rows `gap` elements further apart, beginning off a 16-byte boundary; vectors as they are."""
    if t.dim() != 2 or t.dtype == torch.uint8:
        return t.clone()
    wide = torch.full((t.shape[0], t.shape[1] + gap), 7.0, device=t.device, dtype=t.dtype)
    wide[:, 1:1 + t.shape[1]] = t
    return wide[:, 1:1 + t.shape[1]]


HOOKS = {
    "offloaded": lambda: torch.autograd.graph.save_on_cpu(),
    "offloaded, pinned": lambda: torch.autograd.graph.save_on_cpu(pin_memory=True),
    "packed": lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t.contiguous().clone(), lambda t: t),
    "unpacked elsewhere": lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t, elsewhere),
    "by columns": lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.t().contiguous().t() if t.dim() == 2 and t.is_floating_point() else t),
}


def operators_of_strided_tensors():
    """(name, function of leaves, leaves): slices with gaps between their rows, on and off 16-byte boundaries."""
    big, wide = randn(70, 3, 144, seed=1, dtype=BF16), randn(96, 400, seed=8, dtype=BF16, scale=0.1)
    _, _, wu, wd, dy = ffn_inputs(70, 128, 96, 128, BF16, seed=3)
    tall = randn(128, 104, seed=9, dtype=BF16, scale=0.1)
    for name, x, gate, down in (("on", big[:, 1, :128], wide[:, 16:144], tall[:, 8:]), ("off", big[:, 1, 3:131], wide[:, 5:133], wd), ("mixed", big[:, 1, 8:136], wide[:, 5:133], tall[:, 8:]),
                                ("one row", big[:1, 1, :128], wide[:, 16:144], tall[:, :96])):
        yield "block " + name, lambda *t: layers.gated_ffn(*t), (x, gate, wu, down)
    yield "norm on", lambda *t: layers.layer_norm(*t), (big[:, 1, :128], randn(128, seed=2, dtype=BF16), randn(128, seed=4, dtype=BF16))
    yield "norm off", lambda *t: layers.layer_norm(*t), (big[:, 1, 3:131], randn(128, seed=2))
    logits = randn(12, 3, 1200, seed=1, dtype=BF16, scale=2.0)
    for cut in (logits[:, 1, 8:1108], logits[:, 1, 3:1104], logits[:, 0, :30]):
        _, teacher, ids = distill_inputs(12, cut.shape[1], 9, BF16, seed=2)
        yield f"distillation {cut.shape[1]}", lambda t, teacher=teacher, ids=ids: layers.distillation_loss(t, teacher, ids, 2.0), (cut,)


def upstream(out):
    return torch.linspace(-1, 1, out.numel(), device="cuda").view(out.shape).to(out.dtype)


def pass_through(function, leaves, hooks):
    """(result, gradients) with the leaves as they lie"""
    leaves = [t.detach().requires_grad_() for t in leaves]
    with hooks():
        out = function(*leaves)
    return out.detach(), torch.autograd.grad(out, leaves, upstream(out))


@gpu
@pytest.mark.parametrize("how", HOOKS)
def test_hooks_that_lay_saved_tensors_out_anew(how):
    """A slice that was offloaded or packed comes back with other distances between its rows, or off its boundaries: the gradients are the same bits, but for
    layer norm, which adds a row up in an order that goes by whether 16 bytes at a time can be read: there they keep to the formulas' bounds."""
    for name, function, leaves in operators_of_strided_tensors():
        want, want_grads = pass_through(function, leaves, contextlib.nullcontext)
        got, grads = pass_through(function, leaves, HOOKS[how])
        assert torch.equal(got, want), (name, how)
        if name.startswith("norm"):
            exact = norm64(leaves[0], leaves[1], leaves[2] if len(leaves) > 2 else None, upstream(got), 1e-5)
            for g, which in zip(grads, ("dx", "dweight", "dbias")):
                near(g, *exact[which], (name, how, which))
        else:
            assert all(torch.equal(a, b) for a, b in zip(grads, want_grads)), (name, how)
    layers.check_status()


@gpu
def test_recomputed_by_checkpoints():
    from torch.utils.checkpoint import checkpoint

    for name, function, leaves in operators_of_strided_tensors():
        want, want_grads = pass_through(function, leaves, contextlib.nullcontext)
        for reentrant in (False, True):
            got, grads = [t.detach().requires_grad_() for t in leaves], None
            out = checkpoint(function, *got, use_reentrant=reentrant)
            out.backward(upstream(out))
            assert torch.equal(out, want) and all(torch.equal(t.grad, b) for t, b in zip(got, want_grads)), (name, reentrant)


def test_operands_of_a_backward_pass_lie_as_they_are():
    """Host side: addresses and distances of what autograd hands back, not those of the forward pass (matrices that lie right are not copied, so no GPU is
    asked)."""
    big = torch.zeros(70, 3, 144, dtype=BF16)
    forward = [big[:, 1, :128], torch.zeros(96, 128, dtype=BF16), torch.zeros(96, 400, dtype=BF16)[:, 16:144], torch.zeros(128, 96, dtype=BF16)]
    operands = layers._Operands(forward)
    assert operands.apart == [432, 128, 400, 96] and operands.room is None
    back = [t.contiguous() for t in forward]
    lies, _ = operands.again(back, None)
    assert lies == [(t.data_ptr(), t.shape[1]) for t in back]
    # those that were copied stay where the copies are
    operands.at, operands.apart, room = [-1, 0, -1, 4096], [432, 128, 400, 104], torch.zeros(1 << 16, dtype=torch.uint8)
    lies, _ = operands.again(back, room)
    assert lies == [(back[0].data_ptr(), 128), (room.data_ptr(), 128), (back[2].data_ptr(), 128), (room.data_ptr() + 4096, 104)]


# ---------------------------------------------------------------------------------------------------------------------
# forward-mode derivatives
# ---------------------------------------------------------------------------------------------------------------------


def calls_of_each_argument(device):
    """(name, function of one tensor, that tensor) for every argument that numbers go into"""
    make = lambda *shape: torch.ones(*shape, device=device)
    x, w, b, h = make(3, 8), make(8), make(8), make(4, 8).bfloat16()
    ids = torch.zeros(3, 2, device=device, dtype=torch.int64)
    yield "x of a norm", lambda t: layers.layer_norm(t, w, b), x
    yield "weight", lambda t: layers.layer_norm(x, t, b), w
    yield "bias", lambda t: layers.layer_norm(x, w, t), b
    for k, name in enumerate(("x", "w_gate", "w_up", "w_down")):
        args = [make(3, 8).bfloat16(), h, h, h.t().contiguous()]
        yield name, lambda t, k=k, args=args: layers.gated_ffn(*args[:k], t, *args[k + 1:]), args[k]
    for function in (layers.distillation_loss, layers.distillation_loss_and_grad):
        yield "logits", lambda t, f=function: f(t, make(3, 2), ids), x
        yield "teacher", lambda t, f=function: f(x, t, ids), make(3, 2)
        yield "weights", lambda t, f=function: f(x, make(3, 2), ids, weights=t), make(3)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=gpu)])
def test_forward_mode_derivatives_are_refused(device):
    """A dual tensor needs no gradient and holds its tangent beside its values, which is all that a kernel sees."""
    for name, function, t in calls_of_each_argument(device):
        with forward.dual_level():
            dual = forward.make_dual(t, torch.ones_like(t))
            for context in (contextlib.nullcontext, torch.no_grad):
                with context(), pytest.raises(NotImplementedError, match="forward-mode"):
                    function(dual)
            if device == "cuda":
                function(t)   # beside a level that it takes no part in
        if device == "cuda":
            function(t)
    if device == "cuda":
        layers.check_status()


# ---------------------------------------------------------------------------------------------------------------------
# distillation far off centre
# ---------------------------------------------------------------------------------------------------------------------


def check_losses(logits, teacher, ids, T, logits_span, teacher_span):
    """Rows' losses and their sum against 64 bits.  Each p_k is off by two roundings of its exponent, at most 1.45 times the span over T, and by those of the
    sums; each term p_k (log p_k - log q_k) by as much of its size, and the sizes add up to the loss and twice what -sum p log p can be (log K < 7)."""
    want, *_ = distill64(logits.double() - logits.double().median(), teacher.double() - teacher.double().amax(1, keepdim=True), ids, T)
    slack = E * (16 * 1.45 * (logits_span + teacher_span) / T + 64 + logits.shape[1] / 32) * (want + 14 * T * T)
    rows = layers.distillation_loss(logits, teacher, ids, T, reduction="none")
    near(rows, want, slack, "rows")
    loss, _ = layers.distillation_loss_and_grad(logits, teacher, ids, T, reduction="sum")
    near(loss, want.sum(), slack.sum() + 16 * E * want.sum(), "sum")


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, FP16])
@pytest.mark.parametrize("vocab", [60, 5001])
@pytest.mark.parametrize("centre", [1e3, -1e4])
def test_distill_of_logits_far_off_centre_whatever_the_first_entry_is(centre, vocab, dtype):
    """As exact as the logits where the first entry is padding, or has no probability."""
    logits, teacher, ids = distill_inputs(9, vocab, 6, F32, seed=31)
    logits, ids = (logits + centre).to(dtype), ids.clone()
    span = float((logits.double() - logits.double().median()).abs().max())
    teacher = teacher - teacher.amax(1, keepdim=True)
    tspan = float(teacher.abs().max())
    check_losses(logits, teacher, ids, 1.0, span, tspan)
    left_out = teacher.clone()
    left_out[:, 0] = -math.inf
    check_losses(logits, left_out, ids, 2.0, span, tspan)
    ids[:, 0] = -1
    check_losses(logits, teacher, ids, 1.0, span, tspan)
    ids[:, 4] = vocab
    check_losses(logits, teacher.flip(1), ids, 0.5, span, tspan)


@gpu
@pytest.mark.parametrize("vocab,top", [(60, 6), (5001, 6), (5001, 300)])
@pytest.mark.parametrize("mask", [-1e4, -1e9, -1e30])
def test_distill_of_a_first_entry_that_the_student_masks(mask, vocab, top):
    """A class that the student leaves out by a large negative number and the teacher gives next to nothing, first among the entries or last: its term
    is a small probability times a large number, and the other terms do not drown in it."""
    logits, teacher, ids = distill_inputs(7, vocab, min(top, vocab), F32, seed=33)
    top = ids.shape[1]
    teacher = teacher - teacher.amax(1, keepdim=True)
    span = float(logits.abs().max())
    for at in (0, top // 2, top - 1):
        x, t = logits.clone(), teacher.clone()
        t[:, at] = -4.0 - math.log(-mask)      # its term is about e^-4
        x.scatter_(1, ids[:, at:at + 1], mask)
        check_losses(x, t, ids, 1.0, span, float(t.abs().max()))


@gpu
@pytest.mark.parametrize("teacher_type", [F32, BF16, FP16])
@pytest.mark.parametrize("vocab,top", [(60, 6), (1000, 200), (5001, 6), (5001, 300)])
@pytest.mark.parametrize("centre", [1e3, -3e4])
def test_distill_of_a_teacher_far_off_centre(centre, vocab, top, teacher_type):
    """The teacher's probabilities are those of its logits' differences: a centre that all of them have in common takes none of their bits."""
    logits, teacher, ids = distill_inputs(9, vocab, min(top, vocab), F32, seed=35)
    span = float(logits.abs().max())
    teacher = (teacher + centre).to(teacher_type)
    d = teacher.double()
    for T in (1.0, 0.75):
        tspan = float((d.amax(1) - d.amin(1)).max())
        check_losses(logits, teacher, ids, T, span, tspan)
        # the gradient's columns of the entries are probabilities themselves
        _, g = layers.distillation_loss_and_grad(logits, teacher, ids, T, reduction="sum")
        _, _, want, _, slack = distill64(logits, d - d.amax(1, keepdim=True), ids, T)
        near(g, want, slack + 8 * E * want.abs(), "gradient")


@gpu
@pytest.mark.parametrize("vocab", [60, 5001])
def test_distill_of_a_teacher_of_extreme_numbers(vocab):
    """Logits whose differences, or multiples, are beyond fp32: the largest alone counts; equal ones share, however large they are."""
    logits, teacher, ids = distill_inputs(4, vocab, 6, F32, seed=37)
    teacher[0] = torch.tensor([3e38, 1.0, 0.0, -1.0, -3e38, -math.inf], device="cuda")
    teacher[1] = 3.4e38
    teacher[2] = torch.finfo(F32).min
    teacher[3] = torch.tensor([2.5, 2.5, 2.0, -1e30, 2.5, -1e30], device="cuda")
    alike = torch.full_like(teacher, -math.inf)
    alike[0, 0], alike[1], alike[2] = 0.0, 0.0, 0.0
    for T in (2.0 ** -60, 1.0):
        alike[3] = torch.where(teacher[3] == 2.5, 0.0, -math.inf if T < 1 else torch.where(teacher[3] == 2.0, -0.5, -math.inf))
        want, _, _, slack, _ = distill64(logits, alike, ids, T)
        near(layers.distillation_loss(logits, teacher, ids, T, reduction="none"), want, slack, "rows")


# ---------------------------------------------------------------------------------------------------------------------
# first calls of several threads
# ---------------------------------------------------------------------------------------------------------------------


def test_first_calls_of_several_threads_share_a_word(monkeypatch):
    """The word that the block's kernels report in is made once: a second one would leave the first to the allocator with a kernel's pointer to it alive."""
    made = []

    def make():
        time.sleep(0.05)
        made.append(torch.zeros(1, dtype=torch.int32))
        return made[-1]

    monkeypatch.setattr(layers, "_reported", None)
    monkeypatch.setattr(layers, "_pinned_word", make)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    begin = threading.Barrier(8)

    def call():
        begin.wait()
        return layers._status_word()

    with concurrent.futures.ThreadPoolExecutor(8) as pool:
        words = [f.result() for f in [pool.submit(call) for _ in range(8)]]
    assert len(made) == 1 and set(words) == {made[0].data_ptr()}


# ---------------------------------------------------------------------------------------------------------------------
# layer norm of large numbers
# ---------------------------------------------------------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("width", [30, 64, 100, 1000, 1024, 5000])
def test_norm_of_rows_far_off_centre(width, dtype):
    """Means so large that they, over a deviation, are beyond fp32: the differences from them are not, and the gradients are the formula's.  A row of one value
    has differences of 0 (equal powers of two add up exactly), so its gradient is r (q - mean q)."""
    x = torch.full((5, width), 1.0, device="cuda")
    x[0], x[1], x[2], x[3, ::2] = 2.0 ** 114, -(2.0 ** 113), 2.0 ** 105, 2.0
    x = x.to(dtype).requires_grad_()
    dy = randn(5, width, seed=41, dtype=dtype)
    w = (1 + 0.2 * randn(width, seed=42, dtype=dtype)).requires_grad_()
    y = layers.layer_norm(x, w, eps=1e-12)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    on = torch.tensor([True, True, True, False, True], device="cuda")
    q = dy.double() * w.detach().double()
    r = 1e-12 ** -0.5
    mean = q.mean(1, keepdim=True)
    assert not bool(y[on].any())
    near(dx[on], (r * (q - mean))[on], (128 * E * r * (q.abs() + q.abs().mean(1, keepdim=True)))[on], "dx")
    want = norm64(x.detach()[3:4], w.detach(), None, dy[3:4], 1e-12)   # the other rows add nothing to it
    near(dx[3:4], *want["dx"], "dx of the row of two values")
    near(dw, want["dweight"][0], want["dweight"][1] + 8 * E * want["dweight"][0].abs(), "dweight")


# ---------------------------------------------------------------------------------------------------------------------
# forms of the block that large sizes take
# ---------------------------------------------------------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("act", sorted(layers.ACTIVATIONS))
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_ffn_on_pairs(dtype, act):
    """Tiles of two SMs in every launch, both types and all activations."""
    x, *rest = ffn_inputs(1300, 328, 2600, 1608, dtype, seed=51)
    check_ffn(x * 2, *rest, act=act)


@gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_ffn_on_pairs_with_results_off_their_boundaries(dtype):
    """Odd widths: no row of a result but the first begins on a 16-byte boundary, and tiles end inside of rows and columns."""
    check_ffn(*ffn_inputs(2100, 1601, 2603, 1603, dtype, seed=52))


@gpu
@pytest.mark.parametrize("rows", [1, 5, 16, 17, 32, 33, 300, 1300])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_ffn_keeps_rows_apart(rows, dtype):
    """A row that is no number spoils itself alone, in the result and in its own gradient; so does a gradient's."""
    x, wg, wu, wd, dy = ffn_inputs(rows, 1001 if rows < 300 else 1000, 1300, 1608, dtype, seed=53)

    def both(x, dy):
        leaf = x.clone().requires_grad_()
        y = layers.gated_ffn(leaf, wg, wu, wd)
        return y.detach(), torch.autograd.grad(y, leaf, dy)[0]

    y, dx = both(x, dy)
    bad = torch.zeros(rows, dtype=torch.bool, device="cuda")
    bad[rows // 2] = True
    x2, dy2 = x.clone(), dy.clone()
    x2[bad, 3], dy2[bad, 7] = math.nan, math.inf
    y2, dx2 = both(x2, dy2)
    assert bool(y2[bad].isnan().all()) and torch.equal(y2[~bad], y[~bad]) and torch.equal(dx2[~bad], dx[~bad])
    assert not bool(dx2[bad].isfinite().any())
    layers.check_status()


@pytest.mark.parametrize("hidden", [1, 16, 1000, 14336])
def test_what_is_kept_for_a_backward_pass_is_what_the_documentation_says(hidden):
    """8 bytes per hidden value, rows counted in 32s beyond 32, 32 bytes per column up to 16 rows; columns are counted in 16s, planes on boundaries of 256."""
    columns = -(-hidden // 16) * 16
    for rows in (1, 2, 15, 16, 17, 31, 32, 33, 64, 1000, 270_003):
        h = columns * 2 * (rows + 16 if rows <= 16 else rows)
        both = columns * 6 * (rows if rows <= 32 else -(-rows // 32) * 32)
        assert 0 <= L.lib.pylo_b200_gated_ffn_kept(rows, hidden, 0) - h < 256
        assert 0 <= L.lib.pylo_b200_gated_ffn_kept(rows, hidden, 1) - h - both < 3 * 256
        assert 0 <= L.lib.pylo_b200_gated_ffn_workspace(rows, hidden) - 2 * h < 512


# ---------------------------------------------------------------------------------------------------------------------
# refusals at the C entries
# ---------------------------------------------------------------------------------------------------------------------


def test_pointers_off_their_elements_are_refused():
    """An address that no element of its type can have gets a negative code on the host, before anything is launched; so does a reduction that there is not."""
    norm = dict(x=16, weight=16, bias=16, y=16, mean=16, rstd=16, rows=4, width=8, x_stride=8, type=L.FP32, weight_type=L.FP32, eps=1e-5)
    for kind, odd in ((dict(), 18), (dict(type=L.BF16, weight_type=L.BF16), 17), (dict(type=L.FP16, weight_type=L.FP16), 17)):
        for name in ("x", "weight", "bias", "y"):
            assert L.lib.pylo_b200_layer_norm(C.byref(L.Norm(**{**norm, **kind, name: odd})), None) == -1, (kind, name)
    for name in ("mean", "rstd"):
        assert L.lib.pylo_b200_layer_norm(C.byref(L.Norm(**{**norm, name: 18})), None) == -1, name
    assert L.lib.pylo_b200_layer_norm(C.byref(L.Norm(**{**norm, "type": L.BF16, "weight": 18})), None) == -1   # fp32 beside bf16
    back = dict(x=16, dy=16, dx=16, weight=16, dweight=16, dbias=16, mean=16, rstd=16, work=16, work_floats=1 << 20, rows=4, width=8, x_stride=8, dy_stride=8,
                type=L.FP32, weight_type=L.FP32)
    for name in ("x", "dy", "dx", "weight", "dweight", "dbias", "mean", "rstd", "work"):
        assert L.lib.pylo_b200_layer_norm_backward(C.byref(L.Norm(**{**back, name: 18})), None) == -1, name
    distill = dict(logits=16, teacher=16, ids=16, weights=16, loss=16, row_loss=16, grad=16, upstream=16, work=16, work_bytes=1 << 20, rows=4, stride=10, vocab=10,
                   top=3, type=L.FP32, teacher_type=L.FP32, ids_bytes=8, reduction=L.REDUCE_MEAN, temperature=1.0, scale=1.0)
    both = L.DISTILL_LOSS | L.DISTILL_GRAD
    for bad in (*({name: 18} for name in ("teacher", "weights", "loss", "row_loss", "grad", "upstream")), dict(ids=20), dict(ids=18, ids_bytes=4), dict(teacher=17, teacher_type=L.BF16),
                dict(reduction=3), dict(reduction=-1)):
        assert L.lib.pylo_b200_distill(C.byref(L.Distill(**{**distill, **bad})), both, None) == -1, bad
    ffn = dict(x=256, w_gate=256, w_up=256, w_down=256, y=256, kept=256, rows=4, ld_x=8, ld_gate=8, ld_up=8, ld_down=16, width=8, hidden=16, out=8, type=L.BF16)
    for bad in (dict(y=257), dict(status=18), dict(host_status=18)):
        assert L.lib.pylo_b200_gated_ffn(C.byref(L.Ffn(**{**ffn, **bad})), None) == -1, bad
    back = {**ffn, "dy": 256, "ld_dy": 8, "work": 256, "dx": 256}
    for bad in (dict(dx=257), dict(dw_gate=257), dict(dw_up=257), dict(dw_down=257), dict(status=18)):
        assert L.lib.pylo_b200_gated_ffn_backward(C.byref(L.Ffn(**{**back, **bad})), None) == -1, bad


# ---------------------------------------------------------------------------------------------------------------------
# shapes and strides at their ends
# ---------------------------------------------------------------------------------------------------------------------


@gpu
def test_no_rows_of_any_stride():
    """No rows, however far they would be apart: results and gradients are empty, the weights' are zero."""
    w = torch.ones(9, device="cuda", requires_grad=True)
    for x in (torch.empty(1, 9, device="cuda").expand(0, 9), torch.empty(9, 4, device="cuda").t()[:0], torch.empty(0, 3, 9, device="cuda"), torch.empty(4, 0, 9, device="cuda")):
        leaf = x.detach().requires_grad_()
        y = layers.layer_norm(leaf, w)
        (dx, dw) = torch.autograd.grad(y, (leaf, w), torch.ones_like(y))
        assert y.shape == x.shape == dx.shape and not bool(dw.any())
        teacher = torch.empty(*x.shape[:-1], 2, device="cuda")
        for reduction in ("mean", "sum", "none"):
            leaf = x.detach().requires_grad_()
            loss = layers.distillation_loss(leaf, teacher, teacher.long(), reduction=reduction)
            (g,) = torch.autograd.grad(loss, leaf, torch.ones_like(loss))
            assert loss.shape == (x.shape[:-1] if reduction == "none" else ()) and g.shape == x.shape and not bool(loss.any())
        loss, g = layers.distillation_loss_and_grad(x, teacher, teacher.long())
        assert float(loss) == 0 and g.shape == x.shape
        h = torch.ones(5, 9, device="cuda", dtype=BF16, requires_grad=True)
        leaf = x.detach().bfloat16().requires_grad_()
        y = layers.gated_ffn(leaf, h, h, h.t())
        (dx, dh) = torch.autograd.grad(y, (leaf, h), torch.ones_like(y))
        assert y.shape == x.shape == dx.shape and not bool(dh.any())


@gpu
def test_one_column_one_row_and_vectors():
    for x in (randn(7, 1, seed=61), randn(1, 7, seed=61).t(), randn(7, 5, seed=61)[:, 2:3], randn(1, 1, seed=62).expand(7, 1)):
        leaf, w, b = x.detach().requires_grad_(), randn(1, seed=63).requires_grad_(), randn(1, seed=64).requires_grad_()
        y = layers.layer_norm(leaf, w, b)
        dx, dw, db = torch.autograd.grad(y, (leaf, w, b), torch.ones_like(y))
        assert torch.equal(y, b.expand(7, 1)) and not bool(dw.any()) and float(db) == 7
        near(dx, *norm64(x, w.detach(), b.detach(), torch.ones_like(x), 1e-5)["dx"], "dx")   # r q - r q, each rounded
        ids = torch.zeros(7, 1, device="cuda", dtype=torch.int64)
        loss, g = layers.distillation_loss_and_grad(x, torch.zeros(7, 1, device="cuda"), ids)
        assert float(loss) == 0 and not bool(g.any())
        check_ffn(x.to(BF16), *[randn(*s, seed=65 + k, dtype=BF16) for k, s in enumerate(((3, 1), (3, 1), (1, 3), (7, 1)))])
    # one row, whose distance to the next means nothing
    wide = randn(1, 40, seed=66)
    row = wide.as_strided((1, 40), (3, 1))
    assert torch.equal(layers.layer_norm(row), layers.layer_norm(wide))
    teacher, ids = torch.zeros(1, 2, device="cuda"), torch.tensor([[3, 8]], device="cuda")
    assert torch.equal(layers.distillation_loss(row, teacher, ids), layers.distillation_loss(wide, teacher, ids))
    w = randn(6, 40, seed=67, dtype=BF16)
    assert torch.equal(layers.gated_ffn(row.bfloat16().as_strided((1, 40), (3, 1)), w, w, w.t()), layers.gated_ffn(wide.bfloat16(), w, w, w.t()))
    # vectors
    assert torch.equal(layers.layer_norm(wide[0]), layers.layer_norm(wide)[0])
    assert torch.equal(layers.gated_ffn(wide[0].bfloat16(), w, w, w.t()), layers.gated_ffn(wide.bfloat16(), w, w, w.t())[0])
    leaf = wide[0].detach().requires_grad_()
    loss = layers.distillation_loss(leaf, teacher[0], ids[0], reduction="none")
    (g,) = torch.autograd.grad(loss, leaf)
    assert loss.shape == () and torch.equal(loss.detach(), layers.distillation_loss(wide, teacher, ids)) and g.shape == (40,)


@gpu
def test_one_tensor_in_several_places():
    """A leaf's gradient is the sum over the places that it has."""
    w = randn(24, seed=71).requires_grad_()
    dy = randn(5, 24, seed=72)
    x = randn(5, 24, seed=73)
    (both,) = torch.autograd.grad(layers.layer_norm(x, w, w), w, dy)
    a, b = (w.detach().clone().requires_grad_() for _ in range(2))
    assert torch.equal(both, sum(torch.autograd.grad(layers.layer_norm(x, a, b), (a, b), dy)))
    m = randn(16, 16, seed=74, dtype=BF16).requires_grad_()
    (both,) = torch.autograd.grad(layers.gated_ffn(m, m, m, m), m, randn(16, 16, seed=75, dtype=BF16))
    parts = [m.detach().clone().requires_grad_() for _ in range(4)]
    grads = torch.autograd.grad(layers.gated_ffn(*parts), parts, randn(16, 16, seed=75, dtype=BF16))
    # three sums of two, each rounded, in whatever order autograd adds them up
    assert bool(((both.double() - sum(g.double() for g in grads)).abs() <= 4 * 2.0 ** -8 * sum(g.double().abs() for g in grads)).all())


@gpu
def test_upstream_gradients_of_any_stride():
    x, wg, wu, wd, dy = ffn_inputs(40, 72, 136, 80, BF16, seed=81)
    leaves = [t.requires_grad_() for t in (x, wg, wu, wd)]
    y = layers.gated_ffn(*leaves)
    z = layers.layer_norm(x.detach().requires_grad_())
    for cut in (lambda t: t.t().contiguous().t(), lambda t: t[:1].expand_as(t), lambda t: t[:, :1].expand_as(t), lambda t: torch.cat([t, t], 1)[:, t.shape[1]:], lambda t: t.as_strided(t.shape, (8, 1))):
        want = torch.autograd.grad(y, leaves, cut(dy).contiguous(), retain_graph=True)
        got = torch.autograd.grad(y, leaves, cut(dy), retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    logits, teacher, ids = distill_inputs(12, 50, 4, F32, seed=82)
    leaf = logits.requires_grad_()
    rows = layers.distillation_loss(leaf, teacher, ids, reduction="none")
    up = randn(12, 3, seed=83)
    for cut in (up[:, 1], up[:1, 0].expand(12), up.double()[:, 2].float()):
        assert torch.equal(*(torch.autograd.grad(rows, leaf, u, retain_graph=True)[0] for u in (cut, cut.contiguous())))


# ---------------------------------------------------------------------------------------------------------------------
# what must not pass in silence
# ---------------------------------------------------------------------------------------------------------------------


@gpu
def test_saved_arguments_that_are_changed_are_noticed():
    """Every argument that a backward pass reads again: changed in place between the passes, it raises."""
    x, wg, wu, wd, dy = ffn_inputs(40, 72, 136, 80, BF16, seed=91)
    logits, teacher, ids = distill_inputs(12, 50, 4, F32, seed=92)
    weights = torch.ones(12, device="cuda")
    calls = {
        "norm": (lambda x, w, b: layers.layer_norm(x, w, b), [randn(5, 24, seed=93), randn(24, seed=94), randn(24, seed=95)], (0, 1)),
        "block": (lambda *t: layers.gated_ffn(*t), [x, wg, wu, wd], (0, 1, 2, 3)),
        "block, copied": (lambda *t: layers.gated_ffn(*t), [t[..., 1:] if k == 0 else t for k, t in enumerate((randn(40, 73, seed=96, dtype=BF16), wg, wu, wd))], (0, 1, 2, 3)),
        "distillation": (lambda t, a, i, w: layers.distillation_loss(t, a, i, weights=w), [logits, teacher, ids, weights], (0, 1, 2, 3)),
    }
    for name, (function, args, saved) in calls.items():
        for k in saved:
            mine = [t.detach().clone() if not name.endswith("copied") else t.detach() for t in args]
            mine = [t.requires_grad_() if t.is_floating_point() and (not name.startswith("dist") or j == 0) else t for j, t in enumerate(mine)]
            views = [t * 1 if t.requires_grad else t for t in mine]   # no leaves, which must not be changed in place
            out = function(*views)
            with torch.no_grad():
                views[k].add_(1)
            with pytest.raises(RuntimeError, match="modified by an inplace"):
                out.sum().backward()


@gpu
def test_transforms_that_the_calls_do_not_know_are_refused():
    """torch.func's transforms and batched gradients raise instead of computing something else."""
    x, w = randn(4, 6, 24, seed=97), randn(24, seed=98)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: layers.layer_norm(t, w))(x)
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda t: layers.layer_norm(t, w).sum())(x[0])
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(lambda t: layers.layer_norm(t, w), (x[0],), (x[1],))
    leaf = x[0].clone().requires_grad_()
    y = layers.layer_norm(leaf, w)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, leaf, x[:2], is_grads_batched=True)
    h = randn(24, 24, seed=99, dtype=BF16)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: layers.gated_ffn(t, h, h, h))(x.bfloat16())
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: layers.distillation_loss(t, t[:, :2], torch.zeros(6, 2, device="cuda", dtype=torch.int64)))(x)

"""Layer norm, the gated feed-forward block and distillation where calls leave the ordinary: values that are no numbers, tensors that come back
from autograd's hooks, forward-mode derivatives, first calls of several threads."""

import math

import pytest
import torch

from pylo_b200 import layers
from test_layers import BF16, F32, FP16, E, distill64, distill_inputs, near

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

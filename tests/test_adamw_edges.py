"""AdamW and clipping where it is easy to go wrong: codes that hang on one rounding, memory that is exchanged under the same tensors,
arguments at the ends of their ranges."""

import math

import numpy as np
import pytest
import torch

from pylo_b200 import _lib as L
from pylo_b200 import optim
from pylo_b200.optim import AdamW_cuda as A
import test_adamw as T
from test_adamw import BETAS, EPS, LR, WD, random_parts

WIDTHS = [optim.AdamW_CUDA, optim.AdamW8bit_CUDA]


# ---------------------------------------------------------------------------------------------------------------------
# the 8-bit step, operation by operation
# ---------------------------------------------------------------------------------------------------------------------
def written_out(m, u, g, betas=BETAS):
    """New moments and roots in fp32, every operation rounded by itself (on the CPU)."""
    b1, b2 = betas
    return b1 * m + (1 - b1) * g, torch.sqrt(b2 * (u * u) + (1 - b2) * (g * g))


def encoded(x, parts, least):
    """Values of the codes, and the scales' bytes, of finite fp32 values: the sum of a float's bits and random ones, cut off."""
    n = x.numel()
    b = torch.zeros(-(-n // 256) * 256)
    b[:n] = x
    b = b.view(-1, 256)
    e = (b.abs().amax(1).view(torch.int32) >> 23).clamp(min=8)
    t = (b.abs().double() * torch.exp2((141 - 127 - e).double())[:, None]).float()   # rounded once, where it is subnormal
    bits = torch.zeros(b.numel(), dtype=torch.int64)
    bits[:n] = (parts * 2 ** 24).long()
    code = ((t.view(torch.int32).long() << 4) + bits.view(-1, 256)) >> 24
    code = torch.maximum(code, (b != 0) * least)
    value = code.to(torch.uint8).view(torch.float8_e4m3fn).float() * torch.where(b < 0, -1.0, 1.0)
    return value.view(-1)[:n], (e - 7).to(torch.uint8)


def one_step_8(m, u, g, t=10, seed=3, **kw):
    """One step of AdamW8bit_CUDA from moments and roots (fp32 on the CPU) that are rounded to codes first: (optimizer's state, parameter,
    the moments and roots that the codes stood for)."""
    p = torch.nn.Parameter(torch.zeros(g.numel(), device="cuda"))
    p.grad = g.to("cuda", torch.float32)
    opt = optim.AdamW8bit_CUDA([p], **{**dict(lr=LR, betas=BETAS, eps=EPS, weight_decay=WD, seed=seed), **kw})
    st = {"step": torch.tensor(t - 1.0, dtype=torch.float64)}
    old = []
    for name, x in (("exp_avg", m), ("exp_avg_sq_root", u)):
        codes, scales = A.to_blocks(x)
        old.append(A.from_blocks(codes, scales))
        st[name], st[name + "_scale"] = codes.cuda(), scales.cuda()
    opt.state[p] = st
    opt.step()
    return opt.state[p], p.detach().cpu(), old


def check_written_out(st, name, want, n, t, seed, first, least):
    value, scale = encoded(want, random_parts(n, seed, t, first), least)
    assert torch.equal(st[name + "_scale"].cpu().view(torch.uint8), scale)
    assert torch.equal(st[name].cpu().float(), value)


@pytest.mark.gpu
def test_moments_that_cancel_have_the_codes_of_the_operations_written_out():
    """b1 m + (1 - b1) g where both are as large: what is left is their roundings, and one rounding more or less is another code or scale."""
    n = 256 * 64 + 77
    gen = torch.Generator().manual_seed(1)
    m0, u0 = torch.randn(n, generator=gen), torch.rand(n, generator=gen)
    m0 = A.from_blocks(*A.to_blocks(m0))
    g = -9 * m0 * (1 + 1e-6 * torch.randn(n, generator=gen))
    st, _, (m, u) = one_step_8(m0, u0, g)
    want, _ = written_out(m, u, g)
    assert want.abs().max() < 1e-4
    check_written_out(st, "exp_avg", want, n, 10, 3, 8, 0)


def near_powers():
    """Gradients whose root of v, from nothing, is within a few last places of a power of two: on its other side is another scale."""
    blocks = []
    for k in range(-40, 12):
        at = (torch.tensor(2.0 ** k, dtype=torch.float64) / (1 - BETAS[1]) ** 0.5).float()
        g = torch.zeros(17, 256)
        g[:, 0] = (at.view(torch.int32) + torch.arange(-8, 9, dtype=torch.int32)).view(torch.float32)
        blocks.append(g.view(-1))
    return torch.cat(blocks)


def many_sizes():
    """Blocks of gradients from 1 down to where squares have few bits or none, wide blocks and narrow ones."""
    gen = torch.Generator().manual_seed(4)
    block = torch.arange(400)
    size = 10.0 ** -(block % 25)[:, None]
    wide = 10.0 ** (-8 * torch.rand(400, 256, generator=gen) * (block % 2)[:, None])
    return (torch.randn(400, 256, generator=gen) * size * wide).view(-1)


@pytest.mark.gpu
@pytest.mark.parametrize("what", [near_powers, many_sizes, lambda: torch.randn(1 << 23, generator=torch.Generator().manual_seed(5))],
                         ids=["near powers of two", "many sizes", "many"])
def test_roots_have_the_codes_of_the_operations_written_out(what):
    g = what()
    u0 = torch.zeros_like(g) if what is near_powers else g.abs() * torch.rand(g.numel(), generator=torch.Generator().manual_seed(6))
    st, p, (m, u) = one_step_8(g / 3, u0, g)
    want_m, want_u = written_out(m, u, g)
    check_written_out(st, "exp_avg", want_m, g.numel(), 10, 3, 8, 0)
    check_written_out(st, "exp_avg_sq_root", want_u, g.numel(), 10, 3, 0, 1)
    assert bool(p.isfinite().all())


@pytest.mark.parametrize("eps", [1e-40, 1.1e-38, 5e-324])
def test_an_eps_that_is_no_normal_number_is_refused_with_8_bits(eps):
    t = T.item(m_scale=256, v_scale=256)
    assert T.step(T.a_call(t, T.a_set(eps=eps), bits=8)) < 0
    assert T.COUNT[0] == 0
    if torch.cuda.is_available():
        with pytest.raises(ValueError, match="eps"):
            optim.AdamW8bit_CUDA([torch.nn.Parameter(torch.zeros(3, device="cuda"))], eps=eps)


@pytest.mark.gpu
@pytest.mark.parametrize("eps", [2.0 ** -126, 1e-30, 1e-20, 1e-15, 1e-8])
def test_an_eps_that_is_smaller_than_roots(eps):
    """Gradients whose squares are no normal numbers, beside ones of 1 and none at all: the update goes by their roots, not by eps alone."""
    g = torch.zeros(5, 256)
    g[0] = torch.linspace(1, 2, 256) * 1e-20
    g[1, :128] = 1.0
    g[1, 128:] = torch.linspace(1, 2, 128) * 1e-21
    g[2, ::3] = -3e-19
    g[3] = torch.logspace(-22, 0, 256)
    g = g.view(-1)
    zero = torch.zeros_like(g)
    st, p, _ = one_step_8(zero, zero, g, t=1, eps=eps, weight_decay=0.0)
    m, u = (x.double() for x in written_out(zero, zero, g))
    want = -LR / (1 - BETAS[0]) * m / (u / (1 - BETAS[1]) ** 0.5 + eps)
    # the factors' roundings: lr / bc1, 1 / root of bc2, product and sum, reciprocal (one place off), quotient, product, result: two half steps each at most
    assert bool(((p.double() - want).abs() <= want.abs() * 16 * 2.0 ** -24 + 2.0 ** -149).all())
    assert bool((p[g == 0] == 0).all())


# ---------------------------------------------------------------------------------------------------------------------
# clipping
# ---------------------------------------------------------------------------------------------------------------------
def test_a_set_without_a_limit_needs_no_norm():
    t = T.item(n=0)   # nothing is launched
    T.COUNT[0] = 0
    assert T.step(T.a_call(t, T.a_set(clip_norm=1.0))) < 0
    for none in (0.0, math.inf, 1e39):
        assert T.step(T.a_call(t, T.a_set(clip_norm=none))) == 0
    T.COUNT[0] = 0


@pytest.mark.gpu
@pytest.mark.parametrize("cls", WIDTHS)
@pytest.mark.parametrize("mixed", [False, True])
@pytest.mark.parametrize("clip_norm", [math.inf, 1e39, 1.7e308])
def test_an_infinite_clipping_norm_clips_nothing(cls, clip_norm, mixed):
    res = []
    for clip in (False, True):
        params = T.params_of([(700,), (30, 40)], torch.float32, 1)
        groups = [dict(params=params[:1], clip_norm=0.1), dict(params=params[1:], clip_grad=clip)] if mixed else params
        opt = cls(groups, clip_grad=clip or mixed, clip_norm=clip_norm)
        for t in range(2):
            T.set_grads(params, torch.float32, 2 + t)
            opt.step()
        res.append(params)
    assert all(torch.equal(x, y) for x, y in zip(*res)) and bool(res[0][0].isfinite().all())


@pytest.mark.gpu
@pytest.mark.parametrize("cls", WIDTHS)
def test_a_clipping_norm_too_small_for_a_float_clips(cls):
    p = torch.nn.Parameter(torch.ones(300, device="cuda"))
    p.grad = torch.ones_like(p)
    opt = cls([p], clip_grad=True, clip_norm=1e-60)
    opt.step()
    assert not opt.state[p]["exp_avg"].float().any()   # 2^-149 / norm is below half of the smallest float


# ---------------------------------------------------------------------------------------------------------------------
# memory that is exchanged under the same tensors
# ---------------------------------------------------------------------------------------------------------------------
def moved(x, how):
    """Other memory with the same values behind a tensor."""
    new = x.detach().clone()
    if how == "data":
        x.data = new
    elif how == "set_":
        x.set_(new)
    else:   # the storage grows, and moves
        x.untyped_storage().resize_(x.untyped_storage().nbytes() + (1 << 20))


def a_plan(bits):
    """The host's table over parameters in the host's memory: nothing can be launched with it, but everything looked at."""
    params = [torch.nn.Parameter(torch.ones(6, 6)), torch.nn.Parameter(torch.ones(40))]
    for p in params:
        p.grad = torch.ones_like(p)
    state = {}
    for p in params:
        n = -(-p.numel() // 256)
        st = {"step": torch.tensor(3.0, dtype=torch.float64)}
        if bits == 32:
            st.update(exp_avg=torch.zeros(p.shape), exp_avg_sq=torch.zeros(p.shape))
        else:
            for name in ("exp_avg", "exp_avg_sq_root"):
                st[name] = torch.zeros(p.shape, dtype=torch.uint8).view(torch.float8_e4m3fn)
                st[name + "_scale"] = torch.ones(n, dtype=torch.uint8).view(torch.float8_e8m0fnu)
        state[p] = st
    flags = [(False, False)]
    plan = A._Plan(params, [0, 0], flags, state, bits)
    assert plan.good_for(params, [0, 0], flags, state)
    return plan, params, flags, state


@pytest.mark.parametrize("how", ["data", "set_", "storage"])
@pytest.mark.parametrize("bits", [32, 8])
def test_a_state_whose_memory_was_exchanged_is_noticed(bits, how):
    for name in list(a_plan(bits)[3].values())[0]:
        for k in (0, 1):
            plan, params, flags, state = a_plan(bits)
            moved(state[params[k]][name], how)
            assert not plan.good_for(params, [0, 0], flags, state), name
    plan, params, flags, state = a_plan(bits)
    state[params[0]]["step"].share_memory_()
    assert not plan.good_for(params, [0, 0], flags, state)


@pytest.mark.parametrize("bits", [32, 8])
def test_strides_that_were_exchanged_are_noticed(bits):
    plan, params, flags, state = a_plan(bits)
    params[0].data = params[0].data.t()
    assert not plan.good_for(params, [0, 0], flags, state)
    for name in ("exp_avg", "exp_avg_sq" if bits == 32 else "exp_avg_sq_root"):
        plan, params, flags, state = a_plan(bits)
        state[params[0]][name].data = state[params[0]][name].data.t()
        assert not plan.good_for(params, [0, 0], flags, state)


def test_gradients_of_another_device_or_size_are_refused():
    plan, params, *_ = a_plan(32)
    look = lambda: plan.look_at([p.grad for p in params], "name")
    look()
    params[0].grad.data = torch.ones(3)
    with pytest.raises(RuntimeError, match="gradient has shape"):
        look()
    params[0].grad.data = torch.ones(6, 6)
    look()
    plan.at = 0   # as if the parameters were on a GPU
    params[1].grad.data = torch.ones(40)
    with pytest.raises(RuntimeError, match="must live on"):
        look()


@pytest.mark.gpu
@pytest.mark.parametrize("cls", WIDTHS)
@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("how", ["data", "set_", "storage"])
def test_a_step_goes_by_the_memory_that_states_have_now(cls, capturable, how):
    shapes = [(40, 40), (300,)]
    a, b = T.params_of(shapes, torch.bfloat16, 1), T.params_of(shapes, torch.bfloat16, 1)
    x, y = (cls(ps, master_weights=True, capturable=capturable) for ps in (a, b))

    def both(t):
        T.set_grads(a, torch.bfloat16, t)
        for p, q in zip(a, b):
            q.grad = p.grad.clone()
        x.step()
        y.step()
        assert all(torch.equal(p, q) for p, q in zip(a, b)), t

    both(0)
    for k, name in enumerate(list(x.state[a[0]])):
        kept = [x.state[p][name].detach().clone() for p in a]
        if how == "storage" and name == "step" and not capturable:
            x.state[a[0]][name].share_memory_()
        else:
            for p in a:
                moved(x.state[p][name], how)
        gone = [torch.full((64, 64), 255, dtype=torch.uint8, device="cuda") for _ in range(64)]   # over what was given back
        both(1 + k)
        if not name.endswith("scale"):   # the new memory is updated
            assert not any(torch.equal(x.state[p][name].float(), z.float()) for p, z in zip(a, kept)), name
        del gone
    # values that come with the other memory count
    x.state[a[0]]["exp_avg"].data = torch.zeros_like(x.state[a[0]]["exp_avg"])
    y.state[b[0]]["exp_avg"] = torch.zeros_like(y.state[b[0]]["exp_avg"])
    both(20)
    # moments that were moved to the host come back
    x.state[a[0]]["exp_avg"].data = x.state[a[0]]["exp_avg"].data.cpu()
    both(21)
    assert x.state[a[0]]["exp_avg"].is_cuda


@pytest.mark.gpu
@pytest.mark.parametrize("cls", WIDTHS)
def test_a_parameter_whose_strides_were_exchanged_is_refused(cls):
    p = torch.nn.Parameter(torch.randn(8, 8, device="cuda"))
    opt = cls([p])
    p.grad = torch.ones_like(p)
    opt.step()
    p.data = p.data.t()
    with pytest.raises(RuntimeError, match="contiguous"):
        opt.step()


@pytest.mark.gpu
@pytest.mark.parametrize("cls", WIDTHS)
def test_a_gradient_that_was_moved_to_the_host_is_refused(cls):
    p, q = T.params_of([(30,), (7,)], torch.float32, 1)
    opt = cls([p, q])
    T.set_grads([p, q], torch.float32, 2)
    opt.step()
    q.grad.data = q.grad.data.cpu()
    with pytest.raises(RuntimeError, match="must live on"):
        opt.step()
    q.grad.data = torch.ones(3, device="cuda")
    with pytest.raises(RuntimeError, match="gradient has shape"):
        opt.step()
    q.grad.data = torch.ones(7, device="cuda")
    opt.step()
    assert float(opt.state[q]["step"]) == 2


# ---------------------------------------------------------------------------------------------------------------------
# states of 32 bits that become ones of 8
# ---------------------------------------------------------------------------------------------------------------------
def test_roots_that_are_not_zero_get_a_code():
    x = torch.logspace(-30, 0, 700)
    x[::7] = 0
    x[5], x[6] = math.nan, math.inf
    codes, scales = A.to_blocks(x, least=1)
    assert torch.equal(codes.float() == 0, x == 0) and bool(codes.float()[5:7].isnan().all())
    nearest = A.to_blocks(x)
    assert torch.equal(scales.view(torch.uint8), nearest[1].view(torch.uint8))
    other = nearest[0].float() != 0
    assert torch.equal(codes.view(torch.uint8)[other], nearest[0].view(torch.uint8)[other])


@pytest.mark.gpu
@pytest.mark.parametrize("g", [0.0, 1e-6])
def test_the_first_step_from_converted_states_is_no_jump(g):
    """One old gradient of 1 among many of 1e-6: the small roots' codes are what keeps their moments from being divided by eps alone."""
    a, b = (torch.nn.Parameter(torch.zeros(512, device="cuda")) for _ in range(2))
    x, y = optim.AdamW_CUDA([a], lr=1.0, weight_decay=0.0), optim.AdamW8bit_CUDA([b], lr=1.0, weight_decay=0.0)
    v = torch.full((512,), 1e-12, device="cuda")
    v[::256] = 1.0
    x.state[a] = {"step": torch.tensor(1000.0, dtype=torch.float64), "exp_avg": torch.full((512,), 1e-6, device="cuda"), "exp_avg_sq": v}
    y.load_state_dict(x.state_dict())
    for p, opt in ((a, x), (b, y)):
        p.grad = torch.full((512,), g, device="cuda")
        opt.step()
    # the moment's nearest code is 2^-4 of it away at most, a root's too where it has one of its own
    assert bool((b.abs() <= a.abs() * (1 + 2.0 ** -4) / (1 - 2.0 ** -4) * (1 + 1e-5)).all())


# ---------------------------------------------------------------------------------------------------------------------
# a learning rate on the device that is replaced by a number
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("cls", WIDTHS)
def test_a_number_in_the_place_of_a_learning_rate_on_the_device(cls):
    """The tensor has no say any more, also where the number is what it said, and the step can be captured."""
    p = torch.nn.Parameter(torch.zeros(100, device="cuda"))
    p.grad = torch.ones_like(p)
    lr = torch.tensor(0.25, device="cuda")
    opt = cls([p], lr=lr, weight_decay=0.0, capturable=True)
    opt.step()
    opt.param_groups[0]["lr"] = 0.25
    opt.step()
    lr.fill_(100.0)
    before = p.detach().clone()
    opt.step()
    assert bool(((p - before).abs() < 1).all())
    opt.param_groups[0]["lr"] = lr
    opt.step()
    opt.param_groups[0]["lr"] = 0.5
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    before = p.detach().clone()
    graph.replay()
    assert bool(((p - before).abs() < 1).all())


@pytest.mark.gpu
@pytest.mark.parametrize("cls", WIDTHS)
def test_a_clipped_steps_workspace_is_its_streams_own(cls):
    """A buffer of another stream's memory would be given back to that stream while this one still reads it."""
    p = T.params_of([(500, 300)], torch.float32, 1)[0]
    T.set_grads([p], torch.float32, 2)
    opt = cls([p], clip_grad=True, clip_norm=0.1)
    opt.step()
    one = opt._plan.norm
    opt.step()
    assert opt._plan.norm is one
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.step()
        assert opt._plan.norm.data_ptr() != one.data_ptr() and opt._plan.call.norm == opt._plan.norm.data_ptr()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    opt = cls([p], clip_grad=True, clip_norm=0.1, capturable=True)
    opt.step()
    with torch.cuda.graph(graph):
        opt.step()
    opt.step()
    assert opt._plan.norm is not None


def test_a_place_for_the_norm_is_needed():
    g, n, t = np.array([512], dtype=np.uint64), np.array([8]), np.array([L.FP32], dtype=np.int32)
    call = lambda root, norm, floats: L.lib.pylo_b200_clip_grads_to(g.ctypes.data, n.ctypes.data, t.ctypes.data, 1, 1.0, root, norm, floats, 0, None)
    assert call(None, 256, 100) == -1 and call(256, None, 100) == -1 and call(256, 512, 2) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("max_norm", [0.1, math.inf])
@pytest.mark.parametrize("shapes", [[(30,)], [(700, 900), (5,)], [(3000, 3000)]])   # few partial sums, and more than a launch adds up itself
def test_the_norm_that_is_returned_keeps_nothing_else(shapes, max_norm):
    grads = T.tensors(shapes, torch.float32, 1)
    before = [g.clone() for g in grads]
    norm = optim.clip_grad_norm_(T.with_grads(grads), max_norm)
    assert norm.untyped_storage().nbytes() == 4
    T.check_clip(grads, before, norm, max_norm)
    again = optim.clip_grad_norm_(T.with_grads(before), max_norm, error_if_nonfinite=True)
    assert again.untyped_storage().nbytes() == 4 and torch.equal(again, norm)


@pytest.mark.gpu
def test_both_forms_of_the_native_call_say_the_same():
    g = T.tensors([(5000,)], torch.float32, 1)[0]
    ptrs, n, t = np.array([g.data_ptr()], dtype=np.uint64), np.array([5000]), np.array([L.FP32], dtype=np.int32)
    for limit in (math.inf, 1e9):   # neither writes to the gradient
        norm, root, other = torch.zeros(100, device="cuda"), torch.zeros(1, device="cuda"), torch.zeros(100, device="cuda")
        L.check(L.lib.pylo_b200_clip_grads(ptrs.ctypes.data, n.ctypes.data, t.ctypes.data, 1, limit, norm.data_ptr(), 100, 0, None), "clip_grads")
        L.check(L.lib.pylo_b200_clip_grads_to(ptrs.ctypes.data, n.ctypes.data, t.ctypes.data, 1, limit, root.data_ptr(), other.data_ptr(), 100, 0, None), "clip_grads_to")
        torch.cuda.synchronize()
        assert torch.equal(norm[:2], other[:2]) and torch.equal(root, norm[1:2]) and float(root) > 0


@pytest.mark.gpu
def test_a_strided_gradient_that_is_given_twice_counts_once():
    base = torch.randn(20, 30, device="cuda")
    z, y = base[:, ::2], torch.randn(7, device="cuda")
    params = T.with_grads([z, y])
    before, hidden = [z.clone(), y.clone()], base[:, 1::2].clone()
    other = torch.nn.Parameter(torch.zeros(20, 15, device="cuda"))   # another parameter with the same gradient
    other.grad = base[:, ::2]
    norm = optim.clip_grad_norm_(params + params[:1] + [other], 0.3)
    T.check_clip([z, y], before, norm, 0.3)
    assert torch.equal(base[:, 1::2], hidden)


@pytest.mark.gpu
def test_an_expanded_gradient_is_refused_before_anything_is_scaled():
    grads = [torch.ones(7, device="cuda"), torch.randn(1, 4, device="cuda").expand(5, 4)]
    with pytest.raises(RuntimeError, match="share memory"):
        optim.clip_grad_norm_(T.with_grads(grads), 0.1)
    assert bool((grads[0] == 1).all())
    T.check_clip(grads, [g.clone() for g in grads], optim.clip_grad_norm_(T.with_grads(grads), math.inf), math.inf)   # its norm alone


# ---------------------------------------------------------------------------------------------------------------------
# what a state may hold, and sharded steps
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("cls", WIDTHS)
def test_a_state_may_hold_other_things(cls):
    a, b = T.params_of([(30, 20)], torch.float32, 1), T.params_of([(30, 20)], torch.float32, 1)
    x, y = cls(a), cls(b)
    for t in range(3):
        T.set_grads(a + b, torch.float32, 2 + t)
        b[0].grad = a[0].grad.clone()
        x.step()
        y.step()
        x.state[a[0]]["note"] = t
        x.state[a[0]]["mask"] = torch.ones(3, 4).t().to_sparse()
        new = cls(a)
        new.load_state_dict(x.state_dict())
        assert new.state[a[0]]["note"] == t
        x = new
    x.step()
    y.step()
    assert torch.equal(a[0], b[0])


@pytest.mark.gpu
@pytest.mark.parametrize("cls", WIDTHS)
@pytest.mark.parametrize("kind", ["staged", "fused"])
def test_through_the_steps_that_overlap_their_exchange(cls, kind):
    """One rank of one: hooks and layout, no exchange."""
    from pylo_b200.zero import FusedShardedStep, StagedShardedStep

    shapes = [(72, 48), (48,), (30, 200), (7,)]
    shard = StagedShardedStep(shapes, "cuda", blocks=2) if kind == "staged" else FusedShardedStep(shapes, "cuda", push="copies")
    other = [torch.nn.Parameter(p.detach().clone()) for p in shard.params]
    x = cls(shard.param_groups() if kind == "staged" else shard.param_groups(groups=2), clip_grad=True, clip_norm=0.5)
    x.after_group = shard.after_group
    x._sharded = True
    y = cls(other, clip_grad=True, clip_norm=0.5)
    for t in range(3):
        T.set_grads(shard.params, torch.float32, t)
        for p, q in zip(shard.params, other):
            q.grad = p.grad.clone()
        x.step()
        shard.finish()
        y.step()
    assert all(torch.equal(p, q) for p, q in zip(shard.params, other))

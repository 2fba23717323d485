"""AdamW with states of 32 and 8 bits, and clipping by the global norm, against plain evaluations in 64 bits.

Tolerances count roundings: half a step of a type is 2^-24 (fp32), 2^-11 (fp16) or 2^-8 (bf16) of a value."""

import ctypes as C
import math

import numpy as np
import pytest
import torch

from pylo_b200 import _lib as L
from pylo_b200 import optim
from pylo_b200.optim import AdamW_cuda as A

H32 = 2.0 ** -24
HALF = {torch.float32: H32, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}   # half of the smallest step (or all of it)
ROOTS = [(math.isqrt(q << 64) & 0xFFFFFFFF) | 1 for q in (2, 3, 5, 7, 11, 13, 17, 19, 23, 29, 31, 37, 41, 43, 47, 53)]
LR, BETAS, EPS, WD = 1e-2, (0.9, 0.95), 1e-8, 0.1
SIZES = [(1,), (), (7,), (256,), (257,), (3, 341), (64, 128), (40_003,)]


# ---------------------------------------------------------------------------------------------------------------------
# the formulas in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact_step(p, g, m, v, t, lr=LR, betas=BETAS, eps=EPS, wd=WD):
    """(p, m, v, size of the update) after one step, all in 64 bits."""
    b1, b2 = betas
    p, g, m, v = (x.double() for x in (p, g, m, v))
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    upd = lr / (1 - b1 ** t) * m / (v.sqrt() / math.sqrt(1 - b2 ** t) + eps)
    return p * (1 - lr * wd) - upd, m, v, upd.abs()


def close(got, want, bound):
    bad = (got.double() - want).abs() > bound
    assert not bad.any(), ((got.double() - want).abs() / bound).max().item()


def check_32(p, m, v, old, g, t, gs=1.0, gs_err=0.0, **kw):
    """One step's results against the formulas, from the old (p, m, v) and the gradient."""
    g = g.double() * gs
    b1, b2 = kw.get("betas", BETAS)
    pe, me, ve, upd = exact_step(old[0], g, old[1], old[2], t, **kw)
    # a product, a sum; constants and the gradient's scale rounded once each
    bm = (b1 * old[1].double().abs() + (1 - b1) * g.abs()) * (4 * H32 + gs_err) + 2.0 ** -149
    close(m, me, bm)
    close(v, ve, ve * (5 * H32 + 2 * gs_err) + 2.0 ** -148)
    # the update's factors: lr / bc1, m, root, 1 / root of bc2, sum, quotient, product: two half steps each at most, and m's own error
    scale = upd / me.abs().clamp(min=1e-300)
    bp = upd * (16 * H32 + 2 * gs_err) + scale * bm + old[0].double().abs() * 3 * H32
    if p.dtype is torch.float32:
        close(p, pe, bp)
    else:
        close(p, pe, bp + (pe.abs() + bp) * HALF[p.dtype] + TINY[p.dtype])
    return pe, bp


def hashed(x):
    x = x ^ (x >> 16)
    x = (x * ROOTS[0]) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * ROOTS[1]) & 0xFFFFFFFF
    return x ^ (x >> 16)


def random_parts(n, seed, step, first):
    """What is added to the parts of a code step that are cut off: 24 bits each, as a part of 1."""
    i = torch.arange(n)
    base = hashed(((i >> 3) * ROOTS[2] + hashed((seed * ROOTS[3] + step) & 0xFFFFFFFF)) & 0xFFFFFFFF)
    return ((base * torch.tensor(ROOTS[first:first + 8])[i & 7] & 0xFFFFFFFF) >> 8).double() / 2 ** 24


def check_codes(codes, scales, exact, err, parts, least):
    """Codes and scales of one state against its values in 64 bits (off by `err` at most), on the CPU."""
    n = exact.numel()
    nb = -(-n // 256)
    x = torch.zeros(nb * 256, dtype=torch.float64)
    x[:n] = exact.reshape(-1)
    e = torch.zeros_like(x)
    e[:n] = err.reshape(-1)
    x, e = x.view(nb, 256), e.view(nb, 256)
    most = x.abs().amax(1)
    lo, hi = ((most + s * e.amax(1)).clamp(min=1e-300) for s in (-1, 1))
    scale = scales.double()
    bounds = [torch.exp2(torch.floor(torch.log2(b)).clamp(min=8 - 127) - 7) for b in (lo, hi)]
    assert bool(((scale == bounds[0]) | (scale == bounds[1])).all())
    got = torch.zeros(nb * 256, dtype=torch.float64)
    got[:n] = codes.reshape(-1).double()
    y = x.abs() / scale[:, None]
    step = torch.exp2(torch.floor(torch.log2(y.clamp(min=2.0 ** -6))) - 3)   # e4m3: three bits behind the leading one, from 2^-6 on
    u = torch.zeros(nb * 256, dtype=torch.float64)
    u[:n] = parts
    at = y / step + u.view(nb, 256)
    want = torch.floor(at) * step
    if least:
        want = torch.maximum(want, (x > 0) * 2.0 ** -9)
    got = got.view(nb, 256)
    # a value that is no larger than its error may be of either sign: b1 m + (1 - b1) g cancels to what the roundings of its terms leave
    assert bool((torch.signbit(got) == (x < 0))[(got != 0) & (x.abs() > e)].all())
    far = (got.abs() - want).abs()
    slack = e / scale[:, None] / step + 2.0 ** -24 + at * 2 ** -24   # the bits behind the 24, the value's own error
    near = ((at - torch.round(at)).abs() <= slack * 2) & (far <= 1.01 * step)   # a border between two codes is that near
    assert bool(((far == 0) | near).all()), (far > 0).sum()


# ---------------------------------------------------------------------------------------------------------------------
# without a GPU
# ---------------------------------------------------------------------------------------------------------------------
COUNT = np.zeros(1)


def item(**kw):
    t = np.zeros(1, dtype=L.ADAMW_DTYPE)
    for name, value in {**dict(p=256, g=256, m=256, v=256, n=4, step=COUNT.ctypes.data), **kw}.items():
        t[name] = value
    return t


def a_call(t, s, **kw):
    return L.AdamwCall(**{**dict(items=t.ctypes.data, n_items=len(t), sets=C.pointer(s), n_sets=1, bits=32), **kw})


def a_set(**kw):
    s = L.AdamwSet(lr=1e-3, weight_decay=0.0, beta1=0.9, beta2=0.99, eps=1e-8)
    for name, value in kw.items():
        setattr(s, name, value)
    return s


def step(call, phases=L.ADAMW_STEP):
    return L.lib.pylo_b200_adamw_step(C.byref(call), phases, None)


@pytest.mark.parametrize("bad", [dict(n=-1), dict(n=2 ** 34 + 1), dict(set=1), dict(set=-1), dict(p_type=3), dict(g_type=-1), dict(p=0), dict(g=0), dict(m=0),
                                 dict(v=0), dict(p_type=L.BF16, g_type=L.FP16), dict(p_type=L.FP16, g_type=L.BF16), dict(master=256), dict(step=0), dict(m=264), dict(v=260),
                                 dict(p_type=L.BF16, g_type=L.BF16, master=264)])
def test_items_are_checked_before_a_launch(bad):
    t, s = item(**bad), a_set()
    assert step(a_call(t, s)) < 0 and COUNT[0] == 0


@pytest.mark.parametrize("bad", [dict(beta1=1.0), dict(beta1=-0.1), dict(beta2=1.0), dict(eps=-1.0), dict(clip_norm=-1.0), dict(beta1=math.nan), dict(clip_norm=1.0)])
def test_sets_are_checked_before_a_launch(bad):
    t, s = item(), a_set(**bad)   # the last: no place for the norm
    assert step(a_call(t, s)) < 0 and COUNT[0] == 0


def test_calls_are_checked_before_a_launch():
    t, s, none = item(), a_set(), item(n=0, p=0)
    assert L.lib.pylo_b200_adamw_step(None, L.ADAMW_STEP, None) < 0 and step(a_call(t, s), 4) < 0
    for bad in (dict(items=None), dict(n_items=-1), dict(n_sets=-1), dict(n_sets=0), dict(sets=None), dict(bits=16), dict(bits=8)):   # the last: no scales
        assert step(a_call(t, s, **bad)) < 0, bad
    assert step(a_call(t, s), L.ADAMW_NORM) < 0 and step(a_call(t, s, norm=256, norm_floats=2), L.ADAMW_NORM) < 0   # no place for the norm
    assert step(a_call(item(m_scale=256, v_scale=256), a_set(eps=0.0), bits=8)) < 0   # a root of zero is possible
    assert step(a_call(t, s, n_items=0)) == 0 and COUNT[0] == 0
    assert step(a_call(none, s)) == 0 and COUNT[0] == 1   # a tensor without elements takes its step too
    COUNT[0] = 0


def test_gradients_are_checked_before_a_launch():
    g, n, t = np.array([512, 1024], dtype=np.uint64), np.array([128, 5]), np.array([L.FP32, L.BF16], dtype=np.int32)
    call = lambda g=g, n=n, t=t, count=2, limit=1.0, norm=256, floats=100, distinct=0: L.lib.pylo_b200_clip_grads(
        g.ctypes.data if g is not None else None, n.ctypes.data if n is not None else None, t.ctypes.data if t is not None else None, count, limit, norm, floats,
        distinct, None)
    for bad in (dict(g=None), dict(n=None), dict(t=None), dict(count=-1), dict(limit=-1.0), dict(limit=math.nan), dict(norm=None), dict(floats=3), dict(n=np.array([128, -1])),
                dict(t=np.array([0, 3], dtype=np.int32)), dict(t=np.array([-1, 0], dtype=np.int32)), dict(g=np.array([512, 0], dtype=np.uint64))):
        assert call(**bad) == -1, bad
    assert call(n=np.array([129, 5])) == L.ERR_GRADS_OVERLAP and call(g=np.array([1024, 512], dtype=np.uint64), n=np.array([5, 300])) == L.ERR_GRADS_OVERLAP
    many = 1025
    apart = (np.arange(many, 0, -1) * 4096).astype(np.uint64)   # no two share memory, but there are too many to find out
    assert call(g=apart, n=np.ones(many, dtype=np.int64), t=np.zeros(many, dtype=np.int32), count=many) == L.ERR_GRADS_OVERLAP
    assert call(g=apart, n=np.ones(many, dtype=np.int64), t=np.zeros(many, dtype=np.int32), count=many, floats=0) in (-1, L.ERR_GRADS_OVERLAP)


def test_there_is_no_path_without_a_gpu():
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    p = torch.nn.Parameter(torch.zeros(3))
    for cls in (optim.AdamW_CUDA, optim.AdamW8bit_CUDA):
        with pytest.raises(RuntimeError, match="CUDA"):
            cls([p])
    p.grad = torch.ones(3)
    with pytest.raises(RuntimeError, match="CUDA"):
        optim.clip_grad_norm_([p], 1.0)


def test_clipping_refuses_what_it_does_not_do():
    p = torch.nn.Parameter(torch.zeros(3))
    with pytest.raises(ValueError, match="2-norm"):
        optim.clip_grad_norm_([p], 1.0, norm_type=math.inf)
    for bad in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            optim.clip_grad_norm_([p], bad)
    assert float(optim.clip_grad_norm_([p], 1.0)) == 0.0   # no gradients: as torch.nn.utils has it


def test_gradients_that_overlap():
    ptrs, types = [1024, 512, 1024], [L.FP32] * 3
    assert A._distinct(ptrs, [64, 128, 64], types) == ([1024, 512], [64, 128], [L.FP32] * 2)
    assert A._distinct([1024, 512, 0], [64, 128, 0], types)[0] == [1024, 512]
    for sizes in ([64, 129, 64], [64, 128, 65]):
        with pytest.raises(ValueError, match="memory"):
            A._distinct(ptrs, sizes, types)
    with pytest.raises(ValueError, match="memory"):
        A._distinct(ptrs, [64, 128, 128], [L.FP32, L.FP32, L.BF16])


@pytest.mark.parametrize("n", [0, 1, 255, 256, 1000])
def test_blocks_and_back(n):
    x = torch.randn(n, generator=torch.Generator().manual_seed(n)) * 10.0 ** torch.randint(-6, 4, (n,), generator=torch.Generator().manual_seed(1))
    codes, scales = A.to_blocks(x)
    assert codes.shape == x.shape and len(scales) == -(-n // 256)
    back = A.from_blocks(codes, scales).double()
    each = scales.double().repeat_interleave(256)[:n]
    # half a step of e4m3 (2^-4 of the value), or of its subnormal numbers
    assert bool(((back - x.double()).abs() <= x.double().abs() * 2.0 ** -4 + each * 2.0 ** -10).all())
    if n:
        most = codes.double().abs()[: min(n, 256)].max()
        assert 128 <= most <= 256


def test_blocks_with_values_that_are_none():
    x = torch.linspace(1, 2, 300)
    x[3], x[5], x[299] = math.nan, -math.inf, math.inf
    back = A.from_blocks(*A.to_blocks(x))
    bad = torch.tensor([3, 5, 299])
    assert bool(back[bad].isnan().all())
    rest = torch.ones(300, dtype=torch.bool)
    rest[bad] = False
    assert bool(((back - x).abs()[rest] <= x[rest] * 2.0 ** -4).all())
    assert bool((A.from_blocks(*A.to_blocks(torch.zeros(10))) == 0).all())


# ---------------------------------------------------------------------------------------------------------------------
# on the GPU
# ---------------------------------------------------------------------------------------------------------------------
def tensors(shapes, dtype, seed, scale=1.0, odd=False):
    """Random tensors of the shapes; `odd`: views that begin one element behind a boundary."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for s in shapes:
        n = math.prod(s)
        x = (torch.randn(n + odd, device="cuda", generator=gen) * scale * 10.0 ** (torch.rand(n + odd, device="cuda", generator=gen) * 3 - 2)).to(dtype)
        out.append(x[int(odd):].view(s))
    return out


def params_of(shapes, dtype, seed, odd=False):
    return [torch.nn.Parameter(x) for x in tensors(shapes, dtype, seed, 1.0, odd)]


def set_grads(params, dtype, seed, scale=1.0, odd=False):
    for p, g in zip(params, tensors([tuple(p.shape) for p in params], dtype, seed, scale, odd)):
        p.grad_dtype = dtype
        p.grad = g


TYPES = [(torch.float32, torch.float32, False), (torch.float32, torch.bfloat16, False), (torch.float32, torch.float16, False),
         (torch.bfloat16, torch.bfloat16, False), (torch.bfloat16, torch.float32, True), (torch.bfloat16, torch.bfloat16, True), (torch.bfloat16, torch.float32, False),
         (torch.float16, torch.float16, True), (torch.float16, torch.float32, False), (torch.float16, torch.float16, False), (torch.float16, torch.float32, True),
         (torch.bfloat16, torch.float16, True)]   # the last: gradients that are copied


@pytest.mark.gpu
@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("pt,gt,master", TYPES)
def test_steps_with_states_of_32_bits(pt, gt, master, odd):
    params = params_of(SIZES, pt, 1, odd)
    opt = optim.AdamW_CUDA(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=WD, master_weights=master)
    for t in (1, 2, 3):
        set_grads(params, gt, 10 + t, odd=odd)
        grads = [p.grad.clone() for p in params]
        old = []
        for p in params:
            st = opt.state[p]
            z = torch.zeros(p.shape, device="cuda")
            old.append([st["master"].clone() if "master" in st else p.detach().clone(), st["exp_avg"].clone() if st else z, st["exp_avg_sq"].clone() if st else z])
        opt.step()
        for p, g, o in zip(params, grads, old):
            st = opt.state[p]
            assert torch.equal(p.grad, g) and ("master" in st) == master and float(st["step"]) == t
            pe, bp = check_32(p.detach(), st["exp_avg"], st["exp_avg_sq"], o, g, t)
            if master:
                close(st["master"], pe, bp)
                assert torch.equal(p.detach(), st["master"].to(pt))


def check_8(opt, params, old, grads, t, seed, gs=1.0, gs_err=0.0, maximize=False):
    for p, (op, om, ou), g in zip(params, old, grads):
        st = opt.state[p]
        g = g.double() * gs * (-1 if maximize else 1)
        pe, me, ve, upd = exact_step(op, g, om, ou.square(), t)
        b1, b2 = BETAS
        bm = (b1 * om.abs() + (1 - b1) * g.abs()) * (4 * H32 + gs_err)
        ue = ve.sqrt()
        bu = ue * (5 * H32 + gs_err)
        scale = upd / me.abs().clamp(min=1e-300)
        bp = upd * (16 * H32 + 2 * gs_err) + scale * bm + op.double().abs() * 3 * H32
        close(st.get("master", p.detach()) if p.dtype is not torch.float32 and "master" in st else p.detach(), pe,
              bp if "master" in st or p.dtype is torch.float32 else bp + (pe.abs() + bp) * HALF[p.dtype] + TINY[p.dtype])
        if "master" in st:
            assert torch.equal(p.detach(), st["master"].to(p.dtype))
        n = p.numel()
        check_codes(st["exp_avg"].cpu(), st["exp_avg_scale"].cpu(), me.cpu(), bm.cpu(), random_parts(n, seed, t, 8), 0)
        check_codes(st["exp_avg_sq_root"].cpu(), st["exp_avg_sq_root_scale"].cpu(), ue.cpu(), bu.cpu(), random_parts(n, seed, t, 0), 1)


def old_8(opt, params):
    out = []
    for p in params:
        st = opt.state[p]
        z = torch.zeros(p.shape, device="cuda", dtype=torch.float64)
        out.append((st["master"].clone() if "master" in st else p.detach().clone(),
                    A.from_blocks(st["exp_avg"], st["exp_avg_scale"]).double() if st else z,
                    A.from_blocks(st["exp_avg_sq_root"], st["exp_avg_sq_root_scale"]).double() if st else z))
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("pt,gt,master", TYPES)
def test_steps_with_states_of_8_bits(pt, gt, master, odd):
    params = params_of(SIZES, pt, 1, odd)
    opt = optim.AdamW8bit_CUDA(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=WD, master_weights=master, seed=7)
    for t in (1, 2, 3):
        set_grads(params, gt, 10 + t, odd=odd)
        grads = [p.grad.clone() for p in params]
        old = old_8(opt, params)
        opt.step()
        check_8(opt, params, old, grads, t, 7)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, 1e-36, 1e-20, 1e-5, 1e5, 1e15])
def test_states_of_8_bits_of_any_size(scale):
    """Blocks of zeros, and of values near either end of the range (1e5 and more: the factor to the codes needs two steps)."""
    params = params_of([(300,), (5, 512)], torch.float32, 2)
    opt = optim.AdamW8bit_CUDA(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=WD, seed=3)
    for t in (1, 2):
        set_grads(params, torch.float32, 20 + t, scale)
        params[0].grad[:256] = 0
        grads, old = [p.grad.clone() for p in params], old_8(opt, params)
        opt.step()
        if scale < 1e-19:   # squares are below 2^-126, the smallest normal number (1e-20: 1e-40 < 1.2e-38), and have few bits left or none
            for p, g, o in zip(params, grads, old):
                st = opt.state[p]
                me = BETAS[0] * o[1] + (1 - BETAS[0]) * g.double()
                check_codes(st["exp_avg"].cpu(), st["exp_avg_scale"].cpu(), me.cpu(), (me.abs() * 4 * H32 + 2.0 ** -140).cpu(), random_parts(p.numel(), 3, t, 8), 0)
                assert bool(p.isfinite().all())
        else:
            check_8(opt, params, old, grads, t, 3)


@pytest.mark.gpu
def test_values_that_are_none_stay_where_they_are():
    p = torch.nn.Parameter(torch.ones(700, device="cuda"))
    opt = optim.AdamW8bit_CUDA([p], lr=LR, weight_decay=0.0)
    p.grad = torch.ones_like(p)
    p.grad[[3, 300, 699]] = torch.tensor([math.nan, math.inf, -math.inf], device="cuda")
    opt.step()
    p.grad = torch.ones_like(p)
    opt.step()
    st = opt.state[p]
    bad = torch.zeros(700, dtype=torch.bool, device="cuda")
    bad[[3, 300, 699]] = True
    m, u = (A.from_blocks(st[k], st[k + "_scale"]) for k in ("exp_avg", "exp_avg_sq_root"))
    for x in (m, u, p.detach()):
        assert bool(x[bad].isnan().all()) and bool(x[~bad].isfinite().all())
    # nothing else of those blocks is off by more than a step of a code, up or down, in each of two steps
    assert bool(((m[~bad] / (0.1 + 0.09) - 1).abs() <= 2 * 2.0 ** -3).all())


@pytest.mark.gpu
def test_codes_are_right_on_the_average():
    """With one gradient for all elements and steps, the mean of m is b1 m + (1 - b1) g, of u the root of b2 v + (1 - b2) g^2, whatever the
    codes can say."""
    n = 1 << 20
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    opt = optim.AdamW8bit_CUDA([p], lr=0.0, weight_decay=0.0, betas=BETAS)
    p.grad = torch.full_like(p, 0.3)
    p.grad[::256] = 1.0   # the blocks' largest: 0.3 stands in the middle of the codes
    opt.step()
    st = opt.state[p]
    rest = torch.arange(n, device="cuda") % 256 != 0
    m, u = (A.from_blocks(st[k], st[k + "_scale"]).double() for k in ("exp_avg", "exp_avg_sq_root"))
    for x, want in ((m, 0.03), (u, math.sqrt(0.05) * 0.3)):
        step = 2.0 ** (math.floor(math.log2(want)) - 3)
        assert len(x[rest].unique()) == 2
        # six standard deviations of a mean of n values that are one of two a step apart
        assert abs(float(x[rest].mean()) - want) < 6 * 0.5 * step / math.sqrt(n) + want * 8 * H32


@pytest.mark.gpu
def test_a_root_that_is_not_zero_stays_so():
    p = torch.nn.Parameter(torch.zeros(512, device="cuda"))
    opt = optim.AdamW8bit_CUDA([p], lr=1e-3)
    g = torch.full((512,), 1e-9, device="cuda")
    g[0] = 1.0   # the smallest code of its block is far above the others' values
    for _ in range(20):
        p.grad = g.clone()
        opt.step()
    assert bool((opt.state[p]["exp_avg_sq_root"].float() > 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [12, 179, 231, 690])   # a launch takes 180 (8-bit) or 224 of a kind; one kind, or three
def test_many_tensors_and_many_sets(bits, count):
    """More tensors and more sets of hyper-parameters than a launch takes, steps that differ, tensors without elements and without
    gradients: the same as one optimizer for each tensor, to the last bit."""
    cls = optim.AdamW_CUDA if bits == 32 else optim.AdamW8bit_CUDA
    shapes = [(i % 7 * 61,) if i % 5 else (3, i + 1) for i in range(count)]
    kinds = [torch.float32, torch.bfloat16, torch.float16] if count % 10 == 0 else [torch.float32] * 3
    make = lambda: [torch.nn.Parameter(tensors([s], kinds[i % 3], i)[0]) for i, s in enumerate(shapes)]
    a, b = make(), make()
    group = lambda ps, k: dict(params=ps, lr=1e-3 * (k + 1), weight_decay=0.01 * k, betas=(0.8 + 0.01 * k, 0.9))
    opt = cls([group(a[k::11], k) for k in range(11)])
    each = [cls([group([p], i % 11)]) for i, p in enumerate(b)]
    for t in range(3):
        for i, (p, q) in enumerate(zip(a, b)):
            if t == 0 and i % 4 == 1:
                continue
            p.grad = tensors([shapes[i]], kinds[i % 3], 1000 * t + i)[0]
            q.grad = p.grad.clone()
        opt.step()
        for q in b:
            if q.grad is not None:
                each[[x is q for x in b].index(True)].step()
    for i, (p, q) in enumerate(zip(a, b)):
        assert torch.equal(p, q), i
        for name, x in each[i].state[q].items():
            y = opt.state[p][name]
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)) if x.dtype.itemsize == 1 else torch.equal(x, y), (i, name)


@pytest.mark.gpu
@pytest.mark.parametrize("cls", [optim.AdamW_CUDA, optim.AdamW8bit_CUDA])
def test_runs_are_the_same_to_the_last_bit(cls):
    res = []
    for _ in range(2):
        params = params_of(SIZES, torch.float32, 5)
        opt = cls(params, clip_grad=True, clip_norm=0.1)
        for t in range(3):
            set_grads(params, torch.float32, t)
            opt.step()
        res.append([p.detach().clone() for p in params])
    assert all(torch.equal(x, y) for x, y in zip(*res))


@pytest.mark.gpu
@pytest.mark.parametrize("cls", [optim.AdamW_CUDA, optim.AdamW8bit_CUDA])
@pytest.mark.parametrize("maximize", [False, True])
def test_clipping_within_the_step(cls, maximize):
    """The gradients are those of all groups; they stay as they are; a group that does not clip goes without."""
    params = params_of(SIZES, torch.float32, 1) + params_of([(100,)], torch.bfloat16, 2)
    free = params_of([(33,)], torch.float32, 3)
    opt = cls([dict(params=params), dict(params=free, clip_grad=False)], lr=LR, betas=BETAS, eps=EPS, weight_decay=WD, clip_grad=True, clip_norm=0.25, maximize=maximize)
    set_grads(params[:-1], torch.float32, 4)
    set_grads(params[-1:], torch.bfloat16, 5)
    set_grads(free, torch.float32, 6)
    every = params + free
    grads = [p.grad.clone() for p in every]
    old = [p.detach().clone() for p in every]
    norm = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
    assert norm > 1
    opt.step()
    for p, g, o in zip(every, grads, old):
        assert torch.equal(p.grad, g)
        gs = (0.25 / norm if p is not free[0] else 1.0)
        z = torch.zeros(p.shape, device="cuda")
        # the sum of squares: 64 squares a thread at most and five sums over lanes and warps, 2^-24 each, half of it in the root
        if cls is optim.AdamW_CUDA:
            check_32(p.detach(), opt.state[p]["exp_avg"], opt.state[p]["exp_avg_sq"], (o, z, z), -g if maximize else g, 1, gs=gs, gs_err=40 * H32)
        else:
            check_8(opt, [p], [(o, z.double(), z.double())], [g], 1, 0, gs=gs, gs_err=40 * H32, maximize=maximize)


@pytest.mark.gpu
def test_a_norm_below_the_limit_changes_nothing():
    res = []
    for clip in (False, True):
        params = params_of(SIZES, torch.float32, 1)
        opt = optim.AdamW_CUDA(params, clip_grad=clip, clip_norm=1e9)
        set_grads(params, torch.float32, 2)
        opt.step()
        res.append(params)
    assert all(torch.equal(x, y) for x, y in zip(*res))


@pytest.mark.gpu
def test_agrees_with_torch_over_many_steps():
    """Both are within a few roundings of the formulas in every step; the sum of 50 steps' roundings bounds their difference."""
    shapes = [(64, 32), (33,), (5, 7, 3)]
    a, b = params_of(shapes, torch.float32, 1), params_of(shapes, torch.float32, 1)
    kw = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2)
    x, y = optim.AdamW_CUDA(a, **kw), torch.optim.AdamW(b, **kw)
    for t in range(50):
        set_grads(a, torch.float32, t)
        for p, q in zip(a, b):
            q.grad = p.grad.clone()
        x.step()
        y.step()
    for p, q in zip(a, b):
        # a step: 6 half steps of p between the two, an update of at most ~10 lr with 40; m and v carry 10 and 20 half steps of their own
        bound = 50 * (6 * H32 * q.abs().double() + 10e-3 * 80 * H32)
        assert bool(((p.double() - q.double()).abs() <= bound).all())


# ---------------------------------------------------------------------------------------------------------------------
# states, checkpoints, arguments
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("cls", [optim.AdamW_CUDA, optim.AdamW8bit_CUDA])
@pytest.mark.parametrize("capturable", [False, True])
def test_a_checkpoint_goes_on_where_it_was_made(cls, capturable, tmp_path):
    kw = dict(master_weights=True, capturable=capturable)
    a = params_of([(40, 30), (300,)], torch.bfloat16, 1)
    opt = cls(a, **kw)
    for t in range(2):
        set_grads(a, torch.bfloat16, t)
        opt.step()
    torch.save(opt.state_dict(), tmp_path / "c.pt")
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    new = cls(b, **kw)
    new.load_state_dict(torch.load(tmp_path / "c.pt", map_location="cpu"))
    for o, ps in ((opt, a), (new, b)):
        for t in range(2, 4):
            set_grads(ps, torch.bfloat16, t)
            o.step()
    for p, q in zip(a, b):
        assert torch.equal(p, q)
        for name, x in opt.state[p].items():
            y = new.state[q][name]
            assert x.dtype is y.dtype and torch.equal(x.float(), y.float()), name


@pytest.mark.gpu
def test_checkpoints_of_torch_and_of_the_other_width():
    a, b = params_of([(64, 32), (33,)], torch.float32, 1), params_of([(64, 32), (33,)], torch.float32, 1)
    theirs, ours = torch.optim.AdamW(a, lr=1e-3), optim.AdamW_CUDA(b, lr=1e-3)
    for t in range(3):
        set_grads(a, torch.float32, t)
        theirs.step()
    with torch.no_grad():
        for p, q in zip(a, b):
            q.copy_(p)
    ours.load_state_dict(theirs.state_dict())
    set_grads(b, torch.float32, 9)
    old = [(q.detach().clone(), theirs.state[p]["exp_avg"].clone(), theirs.state[p]["exp_avg_sq"].clone()) for p, q in zip(a, b)]
    ours.step()
    for q, o in zip(b, old):
        check_32(q.detach(), ours.state[q]["exp_avg"], ours.state[q]["exp_avg_sq"], o, q.grad, 4, lr=1e-3, betas=(0.9, 0.999), wd=1e-2)
    eight = optim.AdamW8bit_CUDA(b, lr=1e-3)
    eight.load_state_dict(ours.state_dict())
    eight.step()
    assert all(float(eight.state[q]["step"]) == 5 and eight.state[q]["exp_avg"].dtype is torch.float8_e4m3fn for q in b)
    back = optim.AdamW_CUDA(b, lr=1e-3)
    back.load_state_dict(eight.state_dict())
    kept = {q: A.from_blocks(eight.state[q]["exp_avg"], eight.state[q]["exp_avg_scale"]) for q in b}
    set_grads(b, torch.float32, 10)
    back.step()
    for q in b:
        close(back.state[q]["exp_avg"], 0.9 * kept[q].double() + 0.1 * q.grad.double(), (0.9 * kept[q].double().abs() + 0.1 * q.grad.double().abs()) * 4 * H32)
    bad = theirs.state_dict()
    bad["param_groups"][0]["amsgrad"] = True
    with pytest.raises(ValueError, match="amsgrad"):
        optim.AdamW_CUDA(b).load_state_dict(bad)


@pytest.mark.gpu
@pytest.mark.parametrize("cls", [optim.AdamW_CUDA, optim.AdamW8bit_CUDA])
def test_what_is_refused(cls):
    p = torch.nn.Parameter(torch.zeros(8, device="cuda"))
    for bad in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1e-8), dict(weight_decay=-1.0), dict(clip_norm=0.0)):
        with pytest.raises(ValueError):
            cls([p], **bad)

    if cls is optim.AdamW8bit_CUDA:
        with pytest.raises(ValueError, match="eps"):
            cls([p], eps=0.0)

    def refused(params, match, error=RuntimeError):
        for q in params:
            if q.grad is None:
                q.grad = torch.zeros_like(q)
        opt = cls(params)
        with pytest.raises(error, match=match):
            opt.step()

    refused([torch.nn.Parameter(torch.zeros(4))], "CUDA")
    refused([torch.nn.Parameter(torch.zeros(4, device="cuda", dtype=torch.float64))], "fp32, bf16 or fp16")
    refused([torch.nn.Parameter(torch.zeros(4, 4, device="cuda").t()[:, :2])], "contiguous")
    x = torch.zeros(10, device="cuda")
    refused([torch.nn.Parameter(x[:6]), torch.nn.Parameter(x[5:])], "share memory", ValueError)
    q = torch.nn.Parameter(torch.zeros(4, 4, device="cuda"))
    q.grad = torch.zeros(4, 4, device="cuda").to_sparse()
    refused([q], "Sparse")
    q = torch.nn.Parameter(torch.zeros(4, device="cuda"))
    q._pylo_peer_ptrs = [256]
    refused([q], "other rank")
    opt = cls([p])
    p.grad = torch.zeros_like(p)
    opt.step()
    whole, p.data = p.data, p.data[:4]   # at the same address
    with pytest.raises(RuntimeError, match="gradient has shape"):
        opt.step()
    p.data = whole
    opt.step()
    opt.state[p]["exp_avg"] = opt.state[p]["exp_avg"][:4]
    with pytest.raises(ValueError, match="shape"):
        opt.step()


@pytest.mark.gpu
@pytest.mark.parametrize("cls", [optim.AdamW_CUDA, optim.AdamW8bit_CUDA])
def test_gradients_in_other_layouts_and_on_another_stream(cls):
    a, b = params_of([(40, 60), (8, 3, 5, 5)], torch.float32, 1), params_of([(40, 60), (8, 3, 5, 5)], torch.float32, 1)
    x, y = cls(a), cls(b)
    side = torch.cuda.Stream()
    for t in range(2):
        set_grads(a, torch.float32, t)
        b[0].grad = a[0].grad.t().contiguous().t()
        b[1].grad = a[1].grad.contiguous(memory_format=torch.channels_last)
        x.step()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            y.step()
        torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.gpu
@pytest.mark.parametrize("cls", [optim.AdamW_CUDA, optim.AdamW8bit_CUDA])
def test_another_memory_behind_a_parameter(cls):
    """Parameters and gradients that move between steps (resized, cast, set anew) are found where they are now."""
    a, b = params_of([(700,)], torch.float32, 1), params_of([(700,)], torch.float32, 1)
    x, y = cls(a), cls(b)
    for t in range(3):
        set_grads(a, torch.float32, t)
        b[0].data = b[0].data.clone()
        b[0].grad = a[0].grad.clone()
        x.step()
        y.step()
    assert torch.equal(a[0], b[0])
    assert x.state[a[0]]["step"] == 3


@pytest.mark.gpu
@pytest.mark.parametrize("cls", [optim.AdamW_CUDA, optim.AdamW8bit_CUDA])
def test_states_in_the_callers_memory(cls):
    """State tensors set before the first step, views into buffers of the caller's, are the ones that are updated."""
    a, b = params_of([(300,), (1000,)], torch.bfloat16, 1), params_of([(300,), (1000,)], torch.bfloat16, 1)
    x, y = cls(a, master_weights=True), cls(b, master_weights=True)
    set_grads(b, torch.bfloat16, 2)
    y.step()
    buffers = {}
    for p, q in zip(a, b):
        p.grad = q.grad.clone()
        x.state[p] = {}
        for name, v in y.state[q].items():
            if name == "step":
                continue
            room = torch.zeros(v.numel() * v.dtype.itemsize + 64, dtype=torch.uint8, device="cuda")
            at = 3 if name.endswith("scale") else 16
            view = room[at:at + v.numel() * v.dtype.itemsize].view(v.dtype).view(v.shape)
            if name == "master":
                view.copy_(p.detach())
            elif at == 3:
                view.view(torch.uint8).fill_(1)   # the least scale
            x.state[p][name], buffers[p, name] = view, (room, at)
    x.step()
    for p, q in zip(a, b):
        assert torch.equal(p, q)
        for name, v in y.state[q].items():
            if name == "step":
                continue
            room, at = buffers[p, name]
            n = v.numel() * v.dtype.itemsize
            assert torch.equal(room[at:at + n], v.contiguous().view(-1).view(torch.uint8)), name
            assert not room[:at].any() and not room[at + n:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("cls", [optim.AdamW_CUDA, optim.AdamW8bit_CUDA])
def test_states_that_are_taken_away_or_set_anew(cls):
    """A step goes by what the state holds now: cleared, it begins anew; a count or a tensor set by hand counts."""
    a, b = params_of([(300,), (20,)], torch.float32, 1), params_of([(300,), (20,)], torch.float32, 1)
    x, y = cls(a), cls(b)

    def both(t):
        set_grads(a, torch.float32, t)
        for p, q in zip(a, b):
            q.grad = p.grad.clone()
        x.step()
        y.step()

    both(0)
    x.state.clear()
    y = cls(b)
    both(1)
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and float(x.state[a[0]]["step"]) == 1
    x.state[a[0]] = {k: v.clone() for k, v in x.state[a[0]].items()}
    x.state[a[1]]["step"] = 7
    y.state[b[1]]["step"].fill_(7)
    both(2)
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and float(x.state[a[1]]["step"]) == 8
    x.state.pop(a[1])
    y.state.pop(b[1])
    moment = x.state[a[0]]["exp_avg"]
    odd = torch.empty(moment.numel() + 1, dtype=moment.dtype, device="cuda")[1:]
    x.state[a[0]]["exp_avg"] = odd.copy_(moment)   # on no boundary
    both(3)
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and float(x.state[a[0]]["step"]) == 3 and float(x.state[a[1]]["step"]) == 1
    for k, name in enumerate(n for n in y.state[b[0]] if n != "step"):   # each of them by another tensor, what was there gone
        x.state[a[0]][name] = y.state[b[0]][name].clone()
        gone = [torch.full((301,), 255, dtype=torch.uint8, device="cuda") for _ in range(64)]   # over the memory that was given back
        both(4 + k)
        assert all(torch.equal(p, q) for p, q in zip(a, b)), name
        del gone
    x.state[a[1]].popitem()   # the last of all: made anew
    last = list(y.state[b[1]])[-1]
    y.state[b[1]].pop(last)
    both(20)
    assert all(torch.equal(p, q) for p, q in zip(a, b)) and last in x.state[a[1]]


@pytest.mark.gpu
def test_closure_hooks_and_groups():
    p, q = params_of([(10,), (20,)], torch.float32, 1)
    opt = optim.AdamW([p], lr=1e-3)
    opt.add_param_group(dict(params=[q], lr=2e-3))
    seen = []
    opt.before_group, opt.after_group = lambda gi: seen.append(("before", gi)), lambda gi: seen.append(("after", gi))

    def closure():
        assert torch.is_grad_enabled()
        opt.zero_grad()
        loss = (p.sum() * 3 + q.square().sum())
        loss.backward()
        return loss

    before = p.detach().clone()
    loss = opt.step(closure)
    assert loss.requires_grad and not torch.equal(before, p)
    assert seen == [("before", 0), ("before", 1), ("after", 0), ("after", 1)]


# ---------------------------------------------------------------------------------------------------------------------
# captured steps
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("cls", [optim.AdamW_CUDA, optim.AdamW8bit_CUDA])
def test_a_captured_step_counts_on(cls):
    """Replays are the steps that an optimizer without a graph takes, with a learning rate on the device that changes between them and
    a clipping norm of each; steps without the graph in between go on from there."""
    shapes = [(64, 32), (257,)]
    a, b = params_of(shapes, torch.float32, 1), params_of(shapes, torch.float32, 1)
    lr = torch.tensor(1e-2, device="cuda")
    x = cls(a, lr=lr, capturable=True, clip_grad=True, clip_norm=1.0)
    y = cls(b, lr=1e-2, capturable=True, clip_grad=True, clip_norm=1.0)
    grads = [torch.zeros(s, device="cuda") for s in shapes]
    for p, g in zip(a, grads):
        p.grad = g

    def feed(t):
        for g, q, new in zip(grads, b, tensors(shapes, torch.float32, 50 + t)):
            g.copy_(new)
            q.grad = new

    feed(0)
    x.step()
    y.step()
    graph = torch.cuda.CUDAGraph()
    kept = [p.detach().clone() for p in a]
    with torch.cuda.graph(graph):
        x.step()
    assert all(torch.equal(p, k) for p, k in zip(a, kept))
    for t in range(1, 6):
        feed(t)
        lr.fill_(1e-2 / t)
        y.param_groups[0]["lr"] = float(lr)
        if t == 3:
            x.step()
        else:
            graph.replay()
        y.step()
        torch.cuda.synchronize()
        for p, q in zip(a, b):
            assert torch.equal(p, q), t
            assert float(x.state[p]["step"]) == t + 1


@pytest.mark.gpu
@pytest.mark.parametrize("cls", [optim.AdamW_CUDA, optim.AdamW8bit_CUDA])
def test_counting_on_the_device_is_the_same_step(cls):
    """Factors made in 32 bits on the device: within a few roundings of those made in 64 on the host."""
    a, b = params_of([(3000,)], torch.float32, 1), params_of([(3000,)], torch.float32, 1)
    x, y = cls(a, lr=1e-2, capturable=True), cls(b, lr=1e-2)
    for t in range(3):
        set_grads(a, torch.float32, t)
        b[0].grad = a[0].grad.clone()
        old = b[0].detach().clone()
        with torch.no_grad():
            a[0].copy_(b[0])
        if t:
            for name, v in y.state[b[0]].items():
                if name != "step":
                    x.state[a[0]][name].view(torch.uint8).copy_(v.view(torch.uint8)) if v.dtype.itemsize == 1 else x.state[a[0]][name].copy_(v)
        x.step()
        y.step()
        moved = (b[0].double() - old.double()).abs() + 1e-2 * old.double().abs() * 1e-2
        # lr / bc1, 1 / root of bc2 by exponentials: 1 - beta^t is off by 2 half steps of its own and t times that of ln beta, each factor of it
        assert bool(((a[0].double() - b[0].double()).abs() <= moved * 40 * H32 + old.double().abs() * 4 * H32).all())


@pytest.mark.gpu
@pytest.mark.parametrize("cls", [optim.AdamW_CUDA, optim.AdamW8bit_CUDA])
def test_captures_that_are_refused(cls):
    p = params_of([(10,)], torch.float32, 1)[0]
    p.grad = torch.ones_like(p)
    for capturable, match in ((False, "capturable"), (True, "run a step before")):
        opt = cls([p], capturable=capturable)
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match=match):
            with torch.cuda.graph(graph):
                torch.ones(1, device="cuda").add_(1)   # a graph that is empty is a warning
                opt.step()


@pytest.mark.gpu
def test_states_are_not_converted_in_a_capture():
    """Loaded states of the other width would be converted on every replay: refused, and possible after a step."""
    a = params_of([(300,)], torch.float32, 1)
    set_grads(a, torch.float32, 2)
    x = optim.AdamW_CUDA(a)
    x.step()
    y = optim.AdamW8bit_CUDA(a, capturable=True)
    y.load_state_dict(x.state_dict())
    for group in y.param_groups:
        group["capturable"] = True
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="run a step before"):
        with torch.cuda.graph(graph):
            torch.ones(1, device="cuda").add_(1)
            y.step()
    y.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y.step()
    graph.replay()
    torch.cuda.synchronize()
    assert float(y.state[a[0]]["step"]) == 3


@pytest.mark.gpu
def test_two_graphs_of_two_optimizers_run_beside_each_other():
    """Each has its own norm's workspace."""
    runs = []
    for k in range(2):
        a, b = params_of([(400, 300)], torch.float32, k), params_of([(400, 300)], torch.float32, k)
        x, y = (optim.AdamW_CUDA(ps, clip_grad=True, clip_norm=0.5, capturable=True) for ps in (a, b))
        for ps, o in ((a, x), (b, y)):
            set_grads(ps, torch.float32, 10 + k, scale=10.0 ** k)
            o.step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            x.step()
        runs.append((a[0], b[0], y, graph, torch.cuda.Stream(), x))   # x: a graph does not keep the states alive
    torch.cuda.synchronize()
    for _ in range(5):
        for _, _, _, graph, stream, _ in runs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for a, b, y, _, _, _ in runs:
        for _ in range(5):
            y.step()
        assert torch.equal(a, b)


# ---------------------------------------------------------------------------------------------------------------------
# clipping by itself
# ---------------------------------------------------------------------------------------------------------------------
def with_grads(grads):
    params = []
    for g in grads:
        p = torch.nn.Parameter(torch.zeros(g.shape, device="cuda", dtype=g.dtype))
        p.grad = g
        params.append(p)
    return params


def check_clip(grads, before, norm, max_norm):
    exact = math.sqrt(sum(float(b.double().square().sum()) for b in before))
    # 64 squares a thread and the sums over lanes and warps, in fp32, half of it in the root
    assert abs(float(norm) - exact) <= exact * 40 * H32
    by = min(1.0, max_norm / (exact + 1e-6))
    for g, b in zip(grads, before):
        if by == 1.0:
            assert torch.equal(g, b)
        else:
            want = b.double() * by
            close(g, want, want.abs() * (45 * H32 + HALF[g.dtype] * (1 + 1e-3)) + TINY[g.dtype])


@pytest.mark.gpu
@pytest.mark.parametrize("odd", [False, True])
@pytest.mark.parametrize("kinds", [(torch.float32,), (torch.bfloat16,), (torch.float16,), (torch.float32, torch.bfloat16, torch.float16)])
@pytest.mark.parametrize("max_norm", [0.0, 0.1, 1e6])
def test_clipping(kinds, odd, max_norm):
    shapes = SIZES + [(0,), (5, 0), (300, 1000)]
    grads = [tensors([s], kinds[i % len(kinds)], i, odd=odd)[0] for i, s in enumerate(shapes)]
    before = [g.clone() for g in grads]
    norm = optim.clip_grad_norm_(with_grads(grads), max_norm)
    assert norm.dtype is torch.float32 and norm.dim() == 0 and norm.is_cuda
    check_clip(grads, before, norm, max_norm)


@pytest.mark.gpu
@pytest.mark.parametrize("backwards", [False, True])
@pytest.mark.parametrize("count", [44, 801, 1024, 1025, 3200])
def test_clipping_of_many_gradients(count, backwards):
    flat = torch.randn(count * 37, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    grads = [flat[37 * i:37 * i + 30 + i % 8] for i in range(count)][::-1 if backwards else 1]
    before = [g.clone() for g in grads]
    gaps = flat.clone()
    check_clip(grads, before, optim.clip_grad_norm_(with_grads(grads), 0.5), 0.5)
    left = torch.ones(count * 37, dtype=torch.bool, device="cuda")
    for i in range(count):
        left[37 * i:37 * i + 30 + i % 8] = False
    assert torch.equal(flat[left], gaps[left])   # what lies between them


@pytest.mark.gpu
def test_clipping_of_other_layouts_and_of_one_given_twice():
    x = torch.randn(6, 4, 5, 5, device="cuda").contiguous(memory_format=torch.channels_last)
    y = torch.randn(20, 30, device="cuda").t()
    z = torch.randn(20, 30, device="cuda")[:, ::2]
    hidden = z._base.clone()
    grads = [x, y, z]
    before = [g.clone() for g in grads]
    strides = [g.stride() for g in grads]
    params = with_grads(grads)
    check_clip([p.grad for p in params], before, optim.clip_grad_norm_(params + params[:1] + params[1:2], 0.3), 0.3)
    assert [p.grad.stride() for p in params] == strides and torch.equal(z._base[:, 1::2], hidden[:, 1::2])
    one = torch.nn.Parameter(torch.zeros(5, device="cuda"))
    one.grad = torch.full((5,), 2.0, device="cuda")
    assert abs(float(optim.clip_grad_norm_(one, 1.0)) - math.sqrt(20)) < 1e-5 and abs(float(one.grad.norm()) - 1) < 1e-5


@pytest.mark.gpu
def test_norms_that_are_not_finite():
    for value in (math.inf, math.nan):
        g = torch.ones(1000, device="cuda")
        g[7] = value
        p = with_grads([g])
        with pytest.raises(RuntimeError, match="non-finite"):
            optim.clip_grad_norm_(p, 1.0, error_if_nonfinite=True)
        assert bool((g[8:] == 1).all())
        norm = optim.clip_grad_norm_(p, 1.0)
        assert (math.isnan if math.isnan(value) else math.isinf)(float(norm))
        want = torch.ones(1000) * (1.0 / (torch.tensor(value) + 1e-6))
        want[7] = math.nan
        assert torch.equal(g.cpu().isnan(), want.isnan()) and torch.equal(g.cpu().nan_to_num(), want.nan_to_num())
    g = torch.full((10,), 3.0, device="cuda")
    assert float(optim.clip_grad_norm_(with_grads([g]), math.inf)) == pytest.approx(math.sqrt(90)) and bool((g == 3).all())


@pytest.mark.gpu
def test_gradients_that_are_refused():
    for g, match in ((torch.zeros(3, device="cuda", dtype=torch.float64), "fp32, bf16 or fp16"), (torch.zeros(3), "CUDA")):
        p = torch.nn.Parameter(torch.zeros(3, device=g.device, dtype=g.dtype))
        p.grad = g
        with pytest.raises(RuntimeError, match=match):
            optim.clip_grad_norm_([p], 1.0)
    p = torch.nn.Parameter(torch.zeros(3, 3, device="cuda"))
    p.grad = torch.zeros(3, 3, device="cuda").to_sparse()
    with pytest.raises(RuntimeError, match="Sparse"):
        optim.clip_grad_norm_([p], 1.0)


@pytest.mark.gpu
def test_clipping_in_a_graph():
    g = torch.randn(5000, device="cuda")
    p = with_grads([g])
    optim.clip_grad_norm_(p, 1.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = optim.clip_grad_norm_(p, 1.0)
    for t in range(3):
        new = torch.randn(5000, device="cuda", generator=torch.Generator(device="cuda").manual_seed(t))
        g.copy_(new)
        graph.replay()
        check_clip([g], [new], norm, 1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("cls", [optim.AdamW_CUDA, optim.AdamW8bit_CUDA])
def test_elements_behind_the_first_four_billion_bytes(cls):
    """One tensor of more than 2^31 elements: its last ones get the step that a tensor of them alone gets (in 8 bits as far as the random rounding
    goes, which takes an element's place into account), and count in the norm."""
    if torch.cuda.get_device_properties(0).total_memory < 100 << 30:
        pytest.skip("needs 60 GB")
    n, k = 2 ** 31 + 2 ** 20, 2 ** 20 + 300
    p = torch.nn.Parameter(torch.zeros(n, device="cuda", dtype=torch.bfloat16))
    p.grad = torch.zeros_like(p)
    p.grad[-k:] = tensors([(k,)], torch.bfloat16, 1)[0]
    p.data[-k:] = tensors([(k,)], torch.bfloat16, 2)[0]
    q = torch.nn.Parameter(p.detach()[-k:].clone())
    q.grad = p.grad[-k:].clone()
    exact = math.sqrt(float(q.grad.double().square().sum()))
    assert abs(float(optim.clip_grad_norm_(p, math.inf)) - exact) <= exact * 40 * H32
    x, y = cls([p]), cls([q])
    x.step()
    y.step()
    assert torch.equal(p[-k:], q) and not p[:-k].any()
    st, want = x.state[p], y.state[q]
    if cls is optim.AdamW_CUDA:
        assert all(torch.equal(st[name][-k:], want[name]) for name in ("exp_avg", "exp_avg_sq"))
    else:
        assert (n - k) % 256 == 212   # blocks lie otherwise
        for name in ("exp_avg", "exp_avg_sq_root"):
            a, b = A.from_blocks(st[name][-k - 212:], st[name + "_scale"][(n - k) // 256:])[212:], A.from_blocks(want[name], want[name + "_scale"])
            each = want[name + "_scale"].float().repeat_interleave(256)[:k]
            # both within a step of a code: 2^-3 of the value (8 / 7 of the larger code at most), or 2^-9 of a scale (the largest value over 128 at most)
            assert bool(((a - b).abs() <= 2.3 * 2.0 ** -3 * torch.maximum(a.abs(), b.abs()) + 4 * 2.0 ** -9 * torch.maximum(each, a.abs().amax() * 2.0 ** -7)).all())
    del x, y, p, q, st, want
    torch.cuda.empty_cache()


# ---------------------------------------------------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("cls", [optim.AdamW_CUDA, optim.AdamW8bit_CUDA])
def test_a_training_loop(cls):
    """Mixed precision: backward passes, clipping, steps, a learned optimizer before and after on the same kind of loop."""
    torch.manual_seed(0)
    model = torch.nn.Sequential(torch.nn.Linear(24, 48), torch.nn.LayerNorm(48), torch.nn.ReLU(), torch.nn.Linear(48, 8)).cuda()
    model[0].to(torch.bfloat16), model[3].to(torch.bfloat16)
    opt = cls(model.parameters(), lr=1e-3, master_weights=True)
    x, y = torch.randn(64, 24, device="cuda"), torch.randn(64, 8, device="cuda")
    for t in range(3):
        opt.zero_grad()
        h = torch.relu(model[1](model[0](x.bfloat16()).float())).bfloat16()
        loss = (model[3](h).float() - y).square().mean()
        loss.backward()
        before = [p.grad.clone() for p in model.parameters()]
        norm = optim.clip_grad_norm_(model.parameters(), 0.05)
        check_clip([p.grad for p in model.parameters()], before, norm, 0.05)
        old = [p.detach().clone() for p in model.parameters()]
        opt.step()
        assert all(bool(p.isfinite().all()) for p in model.parameters())
        assert any(not torch.equal(p, o) for p, o in zip(model.parameters(), old))
        for p in model.parameters():
            assert ("master" in opt.state[p]) == (p.dtype is torch.bfloat16)


@pytest.mark.gpu
def test_beside_a_learned_optimizer():
    """Matrices through AdafacLO, vectors through AdamW, the gradients of both clipped together: each as by itself."""
    from pylo_b200 import models

    torch.manual_seed(1)
    net = models.MetaMLP()
    shapes = [(96, 64), (96,), (40, 96), (40,)]
    a, b = params_of(shapes, torch.float32, 1), params_of(shapes, torch.float32, 1)
    learned, plain = optim.AdafacLO_CUDA(a[::2], network=net), optim.AdamW8bit_CUDA(a[1::2])
    alone, other = optim.AdafacLO_CUDA(b[::2], network=net), optim.AdamW8bit_CUDA(b[1::2])
    for t in range(3):
        set_grads(a, torch.float32, t)
        for p, q in zip(a, b):
            q.grad = p.grad.clone()
        optim.clip_grad_norm_(a, 0.5)
        plain.step()
        learned.step()
        optim.clip_grad_norm_(b, 0.5)
        torch.cuda.synchronize()
        alone.step()
        torch.cuda.synchronize()
        other.step()
        assert all(torch.equal(p, q) for p, q in zip(a, b)), t


@pytest.mark.gpu
@pytest.mark.parametrize("cls", [optim.AdamW_CUDA, optim.AdamW8bit_CUDA])
def test_through_a_sharded_step(cls):
    from pylo_b200.zero import ShardedStep, consolidate_state_dict, sharded_optimizer

    shapes = [(40, 24), (24,), (300,)]
    a, b = params_of(shapes, torch.float32, 1), params_of(shapes, torch.float32, 1)
    shard = ShardedStep(a)
    x, y = sharded_optimizer(cls, shard, clip_grad=True, clip_norm=0.5), cls(b, clip_grad=True, clip_norm=0.5)
    for t in range(2):
        set_grads(a, torch.float32, t)
        for p, q in zip(a, b):
            q.grad = p.grad.clone()
        x.step()
        shard.gather()
        y.step()
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    full = consolidate_state_dict(x, shard)
    assert sorted(full["state"]) == [0, 1, 2]
    new = cls(b, clip_grad=True, clip_norm=0.5)
    new.load_state_dict(full)
    set_grads(b, torch.float32, 5)
    new.step()


@pytest.mark.gpu
@pytest.mark.parametrize("cls", [optim.AdamW_CUDA, optim.AdamW8bit_CUDA])
@pytest.mark.parametrize("capturable", [False, True])
def test_a_norm_that_is_summed_over_ranks(cls, capturable, monkeypatch):
    """Two optimizers with half of the tensors each, the exchange of their sums of squares played by hand: each rank's sum is that of its own
    gradients, the step goes by both."""
    shapes = [(300, 200), (77,), (1000,), (5, 5)]
    params = params_of(shapes, torch.float32, 1)
    set_grads(params, torch.float32, 2)
    old = [p.detach().clone() for p in params]
    squares = [float(p.grad.double().square().sum()) for p in params]
    norm = math.sqrt(sum(squares))
    said = []
    for mine in ((0, 1), (2, 3)):
        opt = cls([params[i] for i in mine], lr=LR, betas=BETAS, eps=EPS, weight_decay=WD, clip_grad=True, clip_norm=0.5, capturable=capturable)
        opt._sharded = True
        own, rest = (sum(squares[i] for i in range(4) if (i in mine) == side) for side in (True, False))

        def exchange(t, group=None):
            said.append(abs(float(t) - own) <= own * 80 * H32)   # a sum of squares: twice a norm's error
            t.add_(rest)

        monkeypatch.setattr(torch.distributed, "is_initialized", lambda: True)
        monkeypatch.setattr(torch.distributed, "all_reduce", exchange)
        opt.step()
        monkeypatch.undo()
        for i in mine:
            z = torch.zeros(shapes[i], device="cuda")
            if cls is optim.AdamW_CUDA and not capturable:
                st = opt.state[params[i]]
                check_32(params[i].detach(), st["exp_avg"], st["exp_avg_sq"], (old[i], z, z), params[i].grad, 1, gs=0.5 / norm, gs_err=40 * H32)
            else:
                pe, _, _, upd = exact_step(old[i], params[i].grad.double() * 0.5 / norm, z, z, 1)
                close(params[i].detach(), pe, upd * 200 * H32 + old[i].double().abs() * 4 * H32)   # 16 + 2 x 40 of the norm, the device's own factors
    assert said == [True, True]

"""AdamW over many tensors at once, with states in 32 bits or in 8, and clipping by the global norm.

The step that the learned optimizers are compared with, and that a model can be trained with before or after them: the
update and the state keys (``step``, ``exp_avg``, ``exp_avg_sq``) of ``torch.optim.AdamW``, whose checkpoints load.
Parameters are fp32, bf16 or fp16, those of 16 bits with or without an fp32 copy in the state (``master_weights``).

A step is one native call and one launch over the tensors of all param groups (one per combination of types and two hundred
tensors); where gradients are clipped by their global norm, one more before it per type of theirs, and one where there are many.
Nothing of it waits for the device.
"""

from __future__ import annotations

import ctypes as C
import math
from array import array
from collections import OrderedDict
from itertools import chain
from operator import attrgetter, is_

import numpy as np
import torch
from torch.optim import Optimizer

from .. import _lib as L
from ..plan import current_stream_ptr, with_gradients
from ._common import optimizer_step

# for map(): a loop of Python's own is a large part of a small model's step
_numel, _data_ptr, _is_contiguous, _get_device = torch.Tensor.numel, torch.Tensor.data_ptr, torch.Tensor.is_contiguous, torch.Tensor.get_device
_dtype, _grad = attrgetter("dtype"), attrgetter("grad")

TYPES = {torch.float32: L.FP32, torch.bfloat16: L.BF16, torch.float16: L.FP16}
_STATES = ("step", "master", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_root", "exp_avg_sq_root_scale")
_CODES, _SCALES = torch.float8_e4m3fn, torch.float8_e8m0fnu


def blocks_of(n: int) -> int:
    return -(-n // L.ADAMW_BLOCK)


def to_blocks(x: torch.Tensor, least: int = 0):
    """(codes, scales) of the 8-bit states for the values of a tensor: e4m3 codes of its shape, rounded to nearest, and a power of
    two for every 256 of its elements that brings the largest magnitude into [128, 256).  ``least = 1``, for roots: one that is not
    zero gets the smallest code at least, as a step gives it (a moment over a root of zero would be divided by eps alone)."""
    flat = x.detach().to(torch.float32).contiguous().view(-1)
    n = flat.numel()
    b = torch.zeros(blocks_of(n) * L.ADAMW_BLOCK, dtype=torch.float32, device=x.device)
    b[:n] = flat
    b = b.view(-1, L.ADAMW_BLOCK)
    finite = torch.where(b.isfinite(), b, 0.0)
    most = finite.abs().amax(1) if len(b) else b.new_zeros(0)
    scale = ((most.view(torch.int32) >> 23).clamp(min=8) - 7)
    codes = (finite / (scale << 23).view(torch.float32)[:, None]).to(_CODES).view(torch.uint8)
    if least:
        codes = torch.where(finite > 0, codes.clamp(min=least), codes)
    codes = torch.where(b.isfinite(), codes, 0x7F).view(_CODES)
    return codes.view(-1)[:n].view(x.shape), scale.to(torch.uint8).view(_SCALES)


def from_blocks(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The fp32 values that codes and scales of an 8-bit state stand for."""
    each = scales.to(torch.float32).repeat_interleave(L.ADAMW_BLOCK)[: codes.numel()]
    return codes.to(torch.float32) * each.view(codes.shape)


def _gradient(g: torch.Tensor, p_dtype) -> torch.Tensor:
    """``g`` as the kernels take it beside parameters of a type: itself, or a copy."""
    if not (g.dtype is p_dtype or g.dtype is torch.float32 or (p_dtype is torch.float32 and g.dtype in TYPES)):
        g = g.detach().to(torch.float32)
    return g.contiguous()


class _Kept:
    """A state tensor on its way through ``Optimizer.load_state_dict``, which gives every tensor the parameter's type."""

    def __init__(self, value):
        self.value = value


class _Plan:
    """The host's table of a set of tensors, and what of it the last step has seen."""

    def __init__(self, params, group_of, flags, state, bits):
        self.device = params[0].device if params else torch.device("cuda", torch.cuda.current_device())
        self.at = params[0].get_device() if params else -1
        self.p_ptrs, self.numels, self.p_dtypes = [p.data_ptr() for p in params], [p.numel() for p in params], [p.dtype for p in params]
        self.group_of, self.flags = group_of, flags
        # the table holds the addresses of these tensors: they stay alive with it, and it is good for them only
        self.params, self.every_state = params, list(state.values())
        self.states = states = [state[p] for p in params]
        self.values = list(chain.from_iterable(map(dict.values, states)))
        self.tensors = [st[name] for st in states for name in _STATES if name in st]   # a state may hold other things too
        self.state_ptrs = list(map(_data_ptr, self.tensors))
        self.matrices = [x for x in self.tensors if x.dim() > 1]   # whose strides can change and nothing else
        self.table = t = np.zeros(len(params), dtype=L.ADAMW_DTYPE)
        t["p"], t["n"], t["p_type"] = self.p_ptrs, self.numels, [TYPES[d] for d in self.p_dtypes]
        ptr = lambda name: [st[name].data_ptr() if name in st else 0 for st in states]
        t["master"], t["m"] = ptr("master"), ptr("exp_avg")
        t["v"] = ptr("exp_avg_sq" if bits == 32 else "exp_avg_sq_root")
        t["m_scale"], t["v_scale"] = ptr("exp_avg_scale"), ptr("exp_avg_sq_root_scale")
        t["step_dev"] = [st["step"].data_ptr() if st["step"].is_cuda else 0 for st in states]
        t["step"] = [0 if st["step"].is_cuda else st["step"].data_ptr() for st in states]
        t["set"] = group_of
        self.g_ptrs, self.g_dtypes = None, None
        self.call = L.AdamwCall(items=t.ctypes.data, n_items=len(params), bits=bits, norm_floats=L.norm_floats(len(params), sum(self.numels)))
        self.call_ref = C.byref(self.call)
        self.sets, self.set_key, self.norm, self.norm_stream = None, None, None, None

    def good_for(self, params, group_of, flags, state):
        """Whether the table says where everything is.  A tensor's memory can be exchanged under the same object (``x.data = y``, ``x.set_(y)``,
        ``x.share_memory_()``), so that objects and addresses are both looked at."""
        if not (len(params) == len(self.params) and all(map(is_, params, self.params)) and list(map(_data_ptr, params)) == self.p_ptrs
                and list(map(_numel, params)) == self.numels and list(map(_dtype, params)) == self.p_dtypes and all(map(_is_contiguous, params))
                and group_of == self.group_of
                and flags == self.flags and len(state) == len(self.every_state) and all(map(is_, state.values(), self.every_state))):
            return False
        values = list(chain.from_iterable(map(dict.values, self.states)))
        return (len(values) == len(self.values) and all(map(is_, values, self.values)) and list(map(_data_ptr, self.tensors)) == self.state_ptrs
                and all(map(_is_contiguous, self.matrices)))

    def look_at(self, grads, name):
        """Put the gradients' addresses and types into the table; returns the copies that stand in for some of them."""
        try:
            ptrs = list(map(_data_ptr, grads))
        except RuntimeError:
            if any(g.is_sparse for g in grads):
                raise RuntimeError("Sparse gradients not supported") from None
            raise
        copies = ()
        dtypes = list(map(_dtype, grads))
        if dtypes != self.g_dtypes or not all(map(_is_contiguous, grads)):
            copies = [_gradient(g, d) for g, d in zip(grads, self.p_dtypes)]
            ptrs = [g.data_ptr() for g in copies]
            self.table["g_type"] = [TYPES[g.dtype] for g in copies]
            self.g_dtypes = dtypes if all([c is g for c, g in zip(copies, grads)]) else None
        if ptrs != self.g_ptrs:
            # no gradient of another device or size can be assigned to a parameter, but either's memory can be exchanged
            if set(map(_get_device, grads)) - {self.at}:
                raise RuntimeError(f"{name}: all gradients must live on {self.device}")
            if list(map(_numel, grads)) != self.numels:
                shapes = next((tuple(g.shape), tuple(p.shape)) for g, p in zip(grads, self.params) if g.numel() != p.numel())
                raise RuntimeError(f"{name}: a gradient has shape {shapes[0]}, its parameter {shapes[1]}")
            self.table["g"] = ptrs
            self.g_ptrs = ptrs
        return copies


class _AdamWFamily(Optimizer):
    _bits = 32

    def _setup(self, params, **defaults):
        if not torch.cuda.is_available():
            raise RuntimeError(f"{self._name} requires a CUDA device.")
        self._check(defaults)
        super().__init__(params, defaults)
        self._reset()
        self.process_group = None   # set (or set _sharded) when the tensors of the model are split over ranks
        self._sharded = False
        self.after_group = None     # optional callable(group index), called once the step's kernels are enqueued
        self.before_group = None    # optional callable(group index), called before them

    def _check(self, group):
        b1, b2 = group["betas"]
        for name, value, fine in (("lr", group["lr"], float(group["lr"]) >= 0), ("betas", group["betas"], 0 <= b1 < 1 and 0 <= b2 < 1),
                                  ("eps", group["eps"], group["eps"] >= 0), ("weight_decay", group["weight_decay"], group["weight_decay"] >= 0),
                                  ("clip_norm", group["clip_norm"], group["clip_norm"] > 0)):
            if not fine:
                raise ValueError(f"{self._name}: invalid {name}: {value}")
        if self._bits == 8 and group["eps"] < 2.0 ** -126:
            raise ValueError(f"{self._name}: eps must be positive, 2^-126 at least (the step's reciprocal takes a smaller one for zero)")
        if group.get("amsgrad"):
            raise ValueError(f"{self._name}: amsgrad is not supported")

    def _reset(self):
        self._plan = None

    # ------------------------------------------------------------------ state
    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        self._check(self.param_groups[-1])
        self._reset()

    def __setstate__(self, state):
        super().__setstate__(state)
        for name in ("process_group", "after_group", "before_group"):
            self.__dict__.setdefault(name, None)
        self.__dict__.setdefault("_sharded", False)
        for group in self.param_groups:
            for name, value in self.defaults.items():   # a checkpoint of torch.optim.AdamW has no entry of some names
                group.setdefault(name, value)
            self._check(group)
        for p, st in self.state.items():
            for name, value in st.items() if isinstance(st, dict) else ():
                if isinstance(value, _Kept):
                    own = torch.is_tensor(p) and name != "step"   # entries of no parameter stay as they are
                    st[name] = value.value.detach().to(p.device if own else value.value.device, copy=True)
        self._reset()

    def load_state_dict(self, state_dict):
        """As ``Optimizer.load_state_dict``, but every state tensor keeps its type (the base class gives it the parameter's).

        States of 32 bits load into the class of 8, rounded to nearest, and the other way round."""
        state_dict = state_dict.copy()
        hooks = self._optimizer_load_state_dict_pre_hooks
        for hook in hooks.values():
            changed = hook(self, state_dict)
            if changed is not None:
                state_dict = changed
        keep = lambda v: _Kept(v) if torch.is_tensor(v) else v
        state_dict["state"] = {k: {n: keep(v) for n, v in st.items()} if isinstance(st, dict) else st for k, st in state_dict["state"].items()}
        self._optimizer_load_state_dict_pre_hooks = OrderedDict()
        try:
            super().load_state_dict(state_dict)
        finally:
            self._optimizer_load_state_dict_pre_hooks = hooks

    def _init_state(self, p, st, group, capturing):
        """Make what a parameter's state lacks, and bring what it has into the form the kernels take.  Not in a capture, which would do it
        again on every replay."""
        dev, n = p.device, p.numel()
        capturable = group["capturable"]

        def changes():
            if capturing:
                raise RuntimeError(f"{self._name}: run a step before the one that is captured: a captured step would make its states anew on every replay")

        step, kind = st.get("step", 0.0), torch.float32 if capturable else torch.float64
        if not torch.is_tensor(step) or step.is_cuda != bool(capturable) or step.dim() != 0 or step.dtype is not kind:
            changes()
            step = torch.tensor(float(step), dtype=kind, device=dev if capturable else "cpu")
        elif capturable and step.device != dev:
            changes()
            step = step.to(dev)
        st["step"] = step
        if self._bits == 32:
            if "exp_avg_sq_root" in st:
                changes()
                st["exp_avg_sq"] = from_blocks(st.pop("exp_avg_sq_root"), st.pop("exp_avg_sq_root_scale")).square_()
                st["exp_avg"] = from_blocks(st["exp_avg"], st.pop("exp_avg_scale"))
            wanted = {"exp_avg": (torch.float32, p.shape), "exp_avg_sq": (torch.float32, p.shape)}
        else:
            if "exp_avg_sq" in st:
                changes()
                st["exp_avg_sq_root"], st["exp_avg_sq_root_scale"] = to_blocks(st.pop("exp_avg_sq").to(torch.float32).sqrt(), least=1)
                st["exp_avg"], st["exp_avg_scale"] = to_blocks(st["exp_avg"])
            each = (blocks_of(n),)
            wanted = {"exp_avg": (_CODES, p.shape), "exp_avg_scale": (_SCALES, each),
                      "exp_avg_sq_root": (_CODES, p.shape), "exp_avg_sq_root_scale": (_SCALES, each)}
        if group["master_weights"] and p.dtype is not torch.float32:
            wanted["master"] = (torch.float32, p.shape)
            if "master" not in st:
                changes()
                st["master"] = p.detach().to(torch.float32).contiguous()
        else:
            st.pop("master", None)
        for name, (dtype, shape) in wanted.items():
            x = st.get(name)
            if x is None:
                changes()
                zero = 1 if dtype is _SCALES else 0   # the least scale there is
                x = torch.full(shape, zero, dtype=torch.uint8, device=dev).view(dtype) if dtype.itemsize == 1 else torch.zeros(shape, dtype=dtype, device=dev)
            if tuple(x.shape) != tuple(shape):
                raise ValueError(f"{self._name}: state {name!r} has shape {tuple(x.shape)}, the parameter's needs {tuple(shape)}")
            if x.dtype is not dtype and (dtype.itemsize == 1 or not x.dtype.is_floating_point):
                raise ValueError(f"{self._name}: state {name!r} is {x.dtype}, not {dtype}")
            y = x.to(device=dev, dtype=dtype).contiguous()
            y = y.clone() if y.data_ptr() % 16 and dtype is not _SCALES else y   # the kernels want all but scales on a boundary
            if y is not x:
                changes()
            st[name] = y

    def _build(self, plist, group_of, flags, capturing):
        dev = plist[0].device if plist else None
        for p in plist:
            if not p.is_cuda:
                raise RuntimeError(f"{self._name}: parameters must live on a CUDA device (there is no CPU path)")
            if p.dtype not in TYPES:
                raise RuntimeError(f"{self._name}: parameters must be fp32, bf16 or fp16, got {p.dtype}")
            if not p.is_contiguous():
                raise RuntimeError(f"{self._name}: parameters must be contiguous")
            if p.device != dev:
                raise RuntimeError(f"{self._name}: all parameters must live on one device, got {dev} and {p.device}")
            if getattr(p, "_pylo_peer_ptrs", None):
                raise RuntimeError(f"{self._name}: writes no other rank's copy of a parameter; use ShardedStep or StagedShardedStep, or push='copies'")
        at = np.array([p.data_ptr() for p in plist if p.numel()], dtype=np.uint64)
        end = at + np.array([p.numel() * p.element_size() for p in plist if p.numel()], dtype=np.uint64)
        order = np.argsort(at)
        if len(at) and np.any(at[order][1:] < end[order][:-1]):
            raise ValueError(f"{self._name}: two parameters share memory")
        for p, gi in zip(plist, group_of):
            self._init_state(p, self.state[p], self.param_groups[gi], capturing)
        return _Plan(plist, group_of, flags, self.state, self._bits)

    # ------------------------------------------------------------------ step
    @optimizer_step
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        groups = self.param_groups
        if self.before_group is not None:
            for gi in range(len(groups)):
                self.before_group(gi)
        plist, grads, group_of = [], [], []
        for gi, group in enumerate(groups):
            ps, gs = with_gradients(group["params"])
            plist += ps
            grads += gs
            group_of += [gi] * len(ps)
        clip = any([g["clip_grad"] and g["clip_norm"] < math.inf for g in groups])
        if plist or clip:
            at = plist[0].get_device() if plist else -1
            if at >= 0 and at != torch._C._cuda_getDevice():
                with torch.cuda.device(at):
                    self._run(plist, grads, group_of, clip)
            else:
                self._run(plist, grads, group_of, clip)
        if self.after_group is not None:
            for gi in range(len(groups)):
                self.after_group(gi)
        return loss

    def _run(self, plist, grads, group_of, clip):
        capturing = torch._C._cuda_isCurrentStreamCapturing()
        flags = [(g["capturable"], g["master_weights"]) for g in self.param_groups]
        if capturing and not all([capturable for capturable, _ in flags]):
            raise RuntimeError(f"{self._name}: a step can be captured into a graph only with capturable=True")
        plan = self._plan
        if plan is None or not plan.good_for(plist, group_of, flags, self.state):
            for p, g in zip(plist, grads):
                if g.shape != p.shape:   # of a parameter whose memory was exchanged since
                    raise RuntimeError(f"{self._name}: a gradient has shape {tuple(g.shape)}, its parameter {tuple(p.shape)}")
            plan = self._plan = self._build(plist, group_of, flags, capturing)
        stream = current_stream_ptr()
        copies = plan.look_at(grads, self._name)
        self._fill_sets(plan)
        phases = L.ADAMW_STEP
        if clip:
            phases = L.ADAMW_NORM | L.ADAMW_STEP
            norm = plan.norm
            # a stream has a buffer of its own, which goes back to that stream's memory; a captured step has one from the graph's
            if norm is None or capturing or stream != plan.norm_stream:
                norm = torch.empty(plan.call.norm_floats, dtype=torch.float32, device=plan.device)
                plan.norm, plan.norm_stream = None if capturing else norm, stream
                plan.call.norm = norm.data_ptr()
            if self.process_group is not None or (self._sharded and torch.distributed.is_initialized()):
                L.check(L.lib.pylo_b200_adamw_step(plan.call_ref, L.ADAMW_NORM, stream), "adamw_step")
                torch.distributed.all_reduce(norm[:1], group=self.process_group)  # each rank holds its own tensors' share
                phases = L.ADAMW_STEP
        code = L.lib.pylo_b200_adamw_step(plan.call_ref, phases, stream)
        if code:
            L.check(code, "adamw_step")
        del copies

    def _fill_sets(self, plan):
        """The hyper-parameters of the step, a set per group."""
        key = [(g["lr"], g["betas"], g["eps"], g["weight_decay"], g["clip_norm"] if g["clip_grad"] else 0.0, g["maximize"], g.get("seed", 0))
               for g in self.param_groups]
        tensors = any([torch.is_tensor(k[0]) for k in key])   # whose value, not the object, is the learning rate: looked at anew in every step
        if not tensors and plan.set_key == key:
            return
        plan.sets = (L.AdamwSet * len(key))()
        for s, group, (lr, (b1, b2), eps, wd, clip_norm, maximize, seed) in zip(plan.sets, self.param_groups, key):
            if torch.is_tensor(lr) and lr.is_cuda and group["capturable"]:
                if lr.dtype is not torch.float32 or lr.numel() != 1 or lr.device != plan.device:
                    raise ValueError(f"{self._name}: lr on the device must be one fp32 value on {plan.device}")
                s.lr_dev, lr = lr.data_ptr(), 0.0
            s.lr, s.weight_decay, s.beta1, s.beta2, s.eps, s.clip_norm = float(lr), wd, b1, b2, eps, clip_norm
            s.maximize, s.seed = bool(maximize), seed & 0xFFFFFFFF
        plan.call.sets, plan.call.n_sets = plan.sets, len(key)
        plan.set_key = None if tensors else key


class AdamW_CUDA(_AdamWFamily):
    """AdamW with fp32 moments.

    ``master_weights``: the state of a bf16 or fp16 parameter holds an fp32 copy (``master``), made from it in its first step,
    which the steps update; the parameter is its rounded value.  ``clip_grad``, ``clip_norm``: gradients are scaled by
    ``clip_norm / max(norm, clip_norm)`` within the step, with the norm over the gradients of all groups (they are left as
    they are in memory; ``clip_norm = inf`` clips nothing).  ``capturable``: the step count lives on the device, as may ``lr``, and a step can be captured into a graph."""

    _name = "AdamW_CUDA"

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, maximize=False, master_weights=False,
                 clip_grad=False, clip_norm=1.0, capturable=False):
        self._setup(params, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, maximize=maximize, master_weights=master_weights,
                    clip_grad=clip_grad, clip_norm=clip_norm, capturable=capturable)


class AdamW8bit_CUDA(_AdamWFamily):
    """AdamW with moments in 8 bits: 2 bytes and a sixty-fourth per parameter.

    The first moment (``exp_avg``) and the root of the second (``exp_avg_sq_root``) are ``float8_e4m3fn`` codes; 256 elements of
    a tensor share a power of two (``exp_avg_scale``, ``exp_avg_sq_root_scale``, ``float8_e8m0fnu``); a value is code times scale.
    Codes are rounded up or down at random, so that they are right on the average: the same ``seed``, step and gradients give the same
    codes, however the tensors are grouped or split over ranks.  Other arguments as :class:`AdamW_CUDA`."""

    _name = "AdamW8bit_CUDA"
    _bits = 8

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, maximize=False, master_weights=False,
                 clip_grad=False, clip_norm=1.0, capturable=False, seed=0):
        self._setup(params, lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, maximize=maximize, master_weights=master_weights,
                    clip_grad=clip_grad, clip_norm=clip_norm, capturable=capturable, seed=int(seed))


# ---------------------------------------------------------------------------------------------------------------------
# clipping by the global norm
# ---------------------------------------------------------------------------------------------------------------------
def _dense(g: torch.Tensor) -> bool:
    """Whether the elements of a tensor are one run of memory, in whatever order."""
    step = 1
    for stride, size in sorted((st, sz) for st, sz in zip(g.stride(), g.shape) if sz != 1):
        if stride != step:
            return False
        step *= size
    return True


def _as_runs(grads, scaled):
    """The gradients as runs of memory: themselves, or copies, one for all that are the same elements."""
    copies, parts = {}, []
    for g in grads:
        if not (g.is_contiguous() or _dense(g)):
            if scaled and any([stride == 0 and n > 1 for stride, n in zip(g.stride(), g.shape)]):
                raise RuntimeError(f"clip_grad_norm_: a gradient's elements share memory (shape {tuple(g.shape)}, strides {g.stride()})")
            same = (g.data_ptr(), g.dtype, g.shape, g.stride())
            if same not in copies:
                copies[same] = g.detach().contiguous()
            g = copies[same]
        parts.append(g)
    return parts


def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False) -> torch.Tensor:
    """Scale the gradients of ``parameters`` in place by ``min(1, max_norm / (norm + 1e-6))``, ``norm`` the 2-norm of all of them
    together; returns ``norm`` (fp32, on the device), as ``torch.nn.utils.clip_grad_norm_`` does.

    Gradients may be fp32, bf16 and fp16, mixed; the norm is summed up in fp32 and more whatever their type.  One that is given twice
    counts and is scaled once.  A launch for the norm and one for the scaling per type and 800 gradients, one between them where there are
    many partial sums; no synchronisation (``error_if_nonfinite`` waits for the norm).  The gradients are written only where the norm
    exceeds ``max_norm``."""
    if float(norm_type) != 2.0:
        raise ValueError(f"clip_grad_norm_: only the 2-norm is supported, got norm_type={norm_type}")
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f"clip_grad_norm_: invalid max_norm: {max_norm}")
    grads = [g for g in map(_grad, [parameters] if torch.is_tensor(parameters) else parameters) if g is not None]
    if not grads:
        return torch.tensor(0.0)
    at = grads[0].get_device()
    if at < 0:
        raise RuntimeError("clip_grad_norm_: gradients must live on a CUDA device (there is no CPU path)")
    if set(map(_get_device, grads)) != {at}:
        raise RuntimeError("clip_grad_norm_: all gradients must live on one device")
    dtypes = list(map(_dtype, grads))
    if not TYPES.keys() >= set(dtypes):
        raise RuntimeError(f"clip_grad_norm_: gradients must be fp32, bf16 or fp16, got {next(d for d in dtypes if d not in TYPES)}")
    types = array("i", map(TYPES.__getitem__, dtypes))
    if at != torch._C._cuda_getDevice():
        with torch.cuda.device(at):
            return _clip(grads, types, max_norm, error_if_nonfinite)
    return _clip(grads, types, max_norm, error_if_nonfinite)


def _clip(grads, types, max_norm, error_if_nonfinite):
    parts = grads
    try:
        if not all(map(_is_contiguous, grads)):
            parts = _as_runs(grads, max_norm < math.inf)
        ptrs = array("Q", map(_data_ptr, parts))
    except RuntimeError:
        if any([g.layout is not torch.strided for g in grads]):
            raise RuntimeError("Sparse gradients not supported") from None
        raise
    sizes = array("q", map(_numel, parts))
    stream = current_stream_ptr()
    floats = L.norm_floats(len(ptrs), sum(sizes))
    device = grads[0].device
    total = torch.empty_strided((), (), dtype=torch.float32, device=device)   # by itself: who keeps it keeps no workspace
    norm = torch.empty(floats, dtype=torch.float32, device=device)
    to, at = total.data_ptr(), norm.data_ptr()

    def run(limit, distinct):
        return L.lib.pylo_b200_clip_grads_to(ptrs.buffer_info()[0], sizes.buffer_info()[0], types.buffer_info()[0], len(ptrs), limit, to, at, floats, distinct,
                                             stream)

    limit = math.inf if error_if_nonfinite else max_norm   # the norm is looked at before anything is scaled
    code, distinct = run(limit, 0), 0
    if code == L.ERR_GRADS_OVERLAP:
        ptrs, sizes, types = (array(kind, x) for kind, x in zip("Qqi", _distinct(ptrs, sizes, types)))
        code, distinct = run(limit, 1), 1
    if code:
        L.check(code, "clip_grads")
    if error_if_nonfinite:
        if not math.isfinite(float(total)):
            raise RuntimeError("The total norm of order 2.0 for gradients from `parameters` is non-finite, so it cannot be clipped. To disable this "
                               "error and scale the gradients by the non-finite norm anyway, set `error_if_nonfinite=False`")
        if max_norm < math.inf:
            L.check(run(max_norm, distinct), "clip_grads")
    if parts is not grads and max_norm < math.inf:
        with torch.no_grad():
            for g, part in zip(grads, parts):
                if part is not g:
                    g.copy_(part)
    return total


def _distinct(ptrs, sizes, types):
    """Every gradient once, in the order given; two that share only a part of their memory are refused."""
    g, n, t = np.array(ptrs, dtype=np.uint64), np.array(sizes, dtype=np.uint64), np.array(types, dtype=np.int64)
    order = np.argsort(g, kind="stable")
    order = order[n[order] > 0]
    first, end = g[order], (g + n * np.array([4, 2, 2], dtype=np.uint64)[t])[order]
    over = first[1:] < end[:-1]
    twice = over & (first[1:] == first[:-1]) & (end[1:] == end[:-1]) & (t[order][1:] == t[order][:-1])
    if (over & ~twice).any():
        raise ValueError("clip_grad_norm_: two gradients share a part of their memory")
    keep = np.sort(order[np.concatenate([[True], ~twice])]) if len(order) else order
    return g[keep].tolist(), n[keep].tolist(), t[keep].tolist()

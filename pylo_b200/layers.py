"""What a model's training step needs beside the optimizer, where the gradients come from: layer norm, the gated feed-forward block and the
loss of a distillation from a teacher's largest logits, each with its gradients.

Functions that autograd differentiates once, backward (a forward-mode derivative is refused), and modules that hold their parameters.  They take
CUDA tensors of fp32, bf16 or fp16 (the feed-forward block: bf16 or fp16), run on the current stream of the tensors' device, wait for nothing, and
leave their arguments as they are.  A call can be captured into a CUDA graph, forward and backward, ``gated_ffn`` after one that is not; as with any
other operator, no result of an earlier pass over the same parameters may be alive when a backward pass is captured (autograd would make the capture
wait for that pass's stream).
"""

from __future__ import annotations

import ctypes as C
import math
import threading

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib as L

TYPES = {torch.float32: L.FP32, torch.bfloat16: L.BF16, torch.float16: L.FP16}
ACTIVATIONS = {"silu": L.ACT_SILU, "gelu": L.ACT_GELU, "gelu_tanh": L.ACT_GELU_TANH, "relu": L.ACT_RELU}
REDUCTIONS = {"none": L.REDUCE_NONE, "sum": L.REDUCE_SUM, "mean": L.REDUCE_MEAN}

_Tensor = torch.Tensor
_device_now, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
_sizes = {}   # what the library says of a call's workspace


def _call(function, what, device, *args):
    """A function of the library on the current stream of a device (its number)."""
    if device == _device_now():
        code = function(*args, _raw_stream(device))
    else:
        with torch.cuda.device(device):
            code = function(*args, _raw_stream(device))
    if code:
        L.check(code, what)


def _size(name, device, *args):
    """What a function of the library that asks the current device says for ``device``."""
    key = (name, device, args)
    size = _sizes.get(key)
    if size is None:
        with torch.cuda.device(device):
            size = getattr(L.lib, name)(*args)
        if len(_sizes) > 4096:
            _sizes.clear()
        _sizes[key] = size
    return size


def _check(name, t, device=None, types=TYPES):
    if isinstance(t, _Tensor) and t.is_cuda and (device is None or t.get_device() == device) and t.dtype in types:
        return
    if not isinstance(t, _Tensor):
        raise TypeError(f"{name} has to be a tensor, got {type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"{name} has to be a CUDA tensor, it is on {t.device}")
    if device is not None and t.get_device() != device:
        raise ValueError(f"{name} is on {t.device}, not on cuda:{device}")
    raise TypeError(f"{name} is {t.dtype}, supported are {', '.join(str(d).split('.')[1] for d in types)}")


def _rows(t):
    """A tensor as rows of its last dimension, whose elements follow one another: a view where there is one, else a copy."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 else t.contiguous()


def _like(t):
    """An uninitialised contiguous tensor of the shape, type and device of ``t``."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty_like(t, memory_format=torch.contiguous_format)


def _graph(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


def _refuse_tangents(*tensors):
    """Inside of a forward-mode level: what a kernel makes of a tensor's values has no tangent, so that a derivative would be lost."""
    for t in tensors:
        if isinstance(t, _Tensor) and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError("forward-mode derivatives are not supported, only backward ones")


def _once(backward):
    """``once_differentiable``, whose contexts a plain backward pass does without."""
    guarded = once_differentiable(backward)

    def run(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return run


# ---------------------------------------------------------------------------------------------------------------------
# layer norm
# ---------------------------------------------------------------------------------------------------------------------


def _norm_forward(x, weight, bias, eps, keep):
    n, width = x.shape
    y = _like(x)
    stat = torch.empty(2 * n, dtype=torch.float32, device=x.device) if keep else None   # means, 1 / deviations
    if n:
        mean = stat.data_ptr() if keep else None
        kind = TYPES[x.dtype]
        w = L.Norm(x=x.data_ptr(), weight=None if weight is None else weight.data_ptr(), bias=None if bias is None else bias.data_ptr(), y=y.data_ptr(),
                   mean=mean, rstd=mean + 4 * n if keep else None, rows=n, x_stride=x.stride(0), width=width, type=kind,
                   weight_type=kind if weight is None else TYPES[weight.dtype], eps=eps)
        _call(L.lib.pylo_b200_layer_norm, "layer_norm", x.get_device(), C.byref(w))
    return y, stat


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weight, bias, eps):
        y, stat = _norm_forward(rows, weight, bias, eps, True)
        ctx.save_for_backward(rows, weight, stat)
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        rows, weight, stat = ctx.saved_tensors
        if rows.stride(1) != 1 or not stat.is_contiguous():   # hooks have laid them out anew
            rows, stat = _rows(rows), stat.contiguous()
        n, width = rows.shape
        device = rows.get_device()
        dy = _rows(dy)
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        dx = _like(rows) if need_x else None
        dw = torch.empty_like(weight) if need_w else None
        db = torch.empty_like(weight) if need_b else None
        kind, mean = TYPES[rows.dtype], stat.data_ptr()
        w = L.Norm(x=rows.data_ptr(), dy=dy.data_ptr(), weight=None if weight is None else weight.data_ptr(), mean=mean, rstd=mean + 4 * n,
                   dx=dx.data_ptr() if need_x else None, dweight=dw.data_ptr() if need_w else None, dbias=db.data_ptr() if need_b else None, rows=n,
                   x_stride=rows.stride(0), dy_stride=dy.stride(0), width=width, type=kind, weight_type=kind if weight is None else TYPES[weight.dtype])
        if need_w or need_b:
            size = _size("pylo_b200_layer_norm_workspace", device, n, width)
            work = torch.empty(size, dtype=torch.float32, device=rows.device)
            w.work, w.work_floats = work.data_ptr(), size
        elif not n:
            return dx, dw, db, None
        _call(L.lib.pylo_b200_layer_norm_backward, "layer_norm backward", device, C.byref(w))
        return dx, dw, db, None


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, eps: float = 1e-5) -> torch.Tensor:
    """Layer norm over the last dimension: ``(x - mean) / sqrt(variance + eps) * weight + bias``, of ``x``'s type.

    ``weight`` and ``bias`` are vectors of ``x``'s type or fp32, and their gradients are of that type; a bias needs a weight beside it.  Means,
    variances and the sums of the gradients are fp32, each result is rounded once.  Rows of up to 16384 elements, of any stride."""
    if forward_ad._current_level >= 0:
        _refuse_tangents(x, weight, bias)
    _check("x", x)
    dim, device, dtype = x.dim(), x.get_device(), x.dtype
    width = x.shape[-1] if dim else 0
    if not 1 <= width <= L.NORM_MOST:
        raise ValueError(f"x has to have rows of 1 to {L.NORM_MOST} elements, its shape is {tuple(x.shape)}")
    if not (isinstance(eps, (int, float)) and 0.0 <= eps < math.inf):
        raise ValueError(f"eps has to be a finite number >= 0, got {eps!r}")
    if weight is not None:
        _check("weight", weight, device, (dtype, torch.float32))
        if weight.shape != (width,):
            raise ValueError(f"weight has the shape {tuple(weight.shape)}, x has rows of {width} elements")
        if not weight.is_contiguous():
            weight = weight.contiguous()
    if bias is not None:
        if weight is None:
            raise ValueError("a bias needs a weight beside it")
        _check("bias", bias, device, (weight.dtype,))
        if bias.shape != (width,):
            raise ValueError(f"bias has the shape {tuple(bias.shape)}, x has rows of {width} elements")
        if not bias.is_contiguous():
            bias = bias.contiguous()
    rows = _rows(x)
    y = _LayerNorm.apply(rows, weight, bias, float(eps)) if _graph(x, weight, bias) else _norm_forward(rows, weight, bias, float(eps), False)[0]
    return y if dim == 2 else y.view(x.shape)


class LayerNorm(torch.nn.Module):
    """:func:`layer_norm` with its parameters, as ``torch.nn.LayerNorm`` over the last dimension."""

    def __init__(self, width: int, eps: float = 1e-5, bias: bool = True, device=None, dtype=None):
        super().__init__()
        self.eps = eps
        self.weight = torch.nn.Parameter(torch.ones(width, device=device, dtype=dtype))
        self.bias = torch.nn.Parameter(torch.zeros(width, device=device, dtype=dtype)) if bias else None

    def forward(self, x):
        return layer_norm(x, self.weight, self.bias, self.eps)

    def extra_repr(self):
        return f"{self.weight.numel()}, eps={self.eps}, bias={self.bias is not None}"


# ---------------------------------------------------------------------------------------------------------------------
# the gated feed-forward block
# ---------------------------------------------------------------------------------------------------------------------

_reported = None   # a word in pinned memory that a kernel sets when one of its waits ran out: kernels hold its address, so it is made once for good
_reported_lock = threading.Lock()


def _pinned_word():
    return torch.zeros(1, dtype=torch.int32).pin_memory()


def _status_word():
    global _reported
    if _reported is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("gated_ffn has to run once before it is captured into a CUDA graph")
        with _reported_lock:
            if _reported is None:
                word = _pinned_word()
                _reported = (word, word.numpy(), word.data_ptr())
    if _reported[1][0]:
        raise L.PyloLibError("gated_ffn: a wait in a kernel of an earlier call ran out, its results are incomplete (clear_status() to go on)")
    return _reported[2]


def check_status():
    """Waits for the current device and raises if a kernel of an earlier :func:`gated_ffn` reported a wait that ran out.  Without it, the
    next call does."""
    torch.cuda.synchronize()
    if _reported is not None:
        _status_word()


def clear_status():
    """Forget what :func:`check_status` raises for."""
    if _reported is not None:
        torch.cuda.synchronize()
        _reported[1][0] = 0


def _spacing(t):
    """Elements between the rows of a matrix that lies as the copies to the tensor cores need it, on 16-byte boundaries; else 0."""
    rows, cols = t.shape
    if t.data_ptr() % 16 == 0:
        if cols % 8 == 0 and t.is_contiguous():
            return cols
        apart, beside = t.stride()
        if beside == 1:
            if rows == 1:
                return -(-cols // 8) * 8
            if apart % 8 == 0 and apart >= cols:
                return apart
    return 0


class _Operands:
    """Matrices as the block's products take them: those that do not lie as they should are copied, all in one launch."""

    def __init__(self, tensors):
        self.apart = apart = list(map(_spacing, tensors))   # elements between rows
        self.room, self.at = None, None                     # the copies, and where in them (bytes) each matrix is, or -1
        if 0 not in apart:
            return
        first = tensors[0]
        odd = [k for k, n in enumerate(apart) if not n]
        items, self.at, size = (L.Pad * len(odd))(), [-1] * len(tensors), 0
        for k in odd:
            rows, cols = tensors[k].shape
            apart[k] = ld = -(-cols // 8) * 8
            self.at[k] = size
            size += 2 * ld * rows
        self.room = torch.empty(size, dtype=torch.uint8, device=first.device)
        base = self.room.data_ptr()
        for item, k in zip(items, odd):
            t = tensors[k]
            item.src, item.dst = t.data_ptr(), base + self.at[k]
            item.rows, item.cols = t.shape
            item.row_stride, item.col_stride = t.stride()
            item.ld = apart[k]
        _call(L.lib.pylo_b200_pad_rows, "gated_ffn", first.get_device(), items, len(odd))

    def pointers(self, tensors):
        if self.room is None:
            return [t.data_ptr() for t in tensors]
        base = self.room.data_ptr()
        return [t.data_ptr() if at < 0 else base + at for t, at in zip(tensors, self.at)]

    def again(self, tensors, room):
        """((address, elements between rows) of each operand, what holds them) of a backward pass: the forward pass's copies, ``room``, and the other matrices
        as autograd hands them back.  Its hooks may have laid those out anew (a slice that was offloaded comes back without its gaps), so how they lie is
        looked up again."""
        if room is None:
            lies = _Operands(tensors)
            return list(zip(lies.pointers(tensors), lies.apart)), lies
        base, operands, held = room.data_ptr(), [], []
        for t, at, apart in zip(tensors, self.at, self.apart):
            if at >= 0:
                operands.append((base + at, apart))
                continue
            lies = _Operands((t,))
            held.append(lies)
            operands.append((*lies.pointers((t,)), *lies.apart))
        return operands, held


def _ffn_struct(tensors, operands, activation):
    """operands: the tensors' addresses, and elements between their rows"""
    (x, ld_x), (w_gate, ld_gate), (w_up, ld_up), (w_down, ld_down) = operands
    (rows, width), (out, hidden) = tensors[0].shape, tensors[3].shape
    return L.Ffn(x=x, w_gate=w_gate, w_up=w_up, w_down=w_down, rows=rows, ld_x=ld_x, ld_gate=ld_gate, ld_up=ld_up, ld_down=ld_down, width=width,
                 hidden=hidden, out=out, type=TYPES[tensors[0].dtype], activation=activation, host_status=_status_word())


def _ffn_forward(tensors, activation, keep):
    """(y, how the operands lie, what is kept for the backward pass)"""
    rows = tensors[0]
    y = torch.empty((rows.shape[0], tensors[3].shape[0]), dtype=rows.dtype, device=rows.device)
    if not rows.shape[0]:
        return y, None, None
    device = rows.get_device()
    operands = _Operands(tensors)
    f = _ffn_struct(tensors, zip(operands.pointers(tensors), operands.apart), activation)
    kept = torch.empty(_size("pylo_b200_gated_ffn_kept", device, f.rows, f.hidden, keep), dtype=torch.uint8, device=rows.device)
    f.y, f.kept, f.keep = y.data_ptr(), kept.data_ptr(), keep
    _call(L.lib.pylo_b200_gated_ffn, "gated_ffn", device, C.byref(f))
    return y, operands, kept


class _GatedFFN(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, w_gate, w_up, w_down, activation):
        y, operands, kept = _ffn_forward((rows, w_gate, w_up, w_down), activation, 1)
        ctx.save_for_backward(rows, w_gate, w_up, w_down, kept, operands and operands.room)
        if operands:
            operands.room = None   # (it is saved)
        ctx.operands, ctx.activation = operands, activation
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        *tensors, kept, room = ctx.saved_tensors
        rows = tensors[0]
        make = _like if kept is not None else lambda t: torch.zeros(t.shape, dtype=t.dtype, device=t.device)
        grads = [make(t) if wanted else None for wanted, t in zip(ctx.needs_input_grad, tensors)]
        if kept is not None:
            device = rows.get_device()
            dy = _rows(dy)
            lies = _Operands((dy,))
            operands, held = ctx.operands.again(tensors, room)
            f = _ffn_struct(tensors, operands, ctx.activation)
            work = torch.empty(_size("pylo_b200_gated_ffn_workspace", device, f.rows, f.hidden), dtype=torch.uint8, device=rows.device)
            (f.dy,), (f.ld_dy,), f.kept, f.work = lies.pointers((dy,)), lies.apart, kept.data_ptr(), work.data_ptr()
            f.dx, f.dw_gate, f.dw_up, f.dw_down = (None if g is None else g.data_ptr() for g in grads)
            _call(L.lib.pylo_b200_gated_ffn_backward, "gated_ffn backward", device, C.byref(f))
        return *grads, None


def gated_ffn(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, w_down: torch.Tensor, activation: str = "silu") -> torch.Tensor:
    """The gated feed-forward block ``(act(x @ w_gate.T) * (x @ w_up.T)) @ w_down.T``.

    ``x`` is ``[..., width]``, ``w_gate`` and ``w_up`` are ``[hidden, width]``, ``w_down`` is ``[out, hidden]``; all are bf16 or all fp16.
    ``activation``: ``"silu"``, ``"gelu"`` (with the error function), ``"gelu_tanh"`` or ``"relu"``.  Sums are fp32; the hidden values, and backward
    their gradients, are rounded to the type once, where they become operands of the next product (up to 16 rows: to two numbers of the type each).  In
    fp16 one beyond 65504 is infinite.  Sizes and strides are free; matrices whose rows do not begin on 16-byte boundaries are copied first (the copies
    are kept for the backward pass).  For a backward pass 8 bytes are kept per hidden value: the value, and the activation and its slope times the other
    projection in 24 bits each (more than 32 rows are counted in 32s; up to 16 rows take 32 bytes more per column)."""
    code = ACTIVATIONS.get(activation)
    if code is None:
        raise ValueError(f"activation is {activation!r}, supported are {', '.join(ACTIVATIONS)}")
    if forward_ad._current_level >= 0:
        _refuse_tangents(x, w_gate, w_up, w_down)
    _check("x", x, types=(torch.bfloat16, torch.float16))
    for name, t in (("w_gate", w_gate), ("w_up", w_up), ("w_down", w_down)):
        _check(name, t, x.get_device(), (x.dtype,))
        if t.dim() != 2:
            raise ValueError(f"{name} has to be a matrix, got the shape {tuple(t.shape)}")
    if x.dim() == 0 or w_gate.shape != w_up.shape or w_gate.shape[1] != x.shape[-1] or w_down.shape[1] != w_gate.shape[0]:
        raise ValueError(f"the shapes do not fit together: x {tuple(x.shape)}, w_gate {tuple(w_gate.shape)}, w_up {tuple(w_up.shape)}, w_down {tuple(w_down.shape)}")
    if min(*w_gate.shape, *w_down.shape) == 0 or max(*w_gate.shape, *w_down.shape) > 1 << 24 or math.prod(x.shape[:-1]) > 1 << 30:
        raise ValueError("sizes from 1 to 2^24 and up to 2^30 rows are supported")
    rows = _rows(x)
    y = _GatedFFN.apply(rows, w_gate, w_up, w_down, code) if _graph(x, w_gate, w_up, w_down) else _ffn_forward((rows, w_gate, w_up, w_down), code, 0)[0]
    return y if x.dim() == 2 else y.view(*x.shape[:-1], y.shape[1])


class GatedFFN(torch.nn.Module):
    """:func:`gated_ffn` with its parameters, initialised as ``torch.nn.Linear`` without biases."""

    def __init__(self, width: int, hidden: int, out: int | None = None, activation: str = "silu", device=None, dtype=torch.bfloat16):
        super().__init__()
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation is {activation!r}, supported are {', '.join(ACTIVATIONS)}")
        self.activation = activation
        make = lambda rows, cols: torch.nn.Parameter(torch.empty(rows, cols, device=device, dtype=dtype).uniform_(-cols ** -0.5, cols ** -0.5))
        self.w_gate, self.w_up, self.w_down = make(hidden, width), make(hidden, width), make(width if out is None else out, hidden)

    def forward(self, x):
        return gated_ffn(x, self.w_gate, self.w_up, self.w_down, self.activation)

    def extra_repr(self):
        return f"{self.w_gate.shape[1]}, {self.w_gate.shape[0]}, out={self.w_down.shape[0]}, activation={self.activation!r}"


# ---------------------------------------------------------------------------------------------------------------------
# distillation from a teacher's largest logits
# ---------------------------------------------------------------------------------------------------------------------


def _distill_arguments(logits, teacher_logits, teacher_ids, temperature, weights, reduction):
    """Checked arguments: (logits' rows, teacher, ids, weights, code of the reduction)."""
    if forward_ad._current_level >= 0:
        _refuse_tangents(logits, teacher_logits, weights)
    _check("logits", logits)
    device = logits.get_device()
    _check("teacher_logits", teacher_logits, device)
    _check("teacher_ids", teacher_ids, device, (torch.int64, torch.int32))
    if reduction not in REDUCTIONS:
        raise ValueError(f"reduction is {reduction!r}, supported are {', '.join(REDUCTIONS)}")
    if not (isinstance(temperature, (int, float)) and 2.0 ** -60 <= temperature <= 2.0 ** 60):
        raise ValueError(f"temperature has to be a positive number from 2^-60 to 2^60, got {temperature!r}")
    if logits.dim() == 0 or not 1 <= logits.shape[-1] <= 1 << 30:
        raise ValueError("logits need a last dimension of 1 to 2^30 classes")
    lead = logits.shape[:-1]
    if teacher_logits.dim() == 0 or teacher_logits.shape != teacher_ids.shape or teacher_logits.shape[:-1] != lead:
        raise ValueError(f"teacher_logits {tuple(teacher_logits.shape)} and teacher_ids {tuple(teacher_ids.shape)} have to be alike and to begin as logits do, {tuple(lead)}")
    if not 1 <= teacher_logits.shape[-1] <= L.DISTILL_MOST_TOP:
        raise ValueError(f"a teacher gives 1 to {L.DISTILL_MOST_TOP} entries, got {teacher_logits.shape[-1]}")
    if weights is not None:
        _check("weights", weights, device, (*TYPES, torch.bool))
        if weights.shape != lead:
            raise ValueError(f"weights have the shape {tuple(weights.shape)}, the rows of logits {tuple(lead)}")
    if torch.is_grad_enabled() and (teacher_logits.requires_grad or (weights is not None and weights.requires_grad)):
        raise ValueError("teacher_logits and weights are constants here: detach them")
    rows = _rows(logits.detach())
    if rows.shape[0] > 1 and rows.stride(0) < rows.shape[1]:
        rows = rows.contiguous()
    if weights is not None and not (weights.dtype is torch.float32 and weights.is_contiguous()):
        weights = weights.detach().to(torch.float32).contiguous()
    return rows, _contiguous(teacher_logits), _contiguous(teacher_ids), weights, REDUCTIONS[reduction]


def _contiguous(t):
    return t if t.is_contiguous() else t.detach().contiguous()


def _distill_struct(rows, teacher, ids, weights, temperature, reduction, work):
    n, vocab = rows.shape
    return L.Distill(logits=rows.data_ptr(), teacher=teacher.data_ptr(), ids=ids.data_ptr(), weights=None if weights is None else weights.data_ptr(),
                     rows=n, stride=vocab if n <= 1 else rows.stride(0), vocab=vocab, top=ids.shape[-1], type=TYPES[rows.dtype],
                     teacher_type=TYPES[teacher.dtype], ids_bytes=ids.element_size(), reduction=reduction, temperature=temperature, scale=1.0,
                     work=work.data_ptr(), work_bytes=work.numel())


def _distill_work(rows, ids):
    size = _size("pylo_b200_distill_workspace", rows.get_device(), *rows.shape, ids.shape[-1])
    return torch.empty(size, dtype=torch.uint8, device=rows.device)


def _distill_forward(rows, teacher, ids, weights, temperature, reduction, lead):
    """(loss, the workspace, which a gradient is made from)"""
    work = _distill_work(rows, ids)
    d = _distill_struct(rows, teacher, ids, weights, temperature, reduction, work)
    if reduction == L.REDUCE_NONE:
        loss = torch.empty(lead, dtype=torch.float32, device=rows.device)
        d.row_loss = loss.data_ptr()
    else:
        loss = torch.empty((), dtype=torch.float32, device=rows.device)
        d.loss = loss.data_ptr()
    _call(L.lib.pylo_b200_distill, "distillation_loss", rows.get_device(), C.byref(d), L.DISTILL_LOSS)
    return loss, work


class _Distillation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, rows, teacher, ids, weights, temperature, reduction):
        loss, work = _distill_forward(rows, teacher, ids, weights, temperature, reduction, logits.shape[:-1])
        ctx.save_for_backward(rows, teacher, ids, weights, work)
        ctx.temperature, ctx.reduction, ctx.shape = temperature, reduction, logits.shape
        return loss

    @staticmethod
    @_once
    def backward(ctx, upstream):
        rows, teacher, ids, weights, work = ctx.saved_tensors
        if rows.stride(1) != 1 or not (teacher.is_contiguous() and ids.is_contiguous() and (weights is None or weights.is_contiguous())):
            # hooks have laid them out anew
            rows, teacher, ids, weights = _rows(rows), teacher.contiguous(), ids.contiguous(), None if weights is None else weights.contiguous()
        grad = _like(rows)
        if upstream.dtype is not torch.float32 or not upstream.is_contiguous():
            upstream = upstream.to(torch.float32).contiguous()
        d = _distill_struct(rows, teacher, ids, weights, ctx.temperature, ctx.reduction, work)
        d.grad, d.upstream = grad.data_ptr(), upstream.data_ptr()
        _call(L.lib.pylo_b200_distill, "distillation_loss backward", rows.get_device(), C.byref(d), L.DISTILL_GRAD)
        return grad.view(ctx.shape), None, None, None, None, None, None


def distillation_loss(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_ids: torch.Tensor, temperature: float = 1.0,
                      weights: torch.Tensor | None = None, reduction: str = "mean") -> torch.Tensor:
    """The divergence of a student's distribution from that of a teacher's largest logits, times ``temperature ** 2``, in fp32.

    ``logits`` are ``[..., classes]``; ``teacher_logits`` and ``teacher_ids`` (int64 or int32) are ``[..., K]``, K up to 1024: the teacher's
    distribution is the softmax over its K entries.  An id outside of ``[0, classes)`` is padding, whatever stands beside it; one that is given
    twice counts twice.  ``weights`` (``[...]``, a mask or numbers): a row of weight 0 is not looked at and gets a gradient of 0, as does a row
    without any entry.  ``reduction``: ``"mean"`` over the sum of the weights that count (0 where that is 0), ``"sum"``, or ``"none"`` (weighted rows).
    Only ``logits`` are differentiated."""
    rows, teacher, ids, w, code = _distill_arguments(logits, teacher_logits, teacher_ids, temperature, weights, reduction)
    if _graph(logits):
        return _Distillation.apply(logits, rows, teacher, ids, w, float(temperature), code)
    return _distill_forward(rows, teacher, ids, w, float(temperature), code, logits.shape[:-1])[0]


def distillation_loss_and_grad(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_ids: torch.Tensor, temperature: float = 1.0,
                               weights: torch.Tensor | None = None, reduction: str = "mean", scale: float | torch.Tensor = 1.0):
    """:func:`distillation_loss` and ``scale`` times its gradient in one pass over the logits, for ``logits.backward(grad)``: ``(loss, grad)``.

    ``reduction`` is ``"mean"`` or ``"sum"``; ``scale`` a number or a one-element fp32 tensor on the device, such as a loss scale (the
    loss itself is not scaled)."""
    rows, teacher, ids, w, code = _distill_arguments(logits, teacher_logits, teacher_ids, temperature, weights, reduction)
    if code == L.REDUCE_NONE:
        raise ValueError("reduction has to be 'mean' or 'sum'")
    work = _distill_work(rows, ids)
    d = _distill_struct(rows, teacher, ids, w, float(temperature), code, work)
    if isinstance(scale, torch.Tensor):
        if forward_ad._current_level >= 0:
            _refuse_tangents(scale)
        _check("scale", scale, logits.get_device(), (torch.float32,))
        if scale.numel() != 1:
            raise ValueError("scale has to have one element")
        d.upstream = scale.data_ptr()
    else:
        d.scale = float(scale)
    loss = torch.empty((), dtype=torch.float32, device=rows.device)
    grad = _like(rows)
    d.loss, d.grad = loss.data_ptr(), grad.data_ptr()
    _call(L.lib.pylo_b200_distill, "distillation_loss_and_grad", rows.get_device(), C.byref(d), L.DISTILL_LOSS | L.DISTILL_GRAD)
    return loss, grad.view(logits.shape)


class DistillationLoss(torch.nn.Module):
    """:func:`distillation_loss` with its options."""

    def __init__(self, temperature: float = 1.0, reduction: str = "mean"):
        super().__init__()
        self.temperature, self.reduction = temperature, reduction

    def forward(self, logits, teacher_logits, teacher_ids, weights=None):
        return distillation_loss(logits, teacher_logits, teacher_ids, self.temperature, weights, self.reduction)

"""Losses of a language model on MI355X (HIP kernels behind the C ABI): cross-entropy from the head's
operands, without logits, and distillation from a teacher's top logits, from the head's operands or
from logits.

``linear_cross_entropy(x, weight, targets, ignore_index=-100, reduction="mean") -> loss`` — the
softmax cross-entropy of the logits ``x.T @ weight.T`` (the reference takes it of its head's
logits, experiments/mamba_inductionheads.py:129-136), which are not kept: x (features, tokens)
float32 or bfloat16, any non-negative strides (the channel-major stream after the final norm, or the
``.t()`` of token-major rows); weight (vocab, features); targets (tokens,) int64.

``linear_distill_loss(x, weight, ids, teacher, temperature=1.0, reduction="mean") -> loss`` — the same
head towards a teacher: ids (tokens, top) int64, the words of the teacher's largest logits, and
teacher (tokens, top), these logits in float32 or bfloat16.

``distill_loss(logits, ids, teacher, temperature=1.0, reduction="mean") -> loss`` — the same loss from
logits (rows, vocab), float32 or bfloat16.

A list's entry counts if its id is not negative and its logit not -inf; what the others hold is not looked
at. With ``q = softmax(teacher / temperature)`` over the entries that count (a word that stands in a list more
than once has the sum) and ``p = softmax(logits / temperature)`` over the vocabulary, a row's loss is
``temperature**2 * sum(q * (log(q) - log(p)))``. A row without an entry, or with ignore_index for a
target, does not count: its loss and gradients are zeros, whatever x or the logits hold there. A word
outside the vocabulary, or a teacher's logit that is NaN or inf, makes its row's loss and gradients NaN.

``reduction``: "mean" over the rows that count (0 if none does), "sum", or "none" for (rows,)
losses. The loss is float32. Differentiable, once, in x, weight and logits; gradients have their input's
type. ``holder`` (``lm_ops.GradHolder``) takes the weight's float32 gradient instead of autograd. There is no
CPU path. A loss from logits keeps them, and a reduced one their gradient beside them, until its backward pass.

What is held in how many bits, of a head's losses (sums are float32):

* a bfloat16 x: the logits' gradient is rounded to bfloat16 once, as the operands are. A float32 weight is
  read in a bfloat16 copy: ``weight_act``, where the caller keeps one, else a cast.
* The same, a reduced loss, x and weight both requiring gradients, from 512 tokens, 640 features, 1024 words and
  2^25 logits on: the gradients come with the loss, from logits held in 16 bits, that is probabilities to
  less than 2^-10 of themselves, and zeros for those below 2^-38; an upstream gradient that is not a power
  of two rounds them a second time. A second backward pass, ``"none"``, one gradient alone and smaller heads
  form the logits again and have neither.
* a float32 x: an element of x and weight counts to 2^-23 of itself down to 2^-27 of its matrix's largest, and
  to 2^-50 of that below; their products to 2^-22; the logits' gradient to 2^-23 of itself down to 2^-28 and
  to 2^-51 below, with ``"none"`` down to 2^-27 and to 2^-50 of the largest upstream gradient of the rows that
  count. (Float32 operations keep what is smaller still to 2^-24 of itself.)
"""
from __future__ import annotations

import contextlib
import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .selective_scan_hip import _io_tag, _ptr, _require_gpu, _resolved, _stream

__all__ = ["linear_cross_entropy", "linear_distill_loss", "distill_loss"]

_F32, _I64 = torch.float32, torch.int64
_REDUCTIONS = {"none": _lib.MSS_LOSS_NONE, "sum": _lib.MSS_LOSS_SUM, "mean": _lib.MSS_LOSS_MEAN}
_MAX_ENTRIES = 1 << 27
_MAX_ROWS = 1 << 21


def _reduction(name):
    tag = _REDUCTIONS.get(name)
    if tag is None:
        raise ValueError(f'reduction must be "none", "sum" or "mean", got {name!r}')
    return tag


def _check_lists(ids, teacher, rows, temperature):
    """The teacher's type tag."""
    if ids.dtype != _I64 or ids.dim() != 2 or ids.shape[0] != rows:
        raise ValueError(f"ids must be int64 with shape ({rows}, top)")
    if teacher.shape != ids.shape:
        raise ValueError(f"teacher must have the shape of ids, {tuple(ids.shape)}")
    if ids.shape[1] > _lib.MSS_LOSS_MAX_TOP:
        raise ValueError(f"lists have at most {_lib.MSS_LOSS_MAX_TOP} words, got {ids.shape[1]}")
    if ids.numel() > _MAX_ENTRIES:
        raise ValueError(f"lists have at most {_MAX_ENTRIES} words in all, got {ids.numel()}")
    if not (temperature > 0 and math.isfinite(temperature)):
        raise ValueError(f"temperature must be finite and above 0, got {temperature}")
    if torch.is_grad_enabled() and teacher.requires_grad:
        raise RuntimeError("the loss has no gradient for the teacher's logits: detach them")
    return _io_tag(teacher.dtype, "teacher")


_HERE = contextlib.nullcontext()


def _guard(t):
    """Launches go to the device of `t`, whichever is current."""
    return _HERE if t.get_device() == torch.cuda.current_device() else torch.cuda.device(t.device)


def _require_one_gpu(*tensors):
    _require_gpu(*tensors)
    device = tensors[0].device
    for t in tensors:
        if t is not None and t.device != device:
            raise ValueError(f"the operands lie on several devices: {device}, {t.device}")


def _bytes(n, device):
    return torch.empty(n, dtype=torch.uint8, device=device)


def _row_stride(m):
    return m.stride(0) if m.shape[0] > 1 else m.shape[1]


def _rows(m):
    """`m` with contiguous rows that do not overlap."""
    rows, cols = m.shape
    return m.contiguous() if cols > 1 and m.stride(1) != 1 or rows > 1 and m.stride(0) < cols else m


def _upstream(grad, reduction, rows):
    """The upstream gradient as the kernels read it."""
    g = _resolved(grad).to(_F32)
    return g.reshape(1) if reduction != _lib.MSS_LOSS_NONE else g.reshape(rows).contiguous()


class _LinearLoss(torch.autograd.Function):
    """Where the loss is reduced and both gradients are wanted, large heads' come with it, for an upstream gradient of
    1: the logits are formed once. The backward pass multiplies them by another one; a second one makes its own."""

    @staticmethod
    def forward(ctx, x, weight, weight_act, targets, ids, teacher, ignore_index, temperature, reduction, teacher_tag,
                holder, both):
        lib = _lib.register_hip_kernel()
        f, t = x.shape
        w = weight_act
        lists = ids is not None
        a = _lib.LinearLossArgs(tokens=t, features=f, vocab=w.shape[0], top=ids.shape[1] if lists else 0,
                                io_dtype=_io_tag(x.dtype, "x"), teacher_dtype=teacher_tag, reduction=reduction,
                                temperature=temperature, ignore_index=ignore_index,
                                stride_f=x.stride(0) if f > 1 else 0, stride_t=x.stride(1) if t > 1 else 0,
                                ldw=_row_stride(w), x=x.data_ptr(), weight=w.data_ptr(),
                                targets=_ptr(targets), ids=_ptr(ids), teacher=_ptr(teacher))
        dev = x.device
        with _guard(x):
            saved = _bytes(lib.mss_linear_loss_saved_bytes(a), dev)
            need = lib.mss_linear_loss_workspace_bytes(a, 2) if both else 0
            name = "mss_linear_loss_fwd_grad" if need else "mss_linear_loss_fwd"
            ws = _bytes(need or lib.mss_linear_loss_workspace_bytes(a, 0), dev)
            ctx.d = None
            if need:
                dx, dw = torch.empty(f, t, dtype=x.dtype, device=dev), torch.empty(w.shape, dtype=weight.dtype, device=dev)
                a.dx, a.dweight, a.dw_dtype = dx.data_ptr(), dw.data_ptr(), _io_tag(weight.dtype, "weight")
                ctx.d = dx, dw
            loss = torch.empty(t, dtype=_F32, device=dev)
            mean = torch.empty((), dtype=_F32, device=dev)
            a.loss, a.mean, a.saved, a.saved_bytes = loss.data_ptr(), mean.data_ptr(), saved.data_ptr(), saved.numel()
            a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
            _lib.check(getattr(lib, name)(a, _stream(x)), name)
        ctx.save_for_backward(w, saved)
        ctx.args = a
        ctx.x_like = (x.dtype, (f, t))
        ctx.dw_dtype, ctx.holder, ctx.head = weight.dtype, holder, object()
        ctx.set_materialize_grads(False)
        return loss if reduction == _lib.MSS_LOSS_NONE else mean

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        need_x, need_w = ctx.needs_input_grad[:2]
        if grad is None or not (need_x or need_w):
            return (None,) * 12
        lib = _lib.register_hip_kernel()
        w, saved = ctx.saved_tensors
        src = ctx.args
        dtype, shape = ctx.x_like
        dev = w.device
        with _guard(w):
            grad = _upstream(grad, src.reduction, src.tokens)
            a = _lib.LinearLossArgs.from_buffer_copy(src)
            a.x = a.loss = a.mean = a.targets = a.ids = a.teacher = None
            # (Saved-tensor hooks may have put both elsewhere, and the weight's rows at another distance.)
            a.saved, a.saved_bytes = saved.data_ptr(), saved.numel()
            if w.data_ptr() != src.weight or w.stride() != (src.ldw, 1):
                w = _rows(w)
                a.weight, a.ldw = w.data_ptr(), _row_stride(w)
                if saved.numel() < lib.mss_linear_loss_saved_bytes(a):  # it was read in place, and cannot be here
                    w = w.clone(memory_format=torch.contiguous_format)
                    a.weight, a.ldw = w.data_ptr(), _row_stride(w)
            a.dw_dtype = _io_tag(ctx.dw_dtype, "weight")
            d, ctx.d = ctx.d, None  # the caller may write over them
            if d is not None:
                dx, dw = d
                name = "mss_linear_loss_rescale"
            else:
                dx = torch.empty(shape, dtype=dtype, device=dev) if need_x else None
                dw = torch.empty(w.shape, dtype=ctx.dw_dtype, device=dev) if need_w else None
                ws = _bytes(lib.mss_linear_loss_workspace_bytes(a, 1), dev)
                a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
                name = "mss_linear_loss_bwd"
            a.grad, a.dx, a.dweight = grad.data_ptr(), _ptr(dx), _ptr(dw)
            _lib.check(getattr(lib, name)(a, _stream(w)), name)
            dx, dw = dx if need_x else None, dw if need_w else None
        if dw is not None and ctx.holder is not None:
            ctx.holder.put(dw, ctx.head)
            dw = None
        return (dx, dw) + (None,) * 10


def _linear_loss(x, weight, weight_act, holder, targets, ids, teacher, ignore_index, temperature, reduction, teacher_tag):
    if x.dim() != 2 or weight.dim() != 2:
        raise ValueError("x must be a (features, tokens) and weight a (vocab, features) matrix")
    _io_tag(x.dtype, "x")
    _io_tag(weight.dtype, "weight")
    f, t = x.shape
    vocab = weight.shape[0]
    if weight.shape[1] != f:
        raise ValueError(f"weight must have x's {f} features, got {weight.shape[1]}")
    if vocab == 0 or f == 0:
        raise ValueError("the head has no words or no features")
    if weight_act is not None and (weight_act.dtype != x.dtype or weight_act.shape != weight.shape):
        raise ValueError("weight_act must be the weight in x's type")
    if holder is not None and weight.dtype != _F32:
        raise ValueError("a holder takes a float32 weight's gradient")
    _require_one_gpu(x, weight, weight_act, targets, ids, teacher)
    if t == 0 or (ids is not None and ids.shape[1] == 0):
        # No row counts: zeros that depend on the operands.
        none = x.new_zeros(t, dtype=_F32) + 0.0 * (x[:0].sum() + weight[:0].sum()).float()
        return none if reduction == _lib.MSS_LOSS_NONE else none.sum()
    if weight_act is None:
        weight_act = weight.detach() if weight.dtype == x.dtype else weight.detach().to(x.dtype)
    else:
        weight_act = weight_act.detach()
    weight_act = _rows(_resolved(weight_act))
    conform = [None if v is None else _resolved(v).contiguous() for v in (targets, ids, teacher)]
    both = reduction != _lib.MSS_LOSS_NONE and torch.is_grad_enabled() and x.requires_grad and weight.requires_grad
    return _LinearLoss.apply(_resolved(x), weight, weight_act, *conform, ignore_index, temperature, reduction, teacher_tag,
                             holder, both)


def linear_cross_entropy(x, weight, targets, ignore_index=-100, reduction="mean", weight_act=None, holder=None):
    reduction = _reduction(reduction)
    if targets.dtype != _I64 or x.dim() != 2 or tuple(targets.shape) != (x.shape[1],):
        raise ValueError("targets must be int64 with one word for each of x's tokens")
    return _linear_loss(x, weight, weight_act, holder, targets, None, None, int(ignore_index), 1.0, reduction, 0)


def linear_distill_loss(x, weight, ids, teacher, temperature=1.0, reduction="mean", weight_act=None, holder=None):
    reduction, temperature = _reduction(reduction), float(temperature)
    tag = _check_lists(ids, teacher, x.shape[1] if x.dim() == 2 else -1, temperature)
    return _linear_loss(x, weight, weight_act, holder, None, ids, teacher, 0, temperature, reduction, tag)


class _Distill(torch.autograd.Function):
    """Where the loss is reduced and will be differentiated, it and its gradient for an upstream gradient of 1
    come from one reading of the logits; the backward pass writes the gradient anew for another one."""

    @staticmethod
    def forward(ctx, logits, ids, teacher, temperature, reduction, teacher_tag, both):
        lib = _lib.register_hip_kernel()
        rows, vocab = logits.shape
        a = _lib.DistillArgs(rows=rows, vocab=vocab, top=ids.shape[1], io_dtype=_io_tag(logits.dtype, "logits"),
                             teacher_dtype=teacher_tag, reduction=reduction, temperature=temperature,
                             ld=_row_stride(logits), logits=logits.data_ptr(), ids=ids.data_ptr(),
                             teacher=teacher.data_ptr())
        dev = logits.device
        with _guard(logits):
            saved = _bytes(lib.mss_distill_saved_bytes(a), dev)
            loss = torch.empty(rows, dtype=_F32, device=dev)
            mean = torch.empty((), dtype=_F32, device=dev)
            d = torch.empty(rows, vocab, dtype=logits.dtype, device=dev) if both else None
            a.loss, a.mean, a.saved, a.saved_bytes = loss.data_ptr(), mean.data_ptr(), saved.data_ptr(), saved.numel()
            a.dlogits = _ptr(d)
            name = "mss_distill_fwd_grad" if both else "mss_distill_fwd"
            _lib.check(getattr(lib, name)(a, _stream(logits)), name)
        ctx.save_for_backward(logits, saved)
        ctx.args, ctx.d = a, d
        ctx.set_materialize_grads(False)
        return loss if reduction == _lib.MSS_LOSS_NONE else mean

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        if grad is None:
            return (None,) * 7
        lib = _lib.register_hip_kernel()
        logits, saved = ctx.saved_tensors
        src = ctx.args
        with _guard(logits):
            grad = _upstream(grad, src.reduction, src.rows)
            d, ctx.d = ctx.d, None  # the caller may write over it: a second pass makes its own
            name = "mss_distill_bwd" if d is None else "mss_distill_regrad"
            if d is None:
                d = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
            a = _lib.DistillArgs.from_buffer_copy(src)
            a.ids = a.teacher = a.loss = a.mean = None
            # (Saved-tensor hooks may have put both elsewhere, and the rows at another distance.)
            if logits.data_ptr() != src.logits or logits.stride() != (src.ld, 1):
                logits = _rows(logits)
                a.logits, a.ld = logits.data_ptr(), _row_stride(logits)
            a.saved, a.saved_bytes = saved.data_ptr(), saved.numel()
            a.grad, a.dlogits = grad.data_ptr(), d.data_ptr()
            _lib.check(getattr(lib, name)(a, _stream(logits)), name)
        return (d,) + (None,) * 6


def distill_loss(logits, ids, teacher, temperature=1.0, reduction="mean"):
    reduction, temperature = _reduction(reduction), float(temperature)
    if logits.dim() != 2:
        raise ValueError("logits must be a (rows, vocab) matrix")
    _io_tag(logits.dtype, "logits")
    rows, vocab = logits.shape
    if vocab == 0:
        raise ValueError("logits have no words")
    if rows > _MAX_ROWS:
        raise ValueError(f"logits have at most {_MAX_ROWS} rows, got {rows}")
    tag = _check_lists(ids, teacher, rows, temperature)
    _require_one_gpu(logits, ids, teacher)
    if rows == 0 or ids.shape[1] == 0:
        none = logits.new_zeros(rows, dtype=_F32) + 0.0 * logits[:0].sum().float()
        return none if reduction == _lib.MSS_LOSS_NONE else none.sum()
    logits = _rows(_resolved(logits))
    both = reduction != _lib.MSS_LOSS_NONE and torch.is_grad_enabled() and logits.requires_grad
    return _Distill.apply(logits, _resolved(ids).contiguous(), _resolved(teacher).detach().contiguous(), temperature,
                          reduction, tag, both)

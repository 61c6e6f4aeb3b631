"""Losses over a set of classes -- the tokens of a vocabulary, or the depth bins of a pixel -- on the HIP library:

    top_logits(logits, k, temperature)                       what a teacher hands on: its k largest logits of every row
    topk_distillation_loss(logits, values, indices, lse)     a student against them, with the gradient of its logits
    linear_cross_entropy(hidden, weight, target, bias)       cross entropy of a linear head in pieces of the vocabulary,
                                                             logits never kept, with the gradients of hidden, weight, bias

The last dimension is the classes (the features, for ``hidden`` and ``weight``); all others are rows, so a decoder's
[B, C, H, W] maps go in as ``maps.movedim(1, -1)``, which costs no copy in channels-last memory.  Tensors are float32,
bfloat16 or float16 (float64 is cast to float32 on load, as everywhere in this package); rows may be strided, everything
else is made contiguous.  Losses and statistics are float32, gradients have their tensor's type.

A logit of -infinity is a masked class.  A row in which nothing is left adds nothing and gets a zero gradient; NaN or
+infinity in a row, and a target or index outside the vocabulary, make that row's results NaN.  ``"mean"`` over no rows is
0.  Results are deterministic.  No host synchronisation: every call can be captured into a graph.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import _abi

_lib = _abi.lib
_TYPES = {torch.float32: _abi.TYPE_F32, torch.bfloat16: _abi.TYPE_BF16, torch.float16: _abi.TYPE_F16}
_REDUCTIONS = {"none": _abi.REDUCE_NONE, "sum": _abi.REDUCE_SUM, "mean": _abi.REDUCE_MEAN}


class TopLogits(NamedTuple):
    values: torch.Tensor    # [..., k], the logits' type, larger first
    indices: torch.Tensor   # [..., k], int32
    lse: torch.Tensor       # [...], float32: log sum exp(logits / temperature) over the whole vocabulary


# The checks below and the calls run once per loss and step; where rows are few they are most of the time (a few
# microseconds each way), so they ask for whole numbers instead of building torch objects and leave alone what fits.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)


def _floating(t: torch.Tensor, name: str) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError("%s must be a GPU tensor (there is no CPU implementation)" % name)
    if t.dtype not in _TYPES:
        if t.dtype != torch.float64:
            raise ValueError("%s must be float32, bfloat16 or float16, not %s" % (name, t.dtype))
        t = t.float()
    return t


def _matrix(t: torch.Tensor, name: str) -> torch.Tensor:
    """[..., n] as [rows, n] whose rows may be strided and whose elements are not."""
    if t.dim() != 2:
        if t.dim() < 1:
            raise ValueError("%s needs a last dimension of at least 1" % name)
        t = t.reshape(t.shape[:-1].numel(), t.shape[-1])
    if t.shape[1] < 1:
        raise ValueError("%s needs a last dimension of at least 1" % name)
    if t.stride(1) != 1 or t.stride(0) < t.shape[1]:
        t = t.contiguous()
    return t


def _row_stride(t: torch.Tensor) -> int:
    return max(t.stride(0), t.shape[1])


def _on(t: torch.Tensor, name: str, like: torch.Tensor) -> None:
    if t.get_device() != like.get_device():
        raise ValueError("%s is on %s, not on %s" % (name, t.device, like.device))


def _per_row(t: Optional[torch.Tensor], name: str, shape, like: torch.Tensor) -> Optional[torch.Tensor]:
    """A float32 vector with one entry per row, or None."""
    if t is None:
        return None
    _on(t, name, like)
    if t.shape != shape:
        raise ValueError("%s must have the shape of the rows, %s, not %s" % (name, tuple(shape), tuple(t.shape)))
    if t.dim() != 1:
        t = t.reshape(-1)
    return (t if t.dtype == torch.float32 else t.float()).contiguous()


def _once(backward):
    """once_differentiable without its cost where no second derivative can be asked for."""
    with_graph = once_differentiable(backward)

    def call(ctx, g):
        return with_graph(ctx, g) if torch.is_grad_enabled() else backward(ctx, g)

    return call


def _differentiable(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _reduction(name: str) -> int:
    if name not in _REDUCTIONS:
        raise ValueError("reduction must be 'none', 'sum' or 'mean', not %r" % (name,))
    return _REDUCTIONS[name]


def _temperature(value) -> float:
    value = float(value)
    if not 1e-4 <= value <= 1e4:
        raise ValueError("temperature must lie in 1e-4..1e4, not %r" % value)
    return value


def _bytes(n: int, like: torch.Tensor) -> torch.Tensor:
    return torch.empty(n, dtype=torch.uint8, device=like.device)


def _floats(n: int, like: torch.Tensor) -> torch.Tensor:
    return torch.empty(n, dtype=torch.float32, device=like.device)


def _ptr(t: Optional[torch.Tensor]):
    return t.data_ptr() if t is not None else None


def _run(like: torch.Tensor, call, *args) -> None:
    """A library call on the current stream of the tensor's device, which need not be the current device."""
    index = like.get_device()
    if index == torch.cuda.current_device():
        rc = call(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = call(*args, _raw_stream(index))
    if rc:
        _abi.check(rc)


# ------------------------------------------------------------------ top logits
def top_logits(logits: torch.Tensor, k: int, temperature: float = 1.0) -> TopLogits:
    """The ``k`` largest logits of every row, larger first, ties to the lower index, NaN above +infinity, and the log of
    the row's whole sum of exp(logits / temperature); 1 <= k <= min(classes, 256).  One pass over the logits; carries no
    gradient."""
    logits = _floating(logits, "logits").detach()
    shape = logits.shape[:-1]
    x = _matrix(logits, "logits")
    k = int(k)
    if not 1 <= k <= min(x.shape[1], _abi.MAX_TOP):
        raise ValueError("k must lie in 1..min(classes, %d), not %d" % (_abi.MAX_TOP, k))
    d = _abi.TopDesc(rows=x.shape[0], vocab=x.shape[1], stride=_row_stride(x), k=k, type=_TYPES[x.dtype],
                     temperature=_temperature(temperature), logits=x.data_ptr())
    values = torch.empty(shape + (k,), dtype=x.dtype, device=x.device)
    indices = torch.empty(shape + (k,), dtype=torch.int32, device=x.device)
    lse = torch.empty(shape, dtype=torch.float32, device=x.device)
    nbytes = _lib.vsl_top_logits_workspace_bytes(ctypes.byref(d))
    ws = _bytes(nbytes, x)
    _run(x, _lib.vsl_top_logits, ctypes.byref(d), values.data_ptr(), indices.data_ptr(), lse.data_ptr(), ws.data_ptr(), nbytes)
    return TopLogits(values, indices, lse)


# ------------------------------------------------------------------ distillation
def _distill_desc(x, values, indices, lse, weights, temperature, reduction):
    return _abi.DistillDesc(rows=x.shape[0], vocab=x.shape[1], stride=_row_stride(x), k=values.shape[1], type=_TYPES[x.dtype],
                            value_type=_TYPES[values.dtype], index_bytes=indices.element_size(), reduction=reduction,
                            temperature=temperature, logits=x.data_ptr(), teacher_values=values.data_ptr(),
                            teacher_indices=indices.data_ptr(), teacher_lse=_ptr(lse), weights=_ptr(weights))


def _distill_forward(x, values, indices, lse, weights, temperature, reduction):
    """The loss, and what the backward call needs of the rows: statistics and, behind them, the divisor of the mean.  The
    workspace and, where they are summed, the row losses share that allocation: all are small beside the logits."""
    rows = x.shape[0]
    d = _distill_desc(x, values, indices, lse, weights, temperature, reduction)
    nbytes = _lib.vsl_distill_workspace_bytes(ctypes.byref(d))
    head = (4 * (_abi.DISTILL_STATS * rows + 1) + 255) // 256 * 256
    kept = _bytes(head + nbytes + 4 * rows, x)
    base = kept.data_ptr()
    if reduction == _abi.REDUCE_NONE:
        out = _floats(rows, x)
        _run(x, _lib.vsl_distill_fwd, ctypes.byref(d), out.data_ptr(), None, None, base, base + head, nbytes)
    else:
        out = _floats((), x)
        _run(x, _lib.vsl_distill_fwd, ctypes.byref(d), base + head + nbytes, out.data_ptr(),
             base + 4 * _abi.DISTILL_STATS * rows, base, base + head, nbytes)
    return out, kept


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, values, indices, lse, weights, temperature, reduction):
        out, kept = _distill_forward(x, values, indices, lse, weights, temperature, reduction)
        ctx.save_for_backward(x, values, indices, weights, kept)
        ctx.cfg = (temperature, reduction)
        return out

    @staticmethod
    @_once
    def backward(ctx, g):
        # the descriptor is made anew: a saved-tensor hook may have moved what it points to
        x, values, indices, weights, kept = ctx.saved_tensors
        d = _distill_desc(x, values, indices, None, weights, *ctx.cfg)
        g = g.contiguous()
        grad = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        base = kept.data_ptr()
        _run(x, _lib.vsl_distill_bwd, ctypes.byref(d), base, base + 4 * _abi.DISTILL_STATS * x.shape[0], g.data_ptr(),
             grad.data_ptr(), x.shape[1])
        return grad, None, None, None, None, None, None


def topk_distillation_loss(logits: torch.Tensor, teacher_values: torch.Tensor, teacher_indices: torch.Tensor,
                           teacher_lse: Optional[torch.Tensor] = None, *, temperature: float = 1.0,
                           weights: Optional[torch.Tensor] = None, reduction: str = "mean") -> torch.Tensor:
    """temperature^2 * KL(teacher || student) from the teacher's top logits (``top_logits``), with the gradient of
    ``logits`` [..., classes].

    ``teacher_values`` / ``teacher_indices`` [..., k] (int32 or int64).  Without ``teacher_lse`` the teacher is the softmax
    of its k values / temperature.  With it ([...], the log of its whole sum at this temperature) the k classes keep their
    probabilities and what is left is one further class, against which the student puts the sum of its other
    probabilities; it is left out of a row where the student has no other class.  ``weights`` [...]: a row of weight 0 is
    not looked at; ``"mean"`` divides by their sum.  The teacher's tensors and the weights carry no gradient."""
    logits = _floating(logits, "logits")
    values, indices, shape = _floating(teacher_values, "teacher_values"), teacher_indices, logits.shape[:-1]
    _on(values, "teacher_values", logits)
    _on(indices, "teacher_indices", logits)
    if indices.dtype not in (torch.int32, torch.int64):
        raise ValueError("teacher_indices must be int32 or int64, not %s" % indices.dtype)
    if values.shape != indices.shape or values.dim() < 1 or values.shape[:-1] != shape:
        raise ValueError("teacher_values and teacher_indices must both be [..., k] over the rows of logits")
    x = _matrix(logits, "logits")
    k = values.shape[-1]
    if not 1 <= k <= min(x.shape[1], _abi.MAX_TOP):
        raise ValueError("the teacher's k must lie in 1..min(classes, %d), not %d" % (_abi.MAX_TOP, k))
    if values.dim() != 2:
        values, indices = values.reshape(x.shape[0], k), indices.reshape(x.shape[0], k)
    args = (x, values.contiguous(), indices.contiguous(), _per_row(teacher_lse, "teacher_lse", shape, logits),
            _per_row(weights, "weights", shape, logits), _temperature(temperature), _reduction(reduction))
    loss = _Distill.apply(*args) if _differentiable(x) else _distill_forward(*args)[0]
    return loss.reshape(shape) if reduction == "none" and len(shape) != 1 else loss


# ------------------------------------------------------------------ linear cross entropy
def _linear_ce_desc(hidden, weight, bias, target, ignore_index, z_loss, reduction):
    return _abi.LinearCeDesc(rows=hidden.shape[0], vocab=weight.shape[0], dim=hidden.shape[1], hidden_stride=_row_stride(hidden),
                             weight_stride=_row_stride(weight), ignore_index=ignore_index, type=_TYPES[hidden.dtype],
                             reduction=reduction, z_loss=z_loss, hidden=hidden.data_ptr(), weight=weight.data_ptr(),
                             bias=_ptr(bias), target=target.data_ptr())


def _linear_ce_forward(hidden, weight, bias, target, ignore_index, z_loss, reduction):
    """The loss, and what the backward call needs of the rows: statistics and, behind them, the divisor of the mean."""
    d = _linear_ce_desc(hidden, weight, bias, target, ignore_index, z_loss, reduction)
    rows = hidden.shape[0]
    kept = _floats(2 * rows + 1, hidden)
    nbytes = _lib.vsl_linear_ce_fwd_workspace_bytes(ctypes.byref(d))
    if reduction == _abi.REDUCE_NONE:
        out, ws = _floats(rows, hidden), _bytes(nbytes, hidden)
        _run(hidden, _lib.vsl_linear_ce_fwd, ctypes.byref(d), out.data_ptr(), kept.data_ptr(), None, None, ws.data_ptr(), nbytes)
    else:
        out, ws = _floats((), hidden), _bytes(nbytes + 4 * rows, hidden)   # the row losses are scratch behind the workspace
        _run(hidden, _lib.vsl_linear_ce_fwd, ctypes.byref(d), ws.data_ptr() + nbytes, kept.data_ptr(), out.data_ptr(),
             kept.data_ptr() + 8 * rows, ws.data_ptr(), nbytes)
    return out, kept


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, bias, target, ignore_index, z_loss, reduction):
        out, kept = _linear_ce_forward(hidden, weight, bias, target, ignore_index, z_loss, reduction)
        ctx.save_for_backward(hidden, weight, bias, target, kept)
        ctx.cfg = (ignore_index, z_loss, reduction)
        return out

    @staticmethod
    @_once
    def backward(ctx, g):
        hidden, weight, bias, target, kept = ctx.saved_tensors
        d = _linear_ce_desc(hidden, weight, bias, target, *ctx.cfg)   # anew: a saved-tensor hook may have moved them
        g = g.contiguous()
        need = ctx.needs_input_grad
        g_hidden = torch.empty(hidden.shape, dtype=hidden.dtype, device=hidden.device) if need[0] else None
        g_weight = torch.empty(weight.shape, dtype=weight.dtype, device=weight.device) if need[1] else None
        g_bias = torch.empty(bias.shape, dtype=bias.dtype, device=bias.device) if bias is not None and need[2] else None
        mask = (g_hidden is not None) | (g_weight is not None) << 1 | (g_bias is not None) << 2
        nbytes = _lib.vsl_linear_ce_bwd_workspace_bytes(ctypes.byref(d), mask)
        ws = _bytes(nbytes, hidden)
        _run(hidden, _lib.vsl_linear_ce_bwd, ctypes.byref(d), kept.data_ptr(), kept.data_ptr() + 8 * hidden.shape[0],
             g.data_ptr(), _ptr(g_hidden), _ptr(g_weight), _ptr(g_bias), ws.data_ptr(), nbytes)
        return g_hidden, g_weight, g_bias, None, None, None, None


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, target: torch.Tensor,
                         bias: Optional[torch.Tensor] = None, *, ignore_index: int = -100, z_loss: float = 0.0,
                         reduction: str = "mean") -> torch.Tensor:
    """Softmax cross entropy of ``hidden @ weight.T + bias`` against ``target``, plus ``z_loss`` times the square of every
    row's log sum, without keeping the logits: the forward pass reduces them tile by tile on the matrix cores, the
    backward pass makes them again in pieces of the vocabulary.

    ``hidden`` [..., dim], ``weight`` [classes, dim] and ``bias`` [classes] share one type; ``target`` [...] holds classes
    or ``ignore_index`` (such a row is left out of the mean and gets a zero gradient).  A class whose bias is -infinity is
    masked out.  Gradients reach ``hidden``, ``weight`` and ``bias``; in 16-bit types the derivative of a logit is rounded
    to that type before the two gradient products, which sum in float32."""
    hidden, weight = _floating(hidden, "hidden"), _floating(weight, "weight")
    _on(weight, "weight", hidden)
    _on(target, "target", hidden)
    if weight.dim() != 2 or hidden.dim() < 1 or weight.shape[1] != hidden.shape[-1] or weight.shape[0] < 1:
        raise ValueError("hidden must be [..., dim] and weight [classes, dim], not %s and %s"
                         % (tuple(hidden.shape), tuple(weight.shape)))
    if weight.dtype != hidden.dtype:
        raise ValueError("hidden and weight must have one type, not %s and %s" % (hidden.dtype, weight.dtype))
    if bias is not None:
        bias = _floating(bias, "bias")
        _on(bias, "bias", hidden)
        if bias.shape != weight.shape[:1] or bias.dtype != hidden.dtype:
            raise ValueError("bias must be [classes] of hidden's type")
        bias = bias.contiguous()
    if target.is_floating_point() or target.is_complex() or target.dtype == torch.bool or target.shape != hidden.shape[:-1]:
        raise ValueError("target must be whole numbers over the rows of hidden, %s" % (tuple(hidden.shape[:-1]),))
    z_loss = float(z_loss)
    if not 0.0 <= z_loss <= 1e30:
        raise ValueError("z_loss must be finite and not negative")
    if target.dim() != 1:
        target = target.reshape(-1)
    args = (_matrix(hidden, "hidden"), _matrix(weight, "weight"), bias, target.long().contiguous(), int(ignore_index), z_loss,
            _reduction(reduction))
    loss = _LinearCrossEntropy.apply(*args) if _differentiable(*args[:3]) else _linear_ce_forward(*args)[0]
    return loss.reshape(hidden.shape[:-1]) if reduction == "none" and hidden.dim() != 2 else loss

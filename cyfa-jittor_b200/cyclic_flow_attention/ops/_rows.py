"""Argument helpers of the row-wise operators: dtype codes, the device guard and
the mapping of a strided tensor's leading dimensions to rows."""

import contextlib

import torch

from .. import _lib

_NO_GUARD = contextlib.nullcontext()
_CODES = {torch.float32: 0, torch.bfloat16: 1}


class _NoSecondDerivative(torch.autograd.Function):
    """A gradient as it is, which refuses to be differentiated."""

    @staticmethod
    def forward(ctx, g, *sources):
        return g.view_as(g)

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError("this operator has no second derivative")


def first_order(backward):
    """For the backward of an operator without a second derivative: under
    create_graph its gradients depend on what they were computed from, and raise
    when they are differentiated.  (``once_differentiable`` would leave out the
    dependence on the saved tensors without a word.)"""

    def run(ctx, *grads):
        if not torch.is_grad_enabled():
            return backward(ctx, *grads)
        with torch.no_grad():
            out = backward(ctx, *grads)
        sources = [t for t in (*grads, *ctx.saved_tensors) if t is not None and t.requires_grad]
        if not sources:
            return out
        return tuple(g if g is None else _NoSecondDerivative.apply(g, *sources) for g in out)

    return run


def dtype_code(name, t):
    code = _CODES.get(t.dtype)
    if code is None:
        raise TypeError(f"{name} must be float32 or bfloat16, got {t.dtype}")
    return code


def same_device(first, *others):
    """Raises unless `first` and the given others are CUDA tensors of one device."""
    device = first.device
    for t in others:
        if t is not None and t.device != device:
            _lib.require_cuda(first, t)
            raise ValueError(f"tensors must be on one device, got {device} and {t.device}")
    if device.type != "cuda":
        _lib.require_cuda(first)


def on_device(t):
    """Makes t's device the current one (the library launches on the current
    device and on its current stream)."""
    if t.device.index == torch._C._cuda_getDevice():
        return _NO_GUARD
    return torch.cuda.device(t.device)


def row_levels(x, most):
    """The leading dimensions of x as at most `most` (size, stride) levels,
    outermost first, when its last dimension is dense; None if they need more."""
    width = x.shape[-1]
    if x.is_contiguous():
        rows = x.numel() // width
        return [(rows, width)] if rows > 1 else []
    if width > 1 and x.stride(-1) != 1:
        return None
    levels = []
    for size, stride in zip(x.shape[:-1], x.stride()[:-1]):
        if size == 1:
            continue
        if levels and levels[-1][1] == size * stride:
            levels[-1] = (levels[-1][0] * size, stride)
        else:
            levels.append((size, stride))
    return levels if len(levels) <= most else None


def as_rows(x):
    """(x, row stride) with x's leading dimensions one evenly spaced run of rows;
    x is copied if they are not."""
    if x.is_contiguous():
        return x, x.shape[-1]
    levels = row_levels(x, 1)
    if levels is None:
        x = x.contiguous()
        return x, x.shape[-1]
    return x, (levels[0][1] if levels else x.shape[-1])


def dense_like(t):
    """An uninitialised dense tensor of t's shape and type (``empty_like`` is the
    cheaper call, but keeps other strides)."""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def f32(t):
    """A dense fp32 tensor with t's values (t itself when it is one)."""
    if t is None or (t.dtype == torch.float32 and t.is_contiguous()):
        return t
    return t.detach().to(torch.float32).contiguous()


def address(t):
    return None if t is None else t.data_ptr()

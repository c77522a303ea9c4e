"""A block's residual add with the norms on both sides of it, with gradients.

The reference writes it as separate framework ops (residual = x + y and RMSNorm,
models/cyfa/modeling_cyfa.py:52-55,64-69; RMSNorm layers/cyfa.py:62-135); here the
add, the branch's gate and scale, and both norms are one libcyfa launch forward
and one, plus the parameter sums, backward.
"""

import ctypes
import math

import torch

from .. import _lib
from ._rows import address, as_rows, dense_like, dtype_code, first_order, on_device, same_device

MAX_WIDTH = 8192


def _dense(g, dtype):
    if g is None or (g.dtype == dtype and g.is_contiguous()):
        return g
    return g.to(dtype).contiguous()


def _param(t):
    """A [D] parameter as a dense fp32 tensor.  The conversion is autograd's own and stands
    outside ResidualNormFunction, which then saves its inputs themselves: a copy made
    inside would cut its gradients off from the parameter."""
    if t is None or (t.dtype == torch.float32 and t.is_contiguous()):
        return t
    return t.to(torch.float32).contiguous()


def _args(x, y, gate, weight, post, scale_vector, scale, eps):
    """The call's argument block and the tensors that have to outlive it."""
    D = x.shape[-1]
    x, sx = as_rows(x)
    sy = sg = 0
    if y is not None:
        y, sy = as_rows(y)
    if gate is not None:
        gate, sg = as_rows(gate)
    p = address
    return _lib.ResidualNormArgs(
        x.numel() // D, D, dtype_code("x", x), p(x), p(y), p(gate), sx, sy, sg, p(weight),
        p(post), p(scale_vector), scale, eps), (x, y, gate)


def _forward(x, y, weight, post, gate, scale_vector, scale, eps, keep):
    """(xn or None, h, rstd_x, rstd_y); the last two, which only the backward
    reads, are None unless `keep`."""
    rows = x.numel() // x.shape[-1]
    h = dense_like(x)
    xn = None if y is None else torch.empty_like(h)
    rstd_x = weight.new_empty(rows) if keep else None
    rstd_y = torch.empty_like(rstd_x) if keep and post is not None else None
    if rows:
        args, _keep = _args(x, y, gate, weight, post, scale_vector, scale, eps)
        with on_device(x):
            _lib.call("cyfa_residual_norm_fwd", ctypes.byref(args), address(xn), h.data_ptr(),
                      address(rstd_x), address(rstd_y), _lib.raw_stream())
    return xn, h, rstd_x, rstd_y


class ResidualNormFunction(torch.autograd.Function):
    """Autograd wrapper over cyfa_residual_norm_fwd / _bwd."""

    @staticmethod
    def forward(ctx, x, y, weight, post, gate, scale_vector, scale, eps):
        ctx.set_materialize_grads(False)
        xn, h, rstd_x, rstd_y = _forward(x, y, weight, post, gate, scale_vector, scale, eps, True)
        plain = post is None and gate is None and scale_vector is None and scale == 1.0
        # the plain sum needs y for no gradient
        ctx.save_for_backward(x if xn is None else xn, None if plain else y, weight, post, gate,
                              scale_vector, rstd_x, rstd_y)
        ctx.meta = (scale, eps, plain, y is not None)
        return (h,) if xn is None else (xn, h)

    @staticmethod
    @first_order
    def backward(ctx, *grads):
        t, y, w, pw, gate, sv, rstd_x, rstd_y = ctx.saved_tensors
        scale, eps, plain, has_y = ctx.meta
        dxn, dh = grads if has_y else (None, grads[0])
        if dxn is None and dh is None:
            return (None,) * 8
        need = ctx.needs_input_grad
        D = t.shape[-1]
        rows = t.numel() // D
        dxn, dh = _dense(dxn, t.dtype), _dense(dh, t.dtype)
        full = has_y and not plain
        want_x = need[0] or (plain and has_y and need[1])
        rowwise = lambda on: dense_like(t) if on else None
        column = lambda on: (torch.empty_like(w) if rows else torch.zeros_like(w)) if on else None
        dx = rowwise(want_x)
        dy = rowwise(full and need[1])
        dgate = rowwise(gate is not None and need[4])
        dw = column(need[2])
        dpost = column(pw is not None and need[3])
        dscale = column(sv is not None and need[5])
        if rows:
            args, _keep = _args(t, y if full else None, gate, w, pw, sv, scale, eps)
            nbytes = _lib.lib().cyfa_residual_norm_bwd_work_bytes(rows, D)
            work = w.new_empty(nbytes // 4)
            P = address
            with on_device(t):
                _lib.call("cyfa_residual_norm_bwd", ctypes.byref(args), rstd_x.data_ptr(),
                          P(rstd_y), P(dxn), P(dh), P(dx), P(dy), P(dgate), P(dw), P(dpost),
                          P(dscale), work.data_ptr(), nbytes, _lib.raw_stream())
        if plain and has_y and need[1]:
            dy = dx
        return dx if need[0] else None, dy, dw, dpost, dgate, dscale, None, None


def residual_norm(x, y, weight, post_weight=None, gate=None, scale=None, eps=1e-6):
    """Adds a block's branch to the residual stream and normalises the sum:

        z  = y, or RMSNorm(y) * post_weight
        x' = x + scale * sigmoid(gate) * z
        h  = RMSNorm(x') * weight

    and returns ``(x', h)``: the new stream and the next branch's input.  ``x``,
    ``y`` and ``gate`` share one shape [..., D] (D <= 8192) and dtype (bf16 or fp32);
    ``weight``, ``post_weight`` [D]; ``scale`` a number, a [D] tensor, or None for 1.
    ``y = None`` is the norm alone (``x'`` is then ``x`` itself).  fp32 arithmetic; x' is rounded to its
    dtype before it is normalised, as the decoder block keeps it.  Gradients flow
    to every tensor; those of the [D] parameters are summed over the rows in fp32
    in a fixed order.  ``gate`` and ``y`` do not broadcast: expand them first
    (the copy and the gradient's sum are then autograd's).
    """
    scale_vector = scale if isinstance(scale, torch.Tensor) else None
    dtype_code("x", x)
    if x.dim() < 1 or not 0 < x.shape[-1] <= MAX_WIDTH:
        raise ValueError(f"x must be [..., D] with 0 < D <= {MAX_WIDTH}, got {tuple(x.shape)}")
    if y is None and (post_weight is not None or gate is not None or scale is not None):
        raise ValueError("post_weight, gate and scale act on y, which is None")
    for name, t in (("y", y), ("gate", gate)):
        if t is not None and (t.shape != x.shape or t.dtype != x.dtype):
            raise ValueError(f"{name} must be {x.dtype} of shape {tuple(x.shape)}, got {t.dtype} "
                             f"of {tuple(t.shape)}")
    for name, t in (("weight", weight), ("post_weight", post_weight), ("scale", scale_vector)):
        if t is not None and (t.dim() != 1 or t.shape[0] != x.shape[-1]):
            raise ValueError(f"{name} must have shape [{x.shape[-1]}], got {tuple(t.shape)}")
        if t is not None and not t.is_floating_point():
            raise TypeError(f"{name} must be a floating-point tensor, got {t.dtype}")
    if x.numel() // x.shape[-1] >= 1 << 31:
        raise ValueError("at most 2^31 - 1 rows per call")
    number = 1.0 if scale is None or scale_vector is not None else float(scale)
    if not (math.isfinite(number) and math.isfinite(eps) and eps >= 0):
        raise ValueError(f"scale and eps must be finite and eps >= 0, got {scale}, {eps}")
    same_device(x, y, weight, post_weight, gate, scale_vector)
    tensors = (x, y, _param(weight), _param(post_weight), gate, _param(scale_vector))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        out = ResidualNormFunction.apply(*tensors, number, float(eps))
        return (x, out[0]) if y is None else out
    xn, h, _, _ = _forward(*tensors, number, float(eps), False)
    return x if xn is None else xn, h

"""Newton-Schulz orthogonalisation of matrix updates, on the tensor cores.

The counterpart for matrices of the element-wise AdamW update (the reference's
only optimizer, training/optim.py:8-124); ``training.optim.Muon`` applies it.
"""

import math

import torch

from .. import _lib
from ._rows import dtype_code, on_device, same_device

QUINTIC = (3.4445, -4.7750, 2.0315)
MAX_SIDE = 1 << 16


def check_iteration(steps, coefficients):
    """Raises on steps or coefficients that ``orthogonalize`` does not take."""
    if len(coefficients) != 3 or not all(math.isfinite(c) for c in coefficients):
        raise ValueError(f"coefficients must be three finite numbers, got {coefficients}")
    if not 0 <= steps <= 64:
        raise ValueError(f"steps must be between 0 and 64, got {steps}")


def orthogonalize(g, steps=5, coefficients=QUINTIC, eps=1e-7):
    """The Newton-Schulz image of each matrix of ``g`` [..., m, n] (bf16 or fp32):

        X = g / (|g|_F + eps);  ``steps`` times  X <- a X + (b A + c A A) X,
        A = X X^T  (X^T X for a tall matrix), (a, b, c) = ``coefficients``

    as bf16 [..., m, n].  With the default coefficients five steps bring every
    singular value that is not tiny to between about 0.7 and 1.2.  Every product
    keeps 22 bits of its operands and accumulates in fp32, so the error is the
    final rounding's (after ten steps or more with the default coefficients, whose
    fixed value 0.868 repels by 1.58 a step, any rounding shows, fp32's too).
    Other coefficients have to keep every entry of X, A and b A + c A A below 16
    in magnitude (beyond that the result is inf or NaN).
    Not differentiable.
    """
    code = dtype_code("g", g)
    if torch.is_grad_enabled() and g.requires_grad:
        raise ValueError("orthogonalize has no backward; call it under torch.no_grad()")
    if g.dim() < 2 or max(g.shape[-2:]) > MAX_SIDE:
        raise ValueError(f"g must be [..., m, n] with sides up to {MAX_SIDE}, got {tuple(g.shape)}")
    check_iteration(steps, coefficients)
    if not (math.isfinite(eps) and eps >= 2.0 ** -126):
        raise ValueError(f"eps must be a positive normal fp32 number, got {eps}")
    m, n = g.shape[-2:]
    L = math.prod(g.shape[:-2])
    if L > 65535:
        raise ValueError(f"at most 65535 matrices per call, got {L}")
    same_device(g)
    out = torch.empty(g.shape, device=g.device, dtype=torch.bfloat16)
    if out.numel() == 0:
        return out
    x = g.contiguous()
    nbytes = _lib.lib().cyfa_newton_schulz_work_bytes(L, m, n)
    work = torch.empty(nbytes, device=g.device, dtype=torch.uint8)
    with on_device(x):
        _lib.call("cyfa_newton_schulz", x.data_ptr(), code, L, m, n, int(steps),
                  *(float(c) for c in coefficients), float(eps), out.data_ptr(), work.data_ptr(),
                  nbytes, _lib.raw_stream())
    return out

"""What the language-model operators' autograd functions refuse, on the CPU: the
launches are replaced by nothing, so the values mean nothing and only the graphs
of the gradients are looked at."""

import contextlib

import pytest
import torch

from cyclic_flow_attention import _lib
from cyclic_flow_attention.ops import norm_ops, residual_norm, token_log_probs, token_ops

BF, F = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _no_device(monkeypatch):
    for module in (norm_ops, token_ops):
        monkeypatch.setattr(module, "same_device", lambda *a: None)
        monkeypatch.setattr(module, "on_device", lambda t: contextlib.nullcontext())
    monkeypatch.setattr(_lib, "call", lambda *a: None)
    monkeypatch.setattr(_lib, "raw_stream", lambda: 0)


def _penalty_is_refused(f, by, of):
    """A loss plus a penalty on the gradient by `by`, differentiated by `of`: the loss
    alone would go through, without the penalty's part."""
    g, = torch.autograd.grad(f().sum(), by, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(f().sum() + g.float().pow(2).sum(), of)


def _weights():
    return [torch.rand(8, requires_grad=True), torch.rand(8, dtype=BF, requires_grad=True),
            torch.rand(16)[::2].requires_grad_(), torch.rand(8, dtype=torch.float64, requires_grad=True)]


@pytest.mark.parametrize("k", range(4))
def test_norm_alone(k):
    """The gradient by x depends on the weight, whatever its type and strides."""
    x, w = torch.randn(4, 8, requires_grad=True), _weights()[k]
    f = lambda: residual_norm(x, None, w)[1]
    _penalty_is_refused(f, x, w)
    _penalty_is_refused(f, x, x)
    _penalty_is_refused(f, w, x)


@pytest.mark.parametrize("k", range(4))
@pytest.mark.parametrize("out", [0, 1])
def test_norm_with_a_branch(k, out):
    x, y, gate = (torch.randn(4, 8, requires_grad=True) for _ in range(3))
    w, post, scale = _weights()[k], _weights()[k], _weights()[k]
    f = lambda: residual_norm(x, y, w, post_weight=post, gate=gate, scale=scale)[out]
    for of in (post, gate, scale, x, y) + ((w,) if out else ()):
        _penalty_is_refused(f, y, of)


def test_gradients_have_their_parameters_types():
    x = torch.randn(4, 8, requires_grad=True)
    for w in _weights():
        for p in torch.autograd.grad(residual_norm(x, x, w, post_weight=w, scale=w)[1].sum(), (x, w)):
            assert p.dtype == (x.dtype if p.dim() == 2 else w.dtype) and p.shape[-1] == 8


@pytest.mark.parametrize("out", [0, 1])
def test_log_probs_of_any_strides(out):
    t = torch.tensor([1, 2, 3])
    for x in (torch.randn(3, 8, requires_grad=True), torch.randn(8, 3).t().requires_grad_(),
              torch.randn(3, 16)[:, ::2].requires_grad_()):
        _penalty_is_refused(lambda: token_log_probs(x, t)[out], x, x)
    x = torch.randn(8, 3, requires_grad=True)
    _penalty_is_refused(lambda: token_log_probs(x.t(), t)[out], x, x)

"""Calls that the language-model operators refuse, on the CPU: the Python checks
raise before any device work, the C entry points return a status."""

import ctypes

import pytest
import torch

from cyclic_flow_attention import _lib
from cyclic_flow_attention.ops import embed_tokens, orthogonalize, residual_norm, token_log_probs

BF, F = torch.bfloat16, torch.float32


def _logits(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("error, match, call", [
    (TypeError, "float32 or bfloat16", lambda: token_log_probs(_logits(2, 5, dtype=torch.float16),
                                                               torch.zeros(2, dtype=torch.long))),
    (TypeError, "int64 or int32", lambda: token_log_probs(_logits(2, 5), torch.zeros(2))),
    (ValueError, "tokens of shape", lambda: token_log_probs(_logits(2, 5),
                                                            torch.zeros(3, dtype=torch.long))),
    (ValueError, "vocabulary", lambda: token_log_probs(_logits(2, 0),
                                                       torch.zeros(2, dtype=torch.long))),
    (ValueError, "top must be", lambda: token_log_probs(_logits(2, 50), torch.zeros(2, dtype=torch.long),
                                                        top=33)),
    (ValueError, "top must be", lambda: token_log_probs(_logits(2, 5), torch.zeros(2, dtype=torch.long),
                                                        top=6)),
    (ValueError, "top must be", lambda: token_log_probs(_logits(2, 5), torch.zeros(2, dtype=torch.long),
                                                        top=-1)),
    (RuntimeError, "no CPU path", lambda: token_log_probs(_logits(2, 5),
                                                          torch.zeros(2, dtype=torch.long))),
    (TypeError, "float32 or bfloat16", lambda: embed_tokens(torch.zeros(2, dtype=torch.long),
                                                            torch.zeros(4, 4, dtype=torch.float64))),
    (TypeError, "int64 or int32", lambda: embed_tokens(torch.zeros(2), torch.zeros(4, 4))),
    (ValueError, "non-empty", lambda: embed_tokens(torch.zeros(2, dtype=torch.long),
                                                   torch.zeros(0, 4))),
    (ValueError, "non-empty", lambda: embed_tokens(torch.zeros(2, dtype=torch.long), torch.zeros(4))),
    (ValueError, "finite", lambda: embed_tokens(torch.zeros(2, dtype=torch.long), torch.zeros(4, 4),
                                                scale=float("inf"))),
    (ValueError, "padding_idx", lambda: embed_tokens(torch.zeros(2, dtype=torch.long),
                                                     torch.zeros(4, 4), padding_idx=4)),
    (ValueError, "padding_idx", lambda: embed_tokens(torch.zeros(2, dtype=torch.long),
                                                     torch.zeros(4, 4), padding_idx=-5)),
    (RuntimeError, "no CPU path", lambda: embed_tokens(torch.zeros(2, dtype=torch.long),
                                                       torch.zeros(4, 4))),
    (TypeError, "float32 or bfloat16", lambda: residual_norm(_logits(2, 8, dtype=torch.float16), None,
                                                             torch.ones(8))),
    (ValueError, "8192", lambda: residual_norm(_logits(2, 8193), None, torch.ones(8193))),
    (ValueError, "y must be", lambda: residual_norm(_logits(2, 8), _logits(1, 8), torch.ones(8))),
    (ValueError, "y must be", lambda: residual_norm(_logits(2, 8), _logits(2, 8, dtype=F),
                                                    torch.ones(8))),
    (ValueError, "gate must be", lambda: residual_norm(_logits(2, 8), _logits(2, 8), torch.ones(8),
                                                       gate=_logits(2, 1))),
    (ValueError, "act on y", lambda: residual_norm(_logits(2, 8), None, torch.ones(8), scale=2.0)),
    (ValueError, "weight must have", lambda: residual_norm(_logits(2, 8), None, torch.ones(7))),
    (ValueError, "scale must have", lambda: residual_norm(_logits(2, 8), _logits(2, 8), torch.ones(8),
                                                          scale=torch.ones(1))),
    (TypeError, "floating-point", lambda: residual_norm(_logits(2, 8), None,
                                                        torch.ones(8, dtype=torch.long))),
    (ValueError, "finite", lambda: residual_norm(_logits(2, 8), _logits(2, 8), torch.ones(8),
                                                 scale=float("nan"))),
    (ValueError, "finite", lambda: residual_norm(_logits(2, 8), None, torch.ones(8), eps=-1.0)),
    (RuntimeError, "no CPU path", lambda: residual_norm(_logits(2, 8), None, torch.ones(8))),
    (TypeError, "float32 or bfloat16", lambda: orthogonalize(torch.zeros(4, 4, dtype=torch.float16))),
    (ValueError, "no backward", lambda: orthogonalize(torch.zeros(4, 4, requires_grad=True))),
    (ValueError, "sides up to", lambda: orthogonalize(torch.zeros(4))),
    (ValueError, "three finite", lambda: orthogonalize(torch.zeros(4, 4), coefficients=(1.0, 2.0))),
    (ValueError, "steps", lambda: orthogonalize(torch.zeros(4, 4), steps=65)),
    (ValueError, "eps", lambda: orthogonalize(torch.zeros(4, 4), eps=0.0)),
    (ValueError, "65535", lambda: orthogonalize(torch.zeros(65536, 1, 1))),
    (RuntimeError, "no CPU path", lambda: orthogonalize(torch.zeros(4, 4))),
])
def test_python_refusals(error, match, call):
    with pytest.raises(error, match=match):
        call()


def test_c_refusals():
    """Null pointers, sizes, types, alignment and workspaces are refused on the
    host; the pointers below are never read."""
    L = _lib.lib()
    P = ctypes.c_void_p
    ok, odd = P(4096), P(4097)
    size = ctypes.c_size_t

    def lp(logits=ok, dtype=1, rows=2, inner=2, so=0, si=8, V=8, tokens=ok, top=0, topp=None):
        return L.cyfa_token_logprobs_fwd(logits, dtype, rows, inner, so, si, V, tokens, -100, top,
                                         ok, ok, ok, topp, topp, None)

    assert lp(logits=None) == 2 and lp(top=1) == 2
    assert lp(rows=0) == 1 and lp(V=0) == 1 and lp(top=33, topp=ok, V=64) == 1
    assert lp(top=9, topp=ok) == 1 and lp(rows=1 << 27) == 1
    assert lp(dtype=2) == 4 and lp(logits=odd) == 3

    def lpb(dlogits=ok, dtype=1, rows=2, V=8):
        return L.cyfa_token_logprobs_bwd(ok, dtype, rows, 2, 0, 8, V, ok, -100, ok, ok, ok, None,
                                         dlogits, None)

    assert lpb(dlogits=None) == 2 and lpb(dlogits=odd) == 3 and lpb(rows=-1) == 1
    assert lpb(rows=1 << 40) == 1 and lpb(dtype=7) == 4
    assert L.cyfa_embed_fwd(None, ok, 1, ok, 4, 4, 4, 1.0, None) == 2
    assert L.cyfa_embed_fwd(ok, ok, 1, ok, 1 << 31, 4, 4, 1.0, None) == 1
    assert L.cyfa_embed_fwd(ok, ok, 1, odd, 4, 4, 4, 1.0, None) == 3
    n = L.cyfa_embed_bwd_work_bytes(4, 8)
    assert n > 0 and L.cyfa_embed_bwd_work_bytes(0, 8) == 0

    def eb(dtype=1, N=4, V=4, work=ok, nbytes=n):
        return L.cyfa_embed_bwd(ok, ok, dtype, ok, N, V, 8, 1.0, -1, work, size(nbytes), None)

    assert eb(work=None) == 2 and eb(N=0) == 1 and eb(V=1 << 31) == 1 and eb(dtype=3) == 4
    assert eb(nbytes=n - 1) == 7 and eb(work=P(4096 + 16)) == 3

    def rn(D=8, rows=2, x=ok, y=ok, post=None, gate=None, xn=ok, rstd_y=None, dtype=1):
        a = _lib.ResidualNormArgs(rows, D, dtype, x, y, gate, D, D, D, ok, post, None, 1.0, 1e-6)
        return L.cyfa_residual_norm_fwd(ctypes.byref(a), xn, ok, ok, rstd_y, None)

    assert rn(x=None) == 2 and rn(xn=None) == 2 and rn(y=None, post=ok) == 2 and rn(y=None, gate=ok) == 2
    assert rn(D=8193) == 1 and rn(rows=0) == 1 and rn(dtype=5) == 4 and rn(x=odd) == 3
    a = _lib.ResidualNormArgs(2, 8, 1, ok, ok, None, 8, 8, 8, ok, None, None, 1.0, 1e-6)
    n = L.cyfa_residual_norm_bwd_work_bytes(2, 8)
    assert L.cyfa_residual_norm_bwd(ctypes.byref(a), ok, None, ok, ok, ok, ok, None, ok, None, None,
                                    ok, size(n - 1), None) == 7
    n = L.cyfa_newton_schulz_work_bytes(2, 8, 16)

    def ns(Lm=2, m=8, nn=16, steps=5, dtype=1, work=ok, nbytes=n):
        return L.cyfa_newton_schulz(ok, dtype, Lm, m, nn, steps, 3.0, -4.0, 2.0, 1e-7, ok, work,
                                    size(nbytes), None)

    assert ns(work=None) == 2 and ns(Lm=65536) == 1 and ns(m=65537) == 1 and ns(steps=65) == 1
    assert ns(dtype=2) == 4 and ns(nbytes=n - 1) == 7 and ns(work=P(64)) == 3


def test_muon_refusals_and_groups():
    from training.optim import Muon

    w = torch.zeros(4, 6, requires_grad=True)
    b = torch.zeros(3, requires_grad=True)
    for kw in (dict(lr=-1.0), dict(momentum=1.0), dict(weight_decay=-0.1), dict(steps=0)):
        with pytest.raises(ValueError, match="Muon"):
            Muon([w], **kw)
    with pytest.raises(ValueError, match="empty"):
        Muon([])
    with pytest.raises(ValueError, match="two-dimensional"):
        Muon([b], matrix=lambda n, p: True)
    with pytest.raises(ValueError, match="sides"):
        Muon([torch.zeros(1 << 17, 1, requires_grad=True)])
    opt = Muon([("x.weight", w), ("lm_head.weight", torch.zeros(4, 6, requires_grad=True)), ("y", b)])
    assert [g["names"] for g in opt.param_groups] == [["x.weight"], ["lm_head.weight", "y"]]
    (w.sum() + b.sum()).backward()
    opt.accumulate_param_grads()
    with pytest.raises(RuntimeError, match="no CPU path"):
        opt.step()
    L = _lib.lib()
    P = ctypes.c_void_p
    piece = (_lib.BucketPiece * 1)(_lib.BucketPiece(4096, 8, 0, 0))
    bad = (_lib.BucketPiece * 1)(_lib.BucketPiece(4096, 8, 4, 0))
    assert L.cyfa_muon_momentum(None, 1, P(4096), P(4096), 0.9, 1, None) == 2
    assert L.cyfa_muon_momentum(bad, 1, P(4096), P(4096), 0.9, 1, None) == 3
    assert L.cyfa_muon_momentum(piece, -1, P(4096), P(4096), 0.9, 1, None) == 1
    assert L.cyfa_muon_apply(piece, None, 1, P(4096), 0.1, 1.0, None) == 2

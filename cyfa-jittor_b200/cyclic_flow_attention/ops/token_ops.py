"""The two ends of the language model: ``embed_tokens`` (scaled lookup, table
gradient summed in a fixed order) and ``token_log_probs`` (log probability of given
tokens, entropy and most likely alternatives straight from the logits).

The reference computes both with framework ops (models/cyfa/modeling_cyfa.py:58-69
for the embedding, :102-116 for the cross entropy over fp32 logits).  Here each
direction is libcyfa kernels that read the logits, or the gradient rows, once and
build no fp32 copy of them.
"""

import math
from typing import NamedTuple, Optional

import torch

from .. import _lib
from ._rows import address, dense_like, dtype_code, f32, first_order, on_device, row_levels, same_device

MAX_TOP = 32
_INTS = (torch.int64, torch.int32)


class TokenLogProbs(NamedTuple):
    """Result of token_log_probs; the top fields are None when top = 0."""

    logp: torch.Tensor
    entropy: torch.Tensor
    top_logp: Optional[torch.Tensor]
    top_tokens: Optional[torch.Tensor]


def _dense_int64(tokens):
    if tokens.dtype == torch.int64 and tokens.is_contiguous():
        return tokens
    return tokens.to(torch.int64).contiguous()


def _addressed(logits):
    """(logits, inner, outer stride, inner stride): row r starts at
    (r // inner) * outer + (r % inner) * inner stride."""
    levels = row_levels(logits, 2)
    if levels is None:
        logits = logits.contiguous()
        levels = row_levels(logits, 2)
    if not levels:
        return logits, 1, 0, 0
    if len(levels) == 1:
        return logits, levels[0][0], 0, levels[0][1]
    return logits, levels[1][0], levels[0][1], levels[1][1]


def _logprobs_fwd(logits, tokens, top, ignore_index, keep):
    """(addressed logits, logp, entropy, stats, top_logp, top_tokens); stats, which
    only the backward reads, is None unless `keep`."""
    rows = tokens.numel()
    x, inner, outer_stride, inner_stride = _addressed(logits)
    logp = torch.empty_like(tokens, dtype=torch.float32)
    entropy = torch.empty_like(logp)
    stats = logp.new_empty((rows, 2)) if keep else None
    top_logp = top_tokens = None
    if top:
        top_logp = logp.new_empty((*tokens.shape, top))
        top_tokens = tokens.new_empty((*tokens.shape, top))
    if rows:
        with on_device(x):
            _lib.call("cyfa_token_logprobs_fwd", x.data_ptr(), dtype_code("logits", x), rows,
                      inner, outer_stride, inner_stride, x.shape[-1], tokens.data_ptr(),
                      ignore_index, top, logp.data_ptr(), entropy.data_ptr(), address(stats),
                      address(top_logp), address(top_tokens), _lib.raw_stream())
    return x, logp, entropy, stats, top_logp, top_tokens


class TokenLogProbsFunction(torch.autograd.Function):
    """Autograd wrapper over cyfa_token_logprobs_fwd / _bwd."""

    @staticmethod
    def forward(ctx, logits, tokens, top, ignore_index):
        ctx.set_materialize_grads(False)
        x, logp, entropy, stats, top_logp, top_tokens = _logprobs_fwd(logits, tokens, top,
                                                                     ignore_index, True)
        ctx.save_for_backward(x, tokens, stats, entropy)
        ctx.ignore_index = ignore_index
        if not top:
            return logp, entropy
        ctx.mark_non_differentiable(top_logp, top_tokens)
        return logp, entropy, top_logp, top_tokens

    @staticmethod
    @first_order
    def backward(ctx, dlogp, dentropy, *_):
        if dlogp is None and dentropy is None:
            return None, None, None, None
        x, tokens, stats, entropy = ctx.saved_tensors
        x, inner, outer_stride, inner_stride = _addressed(x)
        dx = dense_like(x)
        rows = tokens.numel()
        dlogp, dentropy = f32(dlogp), f32(dentropy)
        if rows:
            with on_device(x):
                _lib.call("cyfa_token_logprobs_bwd", x.data_ptr(), dtype_code("logits", x), rows,
                          inner, outer_stride, inner_stride, x.shape[-1], tokens.data_ptr(),
                          ctx.ignore_index, stats.data_ptr(), entropy.data_ptr(),
                          address(dlogp), address(dentropy), dx.data_ptr(), _lib.raw_stream())
        return dx, None, None, None


def token_log_probs(logits, tokens, top=0, ignore_index=-100):
    """Log probabilities of ``tokens`` under softmax(``logits``).

    ``logits`` [..., V] bf16 or fp32 and ``tokens`` [...] int64 or int32, on one
    CUDA device; any strides (rows dense and evenly spaced on up to two levels,
    such as ``logits[:, :-1]``, are read in place).  Returns ``TokenLogProbs``:

    * ``logp`` [...] fp32: log p of each token; 0 where it is ``ignore_index``;
    * ``entropy`` [...] fp32: -sum p log p of each position's distribution;
    * ``top_logp``, ``top_tokens`` [..., top]: the ``top`` (<= 32) most likely
      tokens, by logit and among equals by lowest index; None when ``top`` is 0.

    Gradients flow to the logits from ``logp`` and ``entropy`` (not from the
    alternatives), in the logits' dtype: ``dlogp`` at the token's entry, less the
    probabilities' share.  A masked logit (-inf) has probability 0.  A position with
    no finite logit has logp -inf, entropy 0 and every probability 0, so that only the
    token's entry has a gradient, ``dlogp``; with ``ignore_index`` as its token it has none.
    NaN or +inf makes the position's results NaN.  A token outside the vocabulary
    gives NaN and sets the device error word (``_lib.device_error()`` returns 3).
    """
    dtype_code("logits", logits)
    if tokens.dtype not in _INTS:
        raise TypeError(f"tokens must be int64 or int32, got {tokens.dtype}")
    if logits.dim() < 1 or logits.shape[:-1] != tokens.shape:
        raise ValueError(f"logits {tuple(logits.shape)} need tokens of shape "
                         f"{tuple(logits.shape[:-1])}, got {tuple(tokens.shape)}")
    V = logits.shape[-1]
    if not 0 < V < 1 << 30:
        raise ValueError(f"unsupported vocabulary size {V}")
    if not 0 <= top <= min(MAX_TOP, V):
        raise ValueError(f"top must be between 0 and {min(MAX_TOP, V)}, got {top}")
    if tokens.numel() >= 1 << 27:
        raise ValueError(f"{tokens.numel()} positions; at most {(1 << 27) - 1} per call")
    same_device(logits, tokens)
    top, ignore_index = int(top), int(ignore_index)
    tokens = _dense_int64(tokens)
    if torch.is_grad_enabled() and logits.requires_grad:
        out = TokenLogProbsFunction.apply(logits, tokens, top, ignore_index)
        return TokenLogProbs(*out, *((None, None) if not top else ()))
    _, logp, entropy, _, top_logp, top_tokens = _logprobs_fwd(logits, tokens, top, ignore_index,
                                                              False)
    return TokenLogProbs(logp, entropy, top_logp, top_tokens)


def _embed_fwd(tokens, weight, scale):
    V, D = weight.shape
    out = weight.new_empty((*tokens.shape, D))
    if out.numel():
        with on_device(weight):
            _lib.call("cyfa_embed_fwd", tokens.data_ptr(), weight.data_ptr(),
                      dtype_code("weight", weight), out.data_ptr(), tokens.numel(), V, D, scale,
                      _lib.raw_stream())
    return out


class EmbedTokensFunction(torch.autograd.Function):
    """Autograd wrapper over cyfa_embed_fwd / _bwd."""

    @staticmethod
    def forward(ctx, tokens, weight, scale, padding_idx):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(tokens)
        ctx.meta = (weight.shape, weight.dtype, scale, padding_idx)
        return _embed_fwd(tokens, weight.contiguous(), scale)

    @staticmethod
    @first_order
    def backward(ctx, dout):
        if dout is None:
            return None, None, None, None
        tokens, = ctx.saved_tensors
        (V, D), dtype, scale, padding_idx = ctx.meta
        N = tokens.numel()
        if N == 0:
            return None, torch.zeros(V, D, device=tokens.device, dtype=dtype), None, None
        if dout.dtype != dtype or not dout.is_contiguous():
            dout = dout.to(dtype).contiguous()
        dw = dout.new_empty((V, D))
        nbytes = _lib.lib().cyfa_embed_bwd_work_bytes(N, D)
        work = tokens.new_empty((nbytes + 7) // 8)
        with on_device(dout):
            _lib.call("cyfa_embed_bwd", tokens.data_ptr(), dout.data_ptr(),
                      dtype_code("weight", dw), dw.data_ptr(), N, V, D, scale, padding_idx,
                      work.data_ptr(), nbytes, _lib.raw_stream())
        return None, dw, None, None


def embed_tokens(tokens, weight, scale=1.0, padding_idx=None):
    """``scale * weight[tokens]`` with a deterministic gradient of the table.

    ``tokens`` [...] int64 or int32 and ``weight`` [V, D] bf16 or fp32, on one CUDA
    device; the result [..., D] has the weight's dtype (one rounding after the
    fp32 product).  The gradient is the dense [V, D] table: each row sums its
    tokens' gradient rows in fp32 in a fixed tree over the token order (the tokens are
    sorted, no float atomics) and is rounded once; ``padding_idx`` (as in ``nn.Embedding``) gets a
    zero row.  A token outside the vocabulary reads as zeros, has no gradient and
    sets the device error word (``_lib.device_error()`` returns 3).
    """
    dtype_code("weight", weight)
    if tokens.dtype not in _INTS:
        raise TypeError(f"tokens must be int64 or int32, got {tokens.dtype}")
    if weight.dim() != 2 or 0 in weight.shape:
        raise ValueError(f"weight must be a non-empty [V, D] table, got {tuple(weight.shape)}")
    V, D = weight.shape
    if V >= 1 << 31 or D >= 1 << 22 or tokens.numel() >= 1 << 31:
        raise ValueError(f"unsupported embedding size: {tokens.numel()} tokens of [{V}, {D}]")
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")
    pad = -1
    if padding_idx is not None:
        if not -V <= padding_idx < V:
            raise ValueError(f"padding_idx {padding_idx} is outside a vocabulary of {V}")
        pad = int(padding_idx) % V
    same_device(weight, tokens)
    tokens = _dense_int64(tokens)
    if torch.is_grad_enabled() and weight.requires_grad:
        return EmbedTokensFunction.apply(tokens, weight, float(scale), pad)
    return _embed_fwd(tokens, weight.contiguous(), float(scale))

"""The norms of ``fuse_training()``: each of the model's norm weights takes its own
gradient, at its own place."""

import pytest
import torch

from gpu_util import rel_l2, seeded
from oracle import cyfa_oracle as O
from test_gpu_fused_training import _grads, _model

pytestmark = pytest.mark.gpu


def _distinct_norms(m):
    """Random norm weights, another one for each norm; their names."""
    names = [n for n, _ in m.named_parameters()
             if n.endswith(("attn_norm.weight", "mlp_norm.weight")) or n == "model.norm.weight"]
    assert len(names) == 2 * len(m.model.layers) + 1
    with torch.no_grad():
        for k, n in enumerate(names):
            w = m.get_parameter(n)
            w.copy_(1 + 0.5 * torch.randn(w.shape, generator=seeded(100 + k)))
    return names


def _oracle_grads(cfg, m, ids, labels, names, shift):
    """Gradients of the norm weights; shift: each norm is given the weight that stands so
    many places further on, and that parameter takes the gradient."""
    params = {n: t.detach().float().cpu().requires_grad_() for n, t in m.named_parameters()}
    used = dict(params)
    for k, n in enumerate(names):
        used[n] = params[names[(k + shift) % len(names)]]
    logits = O.cyfa_lm(used, ids.cpu(), cfg.num_hidden_layers, cfg.num_heads, cfg.head_dim, cfg.head_dim)
    torch.nn.functional.cross_entropy(logits[:, :-1].reshape(-1, cfg.vocab_size),
                                      labels[:, 1:].reshape(-1).cpu(), ignore_index=-100).backward()
    return {n: params[n].grad for n in names}


def test_each_norm_weight_takes_its_gradient():
    """Both paths compute in bf16 with the roundings in other places: two draws of one
    noise, whose norms over 256 entries (64 independent ones at least) have a ratio of
    1 within 6 times 2^-3, rounded up to 2, plus one bf16 step.  A norm with its neighbour's
    weight is off by the weights' spread of a half, far outside."""
    cfg, m = _model()
    names = _distinct_norms(m)
    ids = torch.randint(0, cfg.vocab_size, (2, 160), generator=seeded(3)).cuda()
    labels = ids.clone()
    labels[0, 100:] = -100
    loss0, g0 = _grads(m, ids, labels)
    loss1, g1 = _grads(m.fuse_training(), ids, labels)
    ref = _oracle_grads(cfg, m, ids, labels, names, 0)
    planted = _oracle_grads(cfg, m, ids, labels, names, 1)
    assert abs(float(loss1) - float(loss0)) < 2.0 ** -8 * abs(float(loss0))
    for n in names:
        bound = 2 * rel_l2(g0[n], ref[n]) + 2.0 ** -8
        assert rel_l2(g1[n], ref[n]) < bound < rel_l2(planted[n], ref[n]), n


def test_each_norm_weight_of_a_padded_batch():
    """With a mask: at most 40 roundings of 2^-8 one after the other stand between a
    parameter's gradient and the inputs on either path."""
    cfg, m = _model(4)
    names = _distinct_norms(m)
    ids = torch.randint(0, cfg.vocab_size, (3, 130), generator=seeded(5)).cuda()
    mask = torch.ones_like(ids)
    mask[0, 77:] = 0
    labels = ids.masked_fill(mask == 0, -100)
    labels[2] = -100
    got = []
    for on in (False, True):
        m.fuse_training(on).zero_grad(set_to_none=True)
        m(ids, labels=labels, attention_mask=mask)["loss"].backward()
        got.append({n: m.get_parameter(n).grad for n in names})
    for k, n in enumerate(names):
        assert rel_l2(got[1][n], got[0][n]) < 40 * 2.0 ** -8, n
        assert rel_l2(got[0][names[k - 1]], got[0][n]) > 0.5, n

"""How many bits the language-model operators keep, against 64-bit computations."""

import pytest
import torch

from cyclic_flow_attention.ops import residual_norm

pytestmark = pytest.mark.gpu
BF, F = torch.bfloat16, torch.float32
EPS = 1e-6


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


@pytest.mark.parametrize("scale", ["none", "number", "vector"])
@pytest.mark.parametrize("rows, D", [(2, 1207), (5, 3001), (20, 340), (71, 1485), (48, 2216), (327, 246),
                                     (347, 693), (512, 64)])
def test_bf16_weight_gradient(rows, D, scale):
    """The weight's gradient of bf16 rows with a post-norm, from x' rounded once out of
    64 bits.  Its terms dh x' / rms(x') carry the rounding of the reciprocal root and of
    its sum of squares (at most 2^-20) and two products; at most 64 of them are added in
    a row, on any path: together below 2^-17 of the sum of magnitudes.  One entry of x'
    at the neighbouring bf16 value alone would be 2^-8 of its term, more than that for
    these numbers of rows."""
    g = _gen(rows + D)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")
    x, y, w, post = (2 * n(rows, D)).to(BF), n(rows, D).to(BF), 1 + 0.1 * n(D), 1 + 0.1 * n(D)
    sc = {"none": None, "number": 0.5, "vector": 0.5 + 0.1 * n(D)}[scale]
    dh = n(rows, D).to(BF)
    wl = w.clone().requires_grad_()
    h = residual_norm(x, y, wl, post_weight=post, scale=sc, eps=EPS)[1]
    got, = torch.autograd.grad(h, wl, dh)
    yd = y.double()
    z = yd / (yd.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * post.double()
    sd = 1.0 if sc is None else (sc if scale == "number" else sc.double())
    t = (x.double() + sd * z).float().to(BF).double()
    terms = dh.double() * t / (t.pow(2).mean(-1, keepdim=True) + EPS).sqrt()
    bad = ~((got.double() - terms.sum(0)).abs() <= 2.0 ** -17 * terms.abs().sum(0))
    assert not bad.any(), int(bad.sum())

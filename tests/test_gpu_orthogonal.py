"""orthogonalize against the same iteration in 64 bits.

Tolerance.  The result is rounded to bf16: at most 2^-8 relative per entry.  The
operands' 22 bits and the fp32 accumulation leave about 2^-18 per product, which
five steps enlarge by at most 3.4445^5 < 2^9 in the weakest directions: below
2^-9 there, far less over the whole matrix.  So the relative Frobenius error stays
below 2^-8, and its root mean square (rounding alone: 0.41 2^-8) below 0.6 2^-8."""

import math

import pytest
import torch

from cyclic_flow_attention import _lib
from cyclic_flow_attention.ops import orthogonalize

pytestmark = pytest.mark.gpu
BF, F = torch.bfloat16, torch.float32
Q = (3.4445, -4.7750, 2.0315)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _plain(g, steps=5, q=Q, eps=1e-7):
    x = g.double()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    x = x / (x.pow(2).sum((-2, -1), keepdim=True).sqrt() + eps)
    for _ in range(steps):
        A = x @ x.mT
        x = q[0] * x + (q[1] * A + q[2] * A @ A) @ x
    return x.mT if tall else x


def _check(g, **kw):
    out = orthogonalize(g, **kw)
    ref = _plain(g, **kw)
    assert out.dtype == BF and out.shape == g.shape and out.is_contiguous()
    err = (out.double() - ref).norm() / ref.norm()
    assert float(err) < 0.6 * 2.0 ** -8, float(err)
    return out


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("shape", [(1, 1), (1, 7), (9, 1), (3, 5, 5), (2, 64, 64), (127, 509), (509, 127),
                                   (4, 128, 256), (2, 129, 257), (300, 130), (2, 3, 40, 24), (1024, 1024), (80, 100, 1500), (3, 256, 1024), (2, 257, 300), (150, 17, 33), (2, 90, 1025), (1, 5000), (3, 2500, 20), (128, 128), (2, 128, 129), (100, 2049),
                                   (2, 1408, 512), (512, 1408), (700, 2049)])
def test_sizes(dtype, shape):
    _check(torch.randn(shape, generator=_gen(1), device="cuda").to(dtype))


@pytest.mark.parametrize("steps", [0, 1, 2, 3, 7])
def test_steps_and_coefficients(steps):
    g = torch.randn(2, 100, 300, generator=_gen(0), device="cuda")
    _check(g, steps=steps)
    out = orthogonalize(g.mT, steps=steps, coefficients=(1.5, -0.5, 0.0))
    ref = _plain(g.mT, steps, (1.5, -0.5, 0.0))
    assert float((out.double() - ref).norm() / ref.norm()) < 0.6 * 2.0 ** -8


def test_gradient_like_and_singular_values():
    """A few strong directions over noise, and rank one: the strong singular values
    land near 1."""
    u = torch.randn(400, 20, generator=_gen(0), device="cuda")
    v = torch.randn(20, 900, generator=_gen(1), device="cuda")
    g = u @ v * 1e-3 + torch.randn(400, 900, generator=_gen(2), device="cuda") * 1e-3
    out = _check(g)
    s = torch.linalg.svdvals(out.double())
    assert s.max() < 1.25 and s[:20].min() > 0.65
    one = torch.outer(u[:, 0], v[0])
    s = torch.linalg.svdvals(_check(one).double())
    assert 0.65 < s[0] < 1.25


def test_scales_zero_and_special_values():
    g = torch.randn(130, 70, generator=_gen(0), device="cuda")
    for f in (1e-4, 1e30, 1e36):
        _check(g * f)
    assert (orthogonalize(torch.zeros(2, 40, 50, device="cuda")) == 0).all()
    x = torch.randn(3, 40, 50, generator=_gen(1), device="cuda")
    x[1, 3, 4] = math.nan
    out = orthogonalize(x)
    assert out[1].isnan().all() and out[0].isfinite().all() and out[2].isfinite().all()
    assert torch.equal(out[0], orthogonalize(x[:1])[0])
    assert orthogonalize(torch.zeros(0, 4, 5, device="cuda")).shape == (0, 4, 5)
    assert orthogonalize(torch.zeros(4, 0, device="cuda")).shape == (4, 0)


def test_strides():
    g = torch.randn(3, 90, 150, generator=_gen(0), device="cuda")
    for x in (g.mT, g[:, ::2, 1:], g[1], g.expand(2, 3, 90, 150), g.permute(1, 0, 2)):
        assert torch.equal(orthogonalize(x), orthogonalize(x.contiguous()))


def test_stream_graph_and_repeat():
    g = torch.randn(6, 200, 333, generator=_gen(0), device="cuda").to(BF)
    first = orthogonalize(g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = orthogonalize(g)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, second)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = orthogonalize(g)
    g.copy_(torch.randn(6, 200, 333, generator=_gen(1), device="cuda"))
    graph.replay()
    graph.replay()
    assert torch.equal(out, orthogonalize(g))
    assert _lib.device_error() == 0

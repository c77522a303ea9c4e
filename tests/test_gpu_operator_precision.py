"""How many bits the language-model operators keep, against 64-bit computations, and
their values where a mask leaves nothing."""

import math

import pytest
import torch

from cyclic_flow_attention.ops import orthogonalize, residual_norm, token_log_probs

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


@pytest.mark.parametrize("D", [64, 67, 4096])
def test_f32_gate_gradients_over_its_range(D):
    """dy = dx' sigmoid(gate) and dgate = dx' y sigmoid (1 - sigmoid) of fp32 rows, entry by
    entry, for gates from -86 to 86 (nothing leaves the normal range).  expf: 2 ulp = 2^-22,
    its sum 2^-24, the reciprocal 2^-23, their product 2^-24: 2^-21, and dx' = 1 adds nothing.
    dgate: two such factors and six products: below 2^-19.  (z < 0 and z > 0: neither 1 - sigmoid nor the
    exponential's argument may lose bits.)"""
    rows = 4096 // D + 8
    gate = torch.linspace(-86, 86, rows * D, device="cuda").view(rows, D).requires_grad_()
    y = 0.5 + torch.rand(rows, D, generator=_gen(D), device="cuda")
    y = torch.where(torch.rand(rows, D, generator=_gen(1), device="cuda") < 0.5, -y, y).requires_grad_()
    xn, _ = residual_norm(torch.zeros(rows, D, device="cuda"), y, torch.ones(D, device="cuda"), gate=gate)
    dgate, dy = torch.autograd.grad(xn, (gate, y), torch.ones_like(xn))
    z = gate.detach().double()
    q, rest = torch.sigmoid(z), torch.sigmoid(-z)
    assert ((dy.double() - q).abs() <= 2.0 ** -21 * q).all()
    want = y.detach().double() * q * rest
    assert ((dgate.double() - want).abs() <= 2.0 ** -19 * want.abs()).all()


def _newton_schulz(g, steps, q):
    x = g.double()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    x = x / (x.pow(2).sum((-2, -1), keepdim=True).sqrt() + 1e-7)
    for _ in range(steps):
        A = x @ x.mT
        x = q[0] * x + (q[1] * A + q[2] * A @ A) @ x
    return x.mT if tall else x


def _graded(m, n, seed):
    """Singular values from 1 down to 1e-2."""
    k = min(m, n)
    r = lambda *s: torch.randn(*s, generator=_gen(seed), device="cuda", dtype=torch.float64)
    u, v = torch.linalg.qr(r(m, k))[0], torch.linalg.qr(r(n, k))[0]
    return ((u * torch.logspace(0, -2, k, device="cuda", dtype=torch.float64)) @ v.mT).float()


@pytest.mark.parametrize("coefficients", [(3.4445, -4.7750, 2.0315), (1.5, -0.5, 0.0), (1.875, -1.25, 0.375)])
@pytest.mark.parametrize("m, n", [(64, 300), (100, 128), (127, 509), (20, 2500), (128, 2048), (300, 200),
                                  (512, 512), (300, 900)])
def test_newton_schulz_error_is_the_final_rounding(m, n, coefficients):
    """From few steps to many, on Gaussian and graded matrices.  A product of operands of
    22 bits with fp32 accumulation is off by at most 2^-19 of its norm, and the iterates
    settle on values where the map does not enlarge that: 24 steps of three products
    leave 72 2^-19 < 2^-12.8, against 2^-9.3 of the rounding to bf16; the two together are
    at most 1.02 times the rounding alone.  (The graded square matrix is symmetric: its
    iterates go to the identity, whose rounding is 0, and the products' share of 3 steps
    2^-19 |X| is all there is.)

    The default quintic p(s) = a s + b s^3 + c s^5 has the fixed value s^2 = 0.753 (where
    a + b s^2 + c s^4 = 1), at which p'(s) = 3.4445 - 10.79 + 5.77 = -1.58: a singular value
    near it moves away by that factor a step, and so does any error of it.  An error of e |X|
    made in each step has grown to at most e |X| (1.58^(steps - 1) + .. + 1) < 1.73 1.58^steps
    e |X| at the end.  e: the accumulator takes 3 K / 16 additions (three MMAs of 16 columns),
    each cut off at 2^-23 of the sum.  Five steps stay under the plain bound."""
    default = coefficients[0] > 3
    e = 3 * max(m, n) / 16 * 2.0 ** -23
    for g in (torch.randn(m, n, generator=_gen(m), device="cuda"), _graded(m, n, n)):
        for steps in (1, 2, 3, 5, 8, 12, 16, 24):
            ref = _newton_schulz(g, steps, coefficients)
            alone = (ref.to(BF).double() - ref).norm()
            grown = 1.73 * 1.58 ** steps * e * ref.norm() if default and steps > 5 else 0.0
            off = (orthogonalize(g, steps, coefficients).double() - ref).norm()
            plain = torch.maximum(1.02 * alone, 3 * steps * 2.0 ** -19 * ref.norm())
            assert off <= plain + grown, (steps, float(off / alone))


@pytest.mark.parametrize("dtype", [BF, F])
@pytest.mark.parametrize("V", [1, 7, 90, 5000, 40000])
def test_log_probs_rows_without_a_finite_logit(V, dtype):
    """Every probability is 0, so the formula leaves dlogp at the token's entry, exactly
    (one rounding to the logits' type), nothing from the entropy, and nothing at all where
    the token is ignored."""
    x = torch.full((4, V), -math.inf, device="cuda", dtype=dtype)
    x[0] = torch.randn(V, generator=_gen(V), device="cuda").to(dtype)
    x.requires_grad_()
    tokens = torch.tensor([0, V - 1, -100, V // 2], device="cuda")
    r = token_log_probs(x, tokens)
    assert r.logp.tolist()[1:] == [-math.inf, 0, -math.inf] and (r.entropy[1:] == 0).all()
    g, h = torch.randn(2, 4, generator=_gen(V + 1), device="cuda")
    dx, = torch.autograd.grad((r.logp, r.entropy), x, (g, h))
    want = torch.zeros(4, V, device="cuda", dtype=dtype)
    want[1, V - 1], want[3, V // 2] = g[1].to(dtype), g[3].to(dtype)
    assert torch.equal(dx[1:], want[1:]) and dx[0].isfinite().all()
